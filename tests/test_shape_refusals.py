"""Sizes that the library does not take are ValueErrors, as the operators promise, and those that
Python can tell are refused before anything is allocated."""
import pytest
import torch


def test_a_refused_size_is_a_value_error(hip_lib):
    from rnn_kernel_amd import _lib

    assert hip_lib.rka_causal_conv_forward(4096, 0, 0, 4096, None, None, None, 4096, 4096, 65536, 1, 1, 2, 0, 0, None) == 1004
    with pytest.raises(ValueError, match="batch exceeds 65535") as refused:
        _lib.check(1004, "rka_causal_conv_forward")
    assert isinstance(refused.value, _lib.RKAError)
    with pytest.raises(_lib.RKAError) as other:
        _lib.check(1001, "rka_causal_conv_forward")
    assert not isinstance(other.value, ValueError)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(65536, 1), (1, 2 ** 20 + 1)])
def test_sequences_that_the_convolution_does_not_take(gpu, shape):
    from rnn_kernel_amd import SelectiveScan, causal_conv

    x = torch.ones(1, 1, 4, device=gpu).expand(*shape, 4)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    for grad in (False, True):
        w = torch.ones(4, 3, device=gpu, requires_grad=grad)
        with pytest.raises(ValueError, match="at most 65535 rows and 2\\^20 tokens"):
            causal_conv(x, w)
    assert torch.cuda.max_memory_allocated() - before <= 4096
    with pytest.raises(ValueError, match="at most 65535 rows and 2\\^20 tokens"), torch.no_grad():
        SelectiveScan(4, device=gpu)(x)


# rows, vocabulary, type (0: float32, 1: bfloat16), whether a launch takes their logits
LOGITS = [(2 ** 21, 2 ** 18, 1, False), (2 ** 21, 2 ** 17, 0, False), (2 ** 20, 2 ** 21, 1, False), (2 ** 20, 2 ** 18, 1, True),
          (2 ** 20, 2 ** 17, 0, True), (2 ** 21, 5, 1, True), (1, 2 ** 21, 0, True), (2 ** 21, 2 ** 21, 0, False)]


@pytest.mark.parametrize("rows,vocabulary,dtype,taken", LOGITS)
def test_more_logits_than_a_launch_has(hip_lib, rows, vocabulary, dtype, taken):
    """The forward's are refused before anything is launched; the backward has them in pieces."""
    sizes = (rows, 8, vocabulary)
    assert (hip_lib.rka_cross_entropy_forward_workspace_bytes(*sizes, dtype) > 0) == taken
    assert hip_lib.rka_cross_entropy_backward_workspace_bytes(*sizes, dtype) > 0
    if not taken:
        assert hip_lib.rka_cross_entropy_forward(4096, 8, 4096, 8, None, 4096, 1, -100, 4096, 4096, 4096, 2 ** 60, *sizes, 1, dtype,
                                                 None) == 1004
        assert "more logits than a launch" in hip_lib.rka_last_error().decode()


@pytest.mark.gpu
def test_more_logits_than_a_launch_has_in_python(gpu):
    from rnn_kernel_amd import linear_cross_entropy

    x, w = (torch.ones(1, 8, device=gpu, dtype=torch.bfloat16).expand(n, 8) for n in (2 ** 21, 2 ** 18))
    target = torch.zeros(2 ** 21, dtype=torch.int32, device=gpu)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    with pytest.raises(ValueError, match="more than a launch may have"):
        linear_cross_entropy(x, w, target)
    assert torch.cuda.max_memory_allocated() == before


def test_a_scan_for_training_is_refused_where_its_gradients_would_be(hip_lib):
    """(2^24 rows of one token: a launch of the gradients has four wavefronts where the forward's has one.)"""
    import ctypes

    strides, P, sizes = (ctypes.c_longlong * 12)(), 4096, (2 ** 24, 1, 16, 1, 1)
    assert hip_lib.rka_selective_scan_forward(P, P, P, P, P, None, None, None, None, None, P, P, P, P, 2 ** 60, *sizes, strides, 0, 0,
                                              None) == 1004
    assert "more workgroups than a launch may have" in hip_lib.rka_last_error().decode()
    assert hip_lib.rka_selective_scan_backward(P, P, P, P, P, None, None, None, None, P, P, None, P, P, P, P, P, None, None, None, None,
                                               P, 2 ** 60, *sizes, strides, 0, 0, None) == 1004


@pytest.mark.gpu
def test_more_gradients_of_B_and_C_than_a_launch_has_threads(gpu):
    """2^32 of them, of 2^19 tokens that are all alike and forget at once: every token's are those of the
    first, which are products of powers of two."""
    from rnn_kernel_amd import selective_scan

    T, G = 2 ** 19, 64
    x, dt = (torch.full((1, 1, G), v, device=gpu, dtype=torch.bfloat16).expand(1, T, G) for v in (2.0, 1.0))
    Bm, C = (torch.full((1, 1, G, 64), v, device=gpu, dtype=torch.bfloat16).expand(1, T, G, 64).detach() for v in (0.5, 0.25))
    Bm.requires_grad_(True), C.requires_grad_(True)
    y, _ = selective_scan(x, dt, torch.full((G, 64), -1e4, device=gpu), Bm, C)
    dB, dC = torch.autograd.grad(y, [Bm, C], torch.ones(1, 1, 1, device=gpu, dtype=torch.bfloat16).expand(1, T, G))
    for g, want in ((dB, 0.5), (dC, 1.0)):
        assert g.shape == (1, T, G, 64)
        assert all(bool((part == want).all()) for part in g.split(2 ** 16, 1))
