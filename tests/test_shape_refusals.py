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
