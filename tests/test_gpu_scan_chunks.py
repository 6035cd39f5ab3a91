"""The selective scan where its chunks are long or there is one alone, and gradients of states that
grow: against the recurrence in float64 and its own, with the tolerances of
test_gpu_selective_scan.py, whose inputs these are."""
import pytest
import torch

from test_gpu_selective_scan import BF16, GRAD, NAMES, SUMS, VALUE, _call, _formula, _inputs, _rel


def _chunks(lib, B, T, D, N, G):
    """Chunks of a row, from the bytes that the forward keeps of each."""
    nbytes = lib.rka_selective_scan_forward_workspace_bytes(B, T, D, N, G)
    return 1 if nbytes == 0 else round(nbytes / (4 * B * D * (N + 1)))


# B, T, D, N, G, tokens of a chunk: one chunk of ten tiles of 16, chunks of nine tiles, chunks of four with two blocks of states
WIDE = [(32, 150, 2112, 4, 1, 160), (8, 2000, 1040, 6, 2, 144), (5, 900, 1536, 17, 1, 64)]


@pytest.mark.parametrize("shape", WIDE)
def test_shapes_have_the_chunks_they_are_for(hip_lib, shape):
    *of, tokens = shape
    assert _chunks(hip_lib, *of) == -(-of[1] // tokens)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", WIDE)
def test_long_chunks_and_one_alone(gpu, shape, dtype):
    B, T = shape[:2]
    args, up, ups = _inputs(*shape[:5], dtype, device=gpu)
    lengths = (torch.arange(B) * 37 % (T + 1)).to(torch.int32)
    lengths[-1] = T
    lengths = lengths.to(gpu)
    ref = [t.double().requires_grad_(True) for t in args]
    got = [t.requires_grad_(True) for t in args]
    out, want = _call(got, lengths=lengths), _formula(*ref, True, lengths)
    assert _rel(out[0], want[0]) <= (VALUE if dtype == torch.float32 else BF16) and _rel(out[1], want[1]) <= VALUE
    grads = torch.autograd.grad(out, got, [up, ups])
    refs = torch.autograd.grad(want, ref, [up.double(), ups.double()])
    behind = torch.arange(T, device=gpu)[None, :] >= lengths[:, None]
    for name, g, r in zip(NAMES, grads, refs):
        tol = BF16 if g.dtype == torch.bfloat16 else SUMS if name in ("A", "skip", "bias", "dt") else GRAD
        assert _rel(g, r) <= tol, (name, _rel(g, r))
        if g.shape[:2] == (B, T):
            assert (g[behind] == 0).all(), name


@pytest.mark.gpu
def test_gradients_that_grow_over_chunks(gpu):
    """A above 0, backwards: over a chunk (64 tokens here) the growth exp(128) is no float32, but there is
    no gradient of the states until the first 10 tokens, or one so small that the result is a float32."""
    from rnn_kernel_amd import selective_scan

    gen = torch.Generator().manual_seed(2)
    x, B, C = torch.randn(1, 300, 32, generator=gen), torch.randn(1, 300, 1, 16, generator=gen), torch.randn(1, 300, 1, 16, generator=gen)
    x[:, :290] = 0
    up = torch.randn(1, 300, 32, generator=gen)
    up[:, 10:] = 0
    dt, A = torch.ones(1, 300, 32), torch.full((32, 16), 2.0)
    ref = [t.double().requires_grad_(True) for t in (x, dt, A, B, C)]
    got = [t.to(gpu).requires_grad_(True) for t in (x, dt, A, B, C)]
    want = torch.autograd.grad(_formula(*ref, None, None, None, None, False, None)[0], ref, up.double())
    grads = torch.autograd.grad(selective_scan(*got)[0], got, up.to(gpu))
    assert _rel(grads[0], want[0]) <= GRAD and (grads[0][:, 10:] == 0).all() and want[0][:, :10].abs().min() > 0
    for g, r in zip(grads[1:], want[1:]):  # (no state is there yet where the gradients are)
        assert (r == 0).all() and (g == 0).all()

    # exp(0.5 * 300) of 1e-30 is exp(81); each of 300 decays is off by 2^-24 or so: 300 * 2^-24 = 1.8e-5
    s0, A, x = torch.full((1, 32, 16), 1e-30), torch.full((32, 16), 0.5), torch.zeros_like(x)
    ref = [t.double().requires_grad_(True) for t in (x, dt, A, B, C, s0)]
    got = [t.to(gpu).requires_grad_(True) for t in (x, dt, A, B, C, s0)]
    ups = torch.full((1, 32, 16), 1e-30)
    want = torch.autograd.grad(_formula(*ref, None, None, None, False, None)[1], ref, ups.double(), allow_unused=True)
    grads = torch.autograd.grad(selective_scan(*got)[1], got, ups.to(gpu))
    for name, g, r in zip(NAMES, grads, want):
        if name == "C":
            assert (g == 0).all()
        else:
            assert _rel(g, r) <= 300 * 2.0 ** -24 + SUMS, name
