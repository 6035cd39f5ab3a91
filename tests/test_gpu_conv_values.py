"""The causal convolution at values where a product of 0 and infinity would be met."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_gradients_behind_a_row_are_0_whatever_the_weights(gpu, bad, dtype):
    """And an empty row's initial state has the gradient of its final state, which is that state."""
    from rnn_kernel_amd import causal_conv

    B, T, D, W = 3, 70, 10, 4
    gen = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=gen).to(gpu, dtype)  # noqa: E731
    x, w, s0, up, ups = r(B, T, D), r(D, W), r(B, W - 1, D), r(B, T, D), r(B, W - 1, D)
    w[2, 1] = bad
    lengths = torch.tensor([T, 33, 0], dtype=torch.int32, device=gpu)
    x, s0 = x.requires_grad_(True), s0.requires_grad_(True)
    y, s = causal_conv(x, w, None, s0, lengths=lengths)
    dx, ds = torch.autograd.grad([y, s], [x, s0], [up, ups])
    assert (dx[1, 33:] == 0).all() and (dx[2] == 0).all() and torch.equal(ds[2], ups[2])
    rest = torch.arange(D, device=gpu) != 2
    assert torch.isfinite(dx[..., rest]).all() and torch.isfinite(ds[..., rest]).all()
