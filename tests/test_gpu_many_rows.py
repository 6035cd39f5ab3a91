"""More rows than a launch has threads for: norms of 2^26 rows and more, as of many short heads."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_norms_of_many_short_rows(gpu):
    from rnn_kernel_amd import layer_norm

    rows, some = 2 ** 26 + 5, 1000
    gen = torch.Generator(device=gpu).manual_seed(0)
    x = torch.randn(rows, 2, generator=gen, device=gpu, dtype=torch.bfloat16).requires_grad_(True)
    w = torch.tensor([2.0, 0.5], device=gpu, dtype=torch.bfloat16)
    y = layer_norm(x, w)
    up = torch.randn(rows, 2, generator=gen, device=gpu, dtype=torch.bfloat16)
    dx = torch.autograd.grad(y, x, up)[0]
    for at in (0, 2 ** 26 - some // 2, rows - some):  # (the bits of a call with those rows alone)
        part = x.detach()[at:at + some].clone().requires_grad_(True)
        of = layer_norm(part, w)
        assert torch.equal(of, y[at:at + some])
        assert torch.equal(torch.autograd.grad(of, part, up[at:at + some])[0], dx[at:at + some])
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w), y)


def test_convolutions_of_many_rows(gpu):
    """65535 rows of 16385 tokens of one channel, in more than one launch either way: rows are those
    of a call with them alone, and the sums over all those of its parts, in float64."""
    from rnn_kernel_amd import causal_conv

    B, T, some = 65535, 16385, 3
    gen = torch.Generator(device=gpu).manual_seed(1)
    x = torch.randn(B, T, 1, generator=gen, device=gpu, dtype=torch.bfloat16).requires_grad_(True)
    s0 = torch.randn(B, 1, 1, generator=gen, device=gpu, dtype=torch.bfloat16).requires_grad_(True)
    w = torch.tensor([[0.5, -1.5]], device=gpu, dtype=torch.bfloat16).requires_grad_(True)
    lengths = torch.full((B,), T, dtype=torch.int32, device=gpu)
    lengths[::7] = 100
    y, s = causal_conv(x, w, None, s0, lengths=lengths)
    up = torch.randn(B, 1, 1, generator=gen, device=gpu, dtype=torch.bfloat16).expand(B, T, 1)
    ups = torch.ones_like(s)
    dx, dw, ds = torch.autograd.grad([y, s], [x, w, s0], [up, ups])
    for at in (0, 65272, B // 2, 61680, B - some):
        rows = slice(at, at + some)
        part, p0 = (t.detach()[rows].clone().requires_grad_(True) for t in (x, s0))
        out = causal_conv(part, w, None, p0, lengths=lengths[rows])
        assert torch.equal(out[0], y[rows]) and torch.equal(out[1], s[rows])
        grads = torch.autograd.grad(out, [part, p0], [up[rows], ups[rows]])
        assert torch.equal(grads[0], dx[rows]) and torch.equal(grads[1], ds[rows])
    want = torch.zeros(2, dtype=torch.float64, device=gpu)
    live = (torch.arange(T, device=gpu)[None] < lengths[:, None])[..., None]
    for a, l, u, b in zip(x.detach().split(4096), live.split(4096), up.split(4096), s0.detach().split(4096)):
        a, u = a.double(), torch.where(l, u, torch.zeros_like(u)).double()
        want[1] += (a * u).sum()
        want[0] += (torch.cat([b.double(), a[:, :-1]], 1) * u).sum()
    # (float32 sums of 10^9 terms in blocks of 60 and then one after another in eight lines, and one rounding:
    # 2^-8 of the sum; the terms' signs are random, their root sum is what the sums' roundings go by)
    assert ((dw[0].double() - want).abs() <= 1.1 * 2.0 ** -8 * want.abs() + 1e-4 * (B * T) ** 0.5).all()
