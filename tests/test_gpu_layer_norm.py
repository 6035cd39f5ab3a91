"""GPU parity of layer norm with its formulas in float64, by automatic differentiation and
by differences.

Tolerances, as 2-norms of the error over 2-norms of the result, set before the first run.
float32: a mean and a variance of n values carry some log2(n) <= 14 roundings of 2^-24 on
their way through lanes (16 values to a lane at most), a value about ten more: 32 * 2^-24 =
2e-6; gradients of weight and bias are sums over up to 3000 rows in two levels, the
same.  The mean itself adds its rounding times |mean| / deviation, which is at most 8 in these
inputs: 8 * 2^-24 is in it.  bfloat16: one rounding at the end, at most 2^-8 per element, and
1.1 times that leaves the float32 part its room."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = 2e-6, 1.1 * 2.0 ** -8


def _tol(dtype):
    return F32 if dtype == torch.float32 else BF16


def _formula(x, w, b, eps=1e-5):
    c = x - x.mean(-1, keepdim=True)
    y = c / (c.square().mean(-1, keepdim=True) + eps).sqrt()
    y = y if w is None else y * w
    return y if b is None else y + b


def _rel(a, ref):
    a, ref = a.detach().double().cpu(), ref.detach().double()
    assert torch.isfinite(a).all()
    return float((a - ref).norm() / ref.norm().clamp_min(1e-30))


# rows and size: every form (one, four and sixteen wavefronts to a row; one, two, four pieces to
# a lane), sizes that end inside a piece, more rows than workgroups
SHAPES = [(1, 1), (3, 2), (7, 65), (2100, 64), (5, 256), (9, 511), (3000, 129), (6, 1025), (4, 2048), (3, 2049),
          (2, 4097), (2, 8192), (2, 8193), (1, 16383), (2, 16384)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("affine", [(True, True), (True, False), (False, False), (False, True)])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_and_gradients(gpu, shape, affine, dtype):
    from rnn_kernel_amd import layer_norm

    print(f"layer norm {shape} {affine} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(shape[0] * 31 + shape[1])
    x = (torch.randn(shape, generator=gen) + 3 * torch.randn(shape[0], 1, generator=gen).clamp(-2, 2)).to(dtype)
    w, b = ((1 + 0.3 * torch.randn(shape[1], generator=gen)).to(dtype) if on else None for on in affine)
    up = torch.randn(shape, generator=gen).to(dtype)
    ref = [t.double().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    got = [t.to(gpu).requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y, ry = layer_norm(*got), _formula(*ref)
    assert y.dtype == dtype and y.shape == shape
    if shape[1] > 2:
        assert _rel(y, ry) <= _tol(dtype)
        grads = torch.autograd.grad(y, [t for t in got if t is not None], up.to(gpu))
        refs = torch.autograd.grad(ry, [t for t in ref if t is not None], up.double())
        for g, r in zip(grads, refs):
            assert g.dtype == dtype and _rel(g, r) <= _tol(dtype)
    else:  # of one or two elements: the deviation is a difference of neighbours, errors go by eps's size
        assert torch.allclose(y.detach().cpu().double(), ry.detach(), atol=2 * _tol(dtype), rtol=2 * _tol(dtype))


def test_without_gradients_and_with_them_alike(gpu):
    from rnn_kernel_amd import LayerNorm

    layer = LayerNorm(100).to(gpu)
    x = torch.randn(5, 7, 100, device=gpu)
    with torch.no_grad():
        y = layer(x)
    assert torch.equal(y, layer(x)) and y.shape == x.shape


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(gpu, dtype):
    """Any strides of x and of the gradient: the bits of the dense call."""
    from rnn_kernel_amd import layer_norm

    gen = torch.Generator().manual_seed(1)
    wide = torch.randn(6, 5, 77, generator=gen).to(gpu, dtype)
    w = torch.randn(70, generator=gen).to(gpu, dtype)
    up = torch.randn(6, 5, 70, generator=gen).to(gpu, dtype)
    for x in (wide[..., 3:73], wide.transpose(0, 1)[..., 3:73].transpose(0, 1), wide[..., :70][:, ::2],
              wide.permute(2, 1, 0)[:70].permute(2, 1, 0), wide[:1, :, 5:75].expand(6, 5, 70)):
        u = up[:, ::2] if x.size(1) == 3 else up
        want_x = x.detach().contiguous().requires_grad_(True)
        leaf = x.detach().requires_grad_(True)
        y, want = layer_norm(leaf, w), layer_norm(want_x, w)
        assert torch.equal(y, want)
        for g in (u, u.transpose(0, 1).contiguous().transpose(0, 1), u[..., :1].expand_as(u)):
            assert torch.equal(torch.autograd.grad(y, leaf, g, retain_graph=True)[0],
                               torch.autograd.grad(want, want_x, g.contiguous(), retain_graph=True)[0])


def test_rows_without_elements(gpu):
    from rnn_kernel_amd import layer_norm

    x = torch.zeros(0, 4, 8, device=gpu, requires_grad=True)
    w = torch.ones(8, device=gpu, requires_grad=True)
    y = layer_norm(x, w)
    dx, dw = torch.autograd.grad(y.sum(), [x, w])
    assert y.shape == dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w))


def test_special_values(gpu):
    """A NaN or an infinity makes its own row NaN and no other; a constant row gives the
    bias."""
    from rnn_kernel_amd import layer_norm

    x = torch.randn(5, 33, device=gpu)
    x[1, 4], x[3, 32], x[4] = float("nan"), float("inf"), 7.0
    b = torch.randn(33, device=gpu)
    y = layer_norm(x, None, b)
    assert y[1].isnan().all() and y[3].isnan().all() and torch.isfinite(y[[0, 2, 4]]).all()
    assert torch.equal(y[4], b)
    assert torch.equal(y[[0, 2]], layer_norm(x[[0, 2]], None, b))


def test_gradients_by_differences(gpu):
    """d<y, up> along a direction, by a central difference of step h in float64 of the kernel's
    float32 values: the truncation is O(h^2) with third derivatives of order 10, the rounding
    2 * 3e-7 |<y, up>| / h; at h = 1e-2 both stay under 1e-3 of a derivative of order 10."""
    from rnn_kernel_amd import layer_norm

    gen = torch.Generator().manual_seed(3)
    args = [torch.randn(*s, generator=gen).to(gpu) for s in ((4, 40), (40,), (40,))]
    up = torch.randn(4, 40, generator=gen).to(gpu)
    leaves = [t.clone().requires_grad_(True) for t in args]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, up)
    for i, g in enumerate(grads):
        d = torch.randn(args[i].shape, generator=gen).to(gpu)
        d = d * g.norm() / (d * g).sum().abs() if (d * g).sum().abs() < 0.1 * g.norm() else d
        d = d / d.norm()
        h = 1e-2
        side = [(layer_norm(*[t + s * h * d if j == i else t for j, t in enumerate(args)]).double() * up.double()).sum()
                for s in (1, -1)]
        diff = (side[0] - side[1]) / (2 * h)
        assert abs(float(diff - (g.double() * d.double()).sum())) <= 2e-3 * float(g.norm())


def test_graph_replay_and_other_stream(gpu):
    from rnn_kernel_amd import layer_norm

    x, w = torch.randn(300, 200, device=gpu), torch.randn(200, device=gpu)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = layer_norm(x, w)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(want, layer_norm(x, w))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer_norm(x, w)
    for i in range(3):
        x.copy_(torch.randn(300, 200, device=gpu))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, layer_norm(x, w))


def test_same_bits_twice(gpu):
    from rnn_kernel_amd import layer_norm

    x, w, b = (torch.randn(*s, device=gpu).requires_grad_(True) for s in ((3000, 130), (130,), (130,)))
    up = torch.randn(3000, 130, device=gpu)
    first = torch.autograd.grad(layer_norm(x, w, b), [x, w, b], up)
    for a, c in zip(first, torch.autograd.grad(layer_norm(x, w, b), [x, w, b], up)):
        assert torch.equal(a, c)
