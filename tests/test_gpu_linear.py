"""GPU parity of the matrix product with bias, activation and residual, and of its
gradients, with the same in float64.

Tolerances, as 2-norms of the error over 2-norms of the result, set before the
first run.  float32: a sum of n products of random signs carries n roundings of at
most 2^-24 of its partial sums, which add up like a random walk: 2^-24 (8 + 2 sqrt(n)).
bfloat16 outputs are rounded once: 2^-8, and a tenth more for the float32 part.  A
bfloat16 gradient goes through three roundings (of z, of dz and of the result), none
of which moves it by more than 2^-8: 3.3 * 2^-8.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ACTS = ("none", "relu", "gelu", "silu", "sigmoid", "logsigmoid")


def _sigmoid(z):
    """Whose derivative, y sigmoid(-z), cancels nothing (torch's y (1 - y) is off by 1e-3
    at z = 30 in float64 too)."""
    return torch.exp(-torch.logaddexp(-z, torch.zeros_like(z)))


def _act(z, act):
    if act == "relu":
        return torch.relu(z)  # whose slope at 0 is 0
    if act == "gelu":
        return z * 0.5 * torch.erfc(-z / math.sqrt(2.0))
    if act == "silu":
        return z * _sigmoid(z)
    if act == "sigmoid":
        return _sigmoid(z)
    if act == "logsigmoid":
        return -torch.logaddexp(-z, torch.zeros_like(z))
    return z


def _oracle(x, w, b, r, act):
    z = x @ w.t()
    if b is not None:
        z = z + b
    y = _act(z, act)
    return y if r is None else y + r


def _rel(a, ref):
    a, ref = a.detach().double().cpu(), ref.detach().double()
    assert a.shape == ref.shape and torch.isfinite(a).all()
    return float((a - ref).norm() / ref.norm().clamp_min(1e-30))


def _tol(dtype, n, grad=False):
    return 2.0 ** -24 * (8 + 2 * math.sqrt(n)) if dtype == torch.float32 else (3.3 if grad else 1.1) * 2.0 ** -8


def _inputs(m, n, k, dtype, bias=True, residual=True, seed=0):
    gen = torch.Generator().manual_seed(seed + m + 3 * n + 7 * k)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return (r(m, k).to(dtype), (r(n, k) / math.sqrt(k)).to(dtype), r(n).to(dtype) if bias else None,
            r(m, n).to(dtype) if residual else None), r(m, n).to(dtype)


def _check(gpu, m, n, k, dtype, act, bias=True, residual=True):
    from rnn_kernel_amd import linear

    print(f"linear {(m, n, k)} {dtype} {act} bias={bias} residual={residual}", flush=True)
    host, dy = _inputs(m, n, k, dtype, bias, residual)
    dev = [None if t is None else t.to(gpu).requires_grad_(True) for t in host]
    ref = [None if t is None else t.double().requires_grad_(True) for t in host]
    y = linear(*dev[:3], activation=act, residual=dev[3])
    ry = _oracle(*ref, act)
    assert y.dtype == dtype and _rel(y, ry) <= _tol(dtype, k)
    with torch.no_grad():
        assert torch.equal(linear(*dev[:3], activation=act, residual=dev[3]), y)
    got = torch.autograd.grad(y, [t for t in dev if t is not None], dy.to(gpu))
    want = torch.autograd.grad(ry, [t for t in ref if t is not None], dy.double())
    names = [s for s, t in zip(("dx", "dw", "db", "dr"), dev) if t is not None]
    for name, a, b, terms in zip(names, got, want, (n, m, m, 1)):
        assert a.dtype == dtype and _rel(a, b) <= _tol(dtype, max(terms, k), True), (name, _rel(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", [(5, 33, 70), (130, 72, 96)])
def test_every_activation(gpu, m, n, k, act, dtype):
    _check(gpu, m, n, k, dtype, act)


# one row and many, tiles that end inside a block, a sum shorter than a stage and
# one that ends inside a 16-byte piece, odd row lengths, the slices and each tile
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 17, 64), (16, 256, 256), (17, 48, 513), (64, 130, 40), (65, 64, 64),
                                   (100, 3, 9), (129, 129, 129), (300, 7, 2000), (1000, 385, 257), (2048, 512, 64),
                                   (1, 4096, 130), (520, 520, 520), (33, 1030, 300)])
def test_sizes(gpu, m, n, k, dtype):
    _check(gpu, m, n, k, dtype, "silu")
    _check(gpu, m, n, k, dtype, "none", bias=False, residual=False)


# operands that go to LDS directly (whole stages on 16 bytes): one stage, even and odd
# numbers of them, slices, and each tile with an end inside
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(70, 1000, 64), (300, 200, 192), (129, 40, 2048), (257, 31, 128), (2048, 1030, 256)])
def test_aligned_sizes(gpu, m, n, k, dtype):
    _check(gpu, m, n, k, dtype, "gelu")


# few rows on either side of the rule that takes the rows' kernel or tiles in slices
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(1, 40, 9000), (16, 70, 2000), (17, 300, 513), (32, 24, 1500), (32, 24, 5000), (33, 24, 1500)])
def test_few_rows(gpu, m, n, k, dtype):
    _check(gpu, m, n, k, dtype, "relu")


# and few columns, on either side of its rule
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(33, 1, 64), (300, 8, 513), (2000, 16, 2048), (4096, 17, 1000), (70, 32, 200), (700, 33, 200)])
def test_few_columns(gpu, m, n, k, dtype):
    _check(gpu, m, n, k, dtype, "logsigmoid")


@pytest.mark.parametrize("m,n,k", [(4100, 4104, 320), (16384, 1032, 64)])
def test_aligned_large_tiles(gpu, m, n, k):
    _check(gpu, m, n, k, torch.bfloat16, "silu")


@pytest.mark.parametrize("m,n,k", [(4096, 4096, 200), (4100, 4100, 136), (8192, 256, 1000)])
def test_large_tiles(gpu, m, n, k):
    _check(gpu, m, n, k, torch.bfloat16, "gelu")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_leading_dimensions(gpu, dtype):
    """Columns of wider matrices, at addresses that are no multiple of 16, and
    transposed operands: the same bits as dense copies."""
    from rnn_kernel_amd import linear

    for m, n, k in ((40, 50, 70), (200, 136, 96)):
        (x, w, b, r), dy = (lambda a, g: ([t.to(gpu) for t in a], g.to(gpu)))(*_inputs(m, n, k, dtype))

        def wide(t, left):
            full = torch.full((t.size(0), t.size(1) + left + 5), float("nan"), dtype=dtype, device=gpu)
            full[:, left:left + t.size(1)] = t
            return full[:, left:left + t.size(1)]

        want = linear(x, w, b, activation="gelu", residual=r)
        for left in (1, 3, 8):
            assert torch.equal(linear(wide(x, left), wide(w, left), b, activation="gelu", residual=wide(r, left)), want)
        assert torch.equal(linear(x.t().contiguous().t(), w.t().contiguous().t(), b, activation="gelu",
                                  residual=r.t().contiguous().t()), want)
        grads = []
        for lay in (lambda t: t, lambda t: wide(t, 3)):
            leaves = [lay(t).detach().requires_grad_(True) for t in (x, w)] + [b.clone().requires_grad_(True)]
            y = linear(*leaves, activation="gelu")
            grads.append(torch.autograd.grad(y, leaves, lay(dy)))
        for a, c in zip(*grads):
            assert torch.equal(a, c)


def test_leading_shapes_broadcasts_and_partial_gradients(gpu):
    from rnn_kernel_amd import Linear, linear

    (x, w, b, _), _ = _inputs(30, 20, 24, torch.float32)
    x, w, b = x.to(gpu), w.to(gpu), b.to(gpu)
    y = linear(x, w, b, activation="relu")
    assert torch.equal(linear(x.view(2, 3, 5, 24), w, b, activation="relu"), y.view(2, 3, 5, 20))
    assert torch.equal(linear(x[0], w, b), linear(x[:1], w, b)[0])
    # a residual that is expanded over the rows: its gradient is summed over them
    r = torch.randn(20, device=gpu, requires_grad=True)
    up = torch.randn(30, 20, device=gpu)
    dr = torch.autograd.grad(linear(x, w, b, residual=r.expand(30, 20)), r, up)[0]
    assert torch.allclose(dr, up.sum(0), rtol=1e-5, atol=1e-5)
    dx = torch.autograd.grad(linear((xe := x.clone().requires_grad_(True)).expand(3, 30, 24), w, b), xe,
                             torch.ones(3, 30, 20, device=gpu))[0]
    assert _rel(dx, (3 * torch.ones(30, 20) @ w.cpu()).double()) <= 1e-6
    # what nobody wants is not made
    wl = w.clone().requires_grad_(True)
    g1 = torch.autograd.grad(linear(x, wl, b, activation="silu"), wl, up)[0]
    xl, wl2, bl = x.clone().requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    g2 = torch.autograd.grad(linear(xl, wl2, bl, activation="silu"), [xl, wl2, bl], up)[1]
    assert torch.equal(g1, g2)
    # an upstream gradient that is one expanded number
    xl = x.clone().requires_grad_(True)
    g = torch.autograd.grad(linear(xl, w, b).sum(), xl)[0]
    assert _rel(g, (torch.ones(30, 20) @ w.cpu()).double()) <= 1e-6
    mod = Linear(24, 20, activation="silu").to(gpu)
    ref = torch.nn.Linear(24, 20).to(gpu)
    ref.load_state_dict(mod.state_dict())
    assert torch.allclose(mod(x, residual=up), torch.nn.functional.silu(ref(x)) + up, rtol=1e-5, atol=1e-5)


def test_no_rows(gpu):
    from rnn_kernel_amd import linear

    x = torch.empty(0, 24, device=gpu, requires_grad=True)
    w = torch.randn(20, 24, device=gpu, requires_grad=True)
    b = torch.randn(20, device=gpu, requires_grad=True)
    y = linear(x, w, b, activation="silu")
    assert y.shape == (0, 20)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.empty(0, 20, device=gpu))
    assert dx.shape == (0, 24) and (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m", [20, 200])
def test_infinities_and_nan_stay_in_their_rows(gpu, m, dtype):
    from rnn_kernel_amd import linear

    (x, w, b, r), _ = _inputs(m, 70, 90, dtype)
    clean = linear(x.to(gpu), w.to(gpu), b.to(gpu), activation="relu", residual=r.to(gpu))
    x[3, 5], x[11, 0] = float("inf"), float("nan")
    y = linear(x.to(gpu), w.to(gpu), b.to(gpu), activation="relu", residual=r.to(gpu))
    rest = [i for i in range(m) if i not in (3, 11)]
    assert torch.equal(y[rest], clean[rest])
    assert torch.isnan(y[11]).all()
    want = torch.where(w[:, 5].float() > 0, float("inf"), 0.0)
    assert torch.equal(torch.isinf(y[3]).cpu(), torch.isinf(want)) and not torch.isnan(y[3]).any()


def test_saturated_activations(gpu):
    """Large sums of either sign: finite, and without the cancellation of 1 + erf."""
    from rnn_kernel_amd import linear

    z = torch.tensor([[-200.0, -100.0, -30.0, -8.0, -5.0, 0.0, 5.0, 30.0, 100.0, 200.0]])
    w = torch.eye(10).to(gpu)
    for act in ACTS:
        zl = z.to(gpu).requires_grad_(True)
        y = linear(zl, w, activation=act)
        g = torch.autograd.grad(y, zl, torch.ones_like(y))[0]
        zr = z.double().requires_grad_(True)
        ry = _act(zr, act)
        rg = torch.autograd.grad(ry, zr, torch.ones_like(ry))[0]
        for a, b in ((y, ry), (g, rg)):
            # relative to each element (2^-18: exp(-x) of a float32 x carries its 2^-24
            # x), down to where float32 ends
            err = (a.detach().cpu().double() - b.detach()).abs()
            assert (err <= 2.0 ** -18 * b.detach().abs() + 1e-37).all(), act


def test_reproducible_on_another_stream_and_in_a_graph(gpu):
    from rnn_kernel_amd import linear

    (x, w, b, r), dy = (lambda a, g: ([t.to(gpu) for t in a], g.to(gpu)))(*_inputs(700, 256, 1024, torch.bfloat16))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def once():
        y = linear(*leaves, activation="gelu", residual=r)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    first = once()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        again = once()
    stream.synchronize()
    for a, c in zip(first, again):
        assert torch.equal(a, c)
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            y = linear(x, w, b, activation="gelu", residual=r)
        for i in range(3):
            r.copy_(torch.randn(r.shape, generator=torch.Generator().manual_seed(i)).to(r))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, linear(x, w, b, activation="gelu", residual=r))
