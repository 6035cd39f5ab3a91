"""GPU parity of the causal convolution with its formula in float64, and of its gradients
with automatic differentiation and with differences.

Tolerances, as 2-norms of the error over 2-norms of the result, set before the first run.
float32: a sum of at most nine products, an activation of some ten roundings of 2^-24, sums
over up to 400 tokens in levels for the weights: 32 * 2^-24 = 2e-6.  bfloat16: one rounding at
the end, at most 2^-8 per element, and 1.1 times that leaves the float32 part its room (the
final state is copied and exact; a gradient of the initial state is rounded once)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = 2e-6, 1.1 * 2.0 ** -8


def _tol(dtype):
    return F32 if dtype == torch.float32 else BF16


def _formula(x, w, b, s0, act, lengths):
    """float64, differentiable; tokens behind a row's length give 0 and take no part."""
    B, T, D = x.shape
    W = w.size(1)
    n = torch.full((B,), T) if lengths is None else lengths.long().clamp(0, T)
    live = (torch.arange(T)[None, :] < n[:, None])[..., None]
    x = torch.where(live, x, torch.zeros_like(x))
    xs = torch.cat([torch.zeros(B, W - 1, D, dtype=x.dtype) if s0 is None else s0, x], 1)
    z = sum(w[:, j] * xs[:, j:j + T] for j in range(W))
    z = z if b is None else z + b
    y = z * torch.sigmoid(z) if act == "silu" else z
    at = n[:, None] + torch.arange(W - 1)
    return torch.where(live, y, torch.zeros_like(y)), xs.gather(1, at[..., None].expand(-1, -1, D))


def _rel(a, ref):
    a, ref = a.detach().double().cpu(), ref.detach().double()
    assert torch.isfinite(a).all()
    return float((a - ref).norm() / ref.norm().clamp_min(1e-30))


def _inputs(B, T, D, W, dtype, bias, s0, seed=0):
    gen = torch.Generator().manual_seed(seed + 7 * T + D)
    r = lambda *s: torch.randn(*s, generator=gen).to(dtype)  # noqa: E731
    return [r(B, T, D), r(D, W), r(D) if bias else None, r(B, W - 1, D) if s0 else None], r(B, T, D), r(B, W - 1, D)


SHAPES = [  # B, T, D, W
    (1, 1, 1, 2), (2, 1, 7, 4), (3, 2, 8, 8), (2, 31, 64, 3), (2, 32, 65, 4), (1, 33, 512, 4), (2, 128, 513, 5),
    (1, 129, 20, 6), (1, 400, 130, 7), (2, 126, 1030, 2),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act,bias,s0,ragged", [("silu", True, True, True), (None, False, False, False),
                                                ("silu", False, True, False), ("none", True, False, True)])
@pytest.mark.parametrize("shape", SHAPES)
def test_sequences_and_gradients(gpu, shape, act, bias, s0, ragged, dtype):
    from rnn_kernel_amd import causal_conv

    print(f"conv {shape} {act} bias={bias} s0={s0} ragged={ragged} {dtype}", flush=True)
    B, T, D, W = shape
    args, up, ups = _inputs(*shape, dtype, bias, s0)
    lengths = torch.tensor([(5 * i + T // 2) % (T + 1) if i else 0 if B > 2 else T for i in range(B)], dtype=torch.int32) if ragged else None
    ref = [None if t is None else t.double().requires_grad_(True) for t in args]
    got = [None if t is None else t.to(gpu).requires_grad_(True) for t in args]
    y, s = causal_conv(*got, activation=act, lengths=None if lengths is None else lengths.to(gpu))
    ry, rs = _formula(*ref, act, lengths)
    assert y.dtype == s.dtype == dtype and _rel(y, ry) <= _tol(dtype) and torch.equal(s.detach().cpu().double(), rs.detach())
    grads = torch.autograd.grad([y, s], [t for t in got if t is not None], [up.to(gpu), ups.to(gpu)])
    refs = torch.autograd.grad([ry, rs], [t for t in ref if t is not None], [up.double(), ups.double()])
    for g, r in zip(grads, refs):
        assert g.dtype == dtype and g.shape == r.shape
        if r.abs().max() == 0:
            assert torch.equal(g.cpu().double(), r)
        else:
            assert _rel(g, r) <= _tol(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [2, 4, 8])
def test_steps_continue_a_sequence(gpu, width, dtype):
    """A prompt, then token by token from states in a pool, in any order of slots: the
    sequence's outputs and states."""
    from rnn_kernel_amd import causal_conv, causal_conv_step

    B, T, D = 3, 20, 77
    (x, w, b, s0), _, _ = _inputs(B, T, D, width, dtype, True, True)
    x, w, b, s0 = (t.to(gpu) for t in (x, w, b, s0))
    whole, last = causal_conv(x, w, b, s0, activation="silu")
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device=gpu)
    pool = torch.full((6, width - 1, D), 9.0, dtype=dtype, device=gpu)
    y, pool[slots.long()] = causal_conv(x[:, :5], w, b, s0, activation="silu")
    out = [y] + [causal_conv_step(x[:, t], pool, w, b, activation="silu", slots=slots)[:, None] for t in range(5, T)]
    assert torch.equal(torch.cat(out, 1), whole) and torch.equal(pool[slots.long()], last)
    assert (pool[[1, 3, 5]] == 9.0).all()


def test_padding_and_bad_slots(gpu):
    from rnn_kernel_amd import causal_conv_step

    x, w = torch.randn(4, 70, device=gpu), torch.randn(70, 4, device=gpu)
    pool = torch.randn(3, 3, 70, device=gpu)
    before = pool.clone()
    y = causal_conv_step(x, pool, w, slots=torch.tensor([-1, 2, 3, -7], dtype=torch.int32, device=gpu))
    assert (y[[0, 3]] == 0).all() and y[2].isnan().all() and torch.isfinite(y[1]).all()
    assert torch.equal(pool[:2], before[:2]) and torch.equal(pool[2], torch.cat([before[2, 1:], x[1:2]]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts_and_what_lies_behind(gpu, dtype):
    """Any strides, the bits of the dense call; NaN behind a row's length reaches nothing."""
    from rnn_kernel_amd import causal_conv

    gen = torch.Generator().manual_seed(2)
    wide = torch.randn(2, 50, 90, generator=gen).to(gpu, dtype)
    w, b = torch.randn(40, 4, generator=gen).to(gpu, dtype), torch.randn(40, generator=gen).to(gpu, dtype)
    up = torch.randn(2, 50, 40, generator=gen).to(gpu, dtype)
    lengths = torch.tensor([50, 17], dtype=torch.int32, device=gpu)
    for x in (wide[..., 3:43], wide.transpose(0, 1).contiguous().transpose(0, 1)[..., 1:41], wide[..., ::2][..., :40],
              wide[:, :1, 2:42].expand(2, 50, 40)):
        base, spoilt = x.contiguous().requires_grad_(True), x.detach().clone()
        spoilt[1, 17:] = float("nan")
        bad_up = up.clone()
        bad_up[1, 17:] = float("nan")
        wants = causal_conv(base, w, b, activation="silu", lengths=lengths)
        want = torch.autograd.grad(wants, base, [up, up[:, :3]])[0]
        for leaf, u in ((x.detach().requires_grad_(True), up), (spoilt.requires_grad_(True), bad_up)):
            got = causal_conv(leaf, w, b, activation="silu", lengths=lengths)
            assert torch.equal(got[0], wants[0]) and torch.equal(got[1], wants[1])
            assert torch.equal(torch.autograd.grad(got, leaf, [u, up[:, :3]])[0], want)


def test_without_tokens_or_rows(gpu):
    from rnn_kernel_amd import causal_conv

    w = torch.randn(6, 4, device=gpu, requires_grad=True)
    s0 = torch.randn(2, 3, 6, device=gpu, requires_grad=True)
    y, s = causal_conv(torch.zeros(2, 0, 6, device=gpu), w, None, s0)
    assert y.shape == (2, 0, 6) and torch.equal(s, s0)
    up = torch.randn_like(s)
    dw, ds0 = torch.autograd.grad(s, [w, s0], up)
    assert (dw == 0).all() and torch.equal(ds0, up)
    y, s = causal_conv(torch.zeros(0, 5, 6, device=gpu), w)
    assert y.shape == (0, 5, 6) and s.shape == (0, 3, 6)
    assert (torch.autograd.grad(y.sum(), w)[0] == 0).all()


def test_only_one_output_used(gpu):
    from rnn_kernel_amd import causal_conv

    (x, w, b, s0), up, ups = _inputs(2, 9, 12, 4, torch.float32, True, True)
    ref = [t.double().requires_grad_(True) for t in (x, w, b, s0)]
    for which in (0, 1):
        got = [t.to(gpu).requires_grad_(True) for t in (x, w, b, s0)]
        u = (up, ups)[which]
        g = torch.autograd.grad(causal_conv(*got, activation="silu")[which], got, u.to(gpu))
        r = torch.autograd.grad(_formula(*ref, "silu", None)[which], ref, u.double(), allow_unused=True, materialize_grads=True)
        for a, c in zip(g, r):
            assert torch.allclose(a.cpu().double(), c, rtol=1e-5, atol=1e-6)


def test_gradients_by_differences(gpu):
    """Along the gradient's own direction, by a central difference of step h of float32 values
    summed in float64: truncation O(h^2) with a third derivative of order |up|, rounding
    2^-24 |y| |up| / h; at h = 1e-2 both are under 1e-3 of the derivative, the gradient's
    norm."""
    from rnn_kernel_amd import causal_conv

    args, up, ups = _inputs(2, 11, 9, 4, torch.float32, True, True, seed=4)
    args, up, ups = [t.to(gpu) for t in args], up.to(gpu), ups.to(gpu)
    leaves = [t.clone().requires_grad_(True) for t in args]
    grads = torch.autograd.grad(causal_conv(*leaves, activation="silu"), leaves, [up, ups])
    for i, g in enumerate(grads):
        d, h = g / g.norm(), 1e-2
        side = []
        for sign in (1, -1):
            y, s = causal_conv(*[t + sign * h * d if j == i else t for j, t in enumerate(args)], activation="silu")
            side.append((y.double() * up.double()).sum() + (s.double() * ups.double()).sum())
        assert abs(float((side[0] - side[1]) / (2 * h)) - float(g.norm())) <= 2e-3 * float(g.norm())


def test_graph_replays(gpu):
    from rnn_kernel_amd import causal_conv_step

    x, w = torch.randn(5, 64, device=gpu), torch.randn(64, 4, device=gpu)
    pool, check = (torch.zeros(5, 3, 64, device=gpu) for _ in range(2))
    causal_conv_step(x, check, w, activation="silu")
    check.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = causal_conv_step(x, pool, w, activation="silu")
    pool.zero_()
    for _ in range(4):
        x.copy_(torch.randn(5, 64, device=gpu))
        graph.replay()
        want = causal_conv_step(x, check, w, activation="silu")
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(pool, check)
