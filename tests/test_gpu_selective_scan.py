"""GPU parity of the selective scan with its recurrence in float64, token by token, and of its
gradients with automatic differentiation and with differences.

Tolerances, as 2-norms of the error over 2-norms of the result, set before the first run.
float32: a state is a sum over the tokens before it of decays and inputs; each carries some
twenty roundings of 2^-24 (the exponential's argument, up to |s A| <= 16 here, times 2^-23 at
decays that matter less the larger it is), which add up like their root: 64 * 2^-24 = 4e-6
for values; gradients pass through the recurrence twice, 8e-6; dA and the biases' are sums
of up to 1200 such terms of either sign, what cancels of them at most half their norm: 2e-5.
bfloat16: rounded once, at most 2^-8 per element, and 1.1 times that leaves the float32 part
its room."""
import pytest
import torch

pytestmark = pytest.mark.gpu

VALUE, GRAD, SUMS, BF16 = 4e-6, 8e-6, 2e-5, 1.1 * 2.0 ** -8
NAMES = ("x", "dt", "A", "B", "C", "s0", "skip", "gate", "bias")


def _formula(x, dt, A, B, C, s0, skip, gate, bias, softplus, lengths):
    """float64 recurrence (differentiable)."""
    Bn, T, D = x.shape
    G, N = B.shape[2:]
    s = dt if bias is None else dt + bias
    s = torch.nn.functional.softplus(s, threshold=100.0) if softplus else s
    B, C = (t.repeat_interleave(D // G, 2) for t in (B, C))
    h = x.new_zeros(Bn, D, N) if s0 is None else s0
    out = []
    for t in range(T):
        live = torch.ones(Bn, dtype=torch.bool, device=x.device) if lengths is None else t < lengths
        new = torch.exp(s[:, t, :, None] * A) * h + (s[:, t] * x[:, t])[..., None] * B[:, t]
        h = torch.where(live[:, None, None], new, h)
        y = (C[:, t] * h).sum(-1) + (0 if skip is None else skip * x[:, t])
        y = y if gate is None else y * gate[:, t] * torch.sigmoid(gate[:, t])
        out.append(torch.where(live[:, None], y, torch.zeros_like(y)))
    return (torch.stack(out, 1) if out else x), h


def _inputs(Bn, T, D, N, G, dtype, seed=0, s0=True, skip=True, gate=True, bias=True, device="cpu"):
    gen = torch.Generator().manual_seed(seed + 7 * T + D)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    args = [r(Bn, T, D).to(dtype), (0.5 * r(Bn, T, D)).to(dtype), -torch.exp(0.3 * r(D, N)) * torch.arange(1, N + 1).clamp(max=4),
            r(Bn, T, G, N).to(dtype), r(Bn, T, G, N).to(dtype), r(Bn, D, N) if s0 else None, r(D) if skip else None,
            r(Bn, T, D).to(dtype) if gate else None, r(D) - 1 if bias else None]
    return [t if t is None else t.to(device) for t in args], r(Bn, T, D).to(dtype).to(device), r(Bn, D, N).to(device)


def _call(args, softplus=True, lengths=None):
    from rnn_kernel_amd import selective_scan

    x, dt, A, B, C, s0, skip, gate, bias = args
    return selective_scan(x, dt, A, B, C, s0, skip=skip, gate=gate, dt_bias=bias, softplus=softplus, lengths=lengths)


def _rel(a, ref):
    a, ref = a.detach().double().cpu(), ref.detach().double().cpu()
    assert torch.isfinite(a).all()
    return float((a - ref).norm() / ref.norm().clamp_min(1e-30))


SHAPES = [  # B, T, D, N, G
    (1, 1, 1, 1, 1), (2, 2, 3, 16, 1), (1, 15, 16, 3, 2), (2, 16, 40, 16, 2), (3, 17, 64, 5, 1), (1, 130, 65, 17, 1),
    (2, 200, 96, 24, 3), (1, 90, 130, 32, 2), (1, 70, 33, 33, 1), (2, 33, 24, 64, 1), (1, 600, 48, 16, 1),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("options", [dict(), dict(s0=False, skip=False, gate=False, bias=False), dict(s0=False, bias=False),
                                     dict(gate=False, skip=False)])
@pytest.mark.parametrize("shape", SHAPES)
def test_sequences_and_gradients(gpu, shape, options, dtype):
    print(f"scan {shape} {options} {dtype}", flush=True)
    args, up, ups = _inputs(*shape, dtype, **options, device=gpu)
    ref = [None if t is None else t.double().requires_grad_(True) for t in args]
    got = [None if t is None else t.clone().requires_grad_(True) for t in args]
    out, want = _call(got), _formula(*ref, True, None)
    assert out[0].dtype == dtype and out[1].dtype == torch.float32
    assert _rel(out[0], want[0]) <= (VALUE if dtype == torch.float32 else BF16) and _rel(out[1], want[1]) <= VALUE
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(_call(args), out))
    grads = torch.autograd.grad(out, [t for t in got if t is not None], [up, ups])
    refs = torch.autograd.grad(want, [t for t in ref if t is not None], [up.double(), ups.double()])
    for name, g, r in zip([n for n, t in zip(NAMES, got) if t is not None], grads, refs):
        tol = BF16 if g.dtype == torch.bfloat16 else SUMS if name in ("A", "skip", "bias", "dt") else GRAD
        assert g.shape == r.shape and _rel(g, r) <= tol, (name, _rel(g, r))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(5, 50, 40, 16, 2), (4, 1200, 16, 8, 1)])
def test_rows_of_unequal_length(gpu, shape, dtype):
    """NaN and infinities behind a row's length reach nothing; outputs and gradients there are
    0, an empty row keeps its state."""
    B, T = shape[:2]
    args, up, ups = _inputs(*shape, dtype, device=gpu)
    lengths = torch.tensor([0, 1, T // 2, T, 33][:B], dtype=torch.int32, device=gpu)
    behind = torch.arange(T, device=gpu)[None, :] >= lengths[:, None]
    spoilt = [None if t is None else t.clone() for t in args]
    for i, bad in ((0, float("nan")), (1, float("inf")), (3, float("nan")), (4, float("-inf")), (7, float("nan"))):
        spoilt[i][behind] = bad
    bad_up = up.clone()
    bad_up[behind] = float("nan")
    ref = [t.double().requires_grad_(True) for t in args]
    got = [t.requires_grad_(True) for t in spoilt]
    out, want = _call(got, lengths=lengths), _formula(*ref, True, lengths)
    assert (out[0][behind] == 0).all() and torch.equal(out[1][0], args[5][0])
    assert _rel(out[0], want[0]) <= (VALUE if dtype == torch.float32 else BF16) and _rel(out[1], want[1]) <= VALUE
    grads = torch.autograd.grad(out, got, [bad_up, ups])
    refs = torch.autograd.grad(want, ref, [up.double(), ups.double()])
    for name, g, r in zip(NAMES, grads, refs):
        if g.dim() == up.dim() and name not in ("s0",):
            assert (g[behind] == 0).all(), name
        tol = BF16 if g.dtype == torch.bfloat16 else SUMS if name in ("A", "skip", "bias", "dt") else GRAD
        assert _rel(g, r) <= tol, (name, _rel(g, r))


def test_long_sequence_in_chunks(gpu):
    """Many chunks at once, and the same in two calls that hand the state on."""
    args, up, ups = _inputs(1, 3001, 16, 16, 1, torch.float32, device=gpu)
    x, dt, A, B, C, s0, skip, gate, bias = args
    whole = _call(args)
    want = _formula(*[t.double() for t in args], True, None)
    assert _rel(whole[0], want[0]) <= VALUE and _rel(whole[1], want[1]) <= VALUE
    first = _call([t[:, :1111] if t.dim() > 2 and t.size(1) == 3001 else t for t in args])
    second = _call([t[:, 1111:] if t.dim() > 2 and t.size(1) == 3001 else t for t in args[:5]] + [first[1], skip, gate[:, 1111:], bias])
    assert _rel(torch.cat([first[0], second[0]], 1), want[0]) <= VALUE and _rel(second[1], want[1]) <= VALUE


def test_steps_as_they_are(gpu):
    """Without softplus: steps of either sign and of zero."""
    args, up, ups = _inputs(2, 40, 20, 16, 1, torch.float32, device=gpu)
    args[1][:, 3] = 0
    args[8] = None
    ref = [None if t is None else t.double().requires_grad_(True) for t in args]
    got = [None if t is None else t.clone().requires_grad_(True) for t in args]
    out, want = _call(got, softplus=False), _formula(*ref, False, None)
    # (negative steps make states grow: errors go with the largest)
    assert _rel(out[0], want[0]) <= 4 * VALUE and _rel(out[1], want[1]) <= 4 * VALUE
    grads = torch.autograd.grad(out, [t for t in got if t is not None], [up, ups])
    for g, r in zip(grads, torch.autograd.grad(want, [t for t in ref if t is not None], [up.double(), ups.double()])):
        assert _rel(g, r) <= 4 * SUMS


@pytest.mark.parametrize("raw", [-80.0, -30.0, -12.0, -7.0, -1.0, 0.0, 1.0, 20.0, 90.0])
def test_small_and_large_steps_keep_their_bits(gpu, raw):
    """softplus of what is far below 0 is that small number, not 0: read off x's own input to
    the state."""
    x = torch.ones(1, 1, 16, device=gpu)
    dt = raw + torch.linspace(-0.5, 0.5, 16, device=gpu).view(1, 1, 16)
    one = torch.ones(1, 1, 1, 1, device=gpu)
    from rnn_kernel_amd import selective_scan

    y, h = selective_scan(x, dt, -torch.ones(16, 1, device=gpu), one, one, softplus=True)
    want = torch.nn.functional.softplus(dt.double(), threshold=1000.0)
    # the exponential's argument: |raw| log2(e) rounded, 2^-24 |raw| of the result; ten more roundings
    assert (y.double() / want - 1).abs().max() <= (12 + abs(raw)) * 2.0 ** -23 and torch.equal(h.view(-1), y.view(-1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(3, 20, 40, 16, 2), (2, 9, 33, 5, 1), (4, 12, 70, 64, 1), (1, 5, 8, 1, 1), (2, 7, 17, 30, 1),
                                   (2, 6, 300, 8, 3)])
def test_steps_continue_a_sequence(gpu, shape, dtype):
    from rnn_kernel_amd import selective_step

    B, T, D, N, G = shape
    args, _, _ = _inputs(*shape, dtype, device=gpu)
    x, dt, A, Bm, C, s0, skip, gate, bias = args
    want, last = _formula(*[t.double() for t in args], True, None)
    slots = torch.randperm(B + 2, generator=torch.Generator().manual_seed(1))[:B].to(gpu, torch.int32)
    pool = torch.full((B + 2, D, N), 9.0, device=gpu)
    y, pool[slots.long()] = _call([t[:, :3] if t.dim() > 2 and i != 5 else t for i, t in enumerate(args)])
    out = [y]
    for t in range(3, T):
        out.append(selective_step(x[:, t], dt[:, t], A, Bm[:, t], C[:, t], pool, skip=skip, gate=gate[:, t], dt_bias=bias,
                                  softplus=True, slots=slots)[:, None])
    assert _rel(torch.cat(out, 1), want) <= (VALUE if dtype == torch.float32 else BF16)
    assert _rel(pool[slots.long()], last) <= VALUE
    rest = torch.ones(B + 2, dtype=torch.bool, device=gpu)
    rest[slots.long()] = False
    assert (pool[rest] == 9.0).all()


def test_padding_and_bad_slots(gpu):
    from rnn_kernel_amd import selective_step

    args, _, _ = _inputs(4, 1, 20, 16, 1, torch.float32, device=gpu)
    x, dt, A, B, C, _, skip, _, bias = (t[:, 0] if t.dim() > 2 else t for t in args)
    pool = torch.randn(3, 20, 16, device=gpu)
    before = pool.clone()
    slots = torch.tensor([-1, 2, 3, -7], dtype=torch.int32, device=gpu)
    y = selective_step(x, dt, A, B, C, pool, skip=skip, slots=slots, softplus=True)
    assert (y[[0, 3]] == 0).all() and y[2].isnan().all() and torch.isfinite(y[1]).all()
    assert torch.equal(pool[:2], before[:2]) and not torch.equal(pool[2], before[2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(gpu, dtype):
    """Columns of wider rows, other orders of dimensions, broadcast inputs: the bits of dense
    tensors, and the gradients that belong to them."""
    from rnn_kernel_amd import selective_scan

    gen = torch.Generator().manual_seed(3)
    row = torch.randn(2, 37, 140, generator=gen).to(gpu, dtype)
    A = -torch.rand(40, 8, generator=gen).to(gpu)
    up = torch.randn(2, 37, 40, generator=gen).to(gpu, dtype)

    def parts(row):
        return [row[..., 1:41], row[..., 41:81], row[..., 81:97].unflatten(-1, (2, 8)), row[..., 100:116].unflatten(-1, (2, 8))]

    def grads(x, dt, B, C, leaf):
        y, s = selective_scan(x, dt, A, B, C, gate=dt, softplus=True)
        return y, s, torch.autograd.grad([y, s], leaf, [up, torch.ones_like(s)])[0]

    a = row.clone().requires_grad_(True)
    want = grads(*[t.contiguous() for t in parts(a)], a)
    for turned in (row, row.transpose(0, 1).contiguous().transpose(0, 1), row.permute(2, 0, 1).contiguous().permute(1, 2, 0)):
        leaf = turned.detach().requires_grad_(True)
        assert all(torch.equal(p, q) for p, q in zip(grads(*parts(leaf), leaf), want))
    one = torch.randn(1, 37, 1, 8, generator=gen).to(gpu, dtype).requires_grad_(True)
    x = parts(row)[0]
    wide = one.expand(2, 37, 2, 8)
    y1 = selective_scan(x, x, A, wide, wide, softplus=True)[0]
    y2 = selective_scan(x, x, A, wide.contiguous(), wide.contiguous(), softplus=True)[0]
    assert torch.equal(y1, y2)
    assert torch.equal(torch.autograd.grad(y1, one, up)[0], torch.autograd.grad(y2, one, up)[0])


def test_without_tokens_or_rows(gpu):
    args, _, _ = _inputs(2, 0, 20, 16, 1, torch.float32, device=gpu)
    leaves = [t.requires_grad_(True) for t in args]
    y, s = _call(leaves)
    assert y.shape == (2, 0, 20) and torch.equal(s, args[5])
    up = torch.randn_like(s)
    grads = torch.autograd.grad(s, [leaves[2], leaves[5], leaves[6]], up)
    assert (grads[0] == 0).all() and torch.equal(grads[1], up) and (grads[2] == 0).all()
    args, _, _ = _inputs(0, 5, 20, 16, 1, torch.float32, device=gpu)
    leaves = [t.requires_grad_(True) for t in args]
    y, s = _call(leaves)
    assert y.shape == (0, 5, 20) and s.shape == (0, 20, 16)
    assert (torch.autograd.grad(y.sum(), leaves[2])[0] == 0).all()


def test_only_one_output_used(gpu):
    args, up, ups = _inputs(2, 30, 20, 16, 1, torch.float32, device=gpu)
    for which, u in ((0, up), (1, ups)):
        ref = [t.double().requires_grad_(True) for t in args]
        got = [t.clone().requires_grad_(True) for t in args]
        g = torch.autograd.grad(_call(got)[which], got, u)
        r = torch.autograd.grad(_formula(*ref, True, None)[which], ref, u.double(), allow_unused=True, materialize_grads=True)
        for name, a, b in zip(NAMES, g, r):
            assert (a == 0).all() if (b == 0).all() else _rel(a, b) <= SUMS, name


def test_gradients_by_differences(gpu):
    """Along each gradient's own direction, by a central difference of step h of float32 values
    summed in float64: rounding 2^-22 |y| |up| / h and truncation h^2 of a third derivative
    over the derivative, at h = 1e-2 each under 2e-3 of it (|y| |up| is at most ten times the
    smallest gradient's norm here)."""
    args, up, ups = _inputs(2, 21, 9, 6, 1, torch.float32, seed=5, device=gpu)
    leaves = [t.clone().requires_grad_(True) for t in args]
    grads = torch.autograd.grad(_call(leaves), leaves, [up, ups])
    for i, g in enumerate(grads):
        d, h, side = g / g.norm(), 1e-2, []
        for sign in (1, -1):
            y, s = _call([t + sign * h * d if j == i else t for j, t in enumerate(args)])
            side.append((y.double() * up.double()).sum() + (s.double() * ups.double()).sum())
        assert abs(float((side[0] - side[1]) / (2 * h)) / float(g.norm()) - 1) <= 5e-3, NAMES[i]


def test_same_bits_twice_and_on_another_stream(gpu):
    args, up, ups = _inputs(2, 500, 40, 16, 1, torch.bfloat16, device=gpu)
    leaves = [t.requires_grad_(True) for t in args]

    def both():
        out = _call(leaves)
        return (*out, *torch.autograd.grad(out, leaves, [up, ups]))

    want = both()
    assert all(torch.equal(a, b) for a, b in zip(both(), want))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = both()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(other, want))


def test_graph_replays(gpu):
    args, _, _ = _inputs(2, 300, 40, 16, 1, torch.float32, device=gpu)
    _call(args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, s = _call(args)
    for i in range(4):
        args[0].copy_(torch.randn_like(args[0]))
        graph.replay()
        want = _call(args)
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(s, want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [3, 16, 24, 64])
def test_what_is_not_finite_stays_with_its_token(gpu, dtype, N):
    """An infinite C is in one token's outputs, a NaN of one channel's x in that channel's from its
    token on, a NaN of dy in the gradients up to its token; all else has the bits of a run without."""
    B, T, D, G, at = 2, 45, 24, 2, 21
    args, dy, _ = _inputs(B, T, D, N, G, dtype, seed=5, device=gpu)
    y0, h0 = _call(args)
    others = torch.arange(T, device=gpu) != at

    C = args[4].clone()
    C[0, at, 0, 0] = float("inf")
    y, h = _call([*args[:4], C, *args[5:]])
    assert torch.equal(y[:, others], y0[:, others]) and torch.equal(h, h0) and torch.equal(y[1], y0[1])
    assert not torch.isfinite(y[0, at, :D // G]).any() and torch.equal(y[0, at, D // G:], y0[0, at, D // G:])

    x = args[0].clone()
    x[0, at, 3] = float("nan")
    y, h = _call([x, *args[1:]])
    assert torch.equal(y[:, :at], y0[:, :at]) and torch.equal(y[1], y0[1])
    assert torch.isnan(y[0, at:, 3]).all() and torch.isnan(h[0, 3]).all()
    rest = torch.arange(D, device=gpu) != 3
    assert torch.equal(y[:, :, rest], y0[:, :, rest]) and torch.equal(h[:, rest], h0[:, rest])

    # (the last token of a row: what lies behind is no part of its state)
    lengths = torch.tensor([at + 1, T], dtype=torch.int32, device=gpu)
    Bm = args[3].clone()
    Bm[0, at, 0, 0] = float("inf")
    _, h = _call([*args[:3], Bm, *args[4:]], lengths=lengths)
    _, clean = _call(args, lengths=lengths)
    assert torch.isinf(h[0, :D // G, 0]).all() and torch.equal(h[0, :, 1:], clean[0, :, 1:]) and torch.equal(h[1], clean[1])

    leaves = [t.clone().requires_grad_(True) for t in args]
    y, _ = _call(leaves)
    pick = [leaves[i] for i in (0, 1, 3, 4, 7)]
    want = torch.autograd.grad(y, pick, dy, retain_graph=True)
    dy = dy.clone()
    dy[0, at, 3] = float("nan")
    for got, ref in zip(torch.autograd.grad(y, pick, dy), want):
        assert torch.equal(got[:, at + 1:], ref[:, at + 1:]) and torch.equal(got[1], ref[1])
        if got.shape[2] == D:
            assert torch.equal(got[:, :, rest], ref[:, :, rest]) and torch.isnan(got[0, at, 3])


def test_growing_states_over_chunks(gpu):
    """A above 0: over a chunk (64 tokens here) the growth exp(128) is no float32, but there is no
    state for it until the last 10 tokens, or one so small that the result is a float32."""
    from rnn_kernel_amd import selective_scan

    gen = torch.Generator().manual_seed(2)
    x, B, C = torch.randn(1, 300, 32, generator=gen), torch.randn(1, 300, 1, 16, generator=gen), torch.randn(1, 300, 1, 16, generator=gen)
    x[:, :290] = 0
    dt, A = torch.ones(1, 300, 32), torch.full((32, 16), 2.0)
    want, h = _formula(*(t.double() for t in (x, dt, A, B, C)), None, None, None, None, False, None)
    y, s = selective_scan(*(t.to(gpu) for t in (x, dt, A, B, C)))
    assert _rel(y, want) <= VALUE and _rel(s, h) <= VALUE

    # exp(0.5 * 300) of 1e-30 is exp(81); each of 300 decays is off by 2^-24 or so: 300 * 2^-24 = 1.8e-5
    s0, A = torch.full((1, 32, 16), 1e-30), torch.full((32, 16), 0.5)
    x = torch.zeros_like(x)
    _, h = _formula(*(t.double() for t in (x, dt, A, B, C)), s0.double(), None, None, None, False, None)
    _, s = selective_scan(*(t.to(gpu) for t in (x, dt, A, B, C)), s0.to(gpu))
    assert _rel(s, h) <= 300 * 2.0 ** -24 + VALUE
