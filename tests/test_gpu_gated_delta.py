"""GPU parity of the gated delta rule with its recurrence in float64, token by
token, and with its gradients by automatic differentiation and by differences.

Tolerances, as 2-norms of the error over 2-norms of the result, set before the
first run: float32 results carry some hundred roundings of 2^-24 each, whose sum
grows like its root or, through a chunk's triangular solve, a few times faster:
32 * 2^-24 = 2e-6 for values, twice that for gradients (which pass through the
solve twice), 1e-5 for dg, whose terms cancel.  bfloat16 results are rounded once:
at most 2^-8 per element, and 1.1 times that leaves the float32 part its room.
A gradient of one element can be what is left of terms that cancel (that of a
normalised single element is all but zero): there the bound goes by the terms.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32_VALUE, F32_GRAD, F32_DG, BF16 = 2e-6, 4e-6, 1e-5, 1.1 * 2.0 ** -8


def _oracle(q, k, v, g, beta, s0=None, lengths=None, scale=None, normalize=False):
    """float64 recurrence on the CPU (differentiable)."""
    q, k, v, g, beta = (t.double() for t in (q, k, v, g, beta))
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2:]
    if normalize:
        q, k = (t / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt() for t in (q, k))
    q = q.repeat_interleave(Hv // Hk, 2) * (Dk ** -0.5 if scale is None else scale)
    k = k.repeat_interleave(Hv // Hk, 2)
    S = torch.zeros(B, Hv, Dk, Dv, dtype=torch.float64) if s0 is None else s0.double()
    out = []
    for t in range(T):
        live = torch.ones(B, dtype=torch.bool) if lengths is None else t < lengths
        Sd = S * g[:, t].exp()[..., None, None]
        e = v[:, t] - torch.einsum("bhd,bhde->bhe", k[:, t], Sd)
        Sn = Sd + torch.einsum("bhd,bhe->bhde", k[:, t], beta[:, t, :, None] * e)
        S = torch.where(live[:, None, None, None], Sn, S)
        o = torch.einsum("bhd,bhde->bhe", q[:, t], S)
        out.append(torch.where(live[:, None, None], o, torch.zeros_like(o)))
    return (torch.stack(out, 1) if out else v.new_zeros(v.shape)), S


def _rel(a, ref):
    a, ref = a.detach().double().cpu(), ref.detach().double()
    assert torch.isfinite(a).all()
    return float((a - ref).norm() / ref.norm().clamp_min(1e-30))


def _inputs(B, T, Hk, Hv, Dk, Dv, dtype, seed=0, s0=True, gate_dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed + 7 * T + Dk)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    q, k, v = (r(B, T, Hk, Dk) / Dk ** 0.5).to(dtype), (r(B, T, Hk, Dk) / Dk ** 0.5).to(dtype), r(B, T, Hv, Dv).to(dtype)
    g = torch.nn.functional.logsigmoid(r(B, T, Hv) + 2.0).to(gate_dtype)
    beta = torch.sigmoid(r(B, T, Hv)).to(gate_dtype)
    return q, k, v, g, beta, r(B, Hv, Dk, Dv) if s0 else None


def _tol(dtype):
    return F32_VALUE if dtype == torch.float32 else BF16


SHAPES = [
    # B, T, Hk, Hv, Dk, Dv
    (1, 1, 1, 1, 1, 1),
    (2, 63, 1, 1, 16, 16),
    (2, 64, 1, 2, 64, 64),
    (1, 65, 2, 2, 17, 33),
    (3, 130, 2, 4, 128, 128),
    (1, 200, 1, 3, 96, 129),
    (1, 97, 2, 2, 160, 24),
    (2, 129, 1, 1, 256, 72),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_rule_matches_the_recurrence(gpu, shape, normalize, dtype):
    from rnn_kernel_amd import gated_delta_rule

    print(f"rule {shape} normalize={normalize} {dtype}", flush=True)
    x = _inputs(*shape, dtype)
    o, s = gated_delta_rule(*[t.to(gpu) for t in x], normalize=normalize)
    ro, rs = _oracle(*x, normalize=normalize)
    assert o.dtype == dtype and s.dtype == torch.float32
    assert _rel(o, ro) <= _tol(dtype) and _rel(s, rs) <= F32_VALUE


def _grads(fn, tensors, do, ds):
    leaves = [t.detach().clone().requires_grad_(True) for t in tensors]
    o, s = fn(*leaves)
    loss = [(t, gr) for t, gr in ((o, do), (s, ds)) if gr is not None]
    return torch.autograd.grad([t for t, _ in loss], leaves, [gr for _, gr in loss])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("shape", SHAPES[1:] + [(2, 1, 1, 2, 16, 16)])
def test_gradients_match_automatic_differentiation(gpu, shape, normalize, dtype):
    from rnn_kernel_amd import gated_delta_rule

    print(f"gradients {shape} normalize={normalize} {dtype}", flush=True)
    B, T, Hk, Hv, Dk, Dv = shape
    x = _inputs(*shape, dtype, seed=3)
    gen = torch.Generator().manual_seed(5)
    do, ds = torch.randn(B, T, Hv, Dv, generator=gen).to(dtype), torch.randn(B, Hv, Dk, Dv, generator=gen)
    ref = _grads(lambda *a: _oracle(*a, normalize=normalize), [t.double() for t in x], do.double(), ds.double())
    got = _grads(lambda *a: gated_delta_rule(*a, normalize=normalize), [t.to(gpu) for t in x], do.to(gpu), ds.to(gpu))
    for name, a, r, t in zip(("dq", "dk", "dv", "dg", "dbeta", "ds0"), got, ref, x):
        assert a.dtype == t.dtype and a.shape == t.shape
        tol = F32_DG if name == "dg" else F32_GRAD if t.dtype == torch.float32 else BF16
        assert _rel(a, r) <= tol, (name, _rel(a, r))


@pytest.mark.parametrize("normalize", [False, True])
def test_gradients_of_single_elements(gpu, normalize):
    """Every tensor has one element: each gradient is a sum of a few products of
    the others, none larger than `terms`."""
    from rnn_kernel_amd import gated_delta_rule

    x = _inputs(1, 1, 1, 1, 1, 1, torch.float32, seed=3)
    do, ds = torch.full((1, 1, 1, 1), 0.7), torch.full((1, 1, 1, 1), -1.3)
    ref = _grads(lambda *a: _oracle(*a, normalize=normalize), [t.double() for t in x], do.double(), ds.double())
    got = _grads(lambda *a: gated_delta_rule(*a, normalize=normalize), [t.to(gpu) for t in x], do.to(gpu), ds.to(gpu))
    size = 1.0 + max(float(t.abs().max()) for t in x)
    inverse = max(1.0, *(1.0 / float(t.abs().max()) for t in x[:2])) if normalize else 1.0
    terms = 2.0 * size ** 4 * inverse
    for name, a, r in zip(("dq", "dk", "dv", "dg", "dbeta", "ds0"), got, ref):
        assert float((a.double().cpu() - r).abs().max()) <= 32 * 2.0 ** -24 * terms, name


@pytest.mark.parametrize("B,T,Hk,Hv,Dk,Dv,slots", [(1, 1, 1, 1, 1, 1, 1), (3, 1, 2, 4, 64, 64, 5), (5, 1, 1, 3, 128, 128, 9),
                                                   (2, 1, 3, 3, 17, 35, 2), (4, 1, 2, 2, 256, 130, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("normalize", [False, True])
def test_step_matches_the_recurrence(gpu, B, T, Hk, Hv, Dk, Dv, slots, dtype, normalize):
    from rnn_kernel_amd import gated_delta_step

    print(f"step {(B, Hk, Hv, Dk, Dv, slots)} {dtype}", flush=True)
    q, k, v, g, beta, _ = _inputs(B, 1, Hk, Hv, Dk, Dv, dtype, seed=11)
    gen = torch.Generator().manual_seed(1)
    pool = torch.randn(slots, Hv, Dk, Dv, generator=gen)
    at = torch.randperm(slots, generator=gen)[:B]
    ro, rs = _oracle(q, k, v, g, beta, pool[at], normalize=normalize)
    state = pool.to(gpu)
    o = gated_delta_step(*[t[:, 0].to(gpu) for t in (q, k, v, g, beta)], state, slots=at.to(gpu, torch.int32),
                         normalize=normalize)
    want = pool.double()
    want[at] = rs
    assert _rel(o, ro[:, 0]) <= _tol(dtype) and _rel(state, want) <= F32_VALUE
    rest = [i for i in range(slots) if i not in at.tolist()]
    assert torch.equal(state.cpu()[rest], pool[rest])


def test_differences_agree_with_the_gradients(gpu):
    """Central differences of the kernel's own outputs, in the direction of the
    gradient: the step of 2^-6 leaves a truncation of its square and a rounding of
    2^-24 over it, both under 2e-3 of the slope."""
    from rnn_kernel_amd import gated_delta_rule

    B, T, Hk, Hv, Dk, Dv = 1, 70, 1, 2, 24, 20
    x = [t.to(gpu) for t in _inputs(B, T, Hk, Hv, Dk, Dv, torch.float32, seed=9)]
    gen = torch.Generator().manual_seed(6)
    do, ds = torch.randn(B, T, Hv, Dv, generator=gen).to(gpu), torch.randn(B, Hv, Dk, Dv, generator=gen).to(gpu)
    grads = _grads(lambda *a: gated_delta_rule(*a), x, do, ds)

    def loss(args):
        o, s = gated_delta_rule(*args)
        return float((o.double() * do).sum() + (s.double() * ds).sum())

    for i, gr in enumerate(grads):
        step = gr / gr.norm() * 2.0 ** -6
        up, down = ([t + sign * step if j == i else t for j, t in enumerate(x)] for sign in (1, -1))
        slope = (loss(up) - loss(down)) / 2 / 2.0 ** -6
        assert abs(slope - float(gr.norm())) <= 2e-3 * float(gr.norm()), i


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_end_at_their_lengths(gpu, dtype):
    """What lies behind a row's length is NaN and infinite: nothing of it may reach
    a result, the outputs and gradients there are exactly 0, an empty row keeps its
    state.  Lengths outside 0 .. T are clamped."""
    from rnn_kernel_amd import gated_delta_rule

    B, T, Hk, Hv, Dk, Dv = 7, 150, 1, 2, 64, 40
    x = list(_inputs(B, T, Hk, Hv, Dk, Dv, dtype, seed=2))
    lens = torch.tensor([0, 1, 64, 65, 150, 400, -3], dtype=torch.int32)
    clamped = lens.clamp(0, T)
    gen = torch.Generator().manual_seed(8)
    do, ds = torch.randn(B, T, Hv, Dv, generator=gen).to(dtype), torch.randn(B, Hv, Dk, Dv, generator=gen)
    ref_o, ref_s = _oracle(*x, lengths=clamped)
    ref = _grads(lambda *a: _oracle(*a, lengths=clamped), [t.double() for t in x], do.double(), ds.double())
    behind = torch.arange(T)[None] >= clamped[:, None]
    for i, bad in zip(range(5), (float("nan"), float("inf"), float("nan"), float("nan"), float("inf"))):
        x[i][behind] = bad
    do[behind] = float("nan")
    args = [t.to(gpu) for t in x]
    o, s = gated_delta_rule(*args, lengths=lens.to(gpu))
    assert _rel(o, ref_o) <= _tol(dtype) and _rel(s, ref_s) <= F32_VALUE
    assert (o.cpu()[behind] == 0).all()
    assert torch.equal(s[0].cpu(), x[5][0]) and torch.equal(s[6].cpu(), x[5][6])
    got = _grads(lambda *a: gated_delta_rule(*a, lengths=lens.to(gpu)), args, do.to(gpu), ds.to(gpu))
    for name, a, r, t in zip(("dq", "dk", "dv", "dg", "dbeta", "ds0"), got, ref, x):
        assert _rel(a, r) <= (F32_DG if name == "dg" else F32_GRAD if t.dtype == torch.float32 else BF16), name
        if name != "ds0":
            assert (a.cpu()[behind] == 0).all(), name


def test_no_tokens_and_no_rows(gpu):
    from rnn_kernel_amd import gated_delta_rule, gated_delta_step

    q, k, v, g, beta, s0 = (t.to(gpu) for t in _inputs(2, 0, 1, 2, 16, 8, torch.bfloat16))
    s0.requires_grad_(True)
    o, s = gated_delta_rule(q, k, v, g, beta, s0)
    assert o.shape == (2, 0, 2, 8) and torch.equal(s, s0)
    ds = torch.randn_like(s)
    assert torch.equal(torch.autograd.grad(s, s0, ds)[0], ds)
    o, s = gated_delta_rule(q, k, v, g, beta)
    assert (s == 0).all()
    x = [t.to(gpu) for t in _inputs(0, 3, 1, 2, 16, 8, torch.bfloat16)]
    o, s = gated_delta_rule(*x)
    assert o.shape == (0, 3, 2, 8) and s.shape == (0, 2, 16, 8)
    o = gated_delta_step(*[t[:, 0] for t in x[:5]], torch.randn(4, 2, 16, 8, device=gpu))
    assert o.shape == (0, 2, 8)


def test_unused_outputs_and_partial_gradients(gpu):
    from rnn_kernel_amd import gated_delta_rule

    shape = (2, 70, 1, 2, 32, 16)
    x = [t.to(gpu) for t in _inputs(*shape, torch.float32, seed=4)]
    gen = torch.Generator().manual_seed(3)
    do, ds = torch.randn(2, 70, 2, 16, generator=gen), torch.randn(2, 2, 32, 16, generator=gen)
    host = [t.cpu().double() for t in x]
    for use_o, use_s in ((do, None), (None, ds)):
        got = _grads(lambda *a: gated_delta_rule(*a), x, None if use_o is None else use_o.to(gpu),
                     None if use_s is None else use_s.to(gpu))
        loss = lambda o, s: (o * use_o.double()).sum() if use_s is None else (s * use_s.double()).sum()  # noqa: E731
        leaves = [t.clone().requires_grad_(True) for t in host]
        ref = torch.autograd.grad(loss(*_oracle(*leaves)), leaves, allow_unused=True)
        for a, r in zip(got, ref):
            if r is None or float(r.norm()) == 0:
                assert (a == 0).all()
            else:
                assert _rel(a, r) <= F32_DG
    v = x[2].clone().requires_grad_(True)
    o, _ = gated_delta_rule(x[0], x[1], v, *x[3:])
    assert _rel(torch.autograd.grad(o, v, do.to(gpu))[0],
                torch.autograd.grad(_oracle(host[0], host[1], (hv := host[2].clone().requires_grad_(True)), *host[3:])[0], hv,
                                    do.double())[0]) <= F32_GRAD


def test_views_and_broadcast_inputs(gpu):
    """Columns of one projection, tokens before batch, a head size that is no
    multiple of the loads' width, expanded gates: strides only, same results bit for
    bit, and the gradient of what is expanded is the sum over its copies."""
    from rnn_kernel_amd import gated_delta_rule, gated_delta_step

    for Dk, Dv, dtype in ((64, 48, torch.bfloat16), (33, 19, torch.bfloat16), (33, 19, torch.float32)):
        B, T, Hk, Hv = 2, 100, 2, 4
        q, k, v, g, beta, s0 = (t.to(gpu) for t in _inputs(B, T, Hk, Hv, Dk, Dv, dtype, seed=1))
        want = gated_delta_rule(q, k, v, g, beta, s0)
        row = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], -1).transpose(0, 1).contiguous().transpose(0, 1)
        qs, ks, vs = row.split([Hk * Dk, Hk * Dk, Hv * Dv], -1)
        views = (qs.unflatten(-1, (Hk, Dk)), ks.unflatten(-1, (Hk, Dk)), vs.unflatten(-1, (Hv, Dv)),
                 g.transpose(1, 2).contiguous().transpose(1, 2), beta.transpose(0, 2).contiguous().transpose(0, 2), s0)
        for a, b in zip(gated_delta_rule(*views), want):
            assert torch.equal(a, b)
        # the elements of a head apart: copied, not refused
        apart = q.transpose(2, 3).contiguous().transpose(2, 3)
        assert torch.equal(gated_delta_rule(apart, k, v, g, beta, s0)[0], want[0])
        p0, p1 = s0.clone(), s0.clone()
        a = gated_delta_step(*[t[:, 3] for t in (q, k, v, g, beta)], p0)
        b = gated_delta_step(*[t[:, 3] for t in views[:5]], p1)
        assert torch.equal(a, b) and torch.equal(p0, p1)
        one = g[:, :, :1].clone().requires_grad_(True)
        full = one.detach().expand(B, T, Hv).contiguous().requires_grad_(True)
        o1 = gated_delta_rule(q, k, v, one.expand(B, T, Hv), beta, s0)[0]
        o2 = gated_delta_rule(q, k, v, full, beta, s0)[0]
        assert torch.equal(o1, o2)
        up = torch.randn_like(o1)
        d1, d2 = torch.autograd.grad(o1, one, up)[0], torch.autograd.grad(o2, full, up)[0].sum(-1, keepdim=True)
        assert torch.allclose(d1, d2, rtol=1e-5, atol=1e-5)


def test_gates_of_either_type_closed_gates_and_no_writes(gpu):
    """bfloat16 gates, a gate that closes (g = -inf empties the state), strong
    decays and beta = 0, forward and backward."""
    from rnn_kernel_amd import gated_delta_rule, gated_delta_step

    B, T, Hk, Hv, Dk, Dv = 2, 140, 1, 2, 48, 32
    for gate_dtype in (torch.float32, torch.bfloat16):
        q, k, v, g, beta, s0 = _inputs(B, T, Hk, Hv, Dk, Dv, torch.bfloat16, seed=5, gate_dtype=gate_dtype)
        g[:, 20], g[:, 21:30], g[0, 64], g[1, 127] = float("-inf"), -90.0, float("-inf"), -300.0
        beta[:, 10:14] = 0
        beta[:, 70] = 0
        x = (q, k, v, g, beta, s0)
        o, s = gated_delta_rule(*[t.to(gpu) for t in x])
        ro, rs = _oracle(*x)
        assert _rel(o, ro) <= BF16 and _rel(s, rs) <= F32_VALUE
        gen = torch.Generator().manual_seed(4)
        do, ds = torch.randn(B, T, Hv, Dv, generator=gen).bfloat16(), torch.randn(B, Hv, Dk, Dv, generator=gen)
        fin = [t.double() for t in x]
        fin[3] = fin[3].clamp_min(-200.0)  # where the oracle's own exp(g) S is not 0 times a slope
        ref = _grads(lambda *a: _oracle(*a), fin, do.double(), ds.double())
        got = _grads(lambda *a: gated_delta_rule(*a), [t.to(gpu) for t in x], do.to(gpu), ds.to(gpu))
        for name, a, r, t in zip(("dq", "dk", "dv", "dg", "dbeta", "ds0"), got, ref, x):
            assert _rel(a, r) <= (BF16 if t.dtype == torch.bfloat16 else F32_DG), name
        state = s0.to(gpu).clone()
        o = gated_delta_step(*[t[:, 20].to(gpu) for t in x[:5]], state)
        ro, rs = _oracle(*[t[:, 20:21] for t in x[:5]], s0)
        assert _rel(o, ro[:, 0]) <= BF16 and _rel(state, rs) <= F32_VALUE


def test_step_with_padding_and_bad_slots(gpu):
    from rnn_kernel_amd import gated_delta_step

    q, k, v, g, beta, _ = (None if t is None else t.to(gpu) for t in _inputs(4, 1, 1, 2, 32, 20, torch.float32, s0=False))
    pool = torch.randn(3, 2, 32, 20, device=gpu)
    state = pool.clone()
    slots = torch.tensor([2, -1, 7, 0], dtype=torch.int32, device=gpu)
    o = gated_delta_step(*[t[:, 0] for t in (q, k, v, g, beta)], state, slots=slots)
    assert (o[1] == 0).all() and torch.isnan(o[2]).all() and torch.isfinite(o[[0, 3]]).all()
    assert torch.equal(state[1], pool[1]) and not torch.equal(state[0], pool[0]) and not torch.equal(state[2], pool[2])


def test_steps_continue_a_sequence(gpu):
    """A prompt, then its continuation token by token, against the whole."""
    from rnn_kernel_amd import gated_delta_rule, gated_delta_step

    x = _inputs(2, 100, 2, 2, 64, 64, torch.float32, seed=12)
    ro, rs = _oracle(*x)
    q, k, v, g, beta, s0 = (t.to(gpu) for t in x)
    o, state = gated_delta_rule(*[t[:, :90] for t in (q, k, v, g, beta)], s0)
    outs = [o] + [gated_delta_step(*[t[:, i] for t in (q, k, v, g, beta)], state)[:, None] for i in range(90, 100)]
    assert _rel(torch.cat(outs, 1), ro) <= F32_VALUE and _rel(state, rs) <= F32_VALUE


def test_results_are_bitwise_reproducible_on_any_stream(gpu):
    from rnn_kernel_amd import gated_delta_rule

    x = [t.to(gpu) for t in _inputs(2, 300, 2, 4, 64, 64, torch.bfloat16, seed=6)]
    gen = torch.Generator().manual_seed(2)
    do, ds = torch.randn(2, 300, 4, 64, generator=gen).bfloat16().to(gpu), torch.randn(2, 4, 64, 64, generator=gen).to(gpu)
    torch.cuda.synchronize()
    first = _grads(lambda *a: gated_delta_rule(*a, normalize=True), x, do, ds)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(stream):
            again = _grads(lambda *a: gated_delta_rule(*a, normalize=True), x, do, ds)
        stream.synchronize()
        for a, b in zip(first, again):
            assert torch.equal(a, b)


def test_graph_replays_match(gpu):
    from rnn_kernel_amd import gated_delta_rule, gated_delta_step

    q, k, v, g, beta, s0 = (t.to(gpu) for t in _inputs(2, 130, 1, 2, 64, 32, torch.bfloat16, seed=6))
    state = s0.clone()
    with torch.no_grad():
        gated_delta_rule(q, k, v, g, beta, s0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o, s = gated_delta_rule(q, k, v, g, beta, s0)
            so = gated_delta_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], state)
        for seed in range(3):
            gen = torch.Generator().manual_seed(seed)
            v.copy_(torch.randn(v.shape, generator=gen).to(v))
            state.copy_(s0)
            graph.replay()
            torch.cuda.synchronize()
            wo, ws = gated_delta_rule(q, k, v, g, beta, s0)
            ref_state = s0.clone()
            wso = gated_delta_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], ref_state)
            torch.cuda.synchronize()
            assert torch.equal(o, wo) and torch.equal(s, ws) and torch.equal(so, wso) and torch.equal(state, ref_state)
