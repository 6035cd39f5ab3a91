"""The selective scan, the convolution, layer norm and the cross entropy where calls meet
autograd, graphs, streams and memory: saved-tensor hooks, forward-mode tangents, states that
count as changed, a captured training step, offsets past 2^31, refusals of tensors that do
not fit.  What is compared is compared bit by bit."""
import pytest
import torch
from torch.autograd import forward_ad


def _inputs(device, dtype=torch.float32):
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    like = lambda *s: r(*s).to(device, dtype)  # noqa: E731
    scan = [like(2, 21, 24), like(2, 21, 24), -torch.rand(24, 5, generator=gen).to(device), like(2, 21, 2, 5), like(2, 21, 2, 5),
            r(2, 24, 5).to(device), r(24).to(device), like(2, 21, 24), r(24).to(device)]
    conv = [like(2, 21, 24), like(24, 4), like(24), like(2, 3, 24)]
    norm = [like(9, 40), like(40), like(40)]
    loss = [like(9, 40), like(70, 40), like(70)]
    return scan, conv, norm, loss


def _calls(device, dtype=torch.float32):
    """(call, its tensors) of each operator that has gradients."""
    from rnn_kernel_amd import causal_conv, layer_norm, linear_cross_entropy, selective_scan

    scan, conv, norm, loss = _inputs(device, dtype)
    lengths = torch.tensor([21, 6], dtype=torch.int32, device=device)
    target = torch.tensor([0, 69, 5, -100, 7, 8, 9, -100, 11], device=device)

    def scanned(x, dt, A, B, C, s0, skip, gate, bias):
        return selective_scan(x, dt, A, B, C, s0, skip=skip, gate=gate, dt_bias=bias, softplus=True, lengths=lengths)

    return [(scanned, scan), (lambda *a: causal_conv(*a, activation="silu", lengths=lengths), conv),
            (lambda *a: (layer_norm(*a),), norm), (lambda x, w, b: (linear_cross_entropy(x, w, target, b),), loss)]


def _steps(device):
    from rnn_kernel_amd import causal_conv_step, selective_step

    scan, conv, _, _ = _inputs(device)
    x, dt, A, B, C, s0, skip, gate, bias = (t[:, 0] if i in (0, 1, 3, 4, 7) else t for i, t in enumerate(scan))
    return [(lambda x, dt, A, B, C, s, skip, gate, bias: selective_step(x, dt, A, B, C, s, skip=skip, gate=gate, dt_bias=bias),
             [x, dt, A, B, C, s0, skip, gate, bias], 5),
            (lambda x, s, w, b: causal_conv_step(x, s, w, b), [conv[0][:, 0], conv[3], conv[1], conv[2]], 1)]


def _refuses_tangents(device):
    for call, tensors in _calls(device) + [s[:2] for s in _steps(device)]:
        with forward_ad.dual_level():
            for i, t in enumerate(tensors):
                args = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else u for j, u in enumerate(tensors)]
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call(*args)


def test_tangents_are_refused():
    _refuses_tangents("cpu")


@pytest.mark.gpu
def test_tangents_are_refused_on_the_gpu(gpu):
    _refuses_tangents(gpu)
    for call, tensors in _calls(gpu):
        with forward_ad.dual_level():
            call(*tensors)


def _apart(t):
    """The same values, neighbouring elements of the last dimension two apart."""
    return torch.stack([t, torch.zeros_like(t)], -1)[..., 0]


def _gradients(call, tensors):
    leaves = [t.detach().clone().requires_grad_(True) for t in tensors]
    out = call(*leaves)
    return out, leaves


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_under_saved_tensor_hooks(gpu, dtype):
    saved = torch.autograd.graph.saved_tensors_hooks
    for call, tensors in _calls(gpu, dtype):
        out, leaves = _gradients(call, tensors)
        up = [torch.ones_like(t) for t in out]
        want = torch.autograd.grad(out, leaves, up)
        for hooks in (saved(lambda t: t.detach().contiguous(), lambda t: t), saved(lambda t: t.detach(), _apart),
                      torch.autograd.graph.save_on_cpu()):
            with hooks:
                out, leaves = _gradients(call, tensors)
            for a, b in zip(torch.autograd.grad(out, leaves, up), want):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_saved_tensors_that_come_back_as_something_else_are_refused(gpu):
    for call, tensors in _calls(gpu):
        for change in (lambda t: t.cpu(), lambda t: t[..., :1], lambda t: t.to(torch.float64)):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), change):
                out, leaves = _gradients(call, tensors)
            with pytest.raises(RuntimeError, match="a saved tensor came back as"):
                torch.autograd.grad(out[0].sum(), leaves)


@pytest.mark.gpu
def test_second_derivatives_are_refused(gpu):
    for call, tensors in _calls(gpu):
        out, leaves = _gradients(call, tensors)
        g = torch.autograd.grad(out[0].square().sum(), leaves[0], create_graph=True)[0]
        with pytest.raises(RuntimeError):
            g.sum().backward()


@pytest.mark.gpu
def test_a_backward_twice_gives_the_same(gpu):
    for call, tensors in _calls(gpu):
        out, leaves = _gradients(call, tensors)
        up = [torch.ones_like(t) for t in out]
        first = torch.autograd.grad(out, leaves, up, retain_graph=True)
        for a, b in zip(torch.autograd.grad(out, leaves, up), first):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_steps_count_as_changes_and_have_no_gradients(gpu):
    w = torch.ones((), device=gpu, requires_grad=True)
    for call, tensors, at in _steps(gpu):
        y = (w * tensors[at]).sum()
        call(*tensors)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        for i, t in enumerate(tensors):
            args = [u.clone().requires_grad_(True) if j == i else u for j, u in enumerate(tensors)]
            with pytest.raises(RuntimeError, match="has no gradients"):
                call(*args)
            with torch.no_grad():
                call(*args)


@pytest.mark.gpu
def test_inputs_changed_before_the_backward_are_noticed(gpu):
    for call, tensors in _calls(gpu):
        leaves = [t.detach().clone() for t in tensors]
        leaves[1].requires_grad_(True)
        out = call(*leaves)
        with torch.no_grad():
            leaves[0].zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out[0].sum(), leaves[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_captured_training_pass_replays(gpu, dtype):
    """Forward and backward of each operator in a graph, replayed on other inputs between eager
    passes: the eager pass's bits."""
    for call, tensors in _calls(gpu, dtype):
        fixed = [t.clone() for t in tensors]

        def both():
            leaves = [t.detach().requires_grad_(True) for t in fixed]
            out = call(*leaves)
            return (*(t.detach() for t in out), *torch.autograd.grad(out, leaves, [torch.ones_like(t) for t in out]))

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            both()
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = both()
        for i in range(4):
            for t in fixed:
                if t.dim() != 2 or t.size(-1) != 5:  # (the scan's decays stay below 0)
                    t.copy_(torch.randn_like(t))
            graph.replay()
            got = [t.clone() for t in held]
            want = both()
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_two_graphs_and_two_streams_at_once(gpu):
    """Calls on two streams, and two graphs, do not share memory."""
    from rnn_kernel_amd import linear_cross_entropy, selective_scan

    gen = torch.Generator().manual_seed(3)
    sets = []
    for _ in range(2):
        x, dt = (torch.randn(1, 2000, 64, generator=gen).to(gpu) for _ in range(2))
        B, C = (torch.randn(1, 2000, 1, 16, generator=gen).to(gpu) for _ in range(2))
        A = -torch.rand(64, 16, generator=gen).to(gpu)
        sets.append((x, dt, A, B, C, torch.randn(300, 64, generator=gen).to(gpu), torch.randn(5000, 64, generator=gen).to(gpu),
                     torch.randint(0, 5000, (300,), generator=gen).to(gpu)))

    def run(x, dt, A, B, C, h, w, t):
        return (*selective_scan(x, dt, A, B, C, softplus=True), linear_cross_entropy(h, w, t))

    want = [run(*s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[], []]
    for _ in range(5):
        for i, (s, stream) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(stream):
                got[i].append(run(*s))
    torch.cuda.synchronize()
    for w, all_ in zip(want, got):
        for g in all_:
            assert all(torch.equal(a, b) for a, b in zip(g, w))
    graphs, held = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(run(*s))
    for order in ((0, 1), (1, 0), (1, 1), (0, 0)):
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in order:
            assert all(torch.equal(a, b) for a, b in zip(held[i], want[i]))


@pytest.mark.gpu
def test_states_far_into_a_pool(gpu):
    from rnn_kernel_amd import causal_conv_step, selective_step

    gen = torch.Generator().manual_seed(4)
    D, N = 2048, 64
    count = 2 ** 31 // (D * N) + 2
    x, dt = (torch.randn(2, D, generator=gen).to(gpu) for _ in range(2))
    A, B, C = -torch.rand(D, N, generator=gen).to(gpu), *(torch.randn(2, 1, N, generator=gen).to(gpu) for _ in range(2))
    near = torch.randn(2, D, N, generator=gen).to(gpu)
    pool = torch.empty(count, D, N, device=gpu)
    pool[count - 1], pool[1], pool[0] = near[0], near[1], 0.0
    slots = torch.tensor([count - 1, 1], dtype=torch.int32, device=gpu)
    far = selective_step(x, dt, A, B, C, pool, softplus=True, slots=slots)
    assert torch.equal(far, selective_step(x, dt, A, B, C, near, softplus=True))
    assert torch.equal(pool[count - 1], near[0]) and torch.equal(pool[1], near[1]) and not pool[0].any()
    del pool
    w, near = torch.randn(8192, 3, generator=gen).to(gpu), torch.randn(2, 2, 8192, generator=gen).to(gpu)
    count = 2 ** 31 // (2 * 8192) + 2
    pool = torch.empty(count, 2, 8192, device=gpu)
    pool[count - 1], pool[1], pool[0] = near[0], near[1], 0.0
    x, slots = torch.randn(2, 8192, generator=gen).to(gpu), torch.tensor([count - 1, 1], dtype=torch.int32, device=gpu)
    assert torch.equal(causal_conv_step(x, pool, w, slots=slots), causal_conv_step(x, near, w))
    assert torch.equal(pool[count - 1], near[0]) and torch.equal(pool[1], near[1]) and not pool[0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("step", [2 ** 21, 2 ** 25])
def test_tokens_far_apart(gpu, step):
    """Up to 2^21 elements from token to token as they are, farther copied."""
    from rnn_kernel_amd import causal_conv, selective_scan

    gen = torch.Generator().manual_seed(5)
    T = 2 ** 31 // step + 6
    base = torch.empty((T - 1) * step + 48, dtype=torch.bfloat16, device=gpu)
    far = base.as_strided((1, T, 48), (base.numel(), step, 1))
    far.copy_(torch.randn(1, T, 48, generator=gen).bfloat16())
    A, w = -torch.rand(16, 8, generator=gen).to(gpu), torch.randn(48, 4, generator=gen).bfloat16().to(gpu)

    assert far.stride(1) * (T - 1) > 2 ** 31
    out = []
    for t in (far, far.contiguous()):
        parts = [t[..., :16], t[..., 16:32], t[..., 32:40].unsqueeze(2), t[..., 40:].unsqueeze(2), t]
        leaves = [p.detach().requires_grad_(True) for p in parts]
        y, s = selective_scan(*leaves[:2], A, *leaves[2:4], softplus=True)
        z, last = causal_conv(leaves[4], w, activation="silu")
        results = (y, s, z, last)
        # (the gradients of the far tensors are dense)
        out.append((*results, *torch.autograd.grad(results, leaves, [torch.ones_like(r) for r in results])))
    for a, b in zip(*out):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_more_than_2_to_the_31_elements(gpu):
    """Rows of a norm and of a vocabulary past 2^31 elements."""
    from rnn_kernel_amd import layer_norm, linear_cross_entropy

    rows, size = 2 ** 31 // 16384 + 3, 16384
    x = torch.empty(rows, size, dtype=torch.bfloat16, device=gpu)
    gen = torch.Generator().manual_seed(6)
    last = torch.randn(3, size, generator=gen).bfloat16().to(gpu)
    x[:-3], x[-3:] = 0.0, last
    assert torch.equal(layer_norm(x)[-3:], layer_norm(last))
    del x
    V, K = 2 ** 20 + 70, 2048
    w = torch.zeros(V, K, dtype=torch.bfloat16, device=gpu)
    w[-70:] = 0.02 * torch.randn(70, K, generator=gen).bfloat16().to(gpu)
    x = torch.randn(3, K, generator=gen).bfloat16().to(gpu)
    target = torch.tensor([V - 1, V - 70, 5], device=gpu)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    loss = linear_cross_entropy(*leaves, target, reduction="none")
    z = x.detach().double() @ w[-70:].detach().double().t()
    lse = torch.log(z.exp().sum(-1) + (V - 70))
    want = lse - torch.stack([z[0, -1], z[1, 0], torch.zeros((), dtype=torch.float64, device=gpu)])
    # (a sum of a million float32 exponentials in levels: 2^-24 times some 40 roundings, of 14)
    assert (loss.double() - want).abs().max() <= 4e-6
    dx, dw = torch.autograd.grad(loss, leaves, torch.ones_like(loss))
    p = torch.exp(z - lse[:, None])
    p[0, -1] -= 1
    p[1, 0] -= 1
    ref = p.t() @ x.detach().double()
    assert (dw[-70:].double() - ref).norm() <= 1.1 * 2 ** 0.5 * 2.0 ** -8 * ref.norm()
    assert torch.isfinite(dx).all() and dw[5].abs().max() > 0


def _refusals(device):
    from rnn_kernel_amd import (causal_conv, causal_conv_step, layer_norm, linear_cross_entropy, selective_scan, selective_step)

    (x, dt, A, B, C, s0, skip, gate, bias), (cx, cw, cb, cs), (nx, nw, nb), (lx, lw, lb) = _inputs(device)
    t = torch.zeros(9, dtype=torch.int64, device=device)
    ints = torch.zeros(2, dtype=torch.int32, device=device)
    step = [x[:, 0], dt[:, 0], A, B[:, 0], C[:, 0]]
    half = lambda a: a.to(torch.float16)  # noqa: E731
    yield RuntimeError, "dt must be float32", lambda: selective_scan(x, dt.bfloat16(), A, B, C)
    yield RuntimeError, "x must be float32 or bfloat16", lambda: selective_scan(half(x), half(dt), A, half(B), half(C))
    yield RuntimeError, "A must be float32", lambda: selective_scan(x, dt, A.double(), B, C)
    yield RuntimeError, "skip must be float32", lambda: selective_scan(x, dt, A, B, C, skip=skip.bfloat16())
    yield RuntimeError, "initial_state must be float32", lambda: selective_scan(x, dt, A, B, C, s0.bfloat16())
    yield RuntimeError, "lengths must be an int32", lambda: selective_scan(x, dt, A, B, C, lengths=ints.long())
    yield ValueError, "lengths must have shape", lambda: selective_scan(x, dt, A, B, C, lengths=ints[:1])
    yield ValueError, "x must have shape", lambda: selective_scan(x[0], dt[0], A, B, C)
    yield ValueError, "A must have shape", lambda: selective_scan(x, dt, A[:3], B, C)
    yield ValueError, "A must have shape", lambda: selective_scan(x, dt, torch.zeros(24, 65, device=device), B, C)
    yield ValueError, "B must have shape", lambda: selective_scan(x, dt, A, B[:, :3], C)
    yield ValueError, "C must have shape", lambda: selective_scan(x, dt, A, B, C[..., :4])
    yield ValueError, "multiple of groups", lambda: selective_scan(x, dt, A, B.repeat(1, 1, 3, 1)[:, :, :5], C.repeat(1, 1, 3, 1)[:, :, :5])
    yield ValueError, "dt must have shape", lambda: selective_scan(x, dt[:, :3], A, B, C)
    yield ValueError, "gate must have shape", lambda: selective_scan(x, dt, A, B, C, gate=gate[..., :3])
    yield ValueError, "dt_bias must have shape", lambda: selective_scan(x, dt, A, B, C, dt_bias=bias[:3])
    yield ValueError, "initial_state must have shape", lambda: selective_scan(x, dt, A, B, C, s0[:1])
    yield ValueError, "state must have shape", lambda: selective_step(*step, s0[:, :3])
    yield ValueError, "state must be contiguous", lambda: selective_step(*step, s0.transpose(1, 2).contiguous().transpose(1, 2))
    yield ValueError, "fewer states than requests", lambda: selective_step(*step, s0[:1])
    yield RuntimeError, "state must be float32", lambda: selective_step(*step, s0.bfloat16())
    yield RuntimeError, "slots must be an int32", lambda: selective_step(*step, s0, slots=ints.long())
    yield RuntimeError, "weight must be float32", lambda: causal_conv(cx, cw.bfloat16())
    yield ValueError, "weight must have shape", lambda: causal_conv(cx, cw[:3])
    yield ValueError, "weight must have shape", lambda: causal_conv(cx, cw[:, :1])
    yield ValueError, "bias must have shape", lambda: causal_conv(cx, cw, cb[:3])
    yield ValueError, "initial_state must have shape", lambda: causal_conv(cx, cw, cb, cs[:, :2])
    yield ValueError, "activation must be", lambda: causal_conv(cx, cw, activation="gelu")
    yield ValueError, "x must have shape", lambda: causal_conv(cx[0], cw)
    yield ValueError, "state must have shape", lambda: causal_conv_step(cx[:, 0], cs[:, :2], cw)
    yield ValueError, "state must be contiguous", lambda: causal_conv_step(cx[:, 0], cs.transpose(1, 2).contiguous().transpose(1, 2), cw)
    yield ValueError, "fewer states than requests", lambda: causal_conv_step(cx[:, 0], cs[:1], cw)
    yield RuntimeError, "weight must be float32", lambda: layer_norm(nx, nw.bfloat16())
    yield RuntimeError, "x must be float32 or bfloat16", lambda: layer_norm(half(nx))
    yield ValueError, "weight must have shape", lambda: layer_norm(nx, nw[:3])
    yield ValueError, "bias must have shape", lambda: layer_norm(nx, None, nb[:3])
    yield ValueError, "last dimension must be", lambda: layer_norm(torch.zeros(2, 16385, device=device))
    yield ValueError, "last dimension must be", lambda: layer_norm(torch.zeros((), device=device))
    yield RuntimeError, "weight must be float32", lambda: linear_cross_entropy(lx, lw.bfloat16(), t)
    yield RuntimeError, "target must be an int64 or int32", lambda: linear_cross_entropy(lx, lw, t.to(torch.int16))
    yield RuntimeError, "target must be an int64 or int32", lambda: linear_cross_entropy(lx, lw, t.cpu() if device != "cpu" else t.float())
    yield ValueError, "reduction must be one of", lambda: linear_cross_entropy(lx, lw, t, reduction="max")
    yield ValueError, "ignore_index must be", lambda: linear_cross_entropy(lx, lw, t, ignore_index=2 ** 63)
    yield ValueError, "weight must have shape", lambda: linear_cross_entropy(lx, lw[0], t)
    yield ValueError, "x must have shape", lambda: linear_cross_entropy(lx[:, :3], lw, t)
    yield ValueError, "target must have shape", lambda: linear_cross_entropy(lx, lw, t[:3])
    yield ValueError, "bias must have shape", lambda: linear_cross_entropy(lx, lw, t, lb[:3])
    yield ValueError, "at most 2\\^21", lambda: linear_cross_entropy(torch.zeros(1, 1, device=device), torch.zeros(2 ** 21 + 1, 1, device=device), t[:1])


@pytest.mark.gpu
def test_refusals(gpu):
    """Every one ends before a launch."""
    for error, message, call in _refusals(gpu):
        with pytest.raises(error, match=message):
            call()
