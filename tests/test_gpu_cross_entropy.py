"""GPU parity of the cross entropy of a product with a vocabulary with its formula in
float64, and of its gradients with theirs and with differences.

Tolerances set before the first run.  A logit is a float32 sum of up to 600 products of size
1 / sqrt(inputs): its error is some 2^-24 sqrt(600) / 2 or 8e-7 of the logits' size, 2 here
(and their largest some 8); a loss is off by that of its target and that of the sum: 4e-6
absolute per row.  Gradients, as 2-norms of the error over that of the result: float32: p is off by
that times p, and sums of up to 3000 terms add some 30 roundings: 1e-5.  bfloat16: dl is rounded
to 2^-9 rms or 2^-8 at most of each element before the products (its errors add up like the
result does, or like its root), and the result once more: sqrt(2) 2^-8 at most, and 1.1 times
that leaves the float32 part its room.  db is summed before dl is rounded: 1.1 * 2^-8."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ROW, GRAD, BF16, BF16_BIAS = 4e-6, 1e-5, 1.1 * 2 ** 0.5 * 2.0 ** -8, 1.1 * 2.0 ** -8


def _formula(x, w, target, b, ignore=-100):
    """Losses of the rows in float64, differentiable."""
    on = target != ignore
    z = torch.where(on[:, None], x, torch.zeros_like(x)) @ w.t()
    z = z if b is None else z + b
    of = z.gather(1, torch.where(on, target, 0).long()[:, None])[:, 0]
    return torch.where(on, torch.logsumexp(z, -1) - of, torch.zeros_like(of))


def _inputs(M, K, V, dtype, bias, ignored, seed=0):
    gen = torch.Generator().manual_seed(seed + M + K + V)
    x, w = torch.randn(M, K, generator=gen).to(dtype), (2 * torch.randn(V, K, generator=gen) / K ** 0.5).to(dtype)
    b = torch.randn(V, generator=gen).to(dtype) if bias else None
    target = torch.randint(0, V, (M,), generator=gen)
    if ignored:
        target[torch.rand(M, generator=gen) < ignored] = -100
        target[M // 2] = V - 1
    return x, w, b, target


def _rel(a, ref):
    a, ref = a.detach().double().cpu(), ref.detach().double()
    assert torch.isfinite(a).all()
    return float((a - ref).norm() / ref.norm().clamp_min(1e-30))


# Rows, inputs and vocabulary around the tiles' edges (64, 128, 256), sums in whole stages and
# not, one column, one row, vocabularies that end inside a tile
SHAPES = [(1, 1, 1), (1, 64, 50), (5, 7, 3), (64, 64, 64), (65, 96, 129), (100, 257, 1007), (130, 128, 300), (257, 320, 2049),
          (33, 600, 5000), (1, 128, 4097), (700, 40, 33), (300, 64, 100), (1500, 128, 65), (2, 33, 20000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bias,ignored", [(False, 0.0), (True, 0.4)])
@pytest.mark.parametrize("shape", SHAPES)
def test_losses_and_gradients(gpu, shape, bias, ignored, dtype):
    from rnn_kernel_amd import linear_cross_entropy

    print(f"cross entropy {shape} bias={bias} ignored={ignored} {dtype}", flush=True)
    x, w, b, target = _inputs(*shape, dtype, bias, ignored)
    ref = [None if t is None else t.double().requires_grad_(True) for t in (x, w, b)]
    want = _formula(ref[0], ref[1], target, ref[2])
    got = [None if t is None else t.to(gpu).requires_grad_(True) for t in (x, w, b)]
    on = target != -100
    up = torch.rand(shape[0], generator=torch.Generator().manual_seed(1)) + 0.5
    for reduction in ("none", "mean", "sum"):
        loss = linear_cross_entropy(got[0], got[1], target.to(gpu), got[2], reduction=reduction)
        assert loss.dtype == torch.float32
        if reduction == "none":
            assert (loss.detach().cpu().double() - want.detach()).abs().max() <= ROW and (loss.cpu()[~on] == 0).all()
            r, g, rg = want, up.to(gpu), up.double()
        else:
            r = want.sum() / (on.sum() if reduction == "mean" else 1)
            assert abs(float(loss) - float(r)) <= ROW * (1 if reduction == "mean" else int(on.sum()))
            g, rg = torch.tensor(0.75, device=gpu), torch.tensor(0.75, dtype=torch.float64)
        grads = torch.autograd.grad(loss, [t for t in got if t is not None], g)
        refs = torch.autograd.grad(r, [t for t in ref if t is not None], rg, retain_graph=True)
        for i, (a, c) in enumerate(zip(grads, refs)):
            tol = GRAD if dtype == torch.float32 else BF16_BIAS if i == 2 else BF16
            if shape[2] == 1:  # one column: the loss and its gradients are 0
                assert a.abs().max() <= 1e-5
            else:
                assert a.dtype == dtype and a.shape == c.shape and _rel(a, c) <= tol, (reduction, i, _rel(a, c))
        assert (grads[0][~on.to(gpu)] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_several_pieces_of_the_vocabulary(gpu, dtype):
    """More than one piece (a piece's gradients take half a GiB): 6000 rows, of which few have
    a target, so that the oracle stays small."""
    from rnn_kernel_amd import linear_cross_entropy

    M, K, V = 6000, 64, 50000
    x, w, b, target = _inputs(M, K, V, dtype, True, 0.97)
    on = target != -100
    ref = [t.double().requires_grad_(True) for t in (x[on], w, b)]
    want = _formula(*ref[:2], target[on], ref[2]).mean()
    refs = torch.autograd.grad(want, ref)
    got = [t.to(gpu).requires_grad_(True) for t in (x, w, b)]
    loss = linear_cross_entropy(got[0], got[1], target.to(gpu), got[2])
    assert abs(float(loss) - float(want)) <= ROW
    grads = torch.autograd.grad(loss, got)
    assert (grads[0][~on.to(gpu)] == 0).all()
    for i, (a, c) in enumerate(zip((grads[0][on.to(gpu)], *grads[1:]), refs)):
        assert _rel(a, c) <= (GRAD if dtype == torch.float32 else BF16_BIAS if i == 2 else BF16), (i, _rel(a, c))


def test_without_a_target_anywhere(gpu):
    from rnn_kernel_amd import linear_cross_entropy

    x, w = (torch.randn(*s, device=gpu).requires_grad_(True) for s in ((70, 32), (90, 32)))
    target = torch.full((70,), -100, device=gpu)
    for reduction in ("none", "mean", "sum"):
        loss = linear_cross_entropy(x, w, target, reduction=reduction)
        assert (loss == 0).all()
        assert all((g == 0).all() for g in torch.autograd.grad(loss.sum(), [x, w]))
    for rows in ((0,), (3, 0)):
        x0 = torch.zeros(*rows, 32, device=gpu, requires_grad=True)
        loss = linear_cross_entropy(x0, w, torch.zeros(*rows, dtype=torch.int64, device=gpu))
        assert loss == 0
        dx, dw = torch.autograd.grad(loss, [x0, w])
        assert dx.shape == x0.shape and (dw == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_what_an_ignored_row_holds_reaches_nothing(gpu, dtype):
    from rnn_kernel_amd import linear_cross_entropy

    x, w, b, target = (t.to(gpu) for t in _inputs(90, 40, 120, dtype, True, 0.5))
    bad = x.clone()
    bad[target == -100] = float("nan")
    out = []
    for rows in (x, bad):
        leaves = [t.clone().requires_grad_(True) for t in (rows, w, b)]
        loss = linear_cross_entropy(leaves[0], leaves[1], target, leaves[2])
        out.append((loss, *torch.autograd.grad(loss, leaves)))
    assert all(torch.equal(p, q) for p, q in zip(*out))


def test_targets_outside_and_of_another_name(gpu):
    """A target outside the vocabulary gives NaN to its row's loss and gradient; int32 targets
    and another ignored number do as int64 and -100."""
    from rnn_kernel_amd import linear_cross_entropy

    x, w, b, target = (t.to(gpu) for t in _inputs(40, 32, 70, torch.float32, True, 0.3))
    want = linear_cross_entropy(x, w, target, b, reduction="none")
    other = torch.where(target == -100, 7777, target).to(torch.int32)
    assert torch.equal(linear_cross_entropy(x, w, other, b, reduction="none", ignore_index=7777), want)
    # with 5 as the ignored number, -100 is a target outside the vocabulary
    five = linear_cross_entropy(x, w, target, b, reduction="none", ignore_index=5)
    usual = (target != -100) & (target != 5)
    assert (five[target == 5] == 0).all() and five[target == -100].isnan().all() and torch.equal(five[usual], want[usual])
    for wrong in (70, -1, 2 ** 40, -2 ** 62):
        bad = target.clone()
        bad[3] = wrong
        leaf = x.clone().requires_grad_(True)
        loss = linear_cross_entropy(leaf, w, bad, b, reduction="none")
        rest = torch.arange(40, device=gpu) != 3
        assert loss[3].isnan() and torch.equal(loss[rest], want[rest])
        g = torch.autograd.grad(loss, leaf, torch.ones_like(loss))[0]
        assert g[3].isnan().all() and torch.isfinite(g[rest]).all()


def test_special_logits(gpu):
    """Columns of -infinity (a masked vocabulary) have no part; a target there costs infinity; a NaN
    row is NaN alone; large logits stay finite."""
    from rnn_kernel_amd import linear_cross_entropy

    x, w, _, target = (None if t is None else t.to(gpu) for t in _inputs(20, 16, 200, torch.float32, False, 0.0))
    b = torch.zeros(200, device=gpu)
    b[64:150] = float("-inf")
    target = target % 64
    leaf = [t.clone().requires_grad_(True) for t in (x, w, b)]
    loss = linear_cross_entropy(leaf[0], leaf[1], target, leaf[2], reduction="none")
    keep = torch.isfinite(b)
    want = _formula(x.double().cpu(), w[keep].double().cpu(), target.cpu(), None)
    assert (loss.detach().cpu().double() - want).abs().max() <= ROW
    dx, dw, db = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    assert torch.isfinite(dx).all() and (dw[64:150] == 0).all() and (db[64:150] == 0).all()
    assert linear_cross_entropy(x[:1], w, torch.tensor([70], device=gpu), b) == float("inf")
    everything = linear_cross_entropy(x[:1], w, torch.tensor([70], device=gpu), torch.full_like(b, float("-inf")))
    assert everything.isnan()
    bad = x.clone()
    bad[4, 3] = float("nan")
    loss = linear_cross_entropy(bad, w, target, reduction="none")
    rest = torch.arange(20, device=gpu) != 4
    assert loss[4].isnan() and torch.equal(loss[rest], linear_cross_entropy(x, w, target, reduction="none")[rest])
    w_nan = w.clone()
    w_nan[100:] = float("nan")
    assert linear_cross_entropy(x, w_nan, target, reduction="none").isnan().all()
    big = linear_cross_entropy(1000 * x, w, target, reduction="none")
    ref = _formula(1000 * x.double().cpu(), w.double().cpu(), target.cpu(), None)
    assert (big.cpu().double() - ref).abs().max() <= 1e-6 * 1000 * 8 and torch.isfinite(big).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(gpu, dtype):
    """Any strides of x, weight, target and the loss's gradient: the bits of dense ones, where
    the weight's rows keep their alignment."""
    from rnn_kernel_amd import linear_cross_entropy

    gen = torch.Generator().manual_seed(4)
    wide = torch.randn(6, 30, 150, generator=gen).to(gpu, dtype)
    ww = torch.randn(130, 144, generator=gen).to(gpu, dtype)
    target = torch.randint(0, 130, (30, 6), generator=gen).to(gpu).t()
    up = torch.rand(1, 30, generator=gen).to(gpu).expand(6, 30)
    for x in (wide[..., 5:133], wide.transpose(0, 1).contiguous().transpose(0, 1)[..., :128], wide[:, :1, :128].expand(6, 30, 128)):
        for w in (ww[:, 8:136], ww[:, :128].t().contiguous().t()):
            leaves = [x.detach().requires_grad_(True), w.detach().requires_grad_(True)]
            dense = [t.detach().contiguous().requires_grad_(True) for t in leaves]
            got = linear_cross_entropy(*leaves, target, reduction="none")
            want = linear_cross_entropy(*dense, target.contiguous(), reduction="none")
            assert got.shape == target.shape and torch.equal(got, want)
            for p, q in zip(torch.autograd.grad(got, leaves, up), torch.autograd.grad(want, dense, up.contiguous())):
                assert torch.equal(p, q)


def test_only_some_gradients(gpu):
    from rnn_kernel_amd import linear_cross_entropy

    x, w, b, target = (t.to(gpu) for t in _inputs(70, 64, 300, torch.float32, True, 0.2))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(linear_cross_entropy(leaves[0], leaves[1], target, leaves[2]), leaves)
    for i in range(3):
        args = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
        g = torch.autograd.grad(linear_cross_entropy(args[0], args[1], target, args[2]), args[i])[0]
        assert torch.equal(g, want[i])


def test_gradients_by_differences(gpu):
    """Along each gradient's own direction, by a central difference of step h of losses summed in
    float64: truncation h^2 / 6 of a third derivative of order the logits' change cubed, rounding
    1e-6 rows / h; the step makes the logits change by about 0.03."""
    from rnn_kernel_amd import linear_cross_entropy

    x, w, b, target = (t.to(gpu) for t in _inputs(50, 24, 90, torch.float32, True, 0.2))
    args = [x, w, b]
    leaves = [t.clone().requires_grad_(True) for t in args]
    grads = torch.autograd.grad(linear_cross_entropy(leaves[0], leaves[1], target, leaves[2], reduction="sum"), leaves)
    for i, (g, h) in enumerate(zip(grads, (0.1, 0.05, 0.1))):
        d, side = g / g.norm(), []
        for sign in (1, -1):
            a = [t + sign * h * d if j == i else t for j, t in enumerate(args)]
            side.append(linear_cross_entropy(a[0], a[1], target, a[2], reduction="none").double().sum())
        assert abs(float((side[0] - side[1]) / (2 * h)) / float(g.norm()) - 1) <= 5e-3, i


def test_same_bits_twice_on_a_stream_and_in_a_graph(gpu):
    from rnn_kernel_amd import LinearCrossEntropy

    torch.manual_seed(3)
    head = LinearCrossEntropy(96, 1000, bias=True, device=gpu)
    x = torch.randn(500, 96, device=gpu, requires_grad=True)
    target = torch.randint(0, 1000, (500,), device=gpu)
    target[::7] = -100

    def both():
        loss = head(x, target)
        return (loss, *torch.autograd.grad(loss, [x, head.weight, head.bias]))

    want = both()
    assert all(torch.equal(a, c) for a, c in zip(both(), want))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = both()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, c) for a, c in zip(other, want))
    with torch.no_grad():
        fixed, t = x.detach().clone(), target.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss = head(fixed, t)
        for i in range(4):
            fixed.copy_(torch.randn_like(fixed))
            t.copy_(torch.where(torch.rand(500, device=gpu) < 0.1 * i, -100, torch.randint(0, 1000, (500,), device=gpu)))
            graph.replay()
            eager = head(fixed, t)
            torch.cuda.synchronize()
            assert torch.equal(loss, eager)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M", [70, 300])
def test_rows_behind_the_last_add_nothing(gpu, dtype, M):
    """A tile's rows past the call's: where all logits are far below 0, or a column's are all
    -infinity, what a row of zeros would have there is not a number.  (float32: logits are sums of 64
    products of size 2, off by at most 2^-24 of each partial sum, 64 * 64 * 2^-24 = 2.5e-4
    altogether, and p by that times p.)"""
    from rnn_kernel_amd import linear_cross_entropy

    gen = torch.Generator().manual_seed(11)
    x = torch.ones(M, 64).to(dtype)
    w = -(2 + 0.01 * torch.randn(256, 64, generator=gen)).to(dtype)
    target = torch.randint(0, 256, (M,), generator=gen)
    for low in (False, True):
        if low:
            x, w = x.clone(), w.clone()
            target = torch.where(target == 9, 10, target)
            w[9, 3] = float("-inf")
        ref = [t.double().requires_grad_(True) for t in (x, w)]
        got = [t.to(gpu).requires_grad_(True) for t in (x, w)]
        want = torch.autograd.grad(_formula(*ref, target, None).mean(), ref[1])[0]
        # (the -infinite column has no part in the others' gradients, nor a gradient)
        dw = torch.autograd.grad(linear_cross_entropy(*got, target.to(gpu)), got[1])[0]
        assert _rel(dw, want) <= (2.5e-4 if dtype == torch.float32 else BF16 + 2.5e-4)
        if low:
            assert (dw[9] == 0).all()
