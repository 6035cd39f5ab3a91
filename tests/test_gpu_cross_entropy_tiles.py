"""The cross entropy with every tile of its products, of whole stages and not, with and without
bias, with many full tiles of rows, remainders, and several pieces of the vocabulary: the form
that each size takes is asked first, so that another rule for it shows here.

Against float64, tolerances set before the first run.  A logit is a float32 sum of K products of
size 2 / sqrt(K): off by 2^-24 sqrt(K) / 2 of their size, 2; a loss by that of its target and of
its largest terms, of thousands of rows at most four deviations, and by some 32 roundings of numbers
of its size: 2^-24 (4 sqrt(K) + 32).  Gradients, as 2-norms of the error over the result's: float32 p is off
by its logit's error times p, and sums of n terms add sqrt(n) / 2 roundings: 2^-24 (sqrt(K) + sqrt(n) / 2
+ 16); bfloat16 rounds dl, once or twice to 2^-8 at most: 1.1 sqrt(2) 2^-8 in all with the result's own
rounding, and db, summed before that, 1.1 2^-8.  The same for each row and column of a gradient by itself, times
three, as of 10^5 of them the worst is looked at: an error of one place is small in the norm of
all."""
import pytest
import torch

F32, BF16 = torch.float32, torch.bfloat16
CODE = {F32: 0, BF16: 1}

# rows, inputs, vocabulary, type, columns in front of the weight, form, edge of the forward, pieces, edges of
# dl, dx and dW, whether the sums of dx and dW are sliced
CASES = [
    (4129, 2048, 50003, BF16, 8, "direct", 256, 2, 256, 256, 256, True, False),
    (4129, 512, 50003, BF16, 8, "direct", 256, 2, 256, 128, 256, True, False),
    (8201, 1024, 20003, BF16, 8, "direct", 256, 2, 256, 128, 64, True, False),
    (8201, 1024, 7001, BF16, 8, "direct", 256, 1, 256, 64, 256, False, True),
    (701, 2048, 50003, BF16, 8, "direct", 256, 1, 256, 256, 256, True, False),
    (2057, 192, 50003, BF16, 8, "direct", 256, 1, 256, 64, 64, True, False),
    (2057, 192, 50003, BF16, 3, "tiles", 256, 1, 256, 64, 64, True, False),
    (2057, 64, 70003, BF16, 8, "direct", 256, 2, 256, 64, 64, True, False),
    (1101, 200, 140003, BF16, 8, "tiles", 256, 2, 256, 64, 128, True, False),
    (8201, 200, 50003, BF16, 8, "tiles", 256, 4, 256, 64, 256, False, True),
    (2057, 512, 3001, BF16, 8, "direct", 128, 1, 128, 64, 64, False, False),
    (2057, 512, 3001, BF16, 3, "tiles", 128, 1, 128, 64, 64, False, False),
    (1101, 2048, 7001, BF16, 8, "direct", 128, 1, 128, 64, 256, False, False),
    (521, 200, 50003, BF16, 8, "tiles", 128, 1, 128, 64, 256, True, False),
    (301, 320, 1003, BF16, 8, "direct", 64, 1, 64, 64, 64, True, False),
    (2101, 1024, 20003, F32, 4, "direct", 128, 1, 128, 128, 128, True, False),
    (1101, 1024, 70003, F32, 4, "direct", 128, 2, 128, 128, 128, True, False),
    (1101, 1024, 20003, F32, 3, "tiles", 128, 1, 128, 64, 128, True, False),
    (1101, 1030, 20003, F32, 4, "tiles", 128, 1, 128, 64, 128, True, False),
    (1101, 544, 20003, F32, 4, "direct", 128, 1, 128, 64, 64, True, False),   # 17 stages: a part of 16 and one more
    (8201, 1024, 7001, F32, 4, "direct", 128, 1, 128, 128, 128, True, True),
    (4201, 128, 50003, F32, 4, "direct", 128, 4, 128, 128, 64, True, True),
    (701, 2048, 50003, F32, 4, "direct", 64, 1, 64, 128, 128, True, False),
    (301, 1024, 3001, F32, 4, "direct", 64, 1, 64, 64, 64, True, False),
]


@pytest.mark.parametrize("case", CASES)
def test_cases_take_the_forms_they_are_for(hip_lib, case):
    from rnn_kernel_amd import _lib

    rows, inputs, vocabulary, dtype, left, *want = case
    aligned = left * torch.finfo(dtype).bits // 8 % 16 == 0
    d = _lib.describe_cross_entropy(rows, inputs, vocabulary, CODE[dtype], aligned)
    assert [d["form"], d["forward"], d["pieces"], d["slopes"], d["grad_x"], d["grad_weight"], d["slices_x"] > 1,
            d["slices_weight"] > 1] == want


def test_descriptions_are_of_sizes_that_are_taken(hip_lib):
    import ctypes

    out = (ctypes.c_int * 9)()
    assert hip_lib.rka_describe_cross_entropy(0, 8, 8, 0, 1, out, 9) == 1001
    assert hip_lib.rka_describe_cross_entropy(2 ** 21 + 1, 8, 8, 0, 1, out, 9) == 1004
    assert hip_lib.rka_describe_cross_entropy(8, 8, 8, 0, 1, None, 9) == 1001
    assert hip_lib.rka_describe_cross_entropy(8, 8, 8, 0, 1, out, 1) == 0 and out[1] == 0


def _inside(t, left):
    """t's values in a matrix that is NaN around them, `left` columns from its left edge."""
    ld = -(-(left + t.size(1) + 1) // 8) * 8
    full = torch.full((t.size(0) + 2, ld), float("nan"), dtype=t.dtype, device=t.device)
    inner = full[1:-1, left:left + t.size(1)]
    inner.copy_(t)
    return inner


def _formula(x, w, b, target, scale):
    """Losses of the rows, and the gradients of their sum weighted by `scale`, in float64."""
    z = x @ w.t()
    if b is not None:
        z += b
    lse = torch.logsumexp(z, 1)
    of = z.gather(1, target[:, None])[:, 0]
    dl = z.sub_(lse[:, None]).exp_()
    dl[torch.arange(len(target), device=x.device), target] -= 1
    dl *= scale[:, None]
    return lse - of, dl @ w, dl.t() @ x, dl.sum(0)


def _fits(got, want, tol):
    err, want = got.double() - want, want
    assert torch.isfinite(got).all()
    assert float(err.norm() / want.norm()) <= tol
    for dim in range(want.dim()) if want.dim() > 1 else ():
        of, ref = err.norm(dim=dim), want.norm(dim=dim)
        assert bool((of <= 3 * tol * ref).all()), (dim, float((of / ref).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("bias,ignored,reduction", [(False, 0.0, "mean"), (False, 0.1, "none"), (True, 0.1, "sum")])
@pytest.mark.parametrize("case", CASES)
def test_losses_and_gradients(gpu, case, bias, ignored, reduction):
    from rnn_kernel_amd import linear_cross_entropy

    M, K, V, dtype, left, *_ = case
    print(f"cross entropy {case} {bias} {ignored} {reduction}", flush=True)
    gen = torch.Generator(device=gpu).manual_seed(M + K + V)
    x = torch.randn(M, K, generator=gen, device=gpu).to(dtype)
    w = (2 * torch.randn(V, K, generator=gen, device=gpu) / K ** 0.5).to(dtype)
    b = torch.randn(V, generator=gen, device=gpu).to(dtype) if bias else None
    target = torch.randint(0, V, (M,), generator=gen, device=gpu)
    target[0], target[-1] = V - 1, 0
    on = torch.rand(M, generator=gen, device=gpu) >= ignored
    on[0] = on[-1] = True
    up = torch.rand(M, generator=gen, device=gpu) + 0.5
    scale = up.double()[on] if reduction == "none" else torch.full((int(on.sum()),), 0.75, dtype=torch.float64, device=gpu)
    scale = scale / (int(on.sum()) if reduction == "mean" else 1)
    losses, dx, dw, db = _formula(x[on].double(), w.double(), None if b is None else b.double(), target[on], scale)

    leaves = [x.clone().requires_grad_(True), _inside(w, left).requires_grad_(True)] + ([b.clone().requires_grad_(True)] if bias else [])
    loss = linear_cross_entropy(leaves[0], leaves[1], torch.where(on, target, -100), leaves[2] if bias else None, reduction=reduction)
    row = 2.0 ** -24 * (4 * K ** 0.5 + 32)
    if reduction == "none":
        assert (loss.detach()[~on] == 0).all() and float((loss.detach()[on].double() - losses).abs().max()) <= row
    else:
        want = losses.mean() if reduction == "mean" else losses.sum()
        assert abs(float(loss) - float(want)) <= row * (1 if reduction == "mean" else len(losses)) + 2.0 ** -24 * float(want)
    grads = torch.autograd.grad(loss, leaves, up if reduction == "none" else torch.tensor(0.75, device=gpu))
    assert (grads[0][~on] == 0).all()
    f32 = 2.0 ** -24 * (K ** 0.5 + max(M, V) ** 0.5 / 2 + 16)
    tol = f32 if dtype == F32 else 1.1 * 2 ** 0.5 * 2.0 ** -8
    _fits(grads[0][on], dx, tol)
    _fits(grads[1], dw, tol)
    if bias:
        _fits(grads[2], db, f32 if dtype == F32 else 1.1 * 2.0 ** -8)
        # (p is above 0: a column's sum of p and its targets are each off by so much)
        size = db.abs() + 2 * 0.75 * torch.bincount(target[on], minlength=V)
        assert bool(((grads[2].double() - db).abs() <= (0 if dtype == F32 else 2.0 ** -8) * db.abs() + 4 * f32 * size).all())
