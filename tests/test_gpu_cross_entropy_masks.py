"""The cross entropy where a bias of -infinity meets a logit that is no number: as the formula has
it, NaN + -infinity is NaN, in the loss as in its gradients."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,at", [(200, 70), (200, 199), (4097, 4096)])
def test_a_nan_in_a_masked_column_is_not_hidden(gpu, V, at, dtype):
    """(Columns past the vocabulary's end, whose sums are another column's, stay without a part: the
    NaN of the last column is in its own.)"""
    from rnn_kernel_amd import linear_cross_entropy

    gen = torch.Generator().manual_seed(V + at)
    x, w = torch.randn(70, 32, generator=gen).to(gpu, dtype), torch.randn(V, 32, generator=gen).to(gpu, dtype)
    b = torch.zeros(V, device=gpu, dtype=dtype)
    b[at] = float("-inf")
    target = torch.randint(0, at, (70,), generator=gen).to(gpu)
    clean = linear_cross_entropy(x, w, target, b, reduction="none")
    assert torch.isfinite(clean).all()
    w[at, 5] = float("nan")
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    loss = linear_cross_entropy(leaves[0], leaves[1], target, leaves[2], reduction="none")
    want = torch.nn.functional.cross_entropy((x.float() @ w.float().t()) + b.float(), target, reduction="none")
    assert want.isnan().all() and loss.isnan().all()
    assert all(g.isnan().any() for g in torch.autograd.grad(loss.sum(), leaves))
    # the same of an infinite logit: infinity + -infinity
    w[at] = 0
    w[at, 5] = float("inf")
    loss = linear_cross_entropy(x, w, target, b, reduction="none")
    want = torch.nn.functional.cross_entropy((x.float() @ w.float().t()) + b.float(), target, reduction="none")
    assert torch.equal(loss.isnan(), want.isnan()) and want.isnan().any() and not want.isnan().all()
    assert torch.equal(loss[~want.isnan()] > 0, want[~want.isnan()] > 0)
