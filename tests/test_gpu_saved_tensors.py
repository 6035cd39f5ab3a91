"""Gradients under saved-tensor hooks that hand the tensors back in another layout (as
keeping them on the host does with every tensor that is not dense): the bits of the
gradients without hooks."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _apart(t):
    """The same values, neighbouring elements of the last dimension two apart."""
    return torch.stack([t, torch.zeros_like(t)], -1)[..., 0]


def _hooks():
    saved = torch.autograd.graph.saved_tensors_hooks
    return (saved(lambda t: t.detach().contiguous(), lambda t: t), saved(lambda t: t.detach(), _apart),
            torch.autograd.graph.save_on_cpu())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,Hk,Hv,Dk,Dv", [(70, 2, 4, 16, 24), (130, 1, 2, 33, 19)])
def test_gradients_of_the_rule(gpu, T, Hk, Hv, Dk, Dv, dtype):
    from rnn_kernel_amd import gated_delta_rule

    gen = torch.Generator().manual_seed(T)
    row = torch.randn(2, T, 2 * Hk * Dk + Hv * Dv + 5, generator=gen).to(gpu, dtype).requires_grad_(True)
    gates = [torch.rand(2, T, 1, generator=gen).to(gpu).requires_grad_(True) for _ in range(2)]
    lengths = torch.tensor([T, 65], dtype=torch.int32, device=gpu)
    up = torch.randn(2, T, Hv, Dv, generator=gen).to(gpu, dtype)

    def run():
        q, k, v = (t.unflatten(-1, (-1, d)) for t, d in
                   zip(row[..., 5:].split([Hk * Dk, Hk * Dk, Hv * Dv], -1), (Dk, Dk, Dv)))
        g, beta = (t.expand(2, T, Hv) for t in gates)
        return gated_delta_rule(q, k, v, -g, beta, normalize=True, lengths=lengths)[0]

    want = torch.autograd.grad(run(), [row, *gates], up)
    for hooks in _hooks():
        with hooks:
            o = run()
        for a, b in zip(torch.autograd.grad(o, [row, *gates], up), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_the_product(gpu, dtype):
    from rnn_kernel_amd import linear

    gen = torch.Generator().manual_seed(1)
    wide = [torch.randn(*s, generator=gen).to(gpu, dtype).requires_grad_(True) for s in ((100, 77), (72, 80), (72,))]
    up = torch.randn(100, 72, generator=gen).to(gpu, dtype)

    def run():
        return linear(wide[0][:, 3:67], wide[1][:, :64], wide[2], activation="gelu")

    want = torch.autograd.grad(run(), wide, up)
    for hooks in _hooks():
        with hooks:
            y = run()
        for a, b in zip(torch.autograd.grad(y, wide, up), want):
            assert torch.equal(a, b)
