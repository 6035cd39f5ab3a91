"""The selective scan at values where a product of 0 and infinity would be met."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _formula(x, dt, A, B, C, lengths):
    """float64 recurrence (differentiable) without skip and gate, one group."""
    h, out = x.new_zeros(x.size(0), *A.shape), []
    for t in range(x.size(1)):
        live = t < lengths
        new = torch.exp(dt[:, t, :, None] * A) * h + (dt[:, t] * x[:, t])[..., None] * B[:, t]
        h = torch.where(live[:, None, None], new, h)
        y = (C[:, t] * h).sum(-1)
        out.append(torch.where(live[:, None], y, torch.zeros_like(y)))
    return torch.stack(out, 1), h


def _inputs(B, T, D, N, device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x, dt = torch.randn(B, T, D, generator=gen), 0.02 * torch.rand(B, T, D, generator=gen) + 0.01
    A = -torch.rand(D, N, generator=gen)
    Bm, C = (torch.randn(B, T, 1, N, generator=gen) for _ in range(2))
    return [t.to(device) for t in (x, dt, A, Bm, C)], torch.randn(B, T, D, generator=gen).to(device)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,at,N", [(45, 21, 16), (45, 21, 40), (200, 150, 16), (200, 150, 20)])
def test_an_infinite_C_in_the_last_token_gives_infinite_gradients(gpu, T, at, N, dtype):
    """(One chunk, and more than one.  Gradients of x are infinite where the formula's are, and no NaN.)"""
    from rnn_kernel_amd import selective_scan

    args, up = _inputs(2, T, 24, N, gpu)
    args = [t if i == 2 else t.to(dtype) for i, t in enumerate(args)]
    args[4][0, at, 0, 0] = float("inf")
    lengths = torch.tensor([at + 1, T], dtype=torch.int32, device=gpu)
    ref = [t.double().requires_grad_(True) for t in args]
    want = torch.autograd.grad(_formula(*ref, lengths)[0], ref[0], up.to(dtype).double())[0]
    got = [t.clone().requires_grad_(True) for t in args]
    grad = torch.autograd.grad(selective_scan(*got, lengths=lengths)[0], got[0], up.to(dtype))[0]
    assert want[0, :at + 1].isinf().all() and not want.isnan().any()
    assert torch.equal(grad.isinf(), want.isinf()) and not grad.isnan().any()
    assert torch.equal(grad[want.isinf()].sign().double(), want[want.isinf()].sign())
