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


@pytest.mark.parametrize("T", [1, 16, 21, 200])
@pytest.mark.parametrize("N", [5, 16, 40])
def test_a_state_whose_A_is_minus_infinity_holds_its_last_token(gpu, T, N):
    """As with A of -1e30, by which exp(s A) is 0 as well: outputs, states and gradients, for rows that
    end inside a tile, at its end, and with a chunk or more behind them."""
    from rnn_kernel_amd import selective_scan, selective_step

    args, up = _inputs(3, T, 24, N, gpu, seed=1)
    s0 = torch.randn(3, 24, N, generator=torch.Generator().manual_seed(2)).to(gpu)
    lengths = torch.tensor([T, (T + 1) // 2, 0], dtype=torch.int32, device=gpu)
    out = []
    for of in (-1e30, float("-inf")):
        leaves = [t.clone() for t in args]
        leaves[2][:, :3] = of
        leaves = [t.requires_grad_(True) for t in (*leaves, s0.clone())]
        y, h = selective_scan(*leaves, lengths=lengths)
        grads = torch.autograd.grad([y, h], leaves, [up, torch.ones_like(h)])
        pool = s0.clone()
        step = selective_step(*(t.detach()[:, 0] if i != 2 else t.detach() for i, t in enumerate(leaves[:5])), pool)
        out.append([y, h, *grads, step, pool])
    for a, b in zip(*out):
        assert torch.isfinite(b).all() and torch.equal(a, b)
    h = out[1][1]
    assert torch.equal(h[2], s0[2])
    last = (args[1] * args[0])[0, T - 1, :, None] * args[3][0, T - 1]
    assert (h[0, :, :3] - last[:, :3]).abs().max() <= 2.0 ** -22 * last.abs().max()
