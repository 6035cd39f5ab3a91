"""Offsets past 2^31 elements: states far into a pool, tokens and rows far apart.  The
results are the bits of the same inputs close together."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_states_far_into_a_pool(gpu):
    from rnn_kernel_amd import gated_delta_step

    gen = torch.Generator().manual_seed(0)
    Dk, Dv = 256, 128
    count = 2 ** 31 // (Dk * Dv) + 2
    q, k, v = (torch.randn(2, 1, d, generator=gen).to(gpu) for d in (Dk, Dk, Dv))
    g, beta = -torch.rand(2, 1, generator=gen).to(gpu), torch.rand(2, 1, generator=gen).to(gpu)
    near = torch.randn(2, 1, Dk, Dv, generator=gen).to(gpu)
    pool = torch.empty(count, 1, Dk, Dv, device=gpu)
    pool[count - 1], pool[1], pool[0] = near[0], near[1], 0.0
    slots = torch.tensor([count - 1, 1], dtype=torch.int32, device=gpu)
    far = gated_delta_step(q, k, v, g, beta, pool, slots=slots, normalize=True)
    assert torch.equal(far, gated_delta_step(q, k, v, g, beta, near, normalize=True))
    assert torch.equal(pool[count - 1], near[0]) and torch.equal(pool[1], near[1]) and not pool[0].any()


def test_tokens_far_apart(gpu):
    from rnn_kernel_amd import gated_delta_rule

    gen = torch.Generator().manual_seed(1)
    T, step = 70, 2 ** 25
    base = torch.empty((T - 1) * step + 48, dtype=torch.bfloat16, device=gpu)
    far = base.as_strided((1, T, 1, 48), (base.numel(), step, 48, 1))
    far.copy_(torch.randn(1, T, 1, 48, generator=gen).bfloat16())
    close = far.contiguous()
    g, beta = -torch.rand(1, T, 1, generator=gen).to(gpu), torch.rand(1, T, 1, generator=gen).to(gpu)

    def run(t):
        q, k, v = (x.detach().requires_grad_(True) for x in t.split(16, dim=-1))
        o, state = gated_delta_rule(q, k, v, g, beta, normalize=True)
        return (o, state, *torch.autograd.grad([o, state], [q, k, v], [torch.ones_like(o), torch.ones_like(state)]))

    assert far.stride(1) * (T - 1) > 2 ** 31
    for a, b in zip(run(far), run(close)):
        assert torch.equal(a, b)


def test_rows_far_apart(gpu):
    from rnn_kernel_amd import linear

    gen = torch.Generator().manual_seed(2)
    rows, ld = 1100, 2 ** 21
    base = torch.empty((rows - 1) * ld + 128, dtype=torch.bfloat16, device=gpu)
    x = base.as_strided((rows, 128), (ld, 1))
    x.copy_(torch.randn(rows, 128, generator=gen).bfloat16())
    close = x.contiguous()
    w = torch.randn(72, 128, generator=gen).bfloat16().to(gpu).requires_grad_(True)
    for cols in (128, 96):  # whole stages, and one that ends inside
        y = linear(x[:, :cols], w[:, :cols], activation="silu")
        z = linear(close[:, :cols], w[:, :cols], activation="silu")
        assert torch.equal(y, z)
        dy = torch.ones_like(y)
        assert torch.equal(*(torch.autograd.grad(t, w, dy)[0] for t in (y, z)))
