"""More rows than a launch has threads for: norms of 2^26 rows and more, as of many short heads."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_norms_of_many_short_rows(gpu):
    from rnn_kernel_amd import layer_norm

    rows, some = 2 ** 26 + 5, 1000
    gen = torch.Generator(device=gpu).manual_seed(0)
    x = torch.randn(rows, 2, generator=gen, device=gpu, dtype=torch.bfloat16).requires_grad_(True)
    w = torch.tensor([2.0, 0.5], device=gpu, dtype=torch.bfloat16)
    y = layer_norm(x, w)
    up = torch.randn(rows, 2, generator=gen, device=gpu, dtype=torch.bfloat16)
    dx = torch.autograd.grad(y, x, up)[0]
    for at in (0, 2 ** 26 - some // 2, rows - some):  # (the bits of a call with those rows alone)
        part = x.detach()[at:at + some].clone().requires_grad_(True)
        of = layer_norm(part, w)
        assert torch.equal(of, y[at:at + some])
        assert torch.equal(torch.autograd.grad(of, part, up[at:at + some])[0], dx[at:at + some])
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w), y)
