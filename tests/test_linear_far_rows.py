"""Rows of a product further apart than the kernels' offsets reach are copied, not refused."""
import importlib

import pytest
import torch

FAR = 2 ** 21 + 8


def _far(t):
    """The same rows, FAR elements apart."""
    base = torch.empty((t.size(0) - 1) * FAR + t.size(1), dtype=t.dtype, device=t.device)
    return base.as_strided(t.shape, (FAR, 1)).copy_(t)


def test_rows_are_copied():
    linear = importlib.import_module("rnn_kernel_amd.linear")  # (the package's `linear` is the function)
    far = _far(torch.randn(3, 8))
    assert linear._rows(far).stride() == (8, 1) and torch.equal(linear._rows(far), far)
    near = torch.empty(3 * linear.MAX_ROW_STRIDE).as_strided((3, 8), (linear.MAX_ROW_STRIDE, 1))
    assert linear._rows(near).data_ptr() == near.data_ptr()
    assert linear._rows(far[:1]).data_ptr() == far.data_ptr()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_far_rows_give_the_bits_of_close_ones(gpu, dtype):
    from rnn_kernel_amd import linear

    gen = torch.Generator().manual_seed(4)
    x, w, r, dy = (torch.randn(*s, generator=gen).to(gpu, dtype) for s in ((5, 40), (7, 40), (5, 7), (5, 7)))
    results = []
    for lay in (lambda t: t.clone(), _far):
        leaves = [lay(t).requires_grad_(True) for t in (x, w)]
        y = linear(*leaves, activation="silu", residual=lay(r))
        results.append((y, *torch.autograd.grad(y, leaves, lay(dy))))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_inputs_and_outputs_past_the_offsets_are_refused(gpu):
    from rnn_kernel_amd import linear

    one = torch.zeros(1, 1, device=gpu)
    for x, w in ((one, one.expand(FAR, 1)), (one.expand(1, FAR), one.expand(1, FAR))):
        with pytest.raises(ValueError, match="at most 2\\^21"):
            linear(x, w)
