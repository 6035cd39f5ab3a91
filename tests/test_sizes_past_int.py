"""Sizes that the library's 32-bit arguments do not hold are refused (they would arrive as
what is left of them modulo 2^32).  The tensors are expanded: nothing of that size is made."""
import ctypes

import pytest
import torch

HUGE = 2 ** 32 + 1


def test_what_an_argument_would_become():
    assert ctypes.c_int(HUGE).value == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_products(gpu, dtype):
    from rnn_kernel_amd import linear

    x, w = torch.randn(1, 1, device=gpu, dtype=dtype), torch.randn(1, 1, device=gpu, dtype=dtype)
    for args in ((x.expand(HUGE, 1), w), (x.expand(3, HUGE, 1), w), (x, w.expand(HUGE, 1)),
                 (x.expand(1, HUGE), w.expand(1, HUGE)), (x[:0].expand(0, 1), w.expand(HUGE, 1))):
        with pytest.raises(ValueError, match="2\\^31"):
            linear(*args)


@pytest.mark.gpu
def test_the_rule_and_its_steps(gpu):
    from rnn_kernel_amd import gated_delta_rule, gated_delta_step

    one, gate = torch.randn(1, 1, 1, 1, device=gpu), torch.rand(1, 1, 1, device=gpu)
    for shape in ((HUGE, 1, 1, 1), (1, HUGE, 1, 1), (1, 1, HUGE, 1), (HUGE, 0, 1, 1)):
        q, g = (one[:, :0] if 0 in shape else one).expand(shape), (gate[:, :0] if 0 in shape else gate).expand(shape[:3])
        with pytest.raises(ValueError, match="2\\^31"):
            gated_delta_rule(q, q, q, g, g)
    with pytest.raises(ValueError, match="2\\^31"):
        gated_delta_rule(one, one, one.expand(1, 1, 1, HUGE), gate, gate)
    step, g = one[0], gate[0]
    with pytest.raises(ValueError, match="2\\^31"):
        gated_delta_step(*[step.expand(HUGE, 1, 1)] * 3, *[g.expand(HUGE, 1)] * 2, one)
    slots = torch.zeros(1, dtype=torch.int32, device=gpu)
    with pytest.raises(ValueError, match="2\\^31"):
        gated_delta_step(step, step, step, g, g, one.expand(HUGE, 1, 1, 1), slots=slots)
