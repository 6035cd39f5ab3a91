"""Every tile of linear's products, unsliced and in slices, with ends inside tiles, in either
type: the form that each size takes is asked of the plan first, so that another rule for it
shows here.

The operands lie in wider matrices that are NaN around them.  Against float64; tolerances set
before the first run.  As 2-norms: float32 2^-24 (8 + 2 sqrt(n)) for a sum of n products;
bfloat16 1.1 * 2^-8 for one rounding, 3.3 * 2^-8 for a gradient behind an activation (three).
For single elements: a rounding of the element, and eight times the 2-norm's part of the rest
(the elements' errors are sums of independent roundings; of 10^7 none is past eight standard
deviations)."""
import math

import pytest
import torch

F32, BF16 = torch.float32, torch.bfloat16
CODE = {F32: 0, BF16: 1}

# rows, outputs, inputs, type, columns in front of the operands, form, edge, in slices
FORWARD = [
    (2057, 5000, 64, BF16, 8, "direct", 256, False),    # one stage
    (2100, 5001, 128, BF16, 8, "direct", 256, False),   # two
    (2057, 5003, 192, BF16, 8, "direct", 256, False),   # three
    (1001, 1543, 16384, BF16, 8, "direct", 256, True),
    (2057, 5003, 200, BF16, 8, "tiles", 256, False),    # a stage that is not whole
    (2057, 5003, 192, BF16, 3, "tiles", 256, False),    # addresses that are no multiple of 16
    (1001, 1543, 16390, BF16, 3, "tiles", 256, True),
    (2057, 3001, 64, BF16, 8, "direct", 128, False),
    (501, 1543, 16384, BF16, 8, "direct", 128, True),
    (2057, 3001, 70, BF16, 3, "tiles", 128, False),
    (501, 1543, 16378, BF16, 3, "tiles", 128, True),
    (2301, 5003, 32, F32, 4, "direct", 128, False),
    (2301, 5003, 96, F32, 4, "direct", 128, False),
    (1001, 2003, 4096, F32, 4, "direct", 128, True),
    (2301, 5003, 50, F32, 3, "tiles", 128, False),
    (1001, 2003, 4093, F32, 3, "tiles", 128, True),
    (65, 129, 64, BF16, 8, "direct", 64, False),
    (65, 129, 1024, BF16, 8, "direct", 64, True),
    (65, 129, 32, F32, 4, "direct", 64, False),
    (65, 129, 1024, F32, 4, "direct", 64, True),
]

# product, rows, outputs, inputs, type, edge, in slices
GRADIENTS = [
    ("grad_x", 2057, 17, 5003, BF16, 256, False),
    ("grad_x", 2057, 200, 5000, BF16, 256, False),
    ("grad_x", 1001, 16390, 1543, BF16, 256, True),
    ("grad_x", 2057, 17, 3001, BF16, 128, False),
    ("grad_x", 257, 8191, 5003, BF16, 128, True),
    ("grad_x", 2057, 17, 3001, F32, 128, False),
    ("grad_x", 501, 4093, 1543, F32, 128, True),
    ("grad_weight", 17, 2057, 5003, BF16, 256, False),
    ("grad_weight", 200, 2057, 5000, BF16, 256, False),
    ("grad_weight", 16390, 1001, 1543, BF16, 256, True),
    ("grad_weight", 8192, 2048, 2048, BF16, 256, True),
    ("grad_weight", 17, 2057, 3001, BF16, 128, False),
    ("grad_weight", 8191, 257, 5003, BF16, 128, True),
    ("grad_weight", 17, 2057, 3001, F32, 128, False),
    ("grad_weight", 4093, 501, 1543, F32, 128, True),
]


def _plan(product, rows, outputs, inputs, dtype, aligned=True):
    from rnn_kernel_amd import _lib

    d = _lib.describe_linear(product, rows, outputs, inputs, CODE[dtype], aligned)
    return d["form"], d["edge"], d["slices"] > 1


@pytest.mark.parametrize("case", FORWARD)
def test_forward_cases_take_the_forms_they_are_for(hip_lib, case):
    rows, outputs, inputs, dtype, left, *want = case
    assert _plan("y", rows, outputs, inputs, dtype, left * torch.finfo(dtype).bits // 8 % 16 == 0) == tuple(want)


@pytest.mark.parametrize("case", GRADIENTS)
def test_gradient_cases_take_the_forms_they_are_for(hip_lib, case):
    product, rows, outputs, inputs, dtype, edge, sliced = case
    assert _plan(product, rows, outputs, inputs, dtype) == ("tiles", edge, sliced)


def _inside(t, left):
    """t's values in a matrix that is NaN around them, `left` columns from its left edge."""
    ld = -(-(left + t.size(1) + 1) // 8) * 8
    full = torch.full((t.size(0) + 2, ld), float("nan"), dtype=t.dtype, device=t.device)
    inner = full[1:-1, left:left + t.size(1)]
    inner.copy_(t)
    return inner


def _check(got, want, norm, rounding):
    err = (got.double() - want).abs()
    rms = want.norm() / math.sqrt(want.numel())
    assert float(err.norm() / want.norm()) <= norm
    assert bool((err <= rounding * want.abs() + 8 * norm * rms).all())


def _rand(gpu, dtype, gen, *shape):
    return torch.randn(*shape, generator=gen, device=gpu).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("case", FORWARD)
def test_forward(gpu, case):
    from rnn_kernel_amd import linear

    rows, outputs, inputs, dtype, left, *form = case
    print(f"forward {case}", flush=True)
    gen = torch.Generator(device=gpu).manual_seed(rows + outputs + inputs)
    x = _rand(gpu, dtype, gen, rows, inputs)
    w = (_rand(gpu, F32, gen, outputs, inputs) / math.sqrt(inputs)).to(dtype)
    b, r = _rand(gpu, dtype, gen, outputs), _rand(gpu, dtype, gen, rows, outputs)
    z = x.double() @ w.double().t() + b.double()
    want = z * 0.5 * torch.erfc(-z / math.sqrt(2.0)) + r.double()
    y = linear(_inside(x, left), _inside(w, left), b, activation="gelu", residual=_inside(r, left))
    f32 = 2.0 ** -24 * (8 + 2 * math.sqrt(inputs))
    if dtype == F32:
        _check(y, want, f32, 2.0 ** -23)
    else:
        _check(y, want, 1.1 * 2.0 ** -8, 2.0 ** -8)
        # the rounding apart, what is left is float32's
        assert bool(((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 8 * f32 + 2.0 ** -20).all())


@pytest.mark.gpu
@pytest.mark.parametrize("case", GRADIENTS)
def test_gradients(gpu, case):
    from rnn_kernel_amd import linear

    product, rows, outputs, inputs, dtype, edge, sliced = case
    print(f"gradients {case}", flush=True)
    gen = torch.Generator(device=gpu).manual_seed(rows + outputs + inputs)
    x = _inside(_rand(gpu, dtype, gen, rows, inputs), 3)
    w = _inside((_rand(gpu, F32, gen, outputs, inputs) / math.sqrt(inputs)).to(dtype), 3)
    dy = _inside(_rand(gpu, dtype, gen, rows, outputs), 3)
    of = x if product == "grad_x" else w
    of.requires_grad_(True)
    terms = outputs if product == "grad_x" else rows
    for act in (None, "silu"):
        (got,) = torch.autograd.grad(linear(x, w, activation=act), of, dy)
        with torch.no_grad():
            dz = dy.double()
            if act:
                z = x.double() @ w.double().t()
                s = torch.sigmoid(z)
                dz = dz * s * (1 + z * (1 - s))
            want = dz @ w.double() if product == "grad_x" else dz.t() @ x.double()
        if dtype == F32:
            _check(got, want, 2.0 ** -24 * (8 + 2 * math.sqrt(max(terms, inputs))), 2.0 ** -23)
        else:
            _check(got, want, (3.3 if act else 1.1) * 2.0 ** -8, 2.0 ** -8)
