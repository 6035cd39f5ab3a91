"""The gated delta rule on more columns than CUs, where a workgroup of its chains takes two
blocks of 16: in either type, for every size of a key, with an odd number of blocks (half of
the last workgroup is empty) and heads that are no multiple of eight.  The form of each shape
is asked of the plan first, so that another rule for it shows here.

Against the recurrence in float64, token by token, and its gradients by automatic
differentiation.  Tolerances, set before the first run, as 2-norms: those of the rule at
fewer columns (float32 32 * 2^-24 for values, twice that for gradients, 1e-5 for dg, whose
terms cancel; bfloat16 1.1 * 2^-8).  For single elements a rounding of the element and 32
times the float32 part, of the tensor's root mean square (heads and tokens differ in size by
a few times, and an element is within a few standard deviations)."""
import math

import pytest
import torch

F32, BF16 = torch.float32, torch.bfloat16
F32_VALUE, F32_GRAD, F32_DG, ROUNDED = 2e-6, 4e-6, 1e-5, 1.1 * 2.0 ** -8

# B, T, Hk, Hv, Dk, Dv
SHAPES = [
    (3, 130, 16, 32, 64, 48),
    (5, 65, 16, 64, 17, 17),
    (3, 130, 16, 32, 128, 40),
    (2, 97, 33, 33, 160, 56),
    (2, 70, 65, 65, 256, 20),
]


@pytest.mark.parametrize("shape", SHAPES)
def test_shapes_take_two_blocks(hip_lib, shape):
    from rnn_kernel_amd import _lib

    B, _, _, Hv, Dk, Dv = shape
    for dtype in (0, 1):
        d = _lib.describe_gated_delta(B, Hv, Dk, Dv, dtype)
        # (float32 operands of the largest keys leave no registers for two)
        columns = 1 if dtype == 0 and Dk > 192 else 2
        assert d["columns"] == columns and d["steps"] == -(-Dk // 64) * 2
        assert d["workgroups"] == -(-B * Hv // 8) * 8 * -(-Dv // (16 * columns))
    few = _lib.describe_gated_delta(1, 16, Dk, 256, 1)
    assert few["columns"] == 1 and few["workgroups"] == 256


def test_describe_refuses(hip_lib):
    import ctypes

    out = (ctypes.c_int * 3)()
    assert hip_lib.rka_describe_gated_delta(1, 1, 16, 16, 2, out, 3) == 1001
    assert hip_lib.rka_describe_gated_delta(1, 1, 16, 16, 0, None, 3) == 1001
    assert hip_lib.rka_describe_gated_delta(1, 1, 257, 16, 0, out, 3) == 1004


def _oracle(q, k, v, g, beta, s0, lengths, normalize):
    if normalize:
        q, k = (t / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt() for t in (q, k))
    rep = v.size(2) // q.size(2)
    q, k = q.repeat_interleave(rep, 2) * q.size(-1) ** -0.5, k.repeat_interleave(rep, 2)
    S, out = s0, []
    for t in range(q.size(1)):
        live = (t < lengths)[:, None, None]
        Sd = S * g[:, t, :, None, None].exp()
        e = v[:, t] - (k[:, t, :, :, None] * Sd).sum(-2)
        Sn = Sd + k[:, t, :, :, None] * (beta[:, t, :, None] * e)[..., None, :]
        S = torch.where(live[..., None], Sn, S)
        out.append(torch.where(live, (q[:, t, :, :, None] * S).sum(-2), 0.0))
    return torch.stack(out, 1), S


def _check(name, got, want, f32):
    assert got.shape == want.shape and bool(torch.isfinite(got).all()), name
    err, rms = (got.double() - want).abs(), float(want.norm()) / math.sqrt(want.numel())
    norm, unit = (ROUNDED, 2.0 ** -8) if got.dtype == BF16 else (f32, 2.0 ** -23)
    assert float(err.norm() / want.norm()) <= norm, name
    assert bool((err <= unit * want.abs() + 32 * f32 * rms).all()), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("normalize,ragged", [(True, True), (False, False)])
@pytest.mark.parametrize("shape", SHAPES)
def test_rule_and_gradients(gpu, shape, normalize, ragged, dtype):
    from rnn_kernel_amd import gated_delta_rule

    print(f"wide {shape} normalize={normalize} ragged={ragged} {dtype}", flush=True)
    B, T, Hk, Hv, Dk, Dv = shape
    gen = torch.Generator(device=gpu).manual_seed(T + Dk)

    def rand(*s):
        return torch.randn(*s, generator=gen, device=gpu)

    q, k = ((rand(B, T, Hk, Dk) / Dk ** 0.5).to(dtype) for _ in range(2))
    x = [q, k, rand(B, T, Hv, Dv).to(dtype), torch.nn.functional.logsigmoid(rand(B, T, Hv) + 2.0),
         torch.sigmoid(rand(B, T, Hv)), rand(B, Hv, Dk, Dv)]
    lengths = torch.tensor([T, 65, 0, 1, 64][:B] if ragged else [T] * B, dtype=torch.int32, device=gpu).clamp(max=T)
    up = [rand(B, T, Hv, Dv).to(dtype), rand(B, Hv, Dk, Dv)]
    with torch.no_grad():
        plain = gated_delta_rule(*x, normalize=normalize, lengths=lengths if ragged else None)
    leaves = [t.clone().requires_grad_(True) for t in x]
    got = gated_delta_rule(*leaves, normalize=normalize, lengths=lengths if ragged else None)
    for a, b in zip(got, plain):
        assert torch.equal(a, b)
    ref = [t.double().requires_grad_(True) for t in x]
    want = _oracle(*ref, lengths, normalize)
    for name, a, b in zip(("o", "state"), got, want):
        _check(name, a.detach(), b.detach(), F32_VALUE)
    grads = torch.autograd.grad(got, leaves, up)
    refs = torch.autograd.grad(want, ref, [t.double() for t in up])
    for name, a, b in zip(("dq", "dk", "dv", "dg", "dbeta", "ds0"), grads, refs):
        _check(name, a, b, F32_DG if name == "dg" else F32_GRAD)
    if ragged:
        behind = torch.arange(T, device=gpu)[None] >= lengths[:, None]
        assert not got[0][behind].any() and all(not t[behind].any() for t in grads[:5])
