"""What the selective scan, the convolution, layer norm and the cross entropy refuse, and say:
in Python and at the C entries, before anything reaches a GPU."""
import ctypes

import pytest
import torch

INVALID, WORKSPACE, SHAPE = 1001, 1002, 1004
P = 4096  # an address that is only looked at


def _scan_inputs(B=2, T=3, D=4, N=5, G=2):
    return [torch.randn(B, T, D), torch.randn(B, T, D), -torch.rand(D, N), torch.randn(B, T, G, N), torch.randn(B, T, G, N)]


def test_cpu_tensors_are_refused():
    from rnn_kernel_amd import (CausalConvFunction, LayerNorm, LayerNormFunction, LinearCrossEntropy, LinearCrossEntropyFunction,
                                SelectiveScan, SelectiveScanFunction, causal_conv, causal_conv_step, layer_norm,
                                linear_cross_entropy, selective_scan, selective_step)

    s = _scan_inputs()
    x, w, t = torch.randn(3, 4), torch.randn(5, 4), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: selective_scan(*s), lambda: selective_step(*[a[:, 0] if a.dim() > 2 else a for a in s], torch.zeros(2, 4, 5)),
                 lambda: SelectiveScanFunction.apply(*s, None, None, None, None, False, None),
                 lambda: causal_conv(s[0], torch.randn(4, 3)), lambda: causal_conv_step(x, torch.zeros(3, 2, 4), torch.randn(4, 3)),
                 lambda: CausalConvFunction.apply(s[0], torch.randn(4, 3), None, None, None, None),
                 lambda: layer_norm(x), lambda: LayerNorm(4)(x), lambda: LayerNormFunction.apply(x, None, None, 1e-5),
                 lambda: linear_cross_entropy(x, w, t), lambda: LinearCrossEntropy(4, 5)(x, t),
                 lambda: LinearCrossEntropyFunction.apply(x, w, t, None, -100, "mean"), lambda: SelectiveScan(4)(s[0])):
        with pytest.raises(RuntimeError, match="x must be a CUDA/HIP tensor"):
            call()


def test_modules_refuse_impossible_sizes():
    from rnn_kernel_amd import LayerNorm, LinearCrossEntropy, SelectiveScan

    for size in (0, 16385):
        with pytest.raises(ValueError, match="size must be in"):
            LayerNorm(size)
    with pytest.raises(ValueError, match="vocabulary must be in"):
        LinearCrossEntropy(4, 0)
    with pytest.raises(ValueError, match="reduction must be one of"):
        LinearCrossEntropy(4, 4, reduction="median")
    with pytest.raises(ValueError, match="multiple of groups"):
        SelectiveScan(8, 9, groups=2)
    with pytest.raises(ValueError, match="states must be at most 64"):
        SelectiveScan(8, states=65)
    with pytest.raises(ValueError, match="width in"):
        SelectiveScan(8, width=9)
    layer = SelectiveScan(8)
    with pytest.raises(ValueError, match="batch, tokens, 8"):
        layer(torch.randn(2, 8))
    with pytest.raises(ValueError, match="requests, 8"):
        layer.step(torch.randn(2, 3, 8), layer.new_states(2))


def test_parameters_are_torchs():
    from rnn_kernel_amd import LayerNorm, LinearCrossEntropy

    norm, ref = LayerNorm(6), torch.nn.LayerNorm(6)
    norm.load_state_dict(ref.state_dict())
    head, lin = LinearCrossEntropy(5, 7, bias=True), torch.nn.Linear(5, 7)
    head.load_state_dict(lin.state_dict())
    assert torch.equal(head.weight, lin.weight) and torch.equal(norm.bias, ref.bias)
    assert LayerNorm(6, bias=False).bias is None and LinearCrossEntropy(5, 7).bias is None


STRIDES = (ctypes.c_longlong * 12)()


def _scan(lib, sizes=(1, 8, 16, 4, 2), x=P, y=P, ws=P, nbytes=1 << 40, dtype=0, strides=STRIDES):
    return lib.rka_selective_scan_forward(x, P, P, P, P, None, None, None, None, None, y, P, None, ws, nbytes, *sizes, strides, 1,
                                          dtype, None)


def _scan_back(lib, sizes=(1, 8, 16, 4, 2), x=P, y=P, ws=P, nbytes=1 << 40, dtype=0, strides=STRIDES):
    return lib.rka_selective_scan_backward(x, P, P, P, P, None, None, None, None, P, P, None, y, P, P, P, P, None, None, None, None,
                                           ws, nbytes, *sizes, strides, 1, dtype, None)


def _scan_step(lib, sizes=(1, 8, 16, 4, 2), x=P, y=P, ws=P, nbytes=1 << 40, dtype=0, strides=STRIDES, num_slots=1):
    return lib.rka_selective_step(x, P, P, P, P, None, None, None, P, None, num_slots, y, sizes[0], *sizes[2:], strides, 1, dtype, None)


@pytest.mark.parametrize("entry", [_scan, _scan_back, _scan_step])
def test_scan_entries_refuse(hip_lib, entry):
    for sizes, status, message in (((-1, 8, 16, 4, 2), INVALID, "batch and tokens"), ((1, 8, 0, 4, 2), INVALID, "multiple of groups"),
                                   ((1, 8, 15, 4, 2), INVALID, "multiple of groups"), ((1, 8, 16, 0, 2), INVALID, "states must be"),
                                   ((1, 8, 16, 65, 2), SHAPE, "more than 64 states"), ((1, 8, 16, 4, 0), INVALID, "groups")):
        assert entry(hip_lib, sizes=sizes) == status, sizes
        assert message in hip_lib.rka_last_error().decode()
    assert entry(hip_lib, dtype=2) == INVALID and entry(hip_lib, strides=None) == INVALID
    assert entry(hip_lib, x=None) == INVALID and entry(hip_lib, y=None) == INVALID
    assert "null tensor" in hip_lib.rka_last_error().decode()


def test_scan_workspaces(hip_lib):
    long = (1, 4096, 64, 16, 1)
    assert hip_lib.rka_selective_scan_forward_workspace_bytes(*long) > 0
    assert _scan(hip_lib, long, nbytes=8) == WORKSPACE and _scan(hip_lib, long, ws=None) == WORKSPACE
    assert _scan(hip_lib, long, ws=P + 8) == INVALID and "multiple of 16" in hip_lib.rka_last_error().decode()
    assert _scan_back(hip_lib, nbytes=8) == WORKSPACE
    assert _scan_step(hip_lib, (2, 1, 16, 4, 2)) == INVALID and "fewer states" in hip_lib.rka_last_error().decode()
    assert _scan(hip_lib, (0, 8, 16, 4, 2), x=None, y=None) == 0
    for sizes in ((1, 8, 15, 4, 2), (1, 8, 16, 65, 2), (-1, 8, 16, 4, 2)):
        for name in ("forward_workspace", "reserve", "backward_workspace"):
            assert getattr(hip_lib, f"rka_selective_scan_{name}_bytes")(*sizes) == 0


def test_conv_entries_refuse(hip_lib):
    def forward(sizes=(1, 8, 16, 4), x=P, act=3, dtype=0):
        return hip_lib.rka_causal_conv_forward(x, 128, 16, P, None, None, None, P, P, *sizes, act, dtype, None)

    def backward(sizes=(1, 8, 16, 4), x=P, act=3, dtype=0, ws=P, nbytes=1 << 40):
        return hip_lib.rka_causal_conv_backward(P, None, x, 128, 16, P, None, None, None, P, P, None, None, ws, nbytes, *sizes, act,
                                                dtype, None)

    def step(sizes=(1, 8, 16, 4), x=P, act=3, dtype=0, slots=1):
        return hip_lib.rka_causal_conv_step(x, 16, P, None, P, None, slots, P, sizes[0], *sizes[2:], act, dtype, None)

    for call in (forward, backward, step):
        assert call((-1, 8, 16, 4)) == INVALID and call((1, 8, 0, 4)) == INVALID
        assert call((1, 8, 16, 1)) == SHAPE and call((1, 8, 16, 9)) == SHAPE and "width" in hip_lib.rka_last_error().decode()
        assert call(act=1) == INVALID and call(dtype=2) == INVALID and call(x=None) == INVALID
    for call in (forward, backward):
        assert call((65536, 8, 16, 4)) == SHAPE and call((1, 1 << 23, 16, 4)) == SHAPE
    assert backward(nbytes=4) == WORKSPACE and backward(ws=None) == WORKSPACE
    assert step((2, 1, 16, 4)) == INVALID and "fewer states" in hip_lib.rka_last_error().decode()
    assert forward((0, 8, 16, 4), x=None) == 0 and step((0, 1, 16, 4), x=None) == 0
    assert hip_lib.rka_causal_conv_backward_workspace_bytes(1, 8, 16, 9) == 0


def test_norm_entries_refuse(hip_lib):
    def forward(rows=2, size=8, x=P, ldx=8, mean=P, dtype=0):
        return hip_lib.rka_layer_norm_forward(x, ldx, None, None, P, mean, P, rows, size, 1e-5, dtype, None)

    def backward(rows=2, size=8, x=P, ldx=8, mean=P, dtype=0, ws=P, nbytes=1 << 40):
        return hip_lib.rka_layer_norm_backward(P, 8, x, ldx, None, mean, P, P, P, None, ws, nbytes, rows, size, dtype, None)

    for call in (forward, backward):
        assert call(rows=-1) == INVALID and call(size=0) == INVALID and call(size=16385) == SHAPE
        assert call(ldx=-1) == INVALID and call(dtype=5) == INVALID and call(x=None) == INVALID and call(mean=None) == INVALID
    assert forward(rows=0, x=None) == 0 and backward(rows=0) == INVALID
    assert backward(nbytes=4) == WORKSPACE and backward(ws=None) == WORKSPACE
    assert hip_lib.rka_layer_norm_backward_workspace_bytes(4, 16385, 0) == 0


def test_cross_entropy_entries_refuse(hip_lib):
    def forward(sizes=(4, 8, 16), x=P, ldx=8, ldw=8, reduction=1, dtype=0, ws=P, nbytes=1 << 40):
        return hip_lib.rka_cross_entropy_forward(x, ldx, P, ldw, None, P, 1, -100, P, P, ws, nbytes, *sizes, reduction, dtype, None)

    def backward(sizes=(4, 8, 16), x=P, ldx=8, ldw=8, reduction=1, dtype=0, ws=P, nbytes=1 << 40):
        return hip_lib.rka_cross_entropy_backward(P, x, ldx, P, ldw, None, P, P, P, None, ws, nbytes, *sizes, reduction, dtype, None)

    for call in (forward, backward):
        for sizes in ((0, 8, 16), (4, 0, 16), (4, 8, 0), (-4, 8, 16)):
            assert call(sizes) == INVALID
        most = (1 << 21) + 1
        for sizes in ((most, 8, 16), (4, most, 16), (4, 8, most)):
            assert call(sizes) == SHAPE and "2^21" in hip_lib.rka_last_error().decode()
        assert call(ldw=most) == SHAPE and call(ldx=-1) == INVALID and call(reduction=3) == INVALID and call(dtype=2) == INVALID
        assert call(x=None) == INVALID and call(nbytes=16) == WORKSPACE and call(ws=None) == WORKSPACE and call(ws=P + 4) == INVALID
    for name in ("forward", "backward"):
        assert getattr(hip_lib, f"rka_cross_entropy_{name}_workspace_bytes")(0, 8, 16, 0) == 0
    assert hip_lib.rka_cross_entropy_reserve_bytes(0) == 0
