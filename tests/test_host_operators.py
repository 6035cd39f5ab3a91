"""What the gated delta rule and the matrix product refuse, and say: in Python and at
the C entries, before anything reaches a GPU."""
import ctypes

import pytest
import torch

INVALID, WORKSPACE, SHAPE = 1001, 1002, 1004


def _delta_inputs(B=2, T=3, Hk=1, Hv=2, Dk=4, Dv=5):
    return [torch.randn(B, T, Hk, Dk), torch.randn(B, T, Hk, Dk), torch.randn(B, T, Hv, Dv), -torch.rand(B, T, Hv),
            torch.rand(B, T, Hv)]


def test_cpu_tensors_are_refused():
    from rnn_kernel_amd import GatedDelta, Linear, gated_delta_rule, gated_delta_step, linear

    q = _delta_inputs()
    with pytest.raises(RuntimeError, match="q must be a CUDA/HIP tensor"):
        gated_delta_rule(*q)
    with pytest.raises(RuntimeError, match="q must be a CUDA/HIP tensor"):
        gated_delta_step(*[t[:, 0] for t in q], torch.zeros(2, 2, 4, 5))
    with pytest.raises(RuntimeError, match="x must be a CUDA/HIP tensor"):
        linear(torch.randn(2, 4), torch.randn(3, 4))
    with pytest.raises(RuntimeError, match="x must be a CUDA/HIP tensor"):
        Linear(4, 3)(torch.randn(2, 4))
    with pytest.raises(RuntimeError, match="CUDA/HIP tensor"):
        GatedDelta(8, 2, 4, 4)(torch.randn(1, 2, 8))


def test_modules_refuse_impossible_sizes():
    from rnn_kernel_amd import GatedDelta, Linear

    with pytest.raises(ValueError, match="in_features"):
        Linear(0, 4)
    with pytest.raises(ValueError, match="activation must be one of"):
        Linear(4, 4, activation="tanh")
    with pytest.raises(ValueError, match="multiple of key_heads"):
        GatedDelta(8, 3, 4, 4, 2)
    with pytest.raises(ValueError, match="sizes must be >= 1"):
        GatedDelta(8, 0, 4, 4)
    layer = GatedDelta(8, 2, 4, 4)
    with pytest.raises(ValueError, match="batch, tokens, 8"):
        layer(torch.randn(2, 8))
    with pytest.raises(ValueError, match="requests, 8"):
        layer.step(torch.randn(2, 3, 8), layer.new_states(2))


def test_linear_has_nn_linears_parameters():
    from rnn_kernel_amd import Linear

    ours, ref = Linear(5, 7), torch.nn.Linear(5, 7)
    ours.load_state_dict(ref.state_dict())
    assert torch.equal(ours.weight, ref.weight) and torch.equal(ours.bias, ref.bias)
    assert Linear(5, 7, bias=False).bias is None


def test_the_command_needs_a_gpu():
    from rnn_kernel_amd.delta_train import main

    with pytest.raises(RuntimeError, match="runs on a GPU"):
        main(["--device", "cpu"])
    with pytest.raises(ValueError, match="--answer"):
        main(["--seq-len", "8", "--answer", "8"])


P = 4096  # an address that is only looked at


def _linear(lib, rows=2, outputs=3, inputs=4, ldx=4, ldw=4, x=P, w=P, y=P, ws=None, nbytes=0, act=0, dtype=0):
    return lib.rka_linear_forward(x, ldx, w, ldw, None, None, 0, y, None, ws, nbytes, rows, outputs, inputs, act, dtype, None)


@pytest.mark.parametrize("change,status,message", [
    (dict(rows=-1), INVALID, "sizes must be >= 1"), (dict(outputs=0), INVALID, "sizes must be >= 1"),
    (dict(inputs=0), INVALID, "sizes must be >= 1"), (dict(act=6), INVALID, "unknown activation"),
    (dict(act=-1), INVALID, "unknown activation"), (dict(dtype=2), INVALID, "dtype must be"),
    (dict(ldx=(1 << 21) + 1), SHAPE, "row strides"), (dict(ldw=-4), SHAPE, "row strides"),
    (dict(x=None), INVALID, "null tensor"), (dict(w=None), INVALID, "null tensor"), (dict(y=None), INVALID, "null tensor"),
    (dict(rows=128, outputs=128, inputs=4096, ldx=4096, ldw=4096), WORKSPACE, "workspace needs")])
def test_linear_entry_refuses(hip_lib, change, status, message):
    assert _linear(hip_lib, **change) == status
    assert message in hip_lib.rka_last_error().decode() and "linear_forward" in hip_lib.rka_last_error().decode()


def test_linear_backward_entry_refuses(hip_lib):
    def call(dy=P, x=P, w=P, z=P, dx=P, dw=P, ws=P, nbytes=1 << 40, sizes=(2, 3, 4), act=3, dtype=0):
        return hip_lib.rka_linear_backward(dy, 3, x, 4, w, 4, z, dx, dw, None, ws, nbytes, *sizes, act, dtype, None)

    assert call(sizes=(0, 3, 4)) == INVALID and call(dtype=9) == INVALID and call(act=7) == INVALID
    for missing in ("dy", "x", "w", "z"):
        assert call(**{missing: None}) == INVALID and "null tensor" in hip_lib.rka_last_error().decode()
    assert call(nbytes=0) == WORKSPACE and call(ws=None) == WORKSPACE


def test_linear_without_rows_does_nothing(hip_lib):
    assert _linear(hip_lib, rows=0, x=None, y=None) == 0
    assert hip_lib.rka_linear_forward_workspace_bytes(0, 4, 4, 0) == 0
    assert hip_lib.rka_linear_backward_workspace_bytes(4, 0, 4, 0) == 0


STRIDES = (ctypes.c_longlong * 15)()


def _forward(lib, sizes=(1, 8, 1, 2, 16, 16), q=P, o=P, ws=P, nbytes=1 << 40, dtype=0, gate=0, strides=STRIDES):
    return lib.rka_gated_delta_forward(q, P, P, P, P, None, None, o, P, None, ws, nbytes, *sizes, strides, dtype, gate, 0, 1.0, None)


def _backward(lib, sizes=(1, 8, 1, 2, 16, 16), reserve=P, dq=P, ws=P, nbytes=1 << 40, dtype=0, gate=0, strides=STRIDES):
    return lib.rka_gated_delta_backward(P, P, P, P, None, reserve, P, None, dq, P, P, P, P, None, ws, nbytes, *sizes, strides,
                                        dtype, gate, 0, 1.0, None)


def _step(lib, sizes=(1, 8, 1, 2, 16, 16), state=P, slots=None, num_slots=1, dtype=0, gate=0, strides=STRIDES):
    batch, _, hk, hv, dk, dv = sizes
    return lib.rka_gated_delta_step(P, P, P, P, P, state, slots, num_slots, P, batch, hk, hv, dk, dv, strides, dtype, gate, 0, 1.0,
                                    None)


@pytest.mark.parametrize("entry", [_forward, _backward, _step])
def test_delta_entries_refuse(hip_lib, entry):
    for sizes, status, message in (((-1, 8, 1, 2, 16, 16), INVALID, "batch and tokens"), ((1, 8, 0, 2, 16, 16), INVALID, "heads"),
                                   ((1, 8, 2, 3, 16, 16), INVALID, "multiple of key heads"),
                                   ((1, 8, 1, 2, 257, 16), SHAPE, "key head size exceeds 256"),
                                   ((1, 8, 1, 2, 16, 0), INVALID, "head sizes"),
                                   ((1 << 20, 8, 1, 1 << 12, 16, 16), SHAPE, "exceeds 2^31")):
        assert entry(hip_lib, sizes=sizes) == status, sizes
        assert message in hip_lib.rka_last_error().decode()
    assert entry(hip_lib, dtype=2) == INVALID and entry(hip_lib, gate=-1) == INVALID
    assert entry(hip_lib, strides=None) == INVALID and "strides" in hip_lib.rka_last_error().decode()


def test_delta_entries_refuse_missing_tensors_and_workspaces(hip_lib):
    assert _forward(hip_lib, q=None) == INVALID and _forward(hip_lib, o=None) == INVALID
    assert _forward(hip_lib, nbytes=1) == WORKSPACE and _forward(hip_lib, ws=None) == WORKSPACE
    assert _backward(hip_lib, reserve=None) == INVALID and _backward(hip_lib, dq=None) == INVALID
    assert _backward(hip_lib, nbytes=1) == WORKSPACE
    assert _step(hip_lib, state=None) == INVALID
    assert _step(hip_lib, sizes=(2, 1, 1, 2, 16, 16)) == INVALID and "fewer states" in hip_lib.rka_last_error().decode()


def test_delta_sizes_of_refused_calls_are_zero(hip_lib):
    for sizes in ((1, 8, 2, 3, 16, 16), (1, 8, 1, 2, 300, 16), (-1, 8, 1, 2, 16, 16)):
        assert hip_lib.rka_gated_delta_forward_workspace_bytes(*sizes, 1) == 0
        assert hip_lib.rka_gated_delta_backward_workspace_bytes(*sizes, 1) == 0
        assert hip_lib.rka_gated_delta_reserve_bytes(*sizes) == 0
