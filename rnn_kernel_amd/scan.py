"""The selective scan, a recurrent layer with a few numbers of state per channel whose decay
and input are made of the token, on the HIP library.

Per channel d of group g and state n, held in float32, with s = softplus(dt + dt_bias) or dt
+ dt_bias:

    h_t = exp(s_t A[d, n]) h_{t-1} + s_t x_t B_t[g, n]
    y_t = (sum_n C_t[g, n] h_t + skip[d] x_t) silu(gate_t)

* ``selective_scan``: whole sequences (training and prompts), with gradients;
* ``selective_step``: one token of each of a batch of requests, the states updated in place
  (answering).

Like the GRU they raise RuntimeError for tensors of other devices or types, ValueError for
shapes, and have no CPU fallback.
"""
from __future__ import annotations

import ctypes
from typing import List, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _args, _lib

MAX_STATES = 64
MAX_TOKENS = 2 ** 30
MAX_TOKEN_STRIDE = 2 ** 21  # elements: the kernels' offsets within a tile are 32-bit


def _fits(x, dt, A, B, C, skip, gate, dt_bias, lead: int) -> bool:
    """Whether the arguments are what the operators take (a call is a few us of the host: one
    expression for all that is right, `_check` to say what is not)."""
    dtype, index, shape = x.dtype, x.get_device(), x.shape
    a, b = A.shape, B.shape
    if len(shape) != lead + 1 or len(a) != 2 or len(b) != lead + 2 or dtype not in _args.DTYPES or not x.is_cuda:
        return False
    channels, states, groups = shape[lead], a[1], b[lead]
    return (index == dt.get_device() == A.get_device() == B.get_device() == C.get_device()
            and dt.dtype is dtype and B.dtype is dtype and C.dtype is dtype and A.dtype is torch.float32
            and dt.shape == shape and C.shape == b and b[:lead] == shape[:lead] and b[lead + 1] == states
            and a[0] == channels and 1 <= states <= MAX_STATES and 1 <= channels <= MAX_TOKEN_STRIDE and groups >= 1
            and channels % groups == 0 and (lead == 1 or shape[1] <= MAX_TOKENS) and shape[0] <= _args.MAX_SIZE
            and (gate is None or (gate.shape == shape and gate.dtype is dtype and gate.get_device() == index))
            and (skip is None or (skip.shape == a[:1] and skip.dtype is torch.float32 and skip.get_device() == index))
            and (dt_bias is None or (dt_bias.shape == a[:1] and dt_bias.dtype is torch.float32 and dt_bias.get_device() == index)))


def _check(what: str, x, dt, A, B, C, skip, gate, dt_bias, tokens: bool) -> None:
    lead = 2 if tokens else 1
    if _fits(x, dt, A, B, C, skip, gate, dt_bias, lead):
        return
    _args.check_dtype(what, x, "x")
    f32 = torch.float32
    _args.check_tensors(what, x, (dt, "dt", x.dtype), (A, "A", f32), (B, "B", x.dtype), (C, "C", x.dtype), (skip, "skip", f32),
                        (gate, "gate", x.dtype), (dt_bias, "dt_bias", f32))
    if x.dim() != lead + 1 or x.size(-1) < 1:
        raise ValueError(f"{what}: x must have shape {'[batch, tokens, channels]' if tokens else '[batch, channels]'}")
    channels = x.size(-1)
    if A.dim() != 2 or A.size(0) != channels or not 1 <= A.size(1) <= MAX_STATES:
        raise ValueError(f"{what}: A must have shape [{channels}, states], states in [1, {MAX_STATES}]")
    if B.dim() != lead + 2 or B.shape[:lead] != x.shape[:lead] or B.size(-1) != A.size(1):
        raise ValueError(f"{what}: B must have shape {[*x.shape[:lead], 'groups', A.size(1)]}")
    if B.size(lead) < 1 or channels % B.size(lead) != 0:
        raise ValueError(f"{what}: channels must be a multiple of groups")
    _args.check_shape(what, C, "C", B.shape)
    for t, name in ((dt, "dt"), (gate, "gate")):
        _args.check_shape(what, t, name, x.shape)
    for t, name in ((skip, "skip"), (dt_bias, "dt_bias")):
        _args.check_shape(what, t, name, (channels,))
    if channels > MAX_TOKEN_STRIDE:
        raise ValueError(f"{what}: at most 2^21 channels")
    if tokens and x.size(1) > MAX_TOKENS:
        raise ValueError(f"{what}: at most 2^30 tokens")
    raise ValueError(f"{what}: sizes must be below 2^31")


def _near(t):
    """``t`` with its last dimension's elements side by side and tokens at most MAX_TOKEN_STRIDE
    apart: a copy where they are not."""
    t = _args.dense_last(t)
    return t if t is None or t.size(1) <= 1 or t.stride(1) <= MAX_TOKEN_STRIDE else t.contiguous()


def _strides(x, dt, gate, B, C):
    """What the C entries take: batch row, token (and group) of each."""
    if x.dim() == 3:
        of_gate = (0, 0) if gate is None else gate.stride()[:2]
        return (ctypes.c_longlong * 12)(*x.stride()[:2], *dt.stride()[:2], *of_gate, *B.stride()[:3], *C.stride()[:3])
    of_gate = 0 if gate is None else gate.stride(0)
    return (ctypes.c_longlong * 12)(x.stride(0), 0, dt.stride(0), 0, of_gate, 0, B.stride(0), 0, B.stride(1), C.stride(0), 0,
                                    C.stride(1))


def _forward(x, dt, A, B, C, initial_state, skip, gate, dt_bias, softplus: bool, lengths, training: bool):
    """Checks, and the forward: y, final_state, what is saved if ``training``, and the inputs as
    they were used."""
    what = "selective_scan"
    _check(what, x, dt, A, B, C, skip, gate, dt_bias, tokens=True)
    batch, tokens, channels = x.shape
    groups, states = B.shape[2:]
    _args.check_tensors(what, x, (initial_state, "initial_state", torch.float32))
    _args.check_shape(what, initial_state, "initial_state", (batch, channels, states))
    _args.check_row_ints(what, lengths, "lengths", batch, x.device)
    x, dt, gate, B, C = (_near(t) for t in (x, dt, gate, B, C))
    A, initial_state, skip, dt_bias, lengths = (_args.dense(t) for t in (A, initial_state, skip, dt_bias, lengths))
    lib, sizes = _lib.load(), (batch, tokens, channels, states, groups)
    y = torch.empty(batch, tokens, channels, dtype=x.dtype, device=x.device)
    final_state = torch.empty(batch, channels, states, dtype=torch.float32, device=x.device)
    nbytes = lib.rka_selective_scan_forward_workspace_bytes(*sizes)
    ws = _args.workspace(nbytes, x.device) if nbytes else None
    reserve = _args.workspace(lib.rka_selective_scan_reserve_bytes(*sizes), x.device) if training else None
    _lib.call(x.get_device(), "rka_selective_scan_forward", x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(),
              C.data_ptr(), _lib.ptr(skip), _lib.ptr(gate), _lib.ptr(dt_bias), _lib.ptr(initial_state), _lib.ptr(lengths),
              y.data_ptr(), final_state.data_ptr(), _lib.ptr(reserve), _lib.ptr(ws), nbytes, *sizes,
              _strides(x, dt, gate, B, C), int(softplus), _args.DTYPES[x.dtype])
    return y, final_state, (x, dt, A, B, C, skip, gate, dt_bias, lengths, reserve)


class SelectiveScanFunction(torch.autograd.Function):
    """apply(x, dt, A, B, C, initial_state, skip, gate, dt_bias, softplus, lengths) -> (y,
    final_state), as selective_scan, with gradients of the first nine."""

    @staticmethod
    def forward(ctx, x, dt, A, B, C, initial_state, skip, gate, dt_bias, softplus, lengths):
        y, final_state, saved = _forward(x, dt, A, B, C, initial_state, skip, gate, dt_bias, softplus, lengths, training=True)
        ctx.save_for_backward(*saved)
        ctx.sizes, ctx.softplus, ctx.device, ctx.dtype = (*x.shape, *A.shape[1:], B.size(2)), bool(softplus), x.device, x.dtype
        ctx.set_materialize_grads(False)
        return y, final_state

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y, grad_state):
        x, dt, A, B, C, skip, gate, dt_bias, lengths, reserve = ctx.saved_tensors
        batch, tokens, channels, states, groups = ctx.sizes
        device, dtype, f32, lib = ctx.device, ctx.dtype, torch.float32, _lib.load()
        wide, of_states, of_a = (batch, tokens, channels), (batch, tokens, groups, states), (channels, states)
        _lib.check_saved("selective_scan", device, (x, dtype, wide), (dt, dtype, wide), (A, f32, of_a), (B, dtype, of_states),
                         (C, dtype, of_states), (skip, f32, (channels,)), (gate, dtype, wide), (dt_bias, f32, (channels,)),
                         (lengths, torch.int32, (batch,)),
                         (reserve, torch.uint8, (max(lib.rka_selective_scan_reserve_bytes(*ctx.sizes), 1),)))
        # (hooks may have given them back in another layout than they were saved in)
        x, dt, gate, B, C = (_near(t) for t in (x, dt, gate, B, C))
        A, skip, dt_bias, lengths, reserve, grad_y, grad_state = (
            _args.dense(t) for t in (A, skip, dt_bias, lengths, reserve, grad_y, grad_state))
        dx, ddt = (torch.empty(wide, dtype=dtype, device=device) for _ in range(2))
        dgate = torch.empty(wide, dtype=dtype, device=device) if gate is not None else None
        dB, dC = (torch.empty(of_states, dtype=dtype, device=device) for _ in range(2))
        dA = torch.empty(of_a, dtype=f32, device=device)
        dskip, dbias = (torch.empty(channels, dtype=f32, device=device) if t is not None else None for t in (skip, dt_bias))
        ds0 = torch.empty(batch, *of_a, dtype=f32, device=device) if ctx.needs_input_grad[5] else None
        if batch == 0:
            for t in (dA, dskip, dbias):
                if t is not None:
                    t.zero_()
            return dx, ddt, dA, dB, dC, ds0, dskip, dgate, dbias, None, None
        nbytes = lib.rka_selective_scan_backward_workspace_bytes(*ctx.sizes)
        ws = _args.workspace(nbytes, device)
        _lib.call(_args.index_of(device), "rka_selective_scan_backward", x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(),
                  C.data_ptr(), _lib.ptr(skip), _lib.ptr(gate), _lib.ptr(dt_bias), _lib.ptr(lengths), reserve.data_ptr(),
                  _lib.ptr(grad_y), _lib.ptr(grad_state), dx.data_ptr(), ddt.data_ptr(), dA.data_ptr(), dB.data_ptr(),
                  dC.data_ptr(), _lib.ptr(dskip), _lib.ptr(dgate), _lib.ptr(dbias), _lib.ptr(ds0), ws.data_ptr(), nbytes,
                  *ctx.sizes, _strides(x, dt, gate, B, C), int(ctx.softplus), _args.DTYPES[dtype])
        return dx, ddt, dA, dB, dC, ds0, dskip, dgate, dbias, None, None


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   initial_state: Optional[torch.Tensor] = None, *, skip: Optional[torch.Tensor] = None,
                   gate: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None, softplus: bool = False,
                   lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The scan over whole sequences: ``(y, final_state)``.

    x, dt and gate (or None) [B, T, D], B and C [B, T, G, N], all float32 or all bfloat16 and
    of any strides, D a multiple of G (channel d is of group d // (D // G)), N at most 64; A
    [D, N], skip and dt_bias [D] (or None) float32; initial_state [B, D, N] float32 or None
    (zeros).  ``softplus``: steps are softplus(dt + dt_bias), else dt + dt_bias.  ``lengths``
    [B] int32: row b ends after lengths[b] tokens; what lies behind is not read, its outputs
    and gradients are 0.  y has x's shape and type; the final state is float32.  States, sums
    and the gradients of A, skip and dt_bias are float32 throughout.  Tensors with forward-mode
    tangents are refused."""
    inputs = (x, dt, A, B, C, initial_state, skip, gate, dt_bias)
    _lib.refuse_tangents("selective_scan", *inputs)
    if _args.wants_grad(*inputs):
        return SelectiveScanFunction.apply(*inputs, softplus, lengths)
    return _forward(*inputs, softplus, lengths, training=False)[:2]


def selective_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, state: torch.Tensor, *,
                   skip: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                   dt_bias: Optional[torch.Tensor] = None, softplus: bool = False,
                   slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of each of B requests: y [B, D]; ``state`` is updated in place.

    x, dt and gate [B, D], B and C [B, G, N], the rest as in selective_scan.  state [M, D, N]
    float32, contiguous: request b has state ``slots[b]`` (int32 [B], distinct), or b if
    ``slots`` is None.  A negative slot marks a request without a state (padding): its output
    is 0; a slot from M up gives NaN; neither touches a state.  No gradients: with grad mode
    on, inputs that require them are refused, and so are forward-mode tangents.  Autograd
    counts the call as a change of ``state``."""
    what = "selective_step"
    _lib.refuse_tangents(what, x, dt, A, B, C, state, skip, gate, dt_bias)
    _check(what, x, dt, A, B, C, skip, gate, dt_bias, tokens=False)
    batch, channels = x.shape
    _, groups, states = B.shape
    of = state.shape
    if len(of) != 3 or of[1] != channels or of[2] != states or state.dtype is not torch.float32 or state.get_device() != x.get_device():
        _args.check_tensors(what, x, (state, "state", torch.float32))
        raise ValueError(f"{what}: state must have shape [slots, {channels}, {states}]")
    slots_held = of[0]
    if slots_held > _args.MAX_SIZE:
        raise ValueError(f"{what}: sizes must be below 2^31")
    if not state.is_contiguous():
        raise ValueError(f"{what}: state must be contiguous")
    if torch.is_grad_enabled() and _args.wants_grad(x, dt, A, B, C, state, skip, gate, dt_bias):
        raise RuntimeError(f"{what} has no gradients; use selective_scan or torch.no_grad()")
    if slots is not None:
        _args.check_row_ints(what, slots, "slots", batch, x.device)
        slots = slots.contiguous()
    elif slots_held < batch:
        raise ValueError(f"{what}: fewer states than requests")
    last = _args.dense_last
    x, dt, B, C, A = last(x), last(dt), last(B), last(C), A.contiguous()
    gate = None if gate is None else last(gate)
    skip = None if skip is None else skip.contiguous()
    dt_bias = None if dt_bias is None else dt_bias.contiguous()
    y = x.new_empty((batch, channels))
    _lib.call(x.get_device(), "rka_selective_step", x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(),
              _lib.ptr(skip), _lib.ptr(gate), _lib.ptr(dt_bias), state.data_ptr(), _lib.ptr(slots), slots_held, y.data_ptr(),
              batch, channels, states, groups, _strides(x, dt, gate, B, C), int(softplus), _args.DTYPES[x.dtype])
    torch.autograd.graph.increment_version(state)  # (a graph that saved it would be wrong)
    return y


__all__: List[str] = ["MAX_STATES", "SelectiveScanFunction", "selective_scan", "selective_step"]
