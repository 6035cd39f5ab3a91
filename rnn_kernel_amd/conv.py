"""The short causal convolution in front of a selective scan, on the HIP library.

Per channel, with the W - 1 inputs before the first token as its state:

    y_t = act(bias + sum_j weight[j] x_{t-W+1+j})

* ``causal_conv``: whole sequences (training and prompts), with gradients;
* ``causal_conv_step``: one token of each of a batch of requests, the states updated in
  place (answering).

float32 or bfloat16, sums in float32 and one rounding in the end.  Like the GRU they raise
RuntimeError for tensors of other devices or types, ValueError for shapes, and have no CPU
fallback.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _args, _lib

MIN_CONV_WIDTH, MAX_CONV_WIDTH = 2, 8
MAX_CONV_BATCH, MAX_CONV_TOKENS = 65535, 2 ** 20  # of whole sequences
_ACTS = {None: 0, "none": 0, "silu": 3}


def _check(what: str, x, weight, bias, activation, lead: int) -> None:
    # (a call is a few us of the host: one expression for all that is right)
    dtype, index, shape, of = x.dtype, x.get_device(), x.shape, weight.shape
    if (x.is_cuda and dtype in _args.DTYPES and weight.dtype is dtype and weight.get_device() == index and activation in _ACTS
            and len(shape) == lead + 1 and len(of) == 2 and of[0] == shape[-1] >= 1 and MIN_CONV_WIDTH <= of[1] <= MAX_CONV_WIDTH
            and (bias is None or (bias.dtype is dtype and bias.get_device() == index and bias.shape == of[:1]))
            and max(shape) <= _args.MAX_SIZE and (lead == 1 or (shape[0] <= MAX_CONV_BATCH and shape[1] <= MAX_CONV_TOKENS))):
        return
    _args.check_dtype(what, x, "x")
    _args.check_tensors(what, x, (weight, "weight", x.dtype), (bias, "bias", x.dtype))
    if x.dim() != lead + 1 or x.size(-1) < 1:
        raise ValueError(f"{what}: x must have shape {'[batch, tokens, channels]' if lead == 2 else '[batch, channels]'}")
    if weight.dim() != 2 or weight.size(0) != x.size(-1) or not MIN_CONV_WIDTH <= weight.size(1) <= MAX_CONV_WIDTH:
        raise ValueError(f"{what}: weight must have shape [{x.size(-1)}, width], width in [{MIN_CONV_WIDTH}, {MAX_CONV_WIDTH}]")
    _args.check_shape(what, bias, "bias", (x.size(-1),))
    if activation not in _ACTS:
        raise ValueError(f"{what}: activation must be none or silu")
    if lead == 2 and (x.size(0) > MAX_CONV_BATCH or x.size(1) > MAX_CONV_TOKENS):
        raise ValueError(f"{what}: at most {MAX_CONV_BATCH} rows and 2^20 tokens")
    raise ValueError(f"{what}: sizes must be below 2^31")


def _forward(x, weight, bias, initial_state, activation, lengths):
    what = "causal_conv"
    _check(what, x, weight, bias, activation, 2)
    batch, tokens, channels = x.shape
    width = weight.size(1)
    _args.check_tensors(what, x, (initial_state, "initial_state", x.dtype))
    _args.check_shape(what, initial_state, "initial_state", (batch, width - 1, channels))
    _args.check_row_ints(what, lengths, "lengths", batch, x.device)
    x = _args.dense_last(x)
    weight, bias, initial_state, lengths = (_args.dense(t) for t in (weight, bias, initial_state, lengths))
    y = torch.empty(batch, tokens, channels, dtype=x.dtype, device=x.device)
    final_state = torch.empty(batch, width - 1, channels, dtype=x.dtype, device=x.device)
    _lib.call(x.get_device(), "rka_causal_conv_forward", x.data_ptr(), x.stride(0), x.stride(1), weight.data_ptr(),
              _lib.ptr(bias), _lib.ptr(initial_state), _lib.ptr(lengths), y.data_ptr(), final_state.data_ptr(), batch, tokens,
              channels, width, _ACTS[activation], _args.DTYPES[x.dtype])
    return y, final_state, (x, weight, bias, initial_state, lengths)


class CausalConvFunction(torch.autograd.Function):
    """apply(x, weight, bias, initial_state, activation, lengths) -> (y, final_state), as
    causal_conv, with gradients of the first four."""

    @staticmethod
    def forward(ctx, x, weight, bias, initial_state, activation, lengths):
        y, final_state, saved = _forward(x, weight, bias, initial_state, activation, lengths)
        ctx.save_for_backward(*saved)
        ctx.sizes, ctx.act, ctx.device, ctx.dtype = (*x.shape, weight.size(1)), _ACTS[activation], x.device, x.dtype
        ctx.set_materialize_grads(False)
        return y, final_state

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y, grad_state):
        x, weight, bias, initial_state, lengths = ctx.saved_tensors
        batch, tokens, channels, width = ctx.sizes
        device, dtype = ctx.device, ctx.dtype
        _lib.check_saved("causal_conv", device, (x, dtype, (batch, tokens, channels)), (weight, dtype, (channels, width)),
                         (bias, dtype, (channels,)), (initial_state, dtype, (batch, width - 1, channels)),
                         (lengths, torch.int32, (batch,)))
        # (hooks may have given them back in another layout than they were saved in)
        x = _args.dense_last(x)
        weight, bias, initial_state, lengths, grad_y, grad_state = (
            _args.dense(t) for t in (weight, bias, initial_state, lengths, grad_y, grad_state))
        needs = ctx.needs_input_grad

        def like(need, *shape):
            return torch.empty(shape, dtype=dtype, device=device) if need else None

        dx, dw, db = like(needs[0], batch, tokens, channels), like(needs[1], channels, width), like(needs[2], channels)
        ds0 = like(needs[3], batch, width - 1, channels)
        if batch == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
            return dx, dw, db, ds0, None, None
        nbytes = _lib.load().rka_causal_conv_backward_workspace_bytes(*ctx.sizes)
        ws = _args.workspace(nbytes, device)
        _lib.call(_args.index_of(device), "rka_causal_conv_backward", _lib.ptr(grad_y), _lib.ptr(grad_state), x.data_ptr(),
                  x.stride(0), x.stride(1), weight.data_ptr(), _lib.ptr(bias), _lib.ptr(initial_state), _lib.ptr(lengths),
                  _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db), _lib.ptr(ds0), ws.data_ptr(), nbytes, *ctx.sizes, ctx.act,
                  _args.DTYPES[dtype])
        return dx, dw, db, ds0, None, None


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                initial_state: Optional[torch.Tensor] = None, *, activation: Optional[str] = None,
                lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The convolution over whole sequences: ``(y, final_state)``.

    x [B, T, D] of any strides, B at most 65535 and T at most 2^20, weight [D, W] with W in
    [2, 8], bias [D] or None, initial_state [B, W - 1, D] (the inputs before the first token)
    or None (zeros), all float32 or all bfloat16; activation "silu" or None.  ``lengths`` [B]
    int32: row b ends after lengths[b] tokens; what lies behind is not read, its outputs and
    gradients are 0.  final_state [B, W - 1, D] holds each row's last W - 1 inputs, those of
    the initial state among them where the row is shorter.  Tensors with forward-mode
    tangents are refused."""
    _lib.refuse_tangents("causal_conv", x, weight, bias, initial_state)
    if _args.wants_grad(x, weight, bias, initial_state):
        return CausalConvFunction.apply(x, weight, bias, initial_state, activation, lengths)
    return _forward(x, weight, bias, initial_state, activation, lengths)[:2]


def causal_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                     activation: Optional[str] = None, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of each of B requests: y [B, D]; ``state`` is updated in place.

    x [B, D]; state [N, W - 1, D] of x's type, contiguous: request b has state ``slots[b]``
    (int32 [B], distinct), or b if ``slots`` is None.  A negative slot marks a request without
    a state (padding): its output is 0; a slot from N up gives NaN; neither touches a state.
    No gradients: with grad mode on, inputs that require them are refused, and so are
    forward-mode tangents.  Autograd counts the call as a change of ``state``."""
    what = "causal_conv_step"
    _lib.refuse_tangents(what, x, state, weight, bias)
    _check(what, x, weight, bias, activation, 1)
    batch, channels = x.shape
    width, of = weight.size(1), state.shape
    if len(of) != 3 or of[1] != width - 1 or of[2] != channels or state.dtype is not x.dtype or state.get_device() != x.get_device():
        _args.check_tensors(what, x, (state, "state", x.dtype))
        raise ValueError(f"{what}: state must have shape [slots, {width - 1}, {channels}]")
    slots_held = of[0]
    if slots_held > _args.MAX_SIZE:
        raise ValueError(f"{what}: sizes must be below 2^31")
    if not state.is_contiguous():
        raise ValueError(f"{what}: state must be contiguous")
    if torch.is_grad_enabled() and _args.wants_grad(x, state, weight, bias):
        raise RuntimeError(f"{what} has no gradients; use causal_conv or torch.no_grad()")
    if slots is not None:
        _args.check_row_ints(what, slots, "slots", batch, x.device)
        slots = slots.contiguous()
    elif slots_held < batch:
        raise ValueError(f"{what}: fewer states than requests")
    x, weight = _args.dense_last(x), weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    y = x.new_empty((batch, channels))
    _lib.call(x.get_device(), "rka_causal_conv_step", x.data_ptr(), x.stride(0), weight.data_ptr(), _lib.ptr(bias),
              state.data_ptr(), _lib.ptr(slots), slots_held, y.data_ptr(), batch, channels, width, _ACTS[activation],
              _args.DTYPES[x.dtype])
    torch.autograd.graph.increment_version(state)  # (a graph that saved it would be wrong)
    return y


__all__: List[str] = ["CausalConvFunction", "MAX_CONV_WIDTH", "MIN_CONV_WIDTH", "causal_conv", "causal_conv_step"]
