"""The gated delta rule, a recurrent layer whose state is a matrix, on the HIP
library.

Per batch row and value head, with the state S [Dk, Dv] in float32:

    S~ = exp(g_t) S_{t-1};  e_t = v_t - S~^T k_t;  S_t = S~ + k_t (beta_t e_t)^T
    o_t = scale * S_t^T q_t

* ``gated_delta_rule``: whole sequences (training and prompts), with gradients;
* ``gated_delta_step``: one token of each of a batch of requests, the states
  updated in place (answering).

Like the GRU they raise RuntimeError for tensors of other devices or types,
ValueError for shapes, and have no CPU fallback.
"""
from __future__ import annotations

import ctypes
from typing import List, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib

MAX_KEY_DIM = 256
MAX_SIZE = 2 ** 31 - 1  # of a dimension: the library takes them as 32-bit integers

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


def _index_of(device) -> int:
    return device.index if device.index is not None else torch.cuda.current_device()


def _check_inputs(q, k, v, g, beta, tokens: bool) -> None:
    """The checks that both entry points share; ``tokens``: with a token
    dimension."""
    lead = 2 if tokens else 1
    index = q.get_device()  # (a tensor's device as an int: a single step is a few us of the host)
    if not (q.is_cuda and k.get_device() == v.get_device() == g.get_device() == beta.get_device() == index):
        for t, name in ((q, "q"), (k, "k"), (v, "v"), (g, "g"), (beta, "beta")):
            if not t.is_cuda:
                raise RuntimeError(f"gated delta rule: {name} must be a CUDA/HIP tensor")
        raise RuntimeError("gated delta rule: all tensors must be on one device")
    dtype, gate = q.dtype, g.dtype
    if dtype not in _DTYPES or k.dtype != dtype or v.dtype != dtype:
        raise RuntimeError("gated delta rule: q, k and v must be all float32 or all bfloat16")
    if beta.dtype != gate or gate not in (torch.float32, dtype):
        raise RuntimeError("gated delta rule: g and beta must be float32 or of q's dtype")
    qs, vs = q.shape, v.shape
    if len(qs) != lead + 2 or k.dim() != lead + 2 or len(vs) != lead + 2:
        name = "q" if len(qs) != lead + 2 else "k" if k.dim() != lead + 2 else "v"
        shape = "[batch, tokens, heads, dim]" if tokens else "[batch, heads, dim]"
        raise ValueError(f"gated delta rule: {name} must have shape {shape}")
    if k.shape != qs:
        raise ValueError("gated delta rule: q and k must have the same shape")
    if vs[0] != qs[0] or vs[lead - 1] != qs[lead - 1]:
        raise ValueError("gated delta rule: v must have q's batch and token dimensions")
    if qs[lead] < 1 or vs[lead] < 1 or vs[lead] % qs[lead] != 0:
        raise ValueError("gated delta rule: v's heads must be a multiple of q's and k's")
    if not 1 <= qs[-1] <= MAX_KEY_DIM or vs[-1] < 1:
        raise ValueError(f"gated delta rule: key dim must be in [1, {MAX_KEY_DIM}] and value dim at least 1")
    # (a size that large shows in the number of elements, or is hidden by a size of 0)
    if not (0 < q.numel() <= MAX_SIZE and 0 < v.numel() <= MAX_SIZE) and max(*qs, *vs) > MAX_SIZE:
        raise ValueError("gated delta rule: sizes must be below 2^31")
    gates = vs[:-1]
    if g.shape != gates or beta.shape != gates:
        raise ValueError("gated delta rule: g and beta must have v's shape without its last dimension")


def _check_state(state, shape, name: str, device) -> None:
    if not state.is_cuda or state.device != device:
        raise RuntimeError(f"gated delta rule: {name} must be on q's device")
    if state.dtype != torch.float32:
        raise RuntimeError(f"gated delta rule: {name} must be float32")
    if tuple(state.shape) != tuple(shape):
        raise ValueError(f"gated delta rule: {name} must have shape {list(shape)}")


def _check_ints(t, batch: int, name: str, device) -> None:
    if not t.is_cuda or t.device != device or t.dtype != torch.int32:
        raise RuntimeError(f"gated delta rule: {name} must be an int32 tensor on q's device")
    if tuple(t.shape) != (batch,):
        raise ValueError(f"gated delta rule: {name} must have shape [batch]")


def _dense_heads(t: torch.Tensor) -> torch.Tensor:
    """``t`` with a head's elements side by side (the other strides are free)."""
    return t if t.size(-1) == 1 or t.stride(-1) == 1 else t.contiguous()


def _strides(q, k, v, g, beta):
    """What the C entries take; ``v`` None: it is not read (the backward)."""
    if q.dim() == 4:
        of_v = (0, 0, 0) if v is None else v.stride()[:3]
        return (ctypes.c_longlong * 15)(*q.stride()[:3], *k.stride()[:3], *of_v, *g.stride(), *beta.stride())
    (qb, qh, _), (kb, kh, _), (vb, vh, _) = q.stride(), k.stride(), v.stride()
    (gb, gh), (bb, bh) = g.stride(), beta.stride()
    return (ctypes.c_longlong * 15)(qb, 0, qh, kb, 0, kh, vb, 0, vh, gb, 0, gh, bb, 0, bh)


def _bytes(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)


def _forward(q, k, v, g, beta, initial_state, lengths, scale: Optional[float], normalize: bool, training: bool):
    """Checks, and the forward: o, final_state, what is saved if ``training``, and q, k,
    lengths and scale as they were used."""
    _check_inputs(q, k, v, g, beta, tokens=True)
    batch, tokens, key_heads, key_dim = q.shape
    if initial_state is not None:
        _check_state(initial_state, (batch, v.size(2), key_dim, v.size(3)), "initial_state", q.device)
        initial_state = initial_state.contiguous()
    if lengths is not None:
        _check_ints(lengths, batch, "lengths", q.device)
        lengths = lengths.contiguous()
    scale = key_dim ** -0.5 if scale is None else float(scale)
    q, k, v = _dense_heads(q), _dense_heads(k), _dense_heads(v)
    lib = _lib.load()
    sizes = (batch, tokens, key_heads, v.size(2), key_dim, v.size(3))
    o = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    final_state = torch.empty(batch, v.size(2), key_dim, v.size(3), dtype=torch.float32, device=v.device)
    ws_bytes = lib.rka_gated_delta_forward_workspace_bytes(*sizes, _DTYPES[q.dtype])
    ws = _bytes(ws_bytes, v.device)
    reserve = _bytes(lib.rka_gated_delta_reserve_bytes(*sizes), v.device) if training else None
    _lib.call(_index_of(v.device), "rka_gated_delta_forward", q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(),
              beta.data_ptr(), _lib.ptr(initial_state), _lib.ptr(lengths), o.data_ptr(), final_state.data_ptr(),
              _lib.ptr(reserve), ws.data_ptr(), ws_bytes, *sizes, _strides(q, k, v, g, beta), _DTYPES[q.dtype],
              _DTYPES[g.dtype], int(normalize), scale)
    return o, final_state, reserve, (q, k, lengths, scale)


class GatedDeltaFunction(torch.autograd.Function):
    """apply(q, k, v, g, beta, initial_state, lengths, scale, normalize) ->
    (o, final_state), as gated_delta_rule, with gradients of the first six."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, initial_state, lengths, scale, normalize):
        o, final_state, reserve, (q, k, lengths, scale) = _forward(q, k, v, g, beta, initial_state, lengths, scale,
                                                                   normalize, training=True)
        ctx.save_for_backward(q, k, g, beta, lengths, reserve)
        ctx.sizes = (*q.shape[:3], v.size(2), q.size(3), v.size(3))
        ctx.device, ctx.dtype, ctx.gate_dtype = q.device, q.dtype, g.dtype
        ctx.scale, ctx.normalize, ctx.has_state = scale, normalize, initial_state is not None
        ctx.set_materialize_grads(False)
        return o, final_state

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_o, grad_state):
        q, k, g, beta, lengths, reserve = ctx.saved_tensors
        batch, tokens, key_heads, value_heads, key_dim, value_dim = ctx.sizes
        lib, device, dtype, gate_dtype = _lib.load(), ctx.device, ctx.dtype, ctx.gate_dtype
        keys, gates = (batch, tokens, key_heads, key_dim), (batch, tokens, value_heads)
        _lib.check_saved("gated delta rule", device, (q, dtype, keys), (k, dtype, keys), (g, gate_dtype, gates),
                         (beta, gate_dtype, gates), (lengths, torch.int32, (batch,)),
                         (reserve, torch.uint8, (max(lib.rka_gated_delta_reserve_bytes(*ctx.sizes), 1),)))
        # (and hooks may have given them back in another layout than they were saved in)
        q, k, reserve = _dense_heads(q), _dense_heads(k), reserve.contiguous()
        lengths = None if lengths is None else lengths.contiguous()
        grad_o = None if grad_o is None else grad_o.contiguous()
        grad_state = None if grad_state is None else grad_state.contiguous()
        dq, dk = (torch.empty(q.shape, dtype=q.dtype, device=device) for _ in range(2))
        dv = torch.empty(batch, tokens, value_heads, value_dim, dtype=q.dtype, device=device)
        dg, dbeta = (torch.empty(g.shape, dtype=g.dtype, device=device) for _ in range(2))
        ds0 = None
        if ctx.has_state and ctx.needs_input_grad[5]:
            ds0 = torch.empty(batch, value_heads, key_dim, value_dim, dtype=torch.float32, device=device)
        ws_bytes = lib.rka_gated_delta_backward_workspace_bytes(*ctx.sizes, _DTYPES[q.dtype])
        ws = _bytes(ws_bytes, device)
        _lib.call(_index_of(device), "rka_gated_delta_backward", q.data_ptr(), k.data_ptr(), g.data_ptr(),
                  beta.data_ptr(), _lib.ptr(lengths), reserve.data_ptr(), _lib.ptr(grad_o), _lib.ptr(grad_state),
                  dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dg.data_ptr(), dbeta.data_ptr(), _lib.ptr(ds0),
                  ws.data_ptr(), ws_bytes, *ctx.sizes, _strides(q, k, None, g, beta), _DTYPES[q.dtype], _DTYPES[g.dtype],
                  int(ctx.normalize), ctx.scale)
        return dq, dk, dv, dg, dbeta, ds0, None, None, None


def gated_delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     initial_state: Optional[torch.Tensor] = None, *, scale: Optional[float] = None,
                     normalize: bool = False, lengths: Optional[torch.Tensor] = None
                     ) -> Tuple[torch.Tensor, torch.Tensor]:
    """The rule over whole sequences: ``(o, final_state)``.

    q, k [B, T, Hk, Dk] and v [B, T, Hv, Dv], float32 or bfloat16, Hv a multiple
    of Hk (value head h uses key head h // (Hv // Hk)), Dk at most 256, of any
    strides; g (log of the decay) and beta [B, T, Hv], float32 or of q's dtype;
    initial_state [B, Hv, Dk, Dv] float32 or None (zeros).  ``scale``: Dk^-0.5 if
    None.  ``normalize``: q and k are divided by sqrt(|.|^2 + 1e-6) first.
    ``lengths`` [B] int32: row b ends after lengths[b] tokens; what lies behind is
    not read, its outputs and gradients are 0.  o has v's shape and type; the
    final state is float32.  Sums and states are held in float32 throughout.

    Tokens are taken in chunks of 64, so a NaN or an infinity in a token may reach
    the outputs of the earlier tokens of its chunk (as NaN; a float32 above 3.39e38, the
    largest bfloat16, counts as an infinity).  Tensors with forward-mode tangents are
    refused."""
    _lib.refuse_tangents("gated_delta_rule", q, k, v, g, beta, initial_state)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, g, beta, initial_state)):
        return GatedDeltaFunction.apply(q, k, v, g, beta, initial_state, lengths, scale, normalize)
    return _forward(q, k, v, g, beta, initial_state, lengths, scale, normalize, training=False)[:2]


def gated_delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     state: torch.Tensor, *, slots: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                     normalize: bool = False) -> torch.Tensor:
    """One token of each of B requests: o [B, Hv, Dv]; ``state`` is updated in place.

    q, k [B, Hk, Dk], v [B, Hv, Dv], g and beta [B, Hv], as in gated_delta_rule.
    state [N, Hv, Dk, Dv] float32, contiguous: request b has state ``slots[b]``
    (int32 [B], distinct), or b if ``slots`` is None.  A negative slot marks a
    request without a state (padding): its output is 0; a slot from N up gives NaN;
    neither touches a state.  No gradients: with grad mode on, inputs that require
    them are refused, and so are forward-mode tangents.  Autograd counts the call as a
    change of ``state``."""
    _lib.refuse_tangents("gated_delta_step", q, k, v, g, beta, state)
    _check_inputs(q, k, v, g, beta, tokens=False)
    batch, _, key_dim = q.shape
    if state.dim() != 4:
        raise ValueError("gated delta rule: state must have shape [slots, heads, key dim, value dim]")
    _check_state(state, (state.size(0), v.size(1), key_dim, v.size(2)), "state", q.device)
    if state.size(0) > MAX_SIZE:
        raise ValueError("gated delta rule: sizes must be below 2^31")
    if not state.is_contiguous():
        raise ValueError("gated delta rule: state must be contiguous")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, g, beta, state)):
        raise RuntimeError("gated_delta_step has no gradients; use gated_delta_rule or torch.no_grad()")
    if slots is not None:
        _check_ints(slots, batch, "slots", q.device)
        slots = slots.contiguous()
    elif state.size(0) < batch:
        raise ValueError("gated delta rule: fewer states than requests")
    q, k, v = _dense_heads(q), _dense_heads(k), _dense_heads(v)
    o = v.new_empty(v.shape)
    _lib.call(v.get_device(), "rka_gated_delta_step", q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(),
              beta.data_ptr(), state.data_ptr(), _lib.ptr(slots), state.size(0), o.data_ptr(), batch, q.size(1),
              v.size(1), key_dim, v.size(2), _strides(q, k, v, g, beta), _DTYPES[q.dtype], _DTYPES[g.dtype],
              int(normalize), key_dim ** -0.5 if scale is None else float(scale))
    torch.autograd.graph.increment_version(state)  # (a graph that saved it would be wrong)
    return o


__all__: List[str] = ["GatedDeltaFunction", "gated_delta_rule", "gated_delta_step"]
