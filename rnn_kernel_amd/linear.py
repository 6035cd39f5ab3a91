"""The matrix product of a layer's projections with its epilogue, on the HIP
library:  y = act(x W^T + b) + r.

* ``linear``: the function, with gradients of x, W, b and r;
* ``Linear``: the module, with nn.Linear's parameter names, shapes and
  initialisation.

float32 or bfloat16, sums in float32 and one rounding in the end.  Like the GRU they
raise RuntimeError for tensors of other devices or types, ValueError for shapes,
and have no CPU fallback.
"""
from __future__ import annotations

import math
from typing import List, Optional

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
MAX_SIZE = 2 ** 31 - 1  # of rows, inputs and outputs: the library takes them as 32-bit integers
MAX_ROW_STRIDE = 2 ** 21  # elements: the kernels' offsets within a tile are 32-bit
ACTIVATIONS = ("none", "relu", "gelu", "silu", "sigmoid", "logsigmoid")
_ACTS = {name: i for i, name in enumerate(ACTIVATIONS)}
_ACTS[None] = 0


def _index_of(device) -> int:
    return device.index if device.index is not None else torch.cuda.current_device()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as a matrix whose rows are dense and at most MAX_ROW_STRIDE apart: a copy where
    they are not."""
    if t.dim() == 2 and t.is_contiguous():
        return t
    m = t if t.dim() == 2 else t.reshape(-1, t.size(-1))
    if (m.size(1) == 1 or m.stride(1) == 1) and (m.size(0) <= 1 or m.size(1) <= m.stride(0) <= MAX_ROW_STRIDE):
        return m
    return m.contiguous()


def _ld(m: torch.Tensor) -> int:
    return m.stride(0) if m.size(0) > 1 else m.size(1)


def _check(x, weight, bias, residual, activation) -> None:
    index, dtype = x.get_device(), x.dtype
    for t, name in ((x, "x"), (weight, "weight"), (bias, "bias"), (residual, "residual")):
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"linear: {name} must be a CUDA/HIP tensor")
        if t.get_device() != index:
            raise RuntimeError("linear: all tensors must be on one device")
        if t.dtype != dtype or dtype not in _DTYPES:
            raise RuntimeError("linear: tensors must be all float32 or all bfloat16")
    if activation not in _ACTS:
        raise ValueError(f"linear: activation must be one of {', '.join(ACTIVATIONS)}")
    if weight.dim() != 2 or weight.size(0) < 1 or weight.size(1) < 1:
        raise ValueError("linear: weight must have shape [outputs, inputs]")
    if x.dim() < 1 or x.size(-1) != weight.size(1):
        raise ValueError(f"linear: x must have shape [..., {weight.size(1)}]")
    if (x.numel() > MAX_SIZE or weight.numel() > MAX_SIZE) and max(x.numel() // x.size(-1), *weight.shape) > MAX_SIZE:
        raise ValueError("linear: rows, inputs and outputs must be below 2^31")
    if weight.numel() > MAX_ROW_STRIDE and max(weight.shape) > MAX_ROW_STRIDE:
        raise ValueError("linear: inputs and outputs must be at most 2^21")
    if bias is not None and bias.shape != (weight.size(0),):
        raise ValueError(f"linear: bias must have shape [{weight.size(0)}]")
    if residual is not None and residual.shape != (*x.shape[:-1], weight.size(0)):
        raise ValueError(f"linear: residual must have shape {[*x.shape[:-1], weight.size(0)]}")


def _bytes(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)


def _forward(x, weight, bias, residual, activation, keep_z: bool):
    _check(x, weight, bias, residual, activation)
    act = _ACTS[activation]
    keep_z = keep_z and act != 0
    lib = _lib.load()
    xm, wm = _rows(x), _rows(weight)
    rows, outputs, inputs = xm.size(0), wm.size(0), wm.size(1)
    bm = None if bias is None else bias.contiguous()
    rm = None if residual is None else _rows(residual)
    y = x.new_empty((*x.shape[:-1], outputs))
    z = x.new_empty((rows, outputs)) if keep_z else None
    dtype = _DTYPES[x.dtype]
    nbytes = lib.rka_linear_forward_workspace_bytes(rows, outputs, inputs, dtype)
    ws = _bytes(nbytes, x.device) if nbytes else None
    _lib.call(x.get_device(), "rka_linear_forward", xm.data_ptr(), _ld(xm), wm.data_ptr(), _ld(wm), _lib.ptr(bm),
              _lib.ptr(rm), 0 if rm is None else _ld(rm), y.data_ptr(), _lib.ptr(z), _lib.ptr(ws), nbytes, rows, outputs,
              inputs, act, dtype)
    return y, z, xm, wm


class LinearFunction(torch.autograd.Function):
    """apply(x, weight, bias, residual, activation) -> y, as ``linear``.  Kept for
    the backward: x, weight, and (with an activation) the sums before it, in x's
    type."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        y, z, xm, wm = _forward(x, weight, bias, residual, activation, keep_z=any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(xm, wm, z)
        ctx.act, ctx.shape, ctx.device, ctx.dtype = _ACTS[activation], x.shape, x.device, x.dtype
        ctx.sizes = (xm.size(0), wm.size(0), wm.size(1))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        xm, wm, z = ctx.saved_tensors
        rows, outputs, inputs = ctx.sizes
        _lib.check_saved("linear", ctx.device, (xm, ctx.dtype, (rows, inputs)), (wm, ctx.dtype, (outputs, inputs)),
                         (z, ctx.dtype, (rows, outputs)))
        # (and hooks may have given them back in another layout than they were saved in)
        xm, wm, z = _rows(xm), _rows(wm), None if z is None else z.contiguous()
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = torch.empty(ctx.shape, dtype=xm.dtype, device=xm.device) if need_x else None
        dw = torch.empty(outputs, inputs, dtype=xm.dtype, device=xm.device) if need_w else None
        db = torch.empty(outputs, dtype=xm.dtype, device=xm.device) if need_b else None
        if rows == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
        elif need_x or need_w or need_b:
            lib, dtype, gm = _lib.load(), _DTYPES[xm.dtype], _rows(grad_y)
            nbytes = lib.rka_linear_backward_workspace_bytes(rows, outputs, inputs, dtype)
            ws = _bytes(nbytes, xm.device)
            _lib.call(_index_of(xm.device), "rka_linear_backward", gm.data_ptr(), _ld(gm), xm.data_ptr(), _ld(xm),
                      wm.data_ptr(), _ld(wm), _lib.ptr(z), _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db), ws.data_ptr(), nbytes,
                      rows, outputs, inputs, ctx.act, dtype)
        return dx, dw, db, grad_y if need_r else None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
           activation: Optional[str] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x W^T + b) + r:  x [..., inputs], weight [outputs, inputs], bias [outputs]
    or None, residual [..., outputs] or None, all float32 or all bfloat16; activation
    one of ACTIVATIONS (gelu is the one with the error function) or None.  Inputs
    and outputs are at most 2^21.  Rows may be any distance apart (more than 2^21 elements:
    they are copied).  Sums, bias, activation and residual are in float32; y is rounded
    once."""
    _lib.refuse_tangents("linear", x, weight, bias, residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return LinearFunction.apply(x, weight, bias, residual, activation)
    return _forward(x, weight, bias, residual, activation, keep_z=False)[0]


class Linear(nn.Module):
    """nn.Linear's parameters and initialisation around ``linear``, with an optional
    activation and, in the call, a residual."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: Optional[str] = None,
                 device=None, dtype=None) -> None:
        super().__init__()
        if in_features < 1 or out_features < 1:
            raise ValueError("Linear: in_features and out_features must be >= 1")
        if activation not in _ACTS:
            raise ValueError(f"Linear: activation must be one of {', '.join(ACTIVATIONS)}")
        self.in_features, self.out_features, self.activation = in_features, out_features, activation
        self.weight = nn.Parameter(torch.empty(out_features, in_features, device=device, dtype=dtype))
        if bias:
            self.bias = nn.Parameter(torch.empty(out_features, device=device, dtype=dtype))
        else:
            self.register_parameter("bias", None)
        self.reset_parameters()

    def reset_parameters(self) -> None:
        nn.init.kaiming_uniform_(self.weight, a=math.sqrt(5))
        if self.bias is not None:
            bound = 1.0 / math.sqrt(self.in_features)
            nn.init.uniform_(self.bias, -bound, bound)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return linear(x, self.weight, self.bias, activation=self.activation, residual=residual)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, "
                f"activation={self.activation}")


__all__: List[str] = ["ACTIVATIONS", "Linear", "LinearFunction", "linear"]
