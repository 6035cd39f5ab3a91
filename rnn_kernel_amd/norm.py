"""Layer norm over the last dimension, on the HIP library.

* ``layer_norm``: the function, with gradients of x, weight and bias;
* ``LayerNorm``: the module, with nn.LayerNorm's parameter names and initialisation.

float32 or bfloat16, sums and statistics in float32 and one rounding in the end.  Like the
GRU they raise RuntimeError for tensors of other devices or types, ValueError for shapes,
and have no CPU fallback.
"""
from __future__ import annotations

from typing import List, Optional

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _args, _lib

MAX_NORM_SIZE = 16384


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as a matrix of dense rows: a copy where its layout has none."""
    if t.dim() == 2 and (t.size(1) == 1 or t.stride(1) == 1) and t.stride(0) >= 0:
        return t
    m = t.reshape(-1, t.size(-1))
    return m if m.size(1) == 1 or m.stride(1) == 1 else m.contiguous()


def _forward(x, weight, bias, eps: float, keep: bool):
    """Checks, and y, the matrix of x's rows, weight as it was used and, with ``keep``, each
    row's mean and 1 / deviation."""
    dtype, index, shape = x.dtype, x.get_device(), x.shape
    # (a call is a few us of the host: one expression for all that is right)
    if not (x.is_cuda and dtype in _args.DTYPES and len(shape) >= 1 and 1 <= shape[-1] <= MAX_NORM_SIZE
            and (weight is None or (weight.dtype is dtype and weight.get_device() == index and weight.shape == shape[-1:]))
            and (bias is None or (bias.dtype is dtype and bias.get_device() == index and bias.shape == shape[-1:]))):
        _args.check_dtype("layer_norm", x, "x")
        _args.check_tensors("layer_norm", x, (weight, "weight", dtype), (bias, "bias", dtype))
        if len(shape) < 1 or not 1 <= shape[-1] <= MAX_NORM_SIZE:
            raise ValueError(f"layer_norm: x's last dimension must be in [1, {MAX_NORM_SIZE}]")
        _args.check_shape("layer_norm", weight, "weight", shape[-1:])
        _args.check_shape("layer_norm", bias, "bias", shape[-1:])
    size = shape[-1]
    if x.numel() // size > _args.MAX_SIZE:
        raise ValueError("layer_norm: rows must be below 2^31")
    xm, weight, bias = _rows(x), _args.dense(weight), _args.dense(bias)
    rows = xm.size(0)
    y = x.new_empty(shape)
    stats = x.new_empty((2, rows), dtype=torch.float32) if keep else None
    if rows:
        mean = stats.data_ptr() if keep else None
        _lib.call(index, "rka_layer_norm_forward", xm.data_ptr(), xm.stride(0), _lib.ptr(weight), _lib.ptr(bias), y.data_ptr(),
                  mean, mean + 4 * rows if keep else None, rows, size, float(eps), _args.DTYPES[dtype])
    return y, xm, weight, stats


class LayerNormFunction(torch.autograd.Function):
    """apply(x, weight, bias, eps) -> y, as ``layer_norm``.  Kept for the backward: x,
    weight, and each row's mean and 1 / deviation in float32."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, xm, wm, stats = _forward(x, weight, bias, eps, keep=True)
        ctx.save_for_backward(xm, wm, stats)
        ctx.shape, ctx.device, ctx.dtype, ctx.matrix = x.shape, x.device, x.dtype, xm.shape
        ctx.has_weight = weight is not None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        xm, weight, stats = ctx.saved_tensors
        (rows, size), device, dtype = ctx.matrix, ctx.device, ctx.dtype
        _lib.check_saved("layer_norm", device, (xm, dtype, ctx.matrix), (weight, dtype, (size,)),
                         (stats, torch.float32, (2, rows)))
        # (hooks may have given them back in another layout than they were saved in)
        xm, weight, stats = _rows(xm), _args.dense(weight), stats.contiguous()
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx = torch.empty(ctx.shape, dtype=dtype, device=device) if need_x else None
        dw = torch.empty(size, dtype=dtype, device=device) if need_w else None
        db = torch.empty(size, dtype=dtype, device=device) if need_b else None
        if rows == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
            return dx, dw, db, None
        gm = _rows(grad_y)
        nbytes = _lib.load().rka_layer_norm_backward_workspace_bytes(rows, size, _args.DTYPES[dtype])
        ws = _args.workspace(nbytes, device)
        _lib.call(_args.index_of(device), "rka_layer_norm_backward", gm.data_ptr(), gm.stride(0), xm.data_ptr(), xm.stride(0),
                  _lib.ptr(weight), stats.data_ptr(), stats.data_ptr() + 4 * rows, _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db),
                  ws.data_ptr(), nbytes, rows, size, _args.DTYPES[dtype])
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over x's last dimension, of at most
    MAX_NORM_SIZE elements; weight and bias of that shape and of x's type, or None.  x may have
    any strides (a copy is made where its rows are not dense); y is dense."""
    _lib.refuse_tangents("layer_norm", x, weight, bias)
    if _args.wants_grad(x, weight, bias):
        return LayerNormFunction.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, keep=False)[0]


class LayerNorm(nn.Module):
    """nn.LayerNorm's parameters and initialisation around ``layer_norm``, for one
    dimension."""

    def __init__(self, size: int, eps: float = 1e-5, bias: bool = True, device=None, dtype=None) -> None:
        super().__init__()
        if not 1 <= size <= MAX_NORM_SIZE:
            raise ValueError(f"LayerNorm: size must be in [1, {MAX_NORM_SIZE}]")
        self.size, self.eps = size, eps
        self.weight = nn.Parameter(torch.ones(size, device=device, dtype=dtype))
        if bias:
            self.bias = nn.Parameter(torch.zeros(size, device=device, dtype=dtype))
        else:
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self) -> str:
        return f"size={self.size}, eps={self.eps}, bias={self.bias is not None}"


__all__: List[str] = ["LayerNorm", "LayerNormFunction", "MAX_NORM_SIZE", "layer_norm"]
