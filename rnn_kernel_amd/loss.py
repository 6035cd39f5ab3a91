"""The cross entropy of a product with a vocabulary, on the HIP library: the loss of a layer
that answers with one of many tokens, without its logits in memory.

    loss = log sum_v exp(x . weight[v] + bias[v]) - (x . weight[target] + bias[target])

* ``linear_cross_entropy``: of each row, or their sum or mean, with gradients of x, weight
  and bias;
* ``LinearCrossEntropy``: the module, with nn.Linear's parameter names and shapes.

float32 or bfloat16, logits, sums and losses in float32.  Like the GRU they raise RuntimeError
for tensors of other devices or types, ValueError for shapes, and have no CPU fallback.
"""
from __future__ import annotations

import math
from typing import List, Optional

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _args, _lib

REDUCTIONS = ("none", "mean", "sum")
MAX_LOSS_SIZE = 2 ** 21  # of rows, inputs and vocabulary
IGNORE_INDEX = -100
_WHAT = "linear_cross_entropy"


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as a matrix of dense rows: a copy where its layout has none."""
    m = t if t.dim() == 2 else t.reshape(-1, t.size(-1))
    return m if m.size(1) == 1 or m.stride(1) == 1 else m.contiguous()


def _weight_rows(w: torch.Tensor) -> torch.Tensor:
    w = _args.dense_last(w)
    return w if w.stride(0) <= MAX_LOSS_SIZE else w.contiguous()


def _forward(x, weight, target, bias, ignore_index: int, reduction: str):
    """Checks, and the loss, x's rows and weight and bias as they were used, and what the
    forward leaves for the backward."""
    _args.check_dtype(_WHAT, x, "x")
    _args.check_tensors(_WHAT, x, (weight, "weight", x.dtype), (bias, "bias", x.dtype))
    if not target.is_cuda or target.get_device() != x.get_device() or target.dtype not in (torch.int64, torch.int32):
        raise RuntimeError(f"{_WHAT}: target must be an int64 or int32 tensor on x's device")
    if reduction not in REDUCTIONS:
        raise ValueError(f"{_WHAT}: reduction must be one of {', '.join(REDUCTIONS)}")
    if not isinstance(ignore_index, int) or not -2 ** 63 <= ignore_index < 2 ** 63:
        raise ValueError(f"{_WHAT}: ignore_index must be a 64-bit integer")
    if weight.dim() != 2 or weight.size(0) < 1 or weight.size(1) < 1:
        raise ValueError(f"{_WHAT}: weight must have shape [vocabulary, inputs]")
    outputs, inputs = weight.shape
    if x.dim() < 1 or x.size(-1) != inputs:
        raise ValueError(f"{_WHAT}: x must have shape [..., {inputs}]")
    _args.check_shape(_WHAT, target, "target", x.shape[:-1])
    _args.check_shape(_WHAT, bias, "bias", (outputs,))
    rows = target.numel()
    if max(rows, inputs, outputs) > MAX_LOSS_SIZE:
        raise ValueError(f"{_WHAT}: rows, inputs and vocabulary must be at most 2^21")
    lib, dtype, nbytes = _lib.load(), _args.DTYPES[x.dtype], 0
    if rows:
        nbytes = lib.rka_cross_entropy_forward_workspace_bytes(rows, inputs, outputs, dtype)
        if nbytes == 0:
            raise ValueError(f"{_WHAT}: {rows} rows of {outputs} logits are more than a launch may have")
    xm, wm, bm, tm = _rows(x), _weight_rows(weight), _args.dense(bias), _args.dense(target)
    loss = torch.empty(target.shape if reduction == "none" else (), dtype=torch.float32, device=x.device)
    if rows == 0:
        return loss.zero_(), xm, wm, bm, None
    reserve = _args.workspace(lib.rka_cross_entropy_reserve_bytes(rows), x.device)
    ws = _args.workspace(nbytes, x.device)
    _lib.call(x.get_device(), "rka_cross_entropy_forward", xm.data_ptr(), xm.stride(0), wm.data_ptr(), wm.stride(0), _lib.ptr(bm),
              tm.data_ptr(), int(tm.dtype == torch.int64), ignore_index, loss.data_ptr(), reserve.data_ptr(), ws.data_ptr(), nbytes,
              rows, inputs, outputs, REDUCTIONS.index(reduction), dtype)
    return loss, xm, wm, bm, reserve


class LinearCrossEntropyFunction(torch.autograd.Function):
    """apply(x, weight, target, bias, ignore_index, reduction) -> loss, as
    linear_cross_entropy.  Kept for the backward: x, weight, bias, and of each row its
    log-sum-exp and three integers."""

    @staticmethod
    def forward(ctx, x, weight, target, bias, ignore_index, reduction):
        loss, xm, wm, bm, reserve = _forward(x, weight, target, bias, ignore_index, reduction)
        ctx.save_for_backward(xm, wm, bm, reserve)
        ctx.shape, ctx.device, ctx.dtype, ctx.reduction = x.shape, x.device, x.dtype, REDUCTIONS.index(reduction)
        ctx.sizes = (xm.size(0), wm.size(1), wm.size(0))
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        xm, wm, bm, reserve = ctx.saved_tensors
        rows, inputs, outputs = ctx.sizes
        device, dtype, lib = ctx.device, ctx.dtype, _lib.load()
        _lib.check_saved(_WHAT, device, (xm, dtype, (rows, inputs)), (wm, dtype, (outputs, inputs)), (bm, dtype, (outputs,)),
                         (reserve, torch.uint8, (lib.rka_cross_entropy_reserve_bytes(rows),)))
        need_x, need_w, _, need_b = ctx.needs_input_grad[:4]
        dx = torch.empty(ctx.shape, dtype=dtype, device=device) if need_x else None
        dw = torch.empty(outputs, inputs, dtype=dtype, device=device) if need_w else None
        db = torch.empty(outputs, dtype=dtype, device=device) if need_b else None
        if rows == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
            return dx, dw, None, db, None, None
        # (hooks may have given them back in another layout than they were saved in)
        xm, wm, bm, reserve, grad_loss = _rows(xm), _weight_rows(wm), _args.dense(bm), reserve.contiguous(), grad_loss.contiguous()
        nbytes = lib.rka_cross_entropy_backward_workspace_bytes(rows, inputs, outputs, _args.DTYPES[dtype])
        ws = _args.workspace(nbytes, device)
        _lib.call(_args.index_of(device), "rka_cross_entropy_backward", grad_loss.data_ptr(), xm.data_ptr(), xm.stride(0),
                  wm.data_ptr(), wm.stride(0), _lib.ptr(bm), reserve.data_ptr(), _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db),
                  ws.data_ptr(), nbytes, rows, inputs, outputs, ctx.reduction, _args.DTYPES[dtype])
        return dx, dw, None, db, None, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                         ignore_index: int = IGNORE_INDEX, reduction: str = "mean") -> torch.Tensor:
    """F.cross_entropy(F.linear(x, weight, bias), target) without the logits in memory: x [...,
    inputs], weight [vocabulary, inputs] and bias [vocabulary] or None, all float32 or all
    bfloat16, target [...] int64 or int32; the loss is float32.

    ``reduction``: "mean" over the rows with a target, "sum" or "none" (a loss for each row). A
    row whose target is ``ignore_index`` has no part in anything: its loss and gradient are 0
    and its x is not read; the mean of no rows is 0.  A row whose target lies outside the
    vocabulary gives NaN.  Rows, inputs and vocabulary are at most 2^21, and the logits 2^38 or so
    in float32, 2^39 in bfloat16 (what a launch may have).  The backward makes the logits again, for a
    piece of the vocabulary at a time, and rounds their gradients to x's type before the products.
    Tensors with forward-mode tangents are refused."""
    _lib.refuse_tangents(_WHAT, x, weight, bias)
    if _args.wants_grad(x, weight, bias):
        return LinearCrossEntropyFunction.apply(x, weight, target, bias, ignore_index, reduction)
    return _forward(x, weight, target, bias, ignore_index, reduction)[0]


class LinearCrossEntropy(nn.Module):
    """nn.Linear's parameters and initialisation around ``linear_cross_entropy``."""

    def __init__(self, in_features: int, vocabulary: int, bias: bool = False, ignore_index: int = IGNORE_INDEX,
                 reduction: str = "mean", device=None, dtype=None) -> None:
        super().__init__()
        if not (1 <= in_features <= MAX_LOSS_SIZE and 1 <= vocabulary <= MAX_LOSS_SIZE):
            raise ValueError("LinearCrossEntropy: in_features and vocabulary must be in [1, 2^21]")
        if reduction not in REDUCTIONS:
            raise ValueError(f"LinearCrossEntropy: reduction must be one of {', '.join(REDUCTIONS)}")
        self.in_features, self.vocabulary, self.ignore_index, self.reduction = in_features, vocabulary, ignore_index, reduction
        bound = 1.0 / math.sqrt(in_features)
        self.weight = nn.Parameter(torch.empty(vocabulary, in_features, device=device, dtype=dtype).uniform_(-bound, bound))
        if bias:
            self.bias = nn.Parameter(torch.empty(vocabulary, device=device, dtype=dtype).uniform_(-bound, bound))
        else:
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
        return linear_cross_entropy(x, self.weight, target, self.bias, ignore_index=self.ignore_index, reduction=self.reduction)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, vocabulary={self.vocabulary}, bias={self.bias is not None}, "
                f"reduction={self.reduction}")


__all__: List[str] = ["LinearCrossEntropy", "LinearCrossEntropyFunction", "linear_cross_entropy"]
