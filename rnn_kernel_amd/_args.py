"""Checks and layouts of arguments that the operators share."""
from __future__ import annotations

import torch

DTYPES = {torch.float32: 0, torch.bfloat16: 1}
MAX_SIZE = 2 ** 31 - 1  # of a dimension: the library takes them as 32-bit integers


def index_of(device) -> int:
    return device.index if device.index is not None else torch.cuda.current_device()


def check_tensors(what: str, device_of: torch.Tensor, *named) -> None:
    """RuntimeError unless every (tensor or None, name, type) is on ``device_of``'s GPU and
    of its type."""
    index = device_of.get_device()
    for t, name, dtype in named:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{what}: {name} must be a CUDA/HIP tensor")
        if t.get_device() != index:
            raise RuntimeError(f"{what}: all tensors must be on one device")
        if t.dtype != dtype:
            raise RuntimeError(f"{what}: {name} must be {str(dtype).split('.')[-1]}, as the call's other tensors ask, "
                               f"not {str(t.dtype).split('.')[-1]}")


def check_dtype(what: str, t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{what}: {name} must be a CUDA/HIP tensor")
    if t.dtype not in DTYPES:
        raise RuntimeError(f"{what}: {name} must be float32 or bfloat16")


def check_shape(what: str, t, name: str, shape) -> None:
    if t is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: {name} must have shape {list(shape)}, not {list(t.shape)}")


def check_row_ints(what: str, t, name: str, batch: int, device) -> None:
    if t is None:
        return
    if not t.is_cuda or t.device != device or t.dtype != torch.int32:
        raise RuntimeError(f"{what}: {name} must be an int32 tensor on x's device")
    if tuple(t.shape) != (batch,):
        raise ValueError(f"{what}: {name} must have shape [batch]")


def wants_grad(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def dense_last(t):
    """``t`` with its last dimension's elements side by side (the other strides are free)."""
    return t if t is None or t.size(-1) == 1 or t.stride(-1) == 1 else t.contiguous()


def dense(t):
    return None if t is None else t.contiguous()


def workspace(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)
