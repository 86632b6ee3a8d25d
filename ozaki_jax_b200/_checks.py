"""Argument checks shared by the 16-bit entry points."""

import torch

from . import _lib as L

DTYPES = {torch.bfloat16: L.OZK_DT_BF16, torch.float16: L.OZK_DT_F16,
          torch.float32: L.OZK_DT_F32}

# The smallest calls take a few microseconds on the device, so the checks look
# each attribute up once and raise from helpers that only a refusal reaches.

def check_matrix(name, x, dtype=None, rows=None, cols=None):
    """x is a 2D tensor [of that type and shape]; returns its shape."""
    if not isinstance(x, torch.Tensor):
        raise ValueError(f"{name} must be a torch tensor, got {type(x).__name__}.")
    shape = x.shape
    if len(shape) != 2:
        raise ValueError(f"{name} must be 2D, got ndim={len(shape)}.")
    if dtype is not None and x.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {x.dtype}.")
    if rows is not None and shape[0] != rows:
        raise ValueError(f"{name} has {shape[0]} rows, expected {rows}.")
    if cols is not None and shape[1] != cols:
        raise ValueError(f"{name} has {shape[1]} columns, expected {cols}.")
    return shape


def check_16bit(name, x):
    """x is a 2D bfloat16 or float16 tensor; returns its shape and type."""
    shape = check_matrix(name, x)
    dtype = x.dtype
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError(f"{name} must be bfloat16 or float16, got {dtype}.")
    return shape, dtype


def check_device(x, *others):
    """All tensors (None skipped) on the CUDA device of x; returns that device."""
    device = x.device
    if not x.is_cuda:
        raise ValueError(f"tensors must be on a CUDA device, got {device}.")
    index = x.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError(f"a tensor is on {t.device}, expected {device}.")
    return device


def row_major(x):
    """(x, its row stride) with adjacent columns and rows that do not overlap
    (copied only when needed; a stride along one element counts for nothing)."""
    rows, cols = x.shape
    step, inner = x.stride()
    if (inner == 1 or cols <= 1) and (step >= cols or rows <= 1):
        return x, step if rows > 1 else max(cols, 1)
    return x.contiguous(), max(cols, 1)
