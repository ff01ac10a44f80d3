"""Entity rows from features: dropout with a counter-based mask.

The framework's scorers read rows of a table; here rows are computed.  Everything is a kernel of the library on the
current CUDA stream.  Gradients are explicit calls, as in cuke_b200.scoring.  No counterpart in the reference, whose
entities are table rows only (apps/kge/data/data_init.py:6-15).
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _lib
from ._lib import DTYPES, check
from .scoring import _dtype_of, _ptr, _stream


def need_here(*ts) -> None:
    """The tensors are on the current CUDA device (the library launches on its current stream)."""
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("expected CUDA tensors")
        if t.device.index != torch.cuda.current_device():
            raise ValueError(f"a tensor is on {t.device}, the current device is cuda:{torch.cuda.current_device()}; "
                             "use torch.cuda.device(...)")


def pitch(t: torch.Tensor, name: str) -> int:
    """Row pitch in elements of a 2-D tensor whose columns are adjacent."""
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    if t.shape[0] <= 1:
        return max(t.shape[1], 1)
    if t.stride(0) < t.shape[1]:
        raise ValueError(f"{name}: rows overlap (stride {t.stride(0)} for {t.shape[1]} columns)")
    return t.stride(0)


def dropout(x: torch.Tensor, p: float, seed: int, stream_id: int = 0, step: Union[int, torch.Tensor] = 0,
            residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x / (1 - p) where an element is kept, 0 where it is dropped, plus `residual` (kge_dropout in include/kge_b200.h).

    x is (rows, dim) or any contiguous shape, float32 or bfloat16; `residual` has its shape and dtype.  The mask is a
    function of (seed, stream_id, step, element number in row-major order) and is not stored: the gradient of x is
    dropout(d_out, p, seed, stream_id, step), the gradient of `residual` is d_out itself.  step may be a one-element int64
    CUDA tensor: it is read when the kernel runs, so a captured graph draws a new mask whenever that tensor is advanced
    between replays.  out may be x or residual itself."""
    need_here(x, residual, out)
    dt = DTYPES[_dtype_of(x)]
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("residual must have the shape and dtype of x")
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif out.shape != x.shape or out.dtype != x.dtype:
        raise ValueError("out must have the shape and dtype of x")
    step_dev = None
    if isinstance(step, torch.Tensor):
        if step.dtype != torch.int64 or step.numel() != 1 or not step.is_cuda:
            raise ValueError("step must be an int or a one-element int64 CUDA tensor")
        need_here(step)
        step_dev, step = step, 0
    if x.dim() == 2 and x.shape[1] > 0:
        rows, dim = x.shape
        ldx, ldo = pitch(x, "x"), pitch(out, "out")
        ldr = 0 if residual is None else pitch(residual, "residual")
    else:
        if not (x.is_contiguous() and out.is_contiguous() and (residual is None or residual.is_contiguous())):
            raise ValueError("tensors that are not 2-D must be contiguous")
        rows, dim = x.numel(), 1
        ldx = ldo = 1
        ldr = 0 if residual is None else 1
    for other, ld in ((x, ldx), (residual, ldr)):
        if other is not None and other.data_ptr() == out.data_ptr() and rows > 1 and ld != ldo:
            raise ValueError("out may be x or residual only with the same row pitch")
    check(_lib.lib().kge_dropout(_ptr(x), dt, rows, dim, ldx, _ptr(residual), ldr, _ptr(out), ldo, float(p),
                                 int(seed) & 0xFFFFFFFFFFFFFFFF, int(stream_id) & 0xFFFFFFFF, int(step) & 0x7FFFFFFF, _ptr(step_dev), _stream()))
    return out
