"""Entity rows from features: a matrix product with bias, activation and residual, and dropout with a counter-based mask.

The framework's scorers read rows of a table; here rows are computed.  Everything is a kernel of the library on the
current CUDA stream.  Gradients are explicit calls, as in cuke_b200.scoring.  No counterpart in the reference, whose
entities are table rows only (apps/kge/data/data_init.py:6-15).
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib
from ._lib import ACTIVATIONS, DTYPES, check
from .scoring import _ptr, _raw_stream


_CODES = {torch.float32: DTYPES["f32"], torch.bfloat16: DTYPES["bf16"]}


def need_here(*ts) -> int:
    """The number of the current CUDA device, which all the tensors are on (the library launches on its current stream)."""
    here = None
    for t in ts:
        if t is not None:
            at = t.get_device()
            if at != here:
                if at < 0:
                    raise ValueError("expected CUDA tensors")
                here = torch.cuda.current_device()
                if at != here:
                    raise ValueError(f"a tensor is on {t.device}, the current device is cuda:{here}; use torch.cuda.device(...)")
    return here


def stream_on(here: int) -> int:
    """Handle of the current stream of device `here`, as need_here returned it."""
    return torch.cuda.current_stream(here).cuda_stream if _raw_stream is None else _raw_stream(here)


def dtype_code(t: torch.Tensor) -> int:
    code = _CODES.get(t.dtype)
    if code is None:
        raise TypeError(f"expected float32 or bfloat16, got {t.dtype}")
    return code


def pitch(t: torch.Tensor, name: str) -> int:
    """Row pitch in elements of a 2-D tensor whose columns are adjacent."""
    rows, cols = t.shape
    if t.is_contiguous():
        return cols or 1
    by_row, by_col = t.stride()
    if cols > 1 and by_col != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    if rows <= 1:
        return cols or 1
    if by_row < cols:
        raise ValueError(f"{name}: rows overlap (stride {by_row} for {cols} columns)")
    return by_row


def dropout(x: torch.Tensor, p: float, seed: int, stream_id: int = 0, step: Union[int, torch.Tensor] = 0,
            residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x / (1 - p) where an element is kept, 0 where it is dropped, plus `residual` (kge_dropout in include/kge_b200.h).

    x is (rows, dim) or any contiguous shape, float32 or bfloat16; `residual` has its shape and dtype.  The mask is a
    function of (seed, stream_id, step, element number in row-major order) and is not stored: the gradient of x is
    dropout(d_out, p, seed, stream_id, step), the gradient of `residual` is d_out itself.  step may be a one-element int64
    CUDA tensor: it is read when the kernel runs, so a captured graph draws a new mask whenever that tensor is advanced
    between replays.  out may be x or residual itself."""
    here = need_here(x, residual, out)
    dt = dtype_code(x)
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("residual must have the shape and dtype of x")
    packed = x.is_contiguous() and (residual is None or residual.is_contiguous())
    if out is None:
        out = torch.empty_like(x) if packed else torch.empty_like(x, memory_format=torch.contiguous_format)
    elif out.shape != x.shape or out.dtype != x.dtype:
        raise ValueError("out must have the shape and dtype of x")
    else:
        packed = packed and out.is_contiguous()
    step_dev = None
    if isinstance(step, torch.Tensor):
        if step.dtype != torch.int64 or step.numel() != 1:
            raise ValueError("step must be an int or a one-element int64 CUDA tensor")
        need_here(step)
        step_dev, step = step.data_ptr(), 0
    ldr = 0
    if packed:
        n = x.numel()                                     # one run of elements, whatever the shape
        rows, dim = (1, n) if n < 1 << 31 else (n, 1)
        ldx = ldo = dim
        if residual is not None:
            ldr = dim
    else:
        if x.dim() != 2:
            raise ValueError("tensors that are not 2-D must be contiguous")
        rows, dim = x.shape
        ldx, ldo = pitch(x, "x"), pitch(out, "out")
        if residual is not None:
            ldr = pitch(residual, "residual")
        for other, ld in ((x, ldx), (residual, ldr)):
            if other is not None and other.data_ptr() == out.data_ptr() and rows > 1 and ld != ldo:
                raise ValueError("out may be x or residual only with the same row pitch")
    check(_lib.lib().kge_dropout(x.data_ptr(), dt, rows, dim, ldx, None if residual is None else residual.data_ptr(), ldr, out.data_ptr(), ldo, p,
                                 int(seed) & 0xFFFFFFFFFFFFFFFF, int(stream_id) & 0xFFFFFFFF, int(step) & 0x7FFFFFFF, step_dev, stream_on(here)))
    return out


def _matrix(t: torch.Tensor, name: str, rows: int, cols: int) -> int:
    """Row pitch of a (rows, cols) bfloat16 matrix."""
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    if t.shape != (rows, cols):
        raise ValueError(f"{name} must be ({rows}, {cols}), got {tuple(t.shape)}")
    return pitch(t, name)


def _act(act: str) -> int:
    if act not in ACTIVATIONS:
        raise ValueError(f"act is one of {sorted(ACTIVATIONS)}")
    return ACTIVATIONS[act]


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, act: str = "none",
           residual: Optional[torch.Tensor] = None, save_preact: bool = False, out: Optional[torch.Tensor] = None):
    """act(x w + bias) + residual: entity rows computed from features (kge_linear_forward in include/kge_b200.h).

    x (M, K), w (K, N) - out[j] = sum_i x[i] w[i][j], as for the relation matrices -, bias (N,) and residual (M, N) are
    bfloat16, accumulation is fp32 with one rounding at the end; K and N are multiples of 8, rows start on 16-byte
    boundaries.  act: "none", "relu", "silu" or "gelu" (tanh form).  With save_preact=True returns (out, preact), preact
    being what linear_backward needs of the pre-activation and not the pre-activation itself: its slope act'(x w + bias), rounded
    to float16 (2^-11 relative), or None for act="none"."""
    here = need_here(x, w, bias, residual, out)
    if x.dim() != 2 or w.dim() != 2:
        raise ValueError("x and w must be matrices")
    (m, k), n = x.shape, w.shape[1]
    code = _act(act)
    ldx, ldw = _matrix(x, "x", m, k), _matrix(w, "w", k, n)
    ldr = 0 if residual is None else _matrix(residual, "residual", m, n)
    if bias is not None and (bias.dtype != torch.bfloat16 or bias.shape != (n,) or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous bfloat16 vector of {n}")
    if out is None:
        out, ldo = x.new_empty(m, n), n
    else:
        ldo = _matrix(out, "out", m, n)
    if residual is not None and residual.data_ptr() == out.data_ptr() and ldr != ldo:
        raise ValueError("out may be residual only with the same row pitch")
    preact = x.new_empty(m, n, dtype=torch.float16) if save_preact and code else None
    L = _lib.lib()
    need = L.kge_linear_workspace_bytes(m, k, n, code, 0)
    ws = x.new_empty((need + 1) // 2) if need else None            # (of two-byte elements: the quickest allocation)
    check(L.kge_linear_forward(x.data_ptr(), ldx, w.data_ptr(), ldw, _ptr(bias), _ptr(residual), ldr, m, k, n, code, out.data_ptr(), ldo,
                               _ptr(preact), _ptr(ws), need, stream_on(here)))
    return (out, preact) if save_preact else out


def linear_backward(dout: torch.Tensor, x: torch.Tensor, w: torch.Tensor, preact: Optional[torch.Tensor] = None, act: str = "none",
                    need_dx: bool = True, need_dw: bool = True,
                    need_dbias: bool = True) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(dx, dw, dbias) of linear, bfloat16, from d(out) (M, N) and the preact it saved; None where not needed.  The gradient
    of `residual` is dout itself.

    preact is what linear(..., save_preact=True) returned, the slopes act'(z): any other float16 tensor of that shape, a
    pre-activation z for one, cannot be told from it and gives wrong gradients.  dz = dout * preact is rounded to bfloat16 before
    the two products, whose sums are fp32 with one rounding of the result: dx and dw are off by 0.0024 of their size where the
    result's rounding alone gives 0.0017.  dbias sums the unrounded dz.  With act="none", dz is dout and nothing is rounded twice."""
    here = need_here(dout, x, w, preact)
    if x.dim() != 2 or w.dim() != 2:
        raise ValueError("x and w must be matrices")
    (m, k), n = x.shape, w.shape[1]
    code = _act(act)
    ldd, ldx, ldw = _matrix(dout, "dout", m, n), _matrix(x, "x", m, k), _matrix(w, "w", k, n)
    if code and (preact is None or preact.dtype != torch.float16 or preact.shape != (m, n) or not preact.is_contiguous()):
        raise ValueError("preact must be what linear(..., save_preact=True) returned")
    dx = x.new_empty(m, k) if need_dx else None
    dw = x.new_empty(k, n) if need_dw else None
    db = x.new_empty(n) if need_dbias else None
    L = _lib.lib()
    need = L.kge_linear_workspace_bytes(m, k, n, code, 1)
    ws = x.new_empty((need + 1) // 2) if need else None            # (of two-byte elements: the quickest allocation)
    check(L.kge_linear_backward(dout.data_ptr(), ldd, x.data_ptr(), ldx, w.data_ptr(), ldw, preact.data_ptr() if code else None, m, k, n, code,
                                _ptr(dx), k, _ptr(dw), _ptr(db), _ptr(ws), need, stream_on(here)))
    return dx, dw, db
