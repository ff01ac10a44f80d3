"""Losses over scores, beside scoring.logistic_loss: preferences between triples and policies over candidates.

Every call returns the loss together with the gradients of its score inputs (as scoring.logistic_loss does), computed by
one or two kernels of the library on the current CUDA stream; nothing is kept between calls and no host read happens.
The scores come from scoring.Scorer.forward (fp32) or from any other scorer of the caller's.  No counterpart in the
reference, which stops at scores (apps/kge/kge.py:273-390).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import PREFERENCE_KINDS, check
from .features import dtype_code, need_here, pitch, stream_on
from .scoring import _id_bits, _ptr


def _floats(t: Optional[torch.Tensor], rows: int, name: str) -> Optional[torch.Tensor]:
    if t is not None and (t.dtype != torch.float32 or t.numel() != rows or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous float32 tensor of {rows} elements")
    return t


def _scale(reduction: str, rows: int) -> float:
    if reduction not in ("sum", "mean"):
        raise ValueError("reduction is 'sum' or 'mean'")
    return 1.0 if reduction == "sum" or rows == 0 else 1.0 / rows


def preference_loss(pos: torch.Tensor, neg: torch.Tensor, ref_pos: Optional[torch.Tensor] = None,
                    ref_neg: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                    weight: Optional[torch.Tensor] = None, kind: str = "logistic", beta: float = 1.0, margin: float = 0.0,
                    smoothing: float = 0.0, reduction: str = "sum") -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(loss (1,), dpos, dneg) of every positive against its negatives (kge_preference_loss in include/kge_b200.h).

    pos (B,) and neg (B, n) - or (chunks, chunk, n), the scorers' chunk-shared layout - are fp32 scores; ref_pos / ref_neg
    the same triples scored by a frozen reference (both or none).  With z = beta ((pos - ref_pos) - (neg - ref_neg)) - margin:
    kind "logistic": (1 - smoothing) softplus(-z) + smoothing softplus(z); "square": z^2.  A positive's pairs are averaged
    over its valid negatives (mask True = valid; a row without any adds nothing), positives are weighted by `weight` (B,)
    and summed, or averaged over B with reduction="mean"."""
    here = need_here(pos, neg, ref_pos, ref_neg, mask, weight)
    rows = pos.numel()
    n = neg.shape[-1] if neg.dim() else 0
    if neg.dim() < 2 or neg.numel() != rows * n:
        raise ValueError("neg must be (B, n) or (chunks, chunk, n) for pos of B elements")
    if kind not in PREFERENCE_KINDS:
        raise ValueError(f"kind is one of {sorted(PREFERENCE_KINDS)}")
    if (ref_pos is None) != (ref_neg is None):
        raise ValueError("ref_pos and ref_neg come together")

    def row_pitch(t, name, dtype):
        if t.dtype != dtype or t.shape != neg.shape:
            raise ValueError(f"{name} must be {dtype} of the shape of neg")
        if t.is_contiguous():
            return n
        if t.dim() != 2:
            raise ValueError(f"{name}: tensors that are not 2-D must be contiguous")
        return pitch(t, name)

    ldn, ldr, ldm = row_pitch(neg, "neg", torch.float32), 0, 0
    _floats(pos, rows, "pos")
    if ref_neg is not None:
        ldr = row_pitch(ref_neg, "ref_neg", torch.float32)
        _floats(ref_pos, rows, "ref_pos")
    if mask is not None:
        ldm = row_pitch(mask, "mask", torch.bool)
    if weight is not None:
        _floats(weight, rows, "weight")
    loss = pos.new_empty(1)
    dpos, dneg = torch.empty_like(pos), torch.empty_like(neg, memory_format=torch.contiguous_format)
    L = _lib.lib()
    need = L.kge_preference_workspace_bytes(rows, n)
    ws = pos.new_empty((need + 3) // 4)
    check(L.kge_preference_loss(pos.data_ptr(), _ptr(ref_pos), neg.data_ptr(), ldn, _ptr(ref_neg), ldr, _ptr(mask), ldm, _ptr(weight), rows, n,
                                PREFERENCE_KINDS[kind], beta, margin, smoothing, _scale(reduction, rows),
                                loss.data_ptr(), dpos.data_ptr(), dneg.data_ptr(), n or 1, ws.data_ptr(), need, stream_on(here)))
    return loss, dpos, dneg


def _candidates(scores, action, n_cand):
    """What every call over candidates passes on first; the tensors' device has been checked."""
    if scores.dim() != 2:
        raise ValueError("scores must be (rows, candidates)")
    rows, n = scores.shape
    if action.numel() != rows or not action.is_contiguous():
        raise ValueError("action must hold one id per row of scores")
    if n_cand is not None and (n_cand.dtype != torch.int32 or n_cand.numel() != rows or not n_cand.is_contiguous()):
        raise ValueError("n_cand must be a contiguous int32 tensor with one count per row of scores")
    return scores.data_ptr(), dtype_code(scores), pitch(scores, "scores"), rows, n, _ptr(n_cand), action.data_ptr(), _id_bits(action)


def log_prob(scores: torch.Tensor, action: torch.Tensor, n_cand: Optional[torch.Tensor] = None,
             temperature: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(logp (rows,) fp32, stats): log softmax(scores / temperature) of the chosen candidate of every row (kge_log_prob).

    scores (rows, n) float32 or bfloat16, n_cand (rows,) int32: row r has its first n_cand[r] columns only; action (rows,)
    int32 / int64, -1 where nothing was chosen (logp 0, zero gradient).  stats is what log_prob_backward needs."""
    here = need_here(scores, action, n_cand)
    how = _candidates(scores, action, n_cand)
    rows, n = how[3], how[4]
    logp = scores.new_empty(rows, dtype=torch.float32)
    stats = logp.new_empty(rows, 3)
    L = _lib.lib()
    need = L.kge_candidates_workspace_bytes(rows, n)
    ws = logp.new_empty((need + 3) // 4)
    check(L.kge_log_prob(*how, temperature, logp.data_ptr(), stats.data_ptr(), ws.data_ptr(), need, stream_on(here)))
    return logp, stats


def log_prob_backward(scores: torch.Tensor, action: torch.Tensor, stats: torch.Tensor, dlogp: torch.Tensor,
                      n_cand: Optional[torch.Tensor] = None, temperature: float = 1.0) -> torch.Tensor:
    """d(scores), in the dtype of scores, from d(logp) (rows,) and the stats of log_prob over the same arguments."""
    here = need_here(scores, action, n_cand, stats, dlogp)
    how = _candidates(scores, action, n_cand)
    _floats(stats, 3 * how[3], "stats"), _floats(dlogp, how[3], "dlogp")
    dscores = torch.empty_like(scores, memory_format=torch.contiguous_format)
    check(_lib.lib().kge_log_prob_backward(*how, temperature, stats.data_ptr(), dlogp.data_ptr(), dscores.data_ptr(), how[4] or 1, stream_on(here)))
    return dscores


def policy_loss(scores: torch.Tensor, action: torch.Tensor, old_logp: torch.Tensor, advantage: torch.Tensor,
                ref_logp: Optional[torch.Tensor] = None, n_cand: Optional[torch.Tensor] = None,
                weight: Optional[torch.Tensor] = None, temperature: float = 1.0, clip_low: float = 0.2, clip_high: float = 0.2,
                kl_coef: float = 0.0, reduction: str = "mean") -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(loss (1,), logp (rows,), kl (rows,), dscores) of a clipped policy step with a KL term (kge_policy_loss).

    ratio = exp(logp - old_logp); per row -min(ratio A, clip(ratio, 1 - clip_low, 1 + clip_high) A) + kl_coef * kl with
    kl = exp(ref_logp - logp) - (ref_logp - logp) - 1 (needs ref_logp; with kl_coef = 0 it is only reported); rows are weighted by
    `weight` (0: the row adds nothing)
    and averaged over their number, or summed with reduction="sum".  scores, action, n_cand, temperature as in log_prob;
    dscores has the dtype of scores."""
    here = need_here(scores, action, n_cand, old_logp, advantage, ref_logp, weight)
    how = _candidates(scores, action, n_cand)
    rows, n = how[3], how[4]
    _floats(old_logp, rows, "old_logp"), _floats(advantage, rows, "advantage")
    if ref_logp is not None:
        _floats(ref_logp, rows, "ref_logp")
    elif kl_coef:
        raise ValueError("kl_coef needs ref_logp")
    if weight is not None:
        _floats(weight, rows, "weight")
    loss = old_logp.new_empty(1)
    logp, kl = old_logp.new_empty(rows), old_logp.new_empty(rows)
    dscores = torch.empty_like(scores, memory_format=torch.contiguous_format)
    L = _lib.lib()
    need = L.kge_candidates_workspace_bytes(rows, n)
    ws = old_logp.new_empty((need + 3) // 4)
    check(L.kge_policy_loss(*how, temperature, old_logp.data_ptr(), _ptr(ref_logp), advantage.data_ptr(), _ptr(weight), clip_low, clip_high,
                            kl_coef, _scale(reduction, rows), loss.data_ptr(), logp.data_ptr(), kl.data_ptr(), dscores.data_ptr(), n or 1,
                            ws.data_ptr(), need, stream_on(here)))
    return loss, logp, kl, dscores
