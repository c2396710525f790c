"""Distillation from a teacher's top logits, forward and backward.

Row ``n`` of the student has ``V`` logits ``x`` and ``K`` stored teacher entries
(logit ``t_k``, token ``id_k``).  With temperature ``T``::

    p = softmax(t / T) over the entries that count
    loss_n = T^2 * sum_k p_k (log p_k - log_softmax(x / T)[id_k])

An entry counts when ``0 <= id_k < V`` and ``t_k`` is not ``-inf``: shorter lists
are padded with the id -1 (what stands in a padded place is not looked at).  A
row without entries has loss 0, gradient 0 and is left out of the mean.  A token
listed twice has the sum of its probabilities.  The teacher gets no gradient.
On CUDA the loss can be differentiated once, in reverse mode (anything else raises).

CUDA (``csrc/kernels/distill.cu``): the forward reads the logits once (twice where a
row's largest value is beyond some 2.9e6 ``T`` either way) and keeps
four numbers a row and the teacher's probabilities; the backward reads them once and writes the gradient; fp32
arithmetic for bf16, fp16 and fp32 logits: a row's loss is off by some ``T^2 2^-20``
times the sizes of its logarithms, which is much beside the loss itself once ``T``
flattens both distributions (hundreds).  The full-vocabulary form is
``VerificationDistillation.temperature_scaled_loss``, which divides by the first
dimension: on ``(N, V)`` logits it is the mean of all tokens listed, on ``(B, S, V)``
it is ``S`` times that.
"""

from __future__ import annotations

import math

import torch

from llm_research_b200._ext import native

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
MAX_TEACHER_ENTRIES = 1024
MIN_TEMPERATURE, MAX_TEMPERATURE = 1e-18, 1e18


def _plain(x, teacher, ids, T, reduction):
    V = x.shape[-1]
    f = torch.float64 if x.dtype == torch.float64 else torch.float32
    x, teacher = x.to(f), teacher.detach().to(f)
    kept = (ids >= 0) & (ids < V) & (teacher != -math.inf)  # what stands in padding is not looked at,
    some = kept.any(dim=-1)
    x = torch.where(some[:, None], x, torch.zeros_like(x))  # nor what a row without entries holds
    x = (x - x.amax(dim=-1, keepdim=True).detach()) / T
    y = torch.where(kept, teacher / T, torch.full_like(teacher, -math.inf))
    y = torch.where(some[:, None], y, torch.zeros_like(y))
    p = torch.where(kept, torch.softmax(y, dim=-1), torch.zeros_like(y))
    log_p = torch.log_softmax(y, dim=-1)
    q = torch.log_softmax(x, dim=-1).gather(1, ids.long().clamp(0, V - 1))
    live = kept & (p != 0)
    zero = torch.zeros_like(p)
    rows = T * T * torch.where(live, torch.where(live, p, zero) * (torch.where(live, log_p, zero) -
                                                                  torch.where(live, q, zero)), zero).sum(-1)
    rows = torch.where(some, rows, torch.zeros_like(rows))
    if reduction == "none":
        return rows
    return rows.sum() if reduction == "sum" else rows.sum() / some.sum().clamp(min=1)


def check_cuda_temperature(T: float) -> None:
    """The kernels hold ``T``, ``T^2`` and ``log2(e) / T`` in fp32: each has to be a normal number."""
    if not MIN_TEMPERATURE <= T <= MAX_TEMPERATURE:
        raise ValueError(f"topk_distillation: temperature must be between {MIN_TEMPERATURE:g} and "
                         f"{MAX_TEMPERATURE:g} on CUDA, got {T:g}")


def topk_distillation(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor,
                      temperature: float = 1.0, reduction: str = "mean") -> torch.Tensor:
    """``logits`` ``(..., V)``; ``teacher_logits``, ``teacher_ids`` ``(..., K)`` with
    the same leading shape (ids int64 or int32).  ``reduction``: ``"mean"`` over the
    rows that have entries (0 without any), ``"sum"``, or ``"none"`` (the leading
    shape), fp32.  ``temperature`` from 1e-18 to 1e18 and at most 1024 entries a row on
    CUDA.  See the module docstring."""
    T = float(temperature)
    if not (T > 0.0 and math.isfinite(T)):
        raise ValueError(f"topk_distillation: temperature must be positive and finite, got {temperature}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"topk_distillation: reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if teacher_ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"topk_distillation: teacher_ids must be int64 or int32, got {teacher_ids.dtype}")
    lead, V = logits.shape[:-1], logits.shape[-1] if logits.dim() else 0
    K = teacher_ids.shape[-1] if teacher_ids.dim() else 0
    if V < 1 or K < 1 or teacher_logits.shape != teacher_ids.shape or teacher_ids.shape[:-1] != lead:
        raise ValueError(f"topk_distillation: logits (..., V) and teacher (..., K) with one leading shape, got "
                         f"{tuple(logits.shape)}, {tuple(teacher_logits.shape)}, {tuple(teacher_ids.shape)}")
    if not logits.is_cuda:
        rows = _plain(logits.reshape(-1, V), teacher_logits.reshape(-1, K), teacher_ids.reshape(-1, K), T, reduction)
        return rows.reshape(lead) if reduction == "none" else rows
    check_cuda_temperature(T)
    if K > MAX_TEACHER_ENTRIES:
        raise ValueError(f"topk_distillation: at most {MAX_TEACHER_ENTRIES} teacher entries on CUDA, got {K}")
    for name, t in (("logits", logits), ("teacher_logits", teacher_logits)):
        if t.dtype not in _DTYPES:
            raise TypeError(f"topk_distillation: {name} must be bf16, fp16 or fp32 on CUDA, got {t.dtype}")
    return native().topk_distillation(logits, teacher_logits, teacher_ids, T, _REDUCTIONS[reduction])
