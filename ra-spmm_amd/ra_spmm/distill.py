"""Distillation of a classifier: a student's logits against a teacher's largest ones, beside labels where there are any.

For a row of logits s with the teacher's kept entries (ids, logits t) and a label:

    p    = softmax(t / T) over the row's entries
    kl   = sum_e p_e (log p_e - log softmax(s / T)[id_e]),    ce = -log softmax(s)[label]
    loss = (1 - hard) T^2 kl + hard ce

Entries with a negative id or t = -inf take no part.  A row without entries has no kl, one with a negative label no ce; with
neither its loss and gradient are 0, whatever its logits are.  An id may stand twice in a row: the probabilities add up.
An id or label that is no class makes its row NaN.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _C


def _check_teacher(name, teacher):
    if torch.is_grad_enabled() and teacher.requires_grad:
        raise RuntimeError(f"{name}: teacher takes no gradient (detach it)")


def distill_loss(logits: torch.Tensor, teacher: torch.Tensor, ids: torch.Tensor, temperature: float = 1.0,
                 labels: Optional[torch.Tensor] = None, hard: float = 0.0, reduction: str = "mean") -> torch.Tensor:
    """The loss above, float32: [rows] for reduction "none", else the mean over all rows or their sum.

    logits [rows, classes] and teacher [rows, kept] (the values of a top-k, kept at most 1024) float32, float16 or bfloat16;
    ids [rows, kept] int32 or int64; labels [rows] int32 or int64; rows possibly strided; 1e-3 <= temperature <= 1e3 and
    0 <= hard <= 1.  Differentiable in logits."""
    _check_teacher("distill_loss", teacher)
    return _C.distill_loss(logits, teacher, ids, temperature, labels, hard, reduction)


def distill_loss_grad(logits: torch.Tensor, teacher: torch.Tensor, ids: torch.Tensor, temperature: float = 1.0,
                      labels: Optional[torch.Tensor] = None, hard: float = 0.0, reduction: str = "mean",
                      factor: Union[None, float, torch.Tensor] = None):
    """(loss, gradient of the logits) in one call that reads the logits once from memory; records no gradient.

    The gradient is that of factor * loss (factor: a number, or one float32 value on the logits' device, such as a loss
    scale; None: 1), for logits.backward(gradient); the loss is without the factor."""
    _check_teacher("distill_loss_grad", teacher)
    if factor is not None and not isinstance(factor, torch.Tensor):
        factor = torch.full((1,), float(factor), dtype=torch.float32, device=logits.device)
    with torch.no_grad():
        loss, _, grad = _C.run_distill(logits, teacher, ids, temperature, labels, hard, reduction, False, True, factor)
    return loss, grad
