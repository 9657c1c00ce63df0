"""Layer norm of every row, alone or of a sum with the residual stream.

    h = x + residual,  n = (h - mean(h)) / sqrt(mean((h - mean(h))^2) + eps),  y = n * weight + bias
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _C


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, residual: Optional[torch.Tensor] = None):
    """Layer norm over the last axis: y, or (y, x + residual) where a residual is given.

    x [.., dim] (dim at most 16384) float32, float16 or bfloat16, its rows possibly strided; residual of x's shape and
    dtype; weight and bias float32 [dim] (None: 1 and 0).  The sum is rounded to the dtype and y is the norm of what is
    returned.  Differentiable in x, residual, weight and bias; statistics and sums are float32, in a fixed order."""
    if residual is not None and residual.shape != x.shape:
        raise RuntimeError(f"layer_norm: residual must have x's shape {tuple(x.shape)}, has {tuple(residual.shape)}")
    if x.dim() == 0:
        raise RuntimeError("layer_norm: x must have at least one axis")
    shape = x.shape
    if len(shape) != 2:
        x = x.reshape(-1, shape[-1])
        residual = None if residual is None else residual.reshape(-1, shape[-1])
    y, total = _C.layer_norm(x, residual, weight, bias, eps)
    if len(shape) != 2:
        y, total = y.view(shape), None if total is None else total.view(shape)
    return y if total is None else (y, total)
