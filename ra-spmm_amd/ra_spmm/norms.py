"""Layer norm of every row, alone or of a sum with the residual stream.

    h = x + residual,  n = (h - mean(h)) / sqrt(mean((h - mean(h))^2) + eps),  y = n * weight + bias
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _C
from .attention import _rows


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        y, total, stats = _C.run_layer_norm(x, residual, weight, bias, eps, True)
        # Without a residual the input itself is kept, else the sum, which the caller has anyway.
        ctx.save_for_backward(x if total is None else total, weight, stats)
        ctx.set_materialize_grads(False)
        return y if total is None else (y, total)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, grad_total=None):
        h, weight, stats = ctx.saved_tensors
        x_grad, residual_grad, weight_grad, bias_grad = ctx.needs_input_grad[:4]
        if grad is None:  # only the sum was used
            dx = grad_total
            dw = torch.zeros_like(weight) if weight_grad else None
            db = torch.zeros(h.size(1), dtype=torch.float32, device=h.device) if bias_grad else None
        else:
            grad_total = None if grad_total is None else grad_total.contiguous()
            dx, dw, db = _C.run_layer_norm_backward(h, weight, stats, grad.contiguous(), grad_total, weight_grad, bias_grad)
        return dx if x_grad else None, dx if residual_grad else None, dw, db, None


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
    x = _rows(x.reshape(-1, shape[-1]) if x.dim() != 2 else x)
    if residual is not None:
        residual = _rows(residual.reshape(-1, shape[-1]) if residual.dim() != 2 else residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight, bias)):
        out = _LayerNorm.apply(x, residual, weight, bias, eps)
    else:
        y, total, _ = _C.run_layer_norm(x, residual, weight, bias, eps, False)
        out = y if total is None else (y, total)
    if len(shape) == 2:
        return out
    return out.view(shape) if residual is None else (out[0].view(shape), out[1].view(shape))
