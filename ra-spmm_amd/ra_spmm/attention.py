"""Differentiable graph attention over CSR neighbour lists.

    out[i, h] = sum_j (softmax(s_1) - lam[h] * softmax(s_2))[j] * v[j, g]
    s_a[j]    = scale * q[i, h, a] . k[j, g, a] + bias[ij],   j over row i's columns

with g = h // (heads / kv_heads).  An edge whose bias is -inf takes no part; a row
without edges (or without one left) gives zeros and takes no gradient.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _C


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t itself where only its rows are strided, else a contiguous copy."""
    run = 1
    for d in range(t.dim() - 1, 0, -1):
        if t.size(d) > 1 and t.stride(d) != run:
            return t.contiguous()
        run *= t.size(d)
    return t if t.size(0) <= 1 or t.stride(0) >= run else t.contiguous()


class _DiffAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, q, k, v, lam, scale, bias):
        out, stats = _C.run_attention_plan_train(plan, q, k, v, lam, scale, bias)
        ctx.plan, ctx.scale = plan, scale
        ctx.save_for_backward(q, k, v, lam, bias, stats)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, lam, bias, stats = ctx.saved_tensors
        dq, dk, dv, dlam = _C.run_attention_plan_backward(ctx.plan, q, k, v, lam, stats, grad.contiguous(), ctx.scale,
                                                          bias)
        return None, dq, dk, dv, dlam, None, None


def diff_attention(plan, q, k, v, lam, scale=None, bias=None) -> torch.Tensor:
    """Differential attention on a kept plan (make_attention_plan), differentiable in q, k, v and lam.

    q [M, heads, 2, head_dim], k [K, kv_heads, 2, head_dim], v [K, kv_heads, value_dim] of one dtype (float32, float16 or
    bfloat16), rows possibly strided; lam float32, one weight or one per head; scale defaults to head_dim ** -0.5; bias
    float32 [nnz] in the plan's edge order, without a gradient.  Returns [M, heads, value_dim]."""
    if bias is not None and bias.requires_grad:
        raise RuntimeError("diff_attention: bias takes no gradient (detach it)")
    q, k, v = _rows(q), _rows(k), _rows(v)
    if q.dim() == 4 and lam.numel() == 1:
        lam = lam.reshape(1).expand(q.size(1))
    lam = lam.contiguous()
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, lam)):
        return _DiffAttention.apply(plan, q, k, v, lam, scale, bias)
    return _C.run_attention_plan(plan, q, k, v, lam, scale, bias)
