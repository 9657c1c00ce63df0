"""Differentiable graph attention over CSR neighbour lists, and the head norms with rotation before it.

Differential attention:

    out[i, h] = sum_j (softmax(s_1) - lam[h] * softmax(s_2))[j] * v[j, g]
    s_a[j]    = scale * q[i, h, a] . k[j, g, a] + bias[ij],   j over row i's columns

with g = h // (heads / kv_heads).  An edge whose bias is -inf takes no part; a row
without edges (or without one left) gives zeros and takes no gradient.
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import _C


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t itself where only its rows are strided, else a contiguous copy."""
    if t.is_neg():  # the imaginary part of a conjugate, say: its memory holds the opposite
        return t.resolve_neg().contiguous()
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
    if bias is not None and bias.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("diff_attention: bias takes no gradient (detach it)")
    q, k, v = _rows(q), _rows(k), _rows(v)
    if q.dim() == 4 and lam.numel() == 1:
        lam = lam.reshape(1).expand(q.size(1))
    lam = lam.contiguous()
    if _C.through_node((q, k, v, lam)):
        return _DiffAttention.apply(plan, q, k, v, lam, scale, bias)
    return _C.run_attention_plan(plan, q, k, v, lam, scale, bias)


def rotation_table(positions: int, rot_dim: int, base: float = 10000.0, scaling: float = 1.0, device=None) -> torch.Tensor:
    """(cos, sin) of the angles p / scaling * base ** (-2 i / rot_dim), float32 [positions, rot_dim / 2, 2], formed in
    64 bits.  scaling > 1 stretches the positions of a longer context over those of a shorter one."""
    if rot_dim < 0 or rot_dim % 2:
        raise RuntimeError(f"rotation_table: rot_dim must be even, got {rot_dim}")
    if not (scaling > 0 and base > 0):
        raise RuntimeError("rotation_table: base and scaling must be positive")
    half = rot_dim // 2
    freq = torch.exp(torch.arange(half, dtype=torch.float64, device=device) * (-2.0 * math.log(base) / max(rot_dim, 1)))
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] / scaling * freq
    return torch.stack([angle.cos(), angle.sin()], dim=-1).float().contiguous()


class _HeadNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, table, positions, eps, layout):
        ctx.save_for_backward(q, k, wq, wk, table, positions)
        ctx.eps, ctx.layout = eps, layout
        ctx.set_materialize_grads(False)
        return _C.run_head_norm(q, k, wq, wk, table, positions, eps, layout)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, wq, wk, table, positions = ctx.saved_tensors
        gq = torch.zeros_like(q, memory_format=torch.contiguous_format) if gq is None else gq.contiguous()
        if k is not None:
            gk = torch.zeros_like(k, memory_format=torch.contiguous_format) if gk is None else gk.contiguous()
        dq, dk, dwq, dwk = _C.run_head_norm_backward(q, k, wq, wk, table, positions, ctx.eps, ctx.layout, gq, gk)
        return dq, dk, dwq, dwk, None, None, None, None


def head_norm_rotate(q, k, wq, wk, table=None, positions=None, eps: float = 1e-6, layout: str = "half"):
    """RMS norm of every query and key head, its weight and the rotation by the row's position, in one pass; (q', k').

    q and k [rows, heads.., head_dim] (k and wk may be None), rows possibly strided; wq, wk float32 [head_dim]; table from
    rotation_table (None: no rotation), its first rot_dim coordinates are rotated, in pairs (i, i + rot_dim / 2) for
    layout "half" and (2 i, 2 i + 1) for "interleaved"; positions int32 [rows], None: the row numbers.  A position outside
    of the table gives NaN.  Differentiable in q, k, wq and wk."""
    q = _rows(q)
    k = None if k is None else _rows(k)
    if _C.through_node((q, k, wq, wk)):
        return _HeadNorm.apply(q, k, wq, wk, table, positions, eps, layout)
    return _C.run_head_norm(q, k, wq, wk, table, positions, eps, layout)
