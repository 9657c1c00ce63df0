"""A graph transformer on the framework's operators: every node attends to its neighbour list.

A layer, on node features x [M, dim]:

    q, k, v  = x W_qkv                                    the input kept in 8 bits for W's gradient (linear8)
    q, k     = rotate(position, rms_norm(q, k))           head_norm_rotate
    o        = (softmax(q_1 k_1) - lam softmax(q_2 k_2)) v over the node's list   diff_attention
    x       += (1 - lam_0) rms_norm(o) W_o                 per head, head_norm_rotate without a table
    x       += relu(x W_1) W_2                             relu8 and linear8: one byte kept per hidden unit

With pre_norm=True the inputs of both branches are layer norms of the stream, the second one formed with the sum before it
(layer_norm with a residual), and the model norms the stream once more before its last map.  With nodes=N the input is a
row of a table for every node (embed, scaled by sqrt(dim)) instead of features.  distill_step trains a model on a
teacher's largest logits (distill_loss_grad).

with lam = exp(a_1 . b_1) - exp(a_2 . b_2) + lam_0 per head, learned.  The gradients of W_qkv, W_o and W_2 are those of the
kept 8-bit inputs, in float32 models too (each value within 1/64 of its group's largest); all others are of the inputs
themselves.  keep8=False keeps the inputs as they are: plain layers, more memory, no such rounding.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from .attention import diff_attention, head_norm_rotate, rotation_table
from .checkpoint8 import linear8, relu8
from .distill import distill_loss_grad
from .embedding import embed
from .norms import layer_norm


class LayerNorm(nn.Module):
    """Weight and bias of layer_norm, float32 whatever the input's type is."""

    def __init__(self, dim: int, eps: float = 1e-5):
        super().__init__()
        self.weight, self.bias, self.eps = nn.Parameter(torch.ones(dim)), nn.Parameter(torch.zeros(dim)), eps

    def forward(self, x, residual=None):
        return layer_norm(x, self.weight.float(), self.bias.float(), self.eps, residual)


class DiffTransformerLayer(nn.Module):
    """One layer; dim = heads * 2 * head_dim, kv_heads shared by heads / kv_heads query heads each."""

    def __init__(self, dim: int, heads: int, kv_heads: int = 0, hidden: int = 0, lam0: float = 0.8, eps: float = 1e-6,
                 keep8: bool = True, pre_norm: bool = False):
        super().__init__()
        kv_heads = kv_heads or heads
        if dim % (2 * heads) or heads % kv_heads:
            raise ValueError(f"dim {dim} must be a multiple of 2 * heads = {2 * heads}, heads of kv_heads = {kv_heads}")
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, dim // (2 * heads)
        self.lam0, self.eps, self.keep8 = lam0, eps, keep8
        d, hidden = self.head_dim, hidden or 2 * dim
        self.qkv = nn.Parameter(torch.empty((2 * heads + 4 * kv_heads) * d, dim))
        self.out = nn.Parameter(torch.empty(dim, dim))
        self.up, self.down = nn.Parameter(torch.empty(hidden, dim)), nn.Parameter(torch.empty(dim, hidden))
        for w in (self.qkv, self.out, self.up, self.down):
            nn.init.kaiming_uniform_(w, a=math.sqrt(5))
        self.q_norm, self.k_norm = nn.Parameter(torch.ones(d)), nn.Parameter(torch.ones(d))
        self.o_norm = nn.Parameter(torch.ones(2 * d))
        self.lam_a, self.lam_b = (nn.Parameter(torch.randn(2, heads, d) * 0.1) for _ in range(2))
        self.in_norm, self.mid_norm = (LayerNorm(dim), LayerNorm(dim)) if pre_norm else (None, None)

    def lam(self) -> torch.Tensor:
        e = (self.lam_a.float() * self.lam_b.float()).sum(-1).exp()
        return e[0] - e[1] + self.lam0

    def forward(self, x, plan, table=None, positions=None, bias=None):
        h, g, d = self.heads, self.kv_heads, self.head_dim
        linear = linear8 if self.keep8 else F.linear
        y = x if self.in_norm is None else self.in_norm(x)
        q, k, v = linear(y, self.qkv).split([2 * h * d, 2 * g * d, 2 * g * d], 1)
        q, k, v = q.unflatten(1, (h, 2, d)), k.unflatten(1, (g, 2, d)), v.unflatten(1, (g, 2 * d))
        q, k = head_norm_rotate(q, k, self.q_norm.float(), self.k_norm.float(), table, positions, eps=self.eps)
        o = diff_attention(plan, q, k, v, self.lam(), bias=bias)
        o, _ = head_norm_rotate(o, None, self.o_norm.float(), None, eps=self.eps)
        o = (1.0 - self.lam0) * linear(o.flatten(1), self.out)
        if self.mid_norm is None:
            x = y = x + o
        else:
            y, x = self.mid_norm(o.to(x.dtype), residual=x)
        u = F.linear(y, self.up)
        if not (self.keep8 and torch.is_grad_enabled()):
            return x + linear(u.relu_(), self.down)
        u, kept = relu8(u)
        return x + linear8(u, self.down, kept)


class DiffTransformer(nn.Module):
    """Node classifier: a linear map in (of features [M, in_dim], or with nodes > 0 a table's rows by node ids [M], -1:
    none), layers, a linear map out.  The plan of the graph (make_attention_plan) is kept by
    the caller, as are the plans of the other models' graphs; positions int32 [M] (None: no rotation)."""

    def __init__(self, in_dim: int, dim: int, out_dim: int, layers: int = 2, heads: int = 4, kv_heads: int = 0,
                 positions: int = 0, keep8: bool = True, pre_norm: bool = False, nodes: int = 0):
        super().__init__()
        self.first = None if nodes else nn.Linear(in_dim, dim, bias=False)
        self.last = nn.Linear(dim, out_dim, bias=False)
        self.layers = nn.ModuleList(DiffTransformerLayer(dim, heads, kv_heads, keep8=keep8, pre_norm=pre_norm)
                                    for _ in range(layers))
        self.last_norm = LayerNorm(dim) if pre_norm else None
        self.nodes = nn.Parameter(torch.randn(nodes, dim) * dim ** -0.5) if nodes else None
        d = dim // (2 * heads)
        self.register_buffer("table", rotation_table(positions, d // 2 * 2) if positions else None, persistent=False)

    def _apply(self, fn, recurse=True):
        """Moves and conversions, after which the table is the float32 one: angles rounded to 16 bits would be off by
        2^-9."""
        table = self.table
        super()._apply(fn, recurse)
        if table is not None and self.table.dtype != table.dtype:
            self.table = table.to(self.table.device)
        return self

    def forward(self, X, plan, positions=None, bias=None):
        if positions is not None and self.table is None:
            raise ValueError("the model was made without positions")
        table = None if positions is None else self.table
        x = embed(X, self.nodes, math.sqrt(self.nodes.size(1)), padding=-1) if self.first is None else self.first(X)
        for layer in self.layers:
            x = layer(x, plan, table, positions, bias)
        return self.last(x if self.last_norm is None else self.last_norm(x))


def train_step(model, plan, X, y, optimizer, positions=None, bias=None) -> torch.Tensor:
    """One forward, backward and optimizer step; the loss."""
    from .gnn import cross_entropy
    optimizer.zero_grad(set_to_none=True)
    loss = cross_entropy(model(X, plan, positions, bias).float(), y)
    loss.backward()
    optimizer.step()
    return loss.detach()


def distill_step(model, plan, X, teacher, ids, optimizer, temperature: float = 1.0, labels=None, hard: float = 0.0,
                 positions=None, bias=None, loss_scale: Optional[float] = None) -> torch.Tensor:
    """One forward, backward and optimizer step on a teacher's largest logits (teacher and ids [M, kept], as of a top-k) and
    the labels of some nodes (-1: none); the loss, distill_loss's.

    The backward pass runs on loss_scale times the loss, and every gradient is divided by it before it is added to its
    parameter's (or X's): a mean over many rows leaves a row's gradient of float16 logits below their smallest steps.  None: 1,
    but for float16 logits of more than 1024 rows the power of two that divides a row's by 1024 at most (1e6 rows: 1024).
    A parameter's gradient is rounded to the parameter's own type after that."""
    if loss_scale is not None and not 0.0 < loss_scale < math.inf:
        raise ValueError(f"distill_step: loss_scale must be positive and finite, got {loss_scale}")
    optimizer.zero_grad(set_to_none=True)
    logits = model(X, plan, positions, bias)
    if loss_scale is None:
        rows = logits.size(0) if logits.dtype == torch.float16 else 1
        loss_scale = max(1.0, 2.0 ** (rows - 1).bit_length() / 1024)
    # A factor of 1 is none: no tensor for it.
    loss, grad = distill_loss_grad(logits.detach(), teacher, ids, temperature, labels, hard,
                                   factor=None if loss_scale == 1.0 else loss_scale)
    leaves = [] if loss_scale == 1.0 else [t for t in (*model.parameters(), X) if t.requires_grad]
    handles = [t.register_hook(lambda g: g * (1.0 / loss_scale)) for t in leaves]
    try:
        logits.backward(grad)
    finally:
        for handle in handles:
            handle.remove()
    optimizer.step()
    return loss
