"""A graph transformer on the framework's operators: every node attends to its neighbour list.

A layer, on node features x [M, dim]:

    q, k, v  = x W_qkv                                    the input kept in 8 bits for W's gradient (linear8)
    q, k     = rotate(position, rms_norm(q, k))           head_norm_rotate
    o        = (softmax(q_1 k_1) - lam softmax(q_2 k_2)) v over the node's list   diff_attention
    x       += (1 - lam_0) rms_norm(o) W_o                 per head, head_norm_rotate without a table
    x       += relu(x W_1) W_2                             relu8 and linear8: one byte kept per hidden unit

with lam = exp(a_1 . b_1) - exp(a_2 . b_2) + lam_0 per head, learned.  The gradients of W_qkv, W_o and W_2 are those of the
kept 8-bit inputs, in float32 models too (each value within 1/64 of its group's largest); all others are of the inputs
themselves.  keep8=False keeps the inputs as they are: plain layers, more memory, no such rounding.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from .attention import diff_attention, head_norm_rotate, rotation_table
from .checkpoint8 import linear8, relu8


class DiffTransformerLayer(nn.Module):
    """One layer; dim = heads * 2 * head_dim, kv_heads shared by heads / kv_heads query heads each."""

    def __init__(self, dim: int, heads: int, kv_heads: int = 0, hidden: int = 0, lam0: float = 0.8, eps: float = 1e-6,
                 keep8: bool = True):
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

    def lam(self) -> torch.Tensor:
        e = (self.lam_a.float() * self.lam_b.float()).sum(-1).exp()
        return e[0] - e[1] + self.lam0

    def forward(self, x, plan, table=None, positions=None, bias=None):
        h, g, d = self.heads, self.kv_heads, self.head_dim
        linear = linear8 if self.keep8 else F.linear
        q, k, v = linear(x, self.qkv).split([2 * h * d, 2 * g * d, 2 * g * d], 1)
        q, k, v = q.unflatten(1, (h, 2, d)), k.unflatten(1, (g, 2, d)), v.unflatten(1, (g, 2 * d))
        q, k = head_norm_rotate(q, k, self.q_norm.float(), self.k_norm.float(), table, positions, eps=self.eps)
        o = diff_attention(plan, q, k, v, self.lam(), bias=bias)
        o, _ = head_norm_rotate(o, None, self.o_norm.float(), None, eps=self.eps)
        x = x + (1.0 - self.lam0) * linear(o.flatten(1), self.out)
        u = F.linear(x, self.up)
        if not (self.keep8 and torch.is_grad_enabled()):
            return x + linear(u.relu_(), self.down)
        u, kept = relu8(u)
        return x + linear8(u, self.down, kept)


class DiffTransformer(nn.Module):
    """Node classifier: a linear map in, layers, a linear map out.  The plan of the graph (make_attention_plan) is kept by
    the caller, as are the plans of the other models' graphs; positions int32 [M] (None: no rotation)."""

    def __init__(self, in_dim: int, dim: int, out_dim: int, layers: int = 2, heads: int = 4, kv_heads: int = 0,
                 positions: int = 0, keep8: bool = True):
        super().__init__()
        self.first, self.last = nn.Linear(in_dim, dim, bias=False), nn.Linear(dim, out_dim, bias=False)
        self.layers = nn.ModuleList(DiffTransformerLayer(dim, heads, kv_heads, keep8=keep8) for _ in range(layers))
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
        x = self.first(X)
        for layer in self.layers:
            x = layer(x, plan, table, positions, bias)
        return self.last(x)


def train_step(model, plan, X, y, optimizer, positions=None, bias=None) -> torch.Tensor:
    """One forward, backward and optimizer step; the loss."""
    from .gnn import cross_entropy
    optimizer.zero_grad(set_to_none=True)
    loss = cross_entropy(model(X, plan, positions, bias).float(), y)
    loss.backward()
    optimizer.step()
    return loss.detach()
