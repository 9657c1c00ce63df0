"""Activations kept in 8 bits between the forward and the backward pass.

Packed8 holds one byte per element and a power-of-two scale per 32 consecutive columns of a row.  A value code * scale has
at most 8 significant bits, so the weight gradient g^T x takes it on the matrix cores without rounding (weight_grad8).  The
codes of a ReLU's output are unsigned and at least 1 where the input was positive: they also hold the ReLU's mask.

    pack8(x)            Packed8, signed
    relu_pack8(x)       (relu(x), Packed8), one pass
    unpack8(p)          code * scale
    relu_grad8(g, p)    gradient through the ReLU
    weight_grad8(g, p)  g^T (code * scale), float32

None of these records a gradient.  relu8 and linear8 are the differentiable forms: a linear layer after a ReLU keeps 1 byte per input element for both of
them, where float32 autograd keeps 4.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _C
from .attention import _rows


class Packed8(NamedTuple):
    codes: torch.Tensor   # uint8 [rows, cols rounded up to 32]
    scales: torch.Tensor  # uint8 [groups, rows rounded up to 8]: exponent + 127, 255 for a group that was not finite
    cols: int
    signed: bool

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()


def pack8(x: torch.Tensor) -> Packed8:
    """x [rows, cols] in 8 bits, signed: round(x / scale) with the group's largest magnitude in [64, 128) scales."""
    codes, scales = _C.pack8(x)
    return Packed8(codes, scales, x.size(1), True)


def relu_pack8(x: torch.Tensor):
    """(relu(x), its 8-bit form): unsigned, the group's largest value in [128, 256) scales, positive values at least 1."""
    y, codes, scales = _C.relu_pack8(x)
    return y, Packed8(codes, scales, x.size(1), False)


def unpack8(p: Packed8, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """code * scale, [rows, cols]."""
    return _C.unpack8(p.codes, p.scales, p.cols, p.signed, dtype)


def relu_grad8(grad: torch.Tensor, p: Packed8) -> torch.Tensor:
    """grad where the ReLU's input was positive, else 0; p from relu_pack8."""
    if p.signed:
        raise RuntimeError("relu_grad8: the codes are signed (pack8); relu_pack8's hold the mask")
    return _C.relu_grad8(grad, p.codes, p.scales, p.cols)


def weight_grad8(grad: torch.Tensor, p: Packed8) -> torch.Tensor:
    """grad^T (code * scale), [out, cols] float32: the weight gradient of y = x W^T with grad [rows, out]."""
    return _C.weight_grad8(grad, p.codes, p.scales, p.cols, p.signed)


class _Relu8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        y, codes, scales = _C.relu_pack8(x)
        ctx.save_for_backward(codes, scales)
        ctx.cols = x.size(1)
        ctx.mark_non_differentiable(codes, scales)
        ctx.set_materialize_grads(False)  # no zeros of the codes' size
        return y, codes, scales

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, _codes, _scales):
        if grad is None:
            return None
        codes, scales = ctx.saved_tensors
        return _C.relu_grad8(_rows(grad), codes, scales, ctx.cols)


def relu8(x: torch.Tensor):
    """relu(x) and its Packed8 for the layer that follows (linear8); its gradient takes the mask from the codes."""
    y, codes, scales = _Relu8.apply(_rows(x))
    return y, Packed8(codes, scales, x.size(1), False)


class _Linear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, codes, scales, signed):
        if codes is None:
            codes, scales = _C.pack8(x)
        ctx.save_for_backward(weight, codes, scales)
        ctx.cols, ctx.signed = x.size(1), signed
        return F.linear(x, weight)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        weight, codes, scales = ctx.saved_tensors
        # Under autocast the output, and so grad, has fewer bits than the weight.
        gx = grad @ weight.to(grad.dtype) if ctx.needs_input_grad[0] else None
        gw = None
        if ctx.needs_input_grad[1]:
            gw = _C.weight_grad8(_rows(grad), codes, scales, ctx.cols, ctx.signed).to(weight.dtype)
        return gx, gw, None, None, None


def linear8(x: torch.Tensor, weight: torch.Tensor, packed: Optional[Packed8] = None) -> torch.Tensor:
    """x W^T that keeps its input in 8 bits: in `packed` where the caller has it (relu8), else packed here.  The weight
    gradient is that of the kept values."""
    if packed is not None and (packed.cols != x.size(1) or packed.codes.size(0) != x.size(0)):
        raise RuntimeError(f"linear8: packed holds [{packed.codes.size(0)}, {packed.cols}], x is {tuple(x.shape)}")
    if not (torch.is_grad_enabled() and weight.requires_grad):
        return F.linear(x, weight)  # nothing to keep
    if packed is None:
        return _Linear8.apply(_rows(x), weight, None, None, True)
    return _Linear8.apply(x, weight, packed.codes, packed.scales, packed.signed)
