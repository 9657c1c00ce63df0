"""Embedding lookup: rows of a table by id, and the table's gradient by sorted ids.

    out[i] = scale * table[ids[i]],    d table[v] = scale * sum over i with ids[i] = v of d out[i]
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _C


def embed(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, padding: Optional[int] = None) -> torch.Tensor:
    """scale * table[ids], of shape [*ids.shape, dim], differentiable in table.

    ids int32 or int64 of any shape; table [rows, dim] float32, float16 or bfloat16, rows possibly strided.  Positions whose
    id is `padding` (any value, inside of the table or not) give zeros and take no gradient; an id outside of the table
    gives NaN and takes none.  The gradient is dense and of the table's type; its sums are float32, and equal inputs give
    equal bits."""
    return _C.embed(ids, table, scale, padding)
