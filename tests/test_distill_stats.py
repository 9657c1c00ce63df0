"""What distillation's forward pass keeps for the backward pass: statistics of long rows only."""
import ctypes

import pytest
import torch

from ra_spmm import capi
from test_model_operators_abi import INVALID, OK, distill


@pytest.mark.parametrize("rows,classes,kept,rows_kept", [
    (0, 50, 5, 0), (1, 50, 5, 1), (1_000_000, 47, 8, 1), (1_000_000, 1024, 8, 1), (5000, 1024, 256, 1), (5000, 1024, 257, 5000),
    (5000, 1025, 8, 5000), (16, 50_000, 32, 16), ((1 << 31) - 1, 2000, 8, (1 << 31) - 1)])
def test_bytes(rows, classes, kept, rows_kept):
    lib, n = capi.load(), ctypes.c_int64(-1)
    s = ctypes.byref(distill(rows=rows, classes=classes, kept=kept, ld_logits=classes, ld_teacher=kept, ld_ids=kept))
    assert lib.ra_distill_stats_bytes(s, ctypes.byref(n)) == OK and n.value == 16 * rows_kept
    assert lib.ra_distill_stats_bytes(s, None) == INVALID and lib.ra_distill_stats_bytes(None, ctypes.byref(n)) == INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("C,kept_bytes", [(47, 0), (300, 0), (3000, 40_000 * 16)])
def test_memory_that_a_graph_keeps(C, kept_bytes):
    """The loss and what it keeps of long rows, in blocks of 512 bytes; 40,000 rows' statistics are 640,000 bytes."""
    import ra_spmm
    x = torch.randn(40_000, C, device="cuda", requires_grad=True)
    t, ids = torch.randn(40_000, 4, device="cuda"), torch.randint(0, C, (40_000, 4), device="cuda")
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    loss = ra_spmm.distill_loss(x, t, ids, 2.0)
    assert torch.cuda.memory_allocated() - before <= kept_bytes + 3 * 512
    g, = torch.autograd.grad(loss, x)
    assert g.shape == x.shape and g.isfinite().all()
