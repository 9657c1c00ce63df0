"""A DiffTransformer converted to 16 bits keeps its rotation table in float32, as head_norm_rotate takes it."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402
from ra_spmm import transformer as T  # noqa: E402


def graph(M):
    dense = torch.rand(M, M, generator=torch.Generator().manual_seed(1)) < 0.1
    rowptr = torch.zeros(M + 1, dtype=torch.int32)
    rowptr[1:] = dense.sum(1).cumsum(0)
    return rowptr.cuda(), dense.nonzero()[:, 1].to(torch.int32).cuda()


@pytest.mark.parametrize("convert", ["to dtype", "half or bfloat16", "to device and dtype", "copy"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_converted_model(dtype, convert):
    M, positions = 150, 5000
    rowptr, colind = graph(M)
    plan = ra_spmm.make_attention_plan(rowptr, colind, M, M)
    torch.manual_seed(2)
    model = T.DiffTransformer(24, 64, 5, heads=2, positions=positions)
    table = ra_spmm.rotation_table(positions, 16)
    if convert == "to dtype":
        model = model.cuda().to(dtype)
    elif convert == "half or bfloat16":
        model = (model.half() if dtype == torch.float16 else model.bfloat16()).cuda()
    elif convert == "to device and dtype":
        model = model.to("cuda", dtype)
    else:
        model = copy.deepcopy(model.to(dtype).cuda())
    assert model.table.dtype == torch.float32 and model.table.is_cuda and torch.equal(model.table.cpu(), table)
    assert all(p.dtype == dtype and p.is_cuda for p in model.parameters())
    assert "table" not in model.state_dict()
    X = torch.randn(M, 24, device="cuda").to(dtype)
    pos = (torch.arange(M, dtype=torch.int32, device="cuda") * 33)
    y = model(X, plan, pos)
    y.float().sum().backward()
    assert y.dtype == dtype and all(p.grad.isfinite().all() for p in model.parameters())


def test_a_model_without_positions_converts():
    model = T.DiffTransformer(8, 16, 2, heads=2).half()
    assert model.table is None and model.first.weight.dtype == torch.float16
