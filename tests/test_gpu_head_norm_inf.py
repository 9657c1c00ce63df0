"""What is not finite at one coordinate of a head, in the coordinates that the rotation leaves alone: each of them has its
own value, whatever lies beside it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,rot", [(16, 8), (20, 12), (24, 0), (9, 4), (64, 32)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_unrotated_coordinates(D, rot, layout, dtype):
    rows = 5
    gen = torch.Generator().manual_seed(D)
    x, g = torch.randn(rows, 2, D, generator=gen), torch.randn(rows, 2, D, generator=gen)
    x[0, 0, rot], x[1, 1, D - 1], x[2, 0, rot + 1] = math.inf, -math.inf, math.inf
    g[3, 0, D - 1], g[4, 1, rot] = math.inf, -math.inf
    x, g, w = x.to(dtype).cuda(), g.to(dtype).cuda(), torch.ones(D, device="cuda", requires_grad=True)
    table = ra_spmm.rotation_table(rows, rot, device="cuda") if rot else None
    xd = x.clone().requires_grad_(True)
    y, _ = ra_spmm.head_norm_rotate(xd, None, w, None, table, None, layout=layout)
    y.backward(g)
    # 1 / rms is 0 where a coordinate is inf: the others are 0, it is inf * 0.
    for row, head, at in ((0, 0, rot), (1, 1, D - 1), (2, 0, rot + 1)):
        got = y.detach()[row, head].float().cpu()
        assert got[at].isnan() and not got[[i for i in range(D) if i != at]].any(), (row, got)
    clean, gc = x.float().cpu(), g.float().cpu()
    # dw of a coordinate sums over the heads; those without a value that is not finite there are finite.
    bad = torch.zeros(D, dtype=torch.bool)
    bad[[rot, D - 1, rot + 1]] = True
    for row, head in ((0, 0), (1, 1), (2, 0)):
        assert clean[row, head].isinf().any()
    for row, head in ((3, 0), (4, 1)):
        assert gc[row, head].isinf().any()
    assert torch.equal(w.grad.cpu().isfinite(), ~bad), w.grad
