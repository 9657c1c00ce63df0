"""weight_grad8 of gradients that are not finite: an output is inf, -inf or NaN where the sum of the products is."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402


@pytest.mark.parametrize("rows", [1, 20, 33, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_gradients_that_are_not_finite(rows, dtype):
    gen = torch.Generator().manual_seed(rows)
    x = torch.randint(-20, 21, (rows, 70), generator=gen).float()
    x[:, ::32] = 64  # a scale of 1: whole numbers are kept as they are
    x[0, 5] = x[rows - 1, 6] = 0
    g = torch.randint(-3, 4, (rows, 50), generator=gen).float()
    g[0, 3], g[rows - 1, 4], g[0, 7] = math.inf, -math.inf, math.nan
    g[0, 9], g[rows // 2, 9] = math.inf, -math.inf if rows > 1 else math.inf
    g[0, 11] = torch.finfo(dtype).max  # finite; times 64 and more past float32 only there
    g = g.to(dtype).cuda()
    if dtype == torch.float32:  # a NaN whose upper half alone would be an inf
        g.view(torch.int32)[0, 13] = 0x7F800001
    p = ra_spmm.pack8(x.cuda())
    assert torch.equal(ra_spmm.unpack8(p).cpu(), x)
    want = (g.double().cpu()[:, :, None] * x.double()[:, None, :]).sum(0).float()  # inf past float32's range
    got = ra_spmm.weight_grad8(g, p).cpu()
    assert torch.equal(got.isnan(), want.isnan())
    ok = ~want.isnan()
    ok[11] = False  # rounded
    assert torch.equal(got[ok], want[ok])
    # Of column 11: one large product and small ones beside it.
    assert torch.equal(got[11].isinf(), want[11].isinf())
    assert torch.allclose(got[11][want[11].isfinite()], want[11][want[11].isfinite()], rtol=1e-6)
