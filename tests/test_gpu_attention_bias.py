"""Finite biases of any size are scores like others, and one of +inf or NaN is what a softmax makes of it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402

MOST = torch.finfo(torch.float32).max
# Two kinds of edges in a row: bias of most of them, bias of a few.
PAIRS = [(-3e38, -2.5e38), (2.1e38, 3e38), (-MOST, -3.3e38), (-MOST, 0.0), (3.3e38, MOST), (-2.2e38, -2.0e38), (1.9e38, 2.3e38),
         (-1e30, -9e29), (-1.1e38, -0.9e38), (0.9e38, 1.1e38), (-1.0e38, -1.01e38), (-MOST, MOST)]


def rows_of(lengths, K, seed):
    gen = torch.Generator().manual_seed(seed)
    rowptr = torch.zeros(len(lengths) + 1, dtype=torch.int32)
    rowptr[1:] = torch.tensor(lengths).cumsum(0)
    return rowptr, torch.cat([torch.randperm(K, generator=gen)[:n].sort().values for n in lengths]).to(torch.int32)


def run(rowptr, colind, K, bias, seed=1):
    gen = torch.Generator().manual_seed(seed)
    M, H, D, Dv = rowptr.numel() - 1, 2, 8, 16
    q, k, v, g = (torch.randn(s, generator=gen) for s in ((M, H, 2, D), (K, H, 2, D), (K, H, Dv), (M, H, Dv)))
    lam = torch.tensor([0.3, 0.6])
    t = [x.cuda().requires_grad_(True) for x in (q, k, v, lam)]
    rp, ci, b = rowptr.cuda(), colind.cuda(), bias.cuda()
    plan = ra_spmm.make_attention_plan(rp, ci, M, K)
    out = ra_spmm.diff_attention(plan, *t, bias=b)
    grads = torch.autograd.grad(out, t, g.cuda())
    with torch.no_grad():
        free = ra_spmm.diff_attention_csr(rp, ci, *t, bias=b)
    return (q, k, v, lam, g), out.detach().cpu(), free.cpu(), [x.cpu() for x in grads]


@pytest.mark.parametrize("pair", PAIRS, ids=str)
def test_two_biases(pair):
    """The row's weight lies on the edges of its larger bias (a score of magnitude 10 does not change one of 1e29)."""
    lengths = [2, 5, 33, 70, 700]
    rowptr, colind = rows_of(lengths, 900, 3)
    bias = torch.empty(colind.numel())
    for i in range(len(lengths)):
        a, b = int(rowptr[i]), int(rowptr[i + 1])
        bias[a:b] = pair[0]
        few = 1 if pair[1] == 0 else 1 + i % 2
        bias[a + (b - a) // 2:b][:few] = pair[1]
    (q, k, v, lam, g), out, free, (dq, dk, dv, dlam) = run(rowptr, colind, 900, bias)
    want, wdv = torch.zeros_like(out, dtype=torch.float64), torch.zeros(v.shape, dtype=torch.float64)
    for i in range(len(lengths)):
        at = slice(int(rowptr[i]), int(rowptr[i + 1]))
        b, j = bias[at].double(), colind[at].long()
        top = b == b.max()
        for h in range(2):
            # A bias of 1e29 and more takes any score up in its rounding: of equal ones, equal weights.
            w = top.double() / top.sum() * (1 - lam[h].double())
            want[i, h] = w @ v[j, h].double()
            wdv[:, h].index_add_(0, j, w[:, None] * g[i, h].double())
    for o in (out, free):
        assert (o.double() - want).abs().max() < 1e-5
    assert (dv.double() - wdv).abs().max() < 1e-5
    assert all(x.isfinite().all() for x in (dq, dk, dlam))


@pytest.mark.parametrize("value", [math.inf, math.nan], ids=str)
def test_biases_without_a_softmax(value):
    """A score of +inf (inf - inf) or NaN: the row is NaN, and no other row."""
    lengths = [1, 5, 33, 700, 6, 600]
    rowptr, colind = rows_of(lengths, 900, 5)
    bias = torch.randn(colind.numel(), generator=torch.Generator().manual_seed(2))
    bad = torch.tensor([True, False, True, True, False, False])
    for i in torch.arange(6)[bad].tolist():
        bias[int(rowptr[i]) + (lengths[i] - 1) // 3] = value
    _, out, free, (dq, _, _, _) = run(rowptr, colind, 900, bias)
    for x in (out, free, dq):
        assert x[bad].isnan().all() and x[~bad].isfinite().all()
