"""Outputs past 256 MB, which are written around the caches, of rows of every kind (parts of a wave, waves and workgroups, whole
packets or not); logits that are columns of wider rows where a lane takes a row; two streams at once, every round compared.

Bounds: those of the operators' own tests.  Where a whole result is compared with the results of its slices instead, both are
within the same bound of the definition: 16-bit values of nearly equal floats are at most one unit in the last place apart, 2 eps |v|
with room (eps = torch.finfo's), or one smallest fp16 step; floats of sums over n terms 2 (n + 40) 2^-24 of their magnitudes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402
from test_gpu_distill import close as close_distill  # noqa: E402
from test_gpu_distill import exact as exact_distill  # noqa: E402
from test_gpu_distill import make as make_distill  # noqa: E402
from test_gpu_layer_norm import HALF_UNIT  # noqa: E402
from test_gpu_layer_norm import exact as exact_norm  # noqa: E402

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def close(got, want, err, what):
    """As test_gpu_layer_norm.close, on the GPU."""
    unit = HALF_UNIT[got.dtype]
    bound = err + unit * (want.abs() + err) + (2.0 ** -25 if unit == 2.0 ** -11 else 1e-30)
    off = (got.detach().double() - want).abs()
    assert (off <= bound).all(), (what, float((off / bound).max()), (~(off <= bound)).nonzero()[0].tolist())


@pytest.mark.parametrize("M,D,dtype", [
    (2_200_000, 64, torch.bfloat16), (600_000, 257, torch.bfloat16), (300_000, 500, torch.float16), (150_000, 900, torch.float16),
    (140_000, 1030, torch.bfloat16), (34_000, 4104, torch.float16), (17_000, 8201, torch.bfloat16), (4_000_000, 19, torch.float32),
    (300_000, 300, torch.float32), (90_000, 1001, torch.float32), (70_000, 1030, torch.float32), (17_000, 4100, torch.float32),
    (8_300, 8201, torch.float32), (5_000, 16_383, torch.float32), (100_000_000, 3, torch.float16)], ids=str)
def test_layer_norm(M, D, dtype):
    assert M * D * torch.finfo(dtype).bits // 8 > 256 << 20
    gen = torch.Generator("cuda").manual_seed(D)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x, res, gy, gh = ((r(M, D) + 0.3).to(dtype) for _ in range(4))
    w, b = 1 + 0.3 * r(D), 0.3 * r(D)
    leaves = [t.requires_grad_(True) for t in (x, res, w, b)]
    y, h = ra_spmm.layer_norm(x, w, b, residual=res)
    dx, dr, dw, db = torch.autograd.grad((y, h), leaves, (gy, gh))
    assert torch.equal(h, (x.detach().float() + res.detach().float()).to(dtype)) and torch.equal(dx, dr)
    step = max(1, 60_000_000 // D)  # rows at a time in 64 bits
    sums = [torch.zeros(D, dtype=torch.float64, device="cuda") for _ in range(4)]
    for lo in range(0, M, step):
        part = slice(lo, lo + step)
        want = exact_norm(h[part].detach(), w.detach(), b.detach(), 1e-5, gy[part], gh[part])
        close(y[part], *want["y"], f"y from {lo}")
        close(dx[part], *want["dx"], f"dx from {lo}")
        n = len(h[part])
        for s, t in zip(sums, (want["dw"][0], want["dw"][1], want["db"][0], want["db"][1])):
            s += t * (M + 3) / (n + 1) if t is want["dw"][1] or t is want["db"][1] else t  # the whole sum has M terms, not n
    close(dw, sums[0], sums[1], "dw")
    close(db, sums[2], sums[3], "db")


@pytest.mark.parametrize("n,V,D,dtype", [
    (1_500_000, 1_500_000, 100, torch.bfloat16), (300_000, 290_000, 257, torch.float32), (40_000_000, 70, 5, torch.float16),
    (9_000, 9_000, 30_001, torch.bfloat16), (1_000, 2_300_000, 129, torch.float16), (2_300_000, 1_000, 129, torch.float16)], ids=str)
def test_embedding(n, V, D, dtype):
    """A product is off by its roundings, to float32 (where the compiler forms it on its own) and to the type; sums of whole
    numbers are exact."""
    assert max(n, V) * D * torch.finfo(dtype).bits // 8 > 256 << 20
    gen = torch.Generator("cuda").manual_seed(D)
    ids = torch.randint(0, V, (n,), generator=gen, device="cuda")
    ids[n // 3:n // 3 + 5] = -1
    table = torch.randn(V, D, generator=gen, device="cuda").to(dtype).requires_grad_(True)
    out = ra_spmm.embed(ids, table, 1.75, padding=-1)
    real = ids >= 0
    for lo in range(0, n, 1 + 50_000_000 // D):
        part = slice(lo, lo + 1 + 50_000_000 // D)
        want = (table.detach()[ids[part].clamp(min=0)].double() * 1.75).masked_fill_(~real[part, None], 0.0)
        close(out[part], want, 2.0 ** -24 * want.abs(), f"out from {lo}")
    # Few rows take many positions: most of their numbers are 0, so that every sum stays a small one.
    g = torch.zeros(n, D, dtype=dtype, device="cuda")
    g[::max(1, n // V)] = torch.randint(-3, 4, g[::max(1, n // V)].shape, generator=gen, device="cuda").to(dtype)
    grad, = torch.autograd.grad(out, table, g)
    sums = torch.zeros(V, D, device="cuda").index_add_(0, ids[real], g[real].float())
    assert torch.equal(grad, (sums * 1.75).to(dtype))


@pytest.mark.parametrize("M,C,dtype", [(1_400, 100_003, torch.bfloat16), (700, 100_001, torch.float32), (9_000, 16_001, torch.float16),
                                       (3, 50_000_017, torch.bfloat16)], ids=str)
def test_long_rows_of_distillation(M, C, dtype):
    """By workgroups and pieces, rows that begin at any address: samples against the definition, everything against slices."""
    assert M * C * torch.finfo(dtype).bits // 8 > 256 << 20
    gen = torch.Generator("cuda").manual_seed(M)
    x = (2 * torch.randn(M, C, generator=gen, device="cuda")).to(dtype)
    t, ids = torch.randn(M, 20, generator=gen, device="cuda"), torch.randint(-1, C, (M, 20), generator=gen, device="cuda")
    labels = torch.randint(-1, C, (M,), generator=gen, device="cuda")
    labels[::5] = ids[::5, 0]
    t[1], ids[2], labels[2] = -math.inf, -1, -1
    loss, grad = ra_spmm.distill_loss_grad(x, t, ids, 2.0, labels, 0.4, "none")
    some = torch.tensor(sorted({0, 1, 2, M // 2, M - 2, M - 1}), device="cuda") if C < 1_000_000 else torch.arange(M, device="cuda")
    want, werr, g, gerr = exact_distill(x[some].cpu(), t[some].cpu(), ids[some].cpu(), 2.0, labels[some].cpu(), 0.4,
                                        torch.ones(len(some), dtype=torch.float64))
    close_distill(loss[some], want, werr, "loss")
    close_distill(grad[some], g, gerr, "gradient")
    leaf = x.detach().requires_grad_(True)
    again, = torch.autograd.grad(ra_spmm.distill_loss(leaf, t, ids, 2.0, labels, 0.4, "none"), leaf, torch.ones(M, device="cuda"))
    eps, smallest = torch.finfo(dtype).eps, 2.0 ** -24 if dtype == torch.float16 else 0.0
    room = max(2 * eps, 4 * (C / 64 + 120) * 2.0 ** -24)  # of sums of C / 64 terms and more in a chain, twice
    for lo in range(0, M, max(1, M // 8)):
        part = slice(lo, lo + max(1, M // 8))
        a, b = grad[part].float(), ra_spmm.distill_loss_grad(x[part], t[part], ids[part], 2.0, labels[part], 0.4, "none")[1].float()
        magnitude = torch.maximum(a.abs(), b.abs())
        # Where an entry's probability is taken off, the difference of two such values is left.
        taken = torch.zeros_like(a).scatter_(1, ids[part].clamp(min=0), 2.0).scatter_(1, labels[part].clamp(min=0)[:, None], 2.0)
        bound = room * (magnitude + taken) + smallest
        assert ((a - b).abs() <= bound).all() and ((a - again[part].float()).abs() <= bound).all(), lo


@pytest.mark.parametrize("extra,begin", [(1, 0), (1, 1), (3, 1), (8, 0), (16, 8)], ids=str)
@pytest.mark.parametrize("C", [7, 40, 47, 64])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_many_strided_rows_of_few_classes(C, dtype, extra, begin):
    """Columns of wider rows, where a lane takes a row."""
    M = 33_001
    x, t, ids, labels = make_distill(M, C, 5, dtype, seed=C)
    some = torch.cat([torch.arange(20), torch.arange(M // 2, M // 2 + 8), torch.arange(M - 12, M)])
    x[3, C - 1], x[5] = math.nan, -math.inf
    ids[7], labels[7], x[7, 0] = -1, -1, math.nan
    wide = torch.full((M, C + extra), math.inf, dtype=dtype, device="cuda")  # what is beside the rows is not read into them
    wide[:, begin:begin + C] = x.cuda()
    rows = wide[:, begin:begin + C]
    assert not rows.is_contiguous()
    up = torch.randn(M, generator=torch.Generator().manual_seed(5))
    for hard in (0.0, 0.4):
        want, werr, grad, gerr = exact_distill(x[some], t[some], ids[some], 2.0, labels[some], hard, up[some].double())
        whole = None
        for at in (rows, x.cuda()):
            leaf = at.detach().requires_grad_(True)
            loss = ra_spmm.distill_loss(leaf, t.cuda(), ids.cuda(), 2.0, labels.cuda(), hard, "none")
            g, = torch.autograd.grad(loss, leaf, up.cuda())
            close_distill(loss[some.cuda()], want, werr, "loss of the rows")
            close_distill(g[some.cuda()], grad, gerr, "gradient of the rows")
            assert torch.equal(loss.isnan(), whole[0].isnan()) if whole else True
            whole = whole or (loss.detach(), g)
        # Sums of at most 64 terms, times an incoming gradient of at most 5, T and the two parts.
        bound = 2 * torch.finfo(dtype).eps * torch.maximum(g.float().abs(), whole[1].float().abs()) + 40 * 200 * 2.0 ** -24
        bad = (g.float() - whole[1].float()).abs() > bound
        assert not bad.any() and torch.equal(g.isnan(), whole[1].isnan())


def test_two_streams_at_once_every_round():
    gen = torch.Generator("cuda").manual_seed(3)
    data = []
    for i in range(2):
        x = torch.randn(4000, 300, generator=gen, device="cuda")
        t, top = torch.randn(4000, 300, generator=gen, device="cuda").topk(6, dim=1)
        data.append((x, torch.randint(0, 4000, (20_000,), generator=gen, device="cuda"),
                     torch.randn(20_000, 300, generator=gen, device="cuda"), t, top))

    def work(x, ids, g, t, top):
        table = x.detach().requires_grad_(True)
        rows = ra_spmm.embed(ids, table)
        y, h = ra_spmm.layer_norm(table, residual=x)
        loss, dx = ra_spmm.distill_loss_grad(y.detach(), t, top, 2.0)
        return [loss, dx, rows.detach(), *torch.autograd.grad((rows, y, h), table, (g, dx, x))]

    want = [work(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    rounds = []
    for _ in range(8):
        rounds.append([])
        for s, d in zip(streams, data):
            with torch.cuda.stream(s):
                rounds[-1].append(work(*d))
    torch.cuda.synchronize()
    for i, got in enumerate(rounds):
        for a, b in zip(want, got):
            assert all(torch.equal(u, v) for u, v in zip(a, b)), i
