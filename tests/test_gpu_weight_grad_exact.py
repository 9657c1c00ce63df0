"""weight_grad8 on whole numbers: every product and every partial sum is exact in float32 (below 2^24), so the result has
to be the float64 product, bit for bit, whatever the order.  A row left out or counted twice, a lost piece of a gradient
or a shifted scale shows."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
BIT = {torch.float32: (1 << 16) + (1 << 8) + 1, torch.float16: (1 << 10) + 1, torch.bfloat16: (1 << 7) + 1}


def kept(rows, cols, signed, gen, largest):
    """Whole numbers up to `largest` (a power of two, and in every group, so that a row's scale is known), halved in every
    second row: kept without rounding."""
    x = torch.randint(-largest + 1, largest, (rows, cols), generator=gen).float()
    x[:, ::32] = largest
    x[1::2] /= 2
    x = x.cuda()
    p = ra_spmm.pack8(x) if signed else ra_spmm.relu_pack8(x)[1]
    want = x if signed else x.relu()
    assert torch.equal(ra_spmm.unpack8(p), want)
    return p, want.double()


def gradients(rows, out, dtype, gen, long):
    """+-1 and +-2 in every row, or (long) ones of every significant bit of the type in three rows of a column: one of the
    first, one of the last, one between."""
    if not long:
        g = torch.randint(1, 3, (rows, out), generator=gen) * (1 - 2 * torch.randint(0, 2, (rows, out), generator=gen))
        return g.to(dtype).cuda()
    g = torch.zeros(rows, out)
    for o in range(out):
        for r in (o % rows, rows - 1 - o % min(rows, 33), int(torch.randint(0, rows, (1,), generator=gen))):
            g[r, o] = BIT[dtype]
    return g.to(dtype).cuda()


def check(rows, out, cols, dtype, signed, seed):
    gen = torch.Generator().manual_seed(seed)
    for long in (False, True):
        largest = 16 if long else 64
        # In steps of a half: the most that a sum can be.
        assert 2 * largest * (3 * BIT[dtype] if long else 2 * rows) < 2 ** 24
        p, x = kept(rows, cols, signed, gen, largest)
        g = gradients(rows, out, dtype, gen, long)
        assert torch.equal(ra_spmm.weight_grad8(g, p).double(), g.double().t() @ x), (rows, out, cols, dtype, signed, long)


# Around the ends of a stage of 32 rows and of a split of 128.
ROWS = [1, 7, 31, 32, 33, 63, 64, 65, 127, 128, 129, 159, 160, 161, 255, 256, 257, 1023, 1055, 1056, 1057]
# One, two and four waves both ways, odd widths, several tiles.
SIZES = [(1, 1), (47, 96), (64, 64), (63, 300), (65, 33), (128, 128), (130, 47), (129, 200), (256, 256), (300, 130), (200, 520)]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_around_stages_and_splits(size, dtype):
    print(f"[weight_grad8] {size} {dtype}", flush=True)
    for n, rows in enumerate(ROWS):
        check(rows, *size, dtype, n % 2 == 0, rows)


@pytest.mark.parametrize("rows,out,cols", [(40_001, 256, 256), (40_031, 47, 96), (33_000, 130, 300), (50_000, 64, 64)])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_many_splits(rows, out, cols, dtype):
    print(f"[weight_grad8] {rows} {out} {cols} {dtype}", flush=True)
    check(rows, out, cols, dtype, False, 1)
    check(rows, out, cols, dtype, True, 2)
