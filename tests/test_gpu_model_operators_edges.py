"""Calls of embedding lookup, layer norm and distillation that a program may make beside the ordinary ones: tensors at odd
addresses, two streams at once, long lists of entries with the same classes, one wide row."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402
from test_gpu_distill import check as check_distill  # noqa: E402
from test_gpu_distill import close  # noqa: E402
from test_gpu_distill import exact as exact_distill  # noqa: E402
from test_gpu_distill import make as make_distill  # noqa: E402

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def odd(t, by):
    """t's values `by` elements past the beginning of an allocation."""
    wide = torch.zeros(t.numel() + by + 3, dtype=t.dtype, device=t.device)
    out = wide[by:by + t.numel()].view(t.shape)
    out.copy_(t)
    return out


@pytest.mark.parametrize("by", [1, 2, 4])
@pytest.mark.parametrize("D", [5, 16, 47, 256, 1100])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_addresses_do_not_change_the_bits(D, dtype, by):
    gen = torch.Generator("cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    x, res, gy, gh = r(37, D), r(37, D), r(37, D), r(37, D)
    w, b = r(D).float(), r(D).float()
    ids = torch.randint(-1, 37, (300,), generator=gen, device="cuda")
    g = r(300, D)
    results = []
    for put in (lambda t: t.clone(), lambda t: odd(t, by)):
        leaves = [put(t).detach().requires_grad_(True) for t in (x, res, w, b)]
        out = ra_spmm.layer_norm(leaves[0], leaves[2], leaves[3], residual=leaves[1])
        grads = torch.autograd.grad(out, leaves, (put(gy), put(gh)))
        table = put(x).detach().requires_grad_(True)
        rows = ra_spmm.embed(put(ids), table, 1.5, padding=-1)
        results.append([t.detach() for t in (*out, *grads, rows, *torch.autograd.grad(rows, table, put(g)))])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("by", [1, 2, 4])
@pytest.mark.parametrize("C", [7, 47, 300, 1500, 20_000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_logits_at_odd_addresses(C, dtype, by):
    x, t, ids, labels = make_distill(9, C, 5, dtype)
    check_distill(x, t, ids, labels, T=2.0, hard=0.3, put=lambda v: odd(v.cuda(), by))


@pytest.mark.parametrize("C", [33, 64, 65, 80, 81, 104, 105, 128, 129, 160, 208, 209, 256, 257, 320, 321, 416, 417, 512, 513, 640,
                               641, 832, 833, 1024])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_lengths_of_many_rows(C, dtype):
    """Row lengths at which the lanes of a row and the classes of a lane change, with rows enough for as few lanes as there
    can be; the first, middle and last rows against the definition."""
    M = 2 ** 20 // C + 77
    x, t, ids, labels = make_distill(M, C, 20, dtype, seed=C)
    some = torch.cat([torch.arange(20), torch.arange(M // 2, M // 2 + 8), torch.arange(M - 12, M)])
    x[3, C - 1], x[5] = math.nan, -math.inf
    ids[7], labels[7], x[7, 0] = -1, -1, math.nan
    up = torch.randn(M, generator=torch.Generator().manual_seed(5))
    for hard in (0.0, 0.4):
        want, werr, grad, gerr = exact_distill(x[some], t[some], ids[some], 2.0, labels[some], hard, up[some].double())
        leaf = x.cuda().requires_grad_(True)
        loss = ra_spmm.distill_loss(leaf, t.cuda(), ids.cuda(), 2.0, labels.cuda(), hard, "none")
        g, = torch.autograd.grad(loss, leaf, up.cuda())
        close(loss[some.cuda()], want, werr, "loss of the rows")
        close(g[some.cuda()], grad, gerr, "gradient of the rows")


@pytest.mark.parametrize("k", [17, 256, 300, 1024])
@pytest.mark.parametrize("C", [1, 5, 700, 3000])
def test_many_entries_of_few_classes(C, k):
    """Every class several times, some entries missing."""
    gen = torch.Generator().manual_seed(k)
    x, t = torch.randn(5, C, generator=gen), torch.randn(5, k, generator=gen)
    ids = torch.randint(-2, C, (5, k), generator=gen)
    check_distill(x, t, ids, torch.randint(-1, C, (5,), generator=gen), T=2.0, hard=0.4)


def test_two_streams_at_once():
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
    got = []
    for _ in range(5):
        got = []
        for s, d in zip(streams, data):
            with torch.cuda.stream(s):
                got.append(work(*d))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_one_wide_row(dtype):
    """n of a row of +-1 is the row, its gradient g - mean(g) - n mean(g n)."""
    D = 16_384
    x = torch.ones(1, D, device="cuda", dtype=dtype)
    x[0, ::2] = -1
    x.requires_grad_(True)
    y = ra_spmm.layer_norm(x, eps=0.0)
    assert torch.equal(y, x)
    g = torch.zeros(1, D, device="cuda", dtype=dtype)
    g[0, 3] = 1
    dx, = torch.autograd.grad(y, x, g)
    assert float(dx[0, 3]) == pytest.approx(1 - 2 / D, rel=2.0 ** -8) and abs(float(dx[0, 2])) < 2.0 ** -20
    assert float(dx[0, 5]) == pytest.approx(-2 / D, rel=2.0 ** -7)


def test_a_table_of_one_row_and_one_position():
    table = torch.randn(1, 1, device="cuda", requires_grad=True)
    out = ra_spmm.embed(torch.zeros(1, dtype=torch.int32, device="cuda"), table, -2.0)
    assert float(out) == -2.0 * float(table)
    assert float(torch.autograd.grad(out, table, torch.full((1, 1), 3.0, device="cuda"))[0]) == -6.0


def test_a_gradient_that_is_scaled_before_it_is_rounded():
    """A mean over many rows in fp16: with a loss scale all bits are there; without one 1 / (70,000 * 40) = 5.99 * 2^-24 is 6 of the
    smallest steps, of which fp16 has no part."""
    M, C = 70_000, 40
    x = torch.zeros(M, C, device="cuda", dtype=torch.float16)
    t, ids = torch.ones(M, 1, device="cuda"), torch.zeros(M, 1, dtype=torch.int64, device="cuda")
    for factor in (65536.0, torch.tensor(65536.0, device="cuda")):
        _, g = ra_spmm.distill_loss_grad(x, t, ids, factor=factor)
        assert math.isclose(float(g[5, 3]), 65536 / (M * C), rel_tol=2.0 ** -9)
    leaf = x.requires_grad_(True)
    (65536.0 * ra_spmm.distill_loss(leaf, t, ids)).backward()
    assert torch.equal(leaf.grad, g)
    assert (ra_spmm.distill_loss_grad(x.detach(), t, ids)[1][:, 1:] == 6 * 2.0 ** -24).all()


def test_an_incoming_gradient_that_has_to_be_copied():
    """The copy must not be given to the gradient that is written from it."""
    M, C = 20_000, 12
    gen = torch.Generator("cuda").manual_seed(2)
    x, up = torch.randn(M, C, generator=gen, device="cuda"), torch.randn(2, M // 2, generator=gen, device="cuda").t()
    t, ids = torch.randn(M, C, generator=gen, device="cuda").topk(3, dim=1)
    _, stats, _ = ra_spmm._C.run_distill(x, t, ids, 2.0, None, 0.0, "none", True, False, None)
    back = lambda g: ra_spmm._C.run_distill_backward(x, t, ids, 2.0, None, 0.0, "none", stats, g)  # noqa: E731
    want = back(up.reshape(-1))
    assert not up.is_contiguous()
    for _ in range(5):
        assert torch.equal(back(up), want)


@pytest.mark.parametrize("scale", [math.inf, -math.inf, math.nan, -2.0, 0.0])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_padding_is_zero_whatever_the_scale_is(dtype, scale):
    """Positive zeros, as of a tensor of zeros; rows and ids outside keep their values."""
    table = torch.ones(5, 11, device="cuda", dtype=dtype).requires_grad_(True)
    out = ra_spmm.embed(torch.tensor([3, -1, 7, 2], device="cuda"), table, scale, padding=-1)
    assert not out[1].any() and not out[1].signbit().any() and out[2].isnan().all()
    assert torch.equal(out[0], torch.full_like(out[0], scale)) or math.isnan(scale) and out[0].isnan().all()
    grad, = torch.autograd.grad(out, table, torch.ones_like(out))
    assert not grad[[0, 1, 4]].any() and torch.equal(grad[2].isnan(), out[0].isnan())
