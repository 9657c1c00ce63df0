"""Activations kept in 8 bits: codes and scales bit for bit against their definition, the ReLU's mask, the weight
gradient against 64 bits.

Tolerance of the weight gradient: every product is exact, so only additions in float32 round.  A result is a sum of at
most 3 * rows products (three pieces of a float32 gradient); an addition is off by at most one unit, 2^-23 of the running
magnitude, whatever its rounding mode: (3 * rows + 8) * 2^-23 of sum |g x|."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def definition(x, relu):
    """(codes int, scale exponent + 127) of x [rows, cols] as numpy float64, in groups of 32 columns."""
    x = x.double().numpy()
    if relu:
        x = np.where(x <= 0, 0.0, x)
    rows, cols = x.shape
    groups = -(-cols // 32)
    codes, scales = np.zeros((rows, groups * 32), np.int64), np.zeros((rows, groups), np.int64)
    for r in range(rows):
        for g in range(groups):
            part = x[r, 32 * g:32 * g + 32]
            if not np.isfinite(part).all():
                scales[r, g] = 255
                if relu:
                    codes[r, 32 * g:32 * g + part.size] = (part > 0) | np.isnan(part)
                continue
            top = np.abs(part).max()
            power = math.frexp(top)[1] - 1 if top > 0 else -1000
            e = max(power - (7 if relu else 6), -126)
            c = np.rint(part / 2.0 ** e)
            c = np.minimum(c, 255) if relu else np.clip(c, -127, 127)
            if relu:
                c = np.where(part > 0, np.maximum(c, 1), c)
            scales[r, g] = e + 127
            codes[r, 32 * g:32 * g + part.size] = c
    return codes, scales


def same_codes(p, x, relu):
    codes, scales = definition(x.cpu(), relu)
    got = p.codes.cpu().numpy()
    got = got.astype(np.int64) if relu else got.view(np.int8).astype(np.int64)
    assert p.scales.shape == (scales.shape[1], -(-x.shape[0] // 8) * 8)
    assert (p.scales.cpu().numpy()[:, :x.shape[0]].T == scales).all()
    assert (got == codes).all()
    bad = np.repeat(scales == 255, 32, axis=1)[:, :x.shape[1]]
    value = codes[:, :x.shape[1]] * np.exp2(np.repeat(scales, 32, axis=1)[:, :x.shape[1]].clip(max=250) - 127.0)
    back = ra_spmm.unpack8(p).cpu().double().numpy()
    assert np.isnan(back[bad]).all() and (back[~bad] == value[~bad]).all()
    for dtype in DTYPES:
        want = torch.from_numpy(np.where(bad, np.nan, value)).float().to(dtype)
        assert torch.equal(ra_spmm.unpack8(p, dtype).cpu().nan_to_num(7.0), want.nan_to_num(7.0)), dtype


def special(rows, cols, dtype, seed):
    """Normal values with ties, zeros, huge and tiny groups."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    x[0::7] *= 1e4
    x[1::7] = (torch.randint(-255, 256, x[1::7].shape, generator=g).float() / 2)  # ties
    x[2::7] = 0
    x[3::7] *= 1e-6
    x[4::7, ::3] = -0.0
    if dtype != torch.float16:
        x[5::7] *= 1e-38
        x[6::7] *= 1e37
    return x.to(dtype)


@pytest.mark.parametrize("cols", [1, 7, 8, 31, 32, 33, 47, 64, 100, 256, 301])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_codes(cols, dtype):
    print(f"[checkpoint8] codes {cols} {dtype}", flush=True)
    x = special(23, cols, dtype, cols)
    same_codes(ra_spmm.pack8(x.cuda()), x, False)
    y, p = ra_spmm.relu_pack8(x.cuda())
    same_codes(p, x, True)
    assert torch.equal(y.cpu(), x.relu())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_extremes(dtype):
    """The type's largest and smallest values, and groups that are not finite."""
    info = torch.finfo(dtype)
    x = torch.randn(8, 96, generator=torch.Generator().manual_seed(1))
    x = x.to(dtype)
    x[0, :32] = info.max
    x[1, 5] = -info.max
    x[2, 33], x[3, 40], x[4, 95], x[5, 0] = math.inf, -math.inf, math.nan, math.nan
    x[6] = info.tiny
    x[7, ::2] = info.smallest_normal / 4
    same_codes(ra_spmm.pack8(x.cuda()), x, False)
    y, p = ra_spmm.relu_pack8(x.cuda())
    same_codes(p, x, True)
    assert torch.equal(y.cpu().nan_to_num(7.0), x.relu().nan_to_num(7.0))


def test_error_of_a_kept_value():
    """Half a step of the group, a whole one at its largest values (and for small positive ones behind a ReLU)."""
    x = torch.randn(1000, 64, generator=torch.Generator().manual_seed(2))
    top = x.view(1000, 2, 32).abs().amax(-1, keepdim=True).expand(-1, -1, 32).reshape(1000, 64)
    err = (ra_spmm.unpack8(ra_spmm.pack8(x.cuda())).cpu() - x).abs()
    assert (err <= top / 64 * 1.0).all() and (err[x.abs() < 0.99 * top] <= top[x.abs() < 0.99 * top] / 128).all()
    y, p = ra_spmm.relu_pack8(x.cuda())
    assert ((ra_spmm.unpack8(p).cpu() - x.relu()).abs() <= top / 128).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("cols", [47, 64])
def test_strided_rows(cols, dtype):
    wide = special(50, cols + 29, dtype, 3).cuda()
    for off in (0, 3, 16):
        x = wide[:, off:off + cols]
        a, b = ra_spmm.pack8(x), ra_spmm.pack8(x.contiguous())
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales[:, :50], b.scales[:, :50])
        y, p = ra_spmm.relu_pack8(x)
        assert torch.equal(y, x.relu())
        assert torch.equal(ra_spmm.relu_grad8(x, p), torch.where(x > 0, x, torch.zeros_like(x)))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_relu_gradient_mask_is_exact(dtype):
    """Positive values far below the group's step keep their gradient."""
    x = torch.randn(300, 100, generator=torch.Generator().manual_seed(4))
    x[:, 0] = 1e4
    x[:, 1] = 1e-7
    x[:, 2] = 0
    x, g = x.to(dtype).cuda(), torch.randn(300, 100).to(dtype).cuda()
    _, p = ra_spmm.relu_pack8(x)
    assert torch.equal(ra_spmm.relu_grad8(g, p), torch.where(x > 0, g, torch.zeros_like(g)))


# rows, out, cols
PRODUCTS = [(1, 1, 1), (5, 3, 7), (32, 64, 64), (33, 65, 33), (127, 47, 256), (1000, 47, 256), (129, 128, 128), (700, 256, 128),
            (64, 300, 300), (5000, 16, 16), (3001, 100, 47), (2000, 256, 256), (1537, 63, 130), (40_000, 47, 96)]


@pytest.mark.parametrize("shape", PRODUCTS, ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_weight_gradient(shape, dtype):
    rows, out, cols = shape
    print(f"[checkpoint8] product {shape} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, cols, generator=gen).to(dtype).cuda()
    g = (torch.randn(rows, out, generator=gen) * 10.0 ** torch.randint(-6, 1, (rows, 1), generator=gen)).to(dtype).cuda()
    for p in (ra_spmm.pack8(x), ra_spmm.relu_pack8(x)[1]):
        kept = ra_spmm.unpack8(p).double()
        got = ra_spmm.weight_grad8(g, p)
        assert got.dtype == torch.float32 and got.shape == (out, cols)
        err = (got.double() - g.double().t() @ kept).abs()
        bound = (3 * rows + 8) * 2.0 ** -23 * (g.double().abs().t() @ kept.abs()) + 1e-37
        assert (err <= bound).all(), float((err / bound).max())
        assert torch.equal(got, ra_spmm.weight_grad8(g, p))


def test_weight_gradient_holds_float32():
    """One row: the products themselves, to float32's last bit."""
    g = torch.randn(1, 70, generator=torch.Generator().manual_seed(1)).cuda()
    p = ra_spmm.pack8(torch.randn(1, 40, generator=torch.Generator().manual_seed(2)).cuda())
    want = (g.double().t() @ ra_spmm.unpack8(p).double())
    err = (ra_spmm.weight_grad8(g, p).double() - want).abs()
    assert (err <= 3 * 2.0 ** -24 * want.abs()).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_weight_gradient_of_strided_rows(dtype):
    p = ra_spmm.pack8(torch.randn(500, 47).cuda())
    wide = torch.randn(500, 131).to(dtype).cuda()
    for off in (0, 1, 2):
        for n in (47, 48):
            g = wide[:, off:off + n]
            assert torch.equal(ra_spmm.weight_grad8(g, p), ra_spmm.weight_grad8(g.contiguous(), p))


def test_groups_that_are_not_finite():
    """NaN reaches the columns of its group and no others."""
    x = torch.randn(200, 96).cuda()
    x[17, 40] = math.nan
    got = ra_spmm.weight_grad8(torch.randn(200, 50).cuda(), ra_spmm.pack8(x))
    assert got[:, 32:64].isnan().all() and got[:, :32].isfinite().all() and got[:, 64:].isfinite().all()


def test_no_rows():
    x = torch.zeros(0, 40, device="cuda")
    y, p = ra_spmm.relu_pack8(x)
    assert y.shape == (0, 40) and p.codes.shape == (0, 64) and ra_spmm.unpack8(p).shape == (0, 40)
    assert ra_spmm.relu_grad8(x, p).shape == (0, 40)
    assert not ra_spmm.weight_grad8(torch.zeros(0, 7, device="cuda"), p).any()


def test_relu_and_linear_layers():
    """relu8 and linear8 against autograd on the kept values: the output from x itself, gradients of the input through
    the exact mask, the weight gradient from what was kept."""
    gen = torch.Generator().manual_seed(5)
    x, w, g = (torch.randn(s, generator=gen) for s in ((400, 100), (47, 100), (400, 47)))
    xd, wd = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    h, kept = ra_spmm.relu8(xd)
    y = ra_spmm.linear8(h, wd, kept)
    y.backward(g.cuda())
    assert torch.equal(h.detach().cpu(), x.relu())
    assert (y.detach().cpu().double() - x.relu().double() @ w.double().t()).abs().max() < 1e-4
    want = (g.double() @ w.double()) * (x > 0)
    assert (xd.grad.cpu().double() - want).abs().max() < 1e-4 and not xd.grad.cpu()[x <= 0].any()
    assert torch.equal(wd.grad, ra_spmm.weight_grad8(g.cuda(), kept))
    w2 = w.cuda().requires_grad_(True)
    ra_spmm.linear8(x.cuda(), w2).backward(g.cuda())
    assert torch.equal(w2.grad, ra_spmm.weight_grad8(g.cuda(), ra_spmm.pack8(x.cuda())))
    off = (w2.grad.cpu().double() - g.double().t() @ x.double()).abs()
    # Each kept value is at most one step, 1/64 of its group's largest, off.
    top = x.abs().max()
    assert (off <= (g.abs().double().sum(0)[:, None] * float(top) / 64)).all()


def test_capture_and_replay():
    x, g = torch.randn(3000, 100).cuda(), torch.randn(3000, 47).cuda()

    def body():
        y, p = ra_spmm.relu_pack8(x)
        s = ra_spmm.pack8(x)
        return y, p.codes, p.scales[:, :3000], s.codes, s.scales[:, :3000], ra_spmm.relu_grad8(x, p), ra_spmm.weight_grad8(g, p), ra_spmm.unpack8(s)

    eager = body()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        body()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = body()
    for _ in range(3):
        junk = torch.randn(1000, 1000, device="cuda") @ torch.randn(1000, 1000, device="cuda")
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))
        del junk


def test_rows_past_32_bit_offsets():
    """Codes and activations whose offsets pass 2^32 elements."""
    rows, cols = 70_000, 65_536
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free memory")
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
    x[-1, -40:] = torch.arange(-20, 20, device="cuda").to(torch.bfloat16)
    x[0, 0] = 3
    y, p = ra_spmm.relu_pack8(x)
    assert torch.equal(y[-1, -40:], x[-1, -40:].relu()) and int(p.codes.count_nonzero()) == 20
    dx = ra_spmm.relu_grad8(x, p)
    assert torch.equal(dx[-1], x[-1].relu()) and float(dx[0, 0]) == 3
    del dx, y, x
    g = torch.ones(rows, 1, device="cuda")
    got = ra_spmm.weight_grad8(g, p)
    assert float(got[0, -1]) == 19 and float(got[0, 0]) == 3 and int(got.count_nonzero()) == 20


@pytest.fixture(scope="module")
def case():
    x = torch.randn(50, 40).cuda()
    return dict(x=x, s=ra_spmm.pack8(x), u=ra_spmm.relu_pack8(x)[1], g=torch.randn(50, 7).cuda())


REFUSED = {
    "x on the host": (lambda c: ra_spmm.pack8(c["x"].cpu()), "CUDA"),
    "x float64": (lambda c: ra_spmm.pack8(c["x"].double()), "float32, float16 or"),
    "x 1-D": (lambda c: ra_spmm.pack8(c["x"][0]), "rows, cols"),
    "x transposed": (lambda c: ra_spmm.relu_pack8(c["x"].t()), "contiguous within"),
    "x without columns": (lambda c: ra_spmm.pack8(c["x"][:, :0]), "rows, cols"),
    "mask of signed codes": (lambda c: ra_spmm.relu_grad8(c["x"], c["s"]), "signed"),
    "gradient of another shape": (lambda c: ra_spmm.relu_grad8(c["x"][:, :39], c["u"]), "packed shape"),
    "gradient of other rows": (lambda c: ra_spmm.weight_grad8(c["g"][:49], c["s"]), "rows"),
    "gradient on the host": (lambda c: ra_spmm.weight_grad8(c["g"].cpu(), c["s"]), "CUDA"),
    "gradient float64": (lambda c: ra_spmm.weight_grad8(c["g"].double(), c["s"]), "float32, float16 or"),
    "codes of another width": (lambda c: ra_spmm.unpack8(c["s"]._replace(cols=70)), "codes"),
    "scales of another shape": (lambda c: ra_spmm.unpack8(c["s"]._replace(scales=c["s"].scales[:, :8].contiguous())), "scales"),
    "unpacked as float64": (lambda c: ra_spmm.unpack8(c["s"], torch.float64), "float32, float16 or"),
    "linear8 with another input's codes": (lambda c: ra_spmm.linear8(c["x"][:49], torch.randn(3, 40).cuda(), c["s"]), "packed"),
}


@pytest.mark.parametrize("name", list(REFUSED))
def test_refusals(case, name):
    fn, match = REFUSED[name]
    with pytest.raises(RuntimeError, match=match):
        fn(case)
    torch.cuda.synchronize()
    assert torch.equal(ra_spmm.pack8(case["x"]).codes, case["s"].codes)
