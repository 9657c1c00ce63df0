"""Layer norm, alone and of a sum, and its gradients against their definition in 64 bits.

Tolerances, u = 2^-24, for rows of D elements.  The mean is off by (D + 1) u mean|h| (dm); h - mean by dm and u of itself; the
variance by 2 dm mean|h - mean| and (D + 6) u of itself; its inverse root by half of that relative to variance + eps and 4 u;
n, y and the gradients follow term by term (`exact`).  Sums over the rows add rows * u of their magnitudes.  16-bit results
add half a unit of their last place (2^-11, 2^-8), or half the smallest fp16 step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402

U = 2.0 ** -24
HALF_UNIT = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def close(got, want, err, what):
    unit = HALF_UNIT[got.dtype]
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    bound = err + unit * (want.abs() + err) + (2.0 ** -25 if unit == 2.0 ** -11 else 1e-30)
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} beyond; first {bad.nonzero()[0].tolist()}, worst "
                           f"{float(((got - want).abs() / bound).nan_to_num(math.inf).max()):.3g} bounds")


def exact(h, w, b, eps, gy=None, gh=None):
    """{name: (value, error bound before the final rounding)}; h as it is kept."""
    h = h.double()
    M, D = h.shape
    w = torch.ones(D, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(D, dtype=torch.float64) if b is None else b.double()
    mean = h.mean(1, keepdim=True)
    dm = (D + 1) * U * h.abs().mean(1, keepdim=True)
    c = h - mean
    var = c.square().mean(1, keepdim=True)
    dv = 2 * dm * c.abs().mean(1, keepdim=True) + dm * dm + (D + 6) * U * var
    r = (var + eps).rsqrt()
    rr = dv / (2 * (var + eps)) + 4 * U
    n = c * r
    dn = r * (dm + U * c.abs()) + n.abs() * (rr + U)
    out = {"y": (n * w + b, w.abs() * dn + 2 * U * ((n * w).abs() + b.abs()))}
    if gy is None:
        return out
    g = gy.double()
    wg = w * g
    s, t = wg.mean(1, keepdim=True), (wg * n).mean(1, keepdim=True)
    ds = (D + 2) * U * wg.abs().mean(1, keepdim=True)
    dt = (D + 3) * U * (wg * n).abs().mean(1, keepdim=True) + (wg.abs() * dn).mean(1, keepdim=True)
    dx = r * (wg - s - n * t)
    err = dx.abs() * rr + r * (U * wg.abs() + ds + dn * t.abs() + n.abs() * dt + 4 * U * (wg.abs() + s.abs() + (n * t).abs()))
    if gh is not None:
        dx = dx + gh.double()
        err = err + U * (dx.abs() + gh.double().abs())
    out["dx"] = (dx, err)
    out["dw"] = ((g * n).sum(0), (g.abs() * dn).sum(0) + (M + 3) * U * (g * n).abs().sum(0))
    out["db"] = (g.sum(0), (M + 1) * U * g.abs().sum(0))
    return out


def make(M, D, dtype, seed=1, shift=0.3):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return ((1.5 * r(M, D) + shift).to(dtype), r(M, D).to(dtype), 1 + 0.3 * r(D), 0.3 * r(D), r(M, D).to(dtype), r(M, D).to(dtype))


def strided(t, extra):
    wide = torch.zeros(t.shape[0], t.shape[1] + extra, dtype=t.dtype, device="cuda")
    wide[:, :t.shape[1]] = t.cuda()
    return wide[:, :t.shape[1]]


def check(M, D, dtype, residual=False, affine="wb", eps=1e-5, extra=0, shift=0.3):
    x, r, w, b, gy, gh = make(M, D, dtype, shift=shift)
    put = (lambda t: strided(t, extra)) if extra else (lambda t: t.cuda())  # noqa: E731
    xd, rd = put(x).detach().requires_grad_(True), put(r).detach().requires_grad_(True)
    wd = w.cuda().requires_grad_(True) if "w" in affine else None
    bd = b.cuda().requires_grad_(True) if "b" in affine else None
    out = ra_spmm.layer_norm(xd, wd, bd, eps=eps, residual=rd if residual else None)
    with torch.no_grad():
        plain = ra_spmm.layer_norm(xd, wd, bd, eps=eps, residual=rd if residual else None)
    leaves = [t for t in (xd, rd if residual else None, wd, bd) if t is not None]
    outs, gs = ((out,), (gy.cuda(),)) if not residual else (out, (gy.cuda(), gh.cuda()))
    assert all(torch.equal(a, c) for a, c in zip(outs, (plain,) if not residual else plain))
    grads = torch.autograd.grad(outs, leaves, gs, retain_graph=True)
    assert all(torch.equal(a, c) for a, c in zip(grads, torch.autograd.grad(outs, leaves, gs))), "the gradients' bits"
    h = x
    if residual:
        h = (x.float() + r.float()).to(dtype)
        assert torch.equal(outs[1].detach().cpu(), h)
    want = exact(h, w if wd is not None else None, b if bd is not None else None, eps, gy, gh if residual else None)
    close(outs[0], *want["y"], "y")
    names = ["dx"] + ["dx"] * residual + ["dw"] * (wd is not None) + ["db"] * (bd is not None)
    for name, g in zip(names, grads):
        close(g, *want[name], name)


WIDTHS = [1, 2, 3, 7, 8, 16, 20, 31, 33, 47, 64, 65, 100, 128, 147, 256, 257, 300, 512, 513, 520, 1000, 1001, 1024, 1025, 1032, 2048, 2049, 4096,
          4097, 4104, 8192, 8193, 8200, 16383, 16384]


@pytest.mark.parametrize("residual", [False, True], ids=["alone", "sum"])
@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_widths_and_types(D, dtype, residual):
    print(f"[layer_norm] {D} {dtype} {residual}", flush=True)
    check(11, D, dtype, residual)


@pytest.mark.parametrize("M", [1, 2, 3, 5, 64, 4097, 20_011])
@pytest.mark.parametrize("D", [16, 100, 147, 256, 1030])
def test_rows(M, D):
    print(f"[layer_norm] {M} x {D}", flush=True)
    check(M, D, torch.bfloat16, True)
    check(M, D, torch.float32)


@pytest.mark.parametrize("affine", ["", "w", "b", "wb"])
def test_without_weight_or_bias(affine):
    check(33, 72, torch.float32, affine=affine)
    check(33, 2000, torch.float16, True, affine=affine)


@pytest.mark.parametrize("extra", [1, 2, 4, 8])
@pytest.mark.parametrize("D", [16, 37, 256, 1032, 5000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_strided_rows(D, extra, dtype):
    check(21, D, dtype, True, extra=extra)


@pytest.mark.parametrize("D", [64, 1024, 6000])
def test_a_mean_far_from_zero(D):
    """The variance is taken around the mean: with squares of h itself nothing would be left of it."""
    check(9, D, torch.float32, shift=3000.0)


def test_rows_of_one_value():
    """No variance: n is 0 and r is 1 / sqrt(eps)."""
    x = torch.full((4, 96), 5.0, device="cuda", requires_grad=True)
    b = torch.randn(96, device="cuda")
    y = ra_spmm.layer_norm(x, torch.ones(96, device="cuda"), b, eps=1e-4)
    assert torch.equal(y, b.expand(4, 96))
    g, = torch.autograd.grad(y, x, torch.ones(4, 96, device="cuda"))
    assert (g.abs() < 1e-3).all()


def test_axes_and_dtype_of_leading_axes():
    x = torch.randn(3, 5, 48, device="cuda", requires_grad=True)
    w, b = torch.rand(48, device="cuda"), torch.rand(48, device="cuda")
    flat = ra_spmm.layer_norm(x.reshape(15, 48), w, b)
    assert torch.equal(ra_spmm.layer_norm(x, w, b), flat.view(3, 5, 48))
    y, h = ra_spmm.layer_norm(x, w, b, residual=x.transpose(0, 1).reshape(3, 5, 48))
    assert y.shape == h.shape == (3, 5, 48)
    one = ra_spmm.layer_norm(x[0, 0], w, b)
    assert one.shape == (48,) and torch.equal(one, flat[0])
    g = torch.randn(3, 5, 48, device="cuda")
    a, = torch.autograd.grad(ra_spmm.layer_norm(x, w, b), x, g)
    c, = torch.autograd.grad(flat, x, g.view(15, 48))
    assert torch.equal(a, c)


def test_gradients_that_are_not_there():
    """Either output alone; inputs without gradients; one tensor as x and as residual."""
    x, r, w, b, gy, gh = (t.cuda() for t in make(40, 64, torch.float32))
    x.requires_grad_(True)
    w.requires_grad_(True)
    y, h = ra_spmm.layer_norm(x, w, b, residual=r)
    dx, dw = torch.autograd.grad(h, (x, w), gh, retain_graph=True, allow_unused=True)
    assert torch.equal(dx, gh) and (dw is None or not dw.any())
    dx, dw = torch.autograd.grad(y, (x, w), gy)
    want = exact(h.detach().cpu(), w.detach().cpu(), b.cpu(), 1e-5, gy.cpu())
    close(dx, *want["dx"], "dx")
    close(dw, *want["dw"], "dw")
    only = b.clone().requires_grad_(True)
    db, = torch.autograd.grad(ra_spmm.layer_norm(x.detach(), None, only), only, gy)
    close(db, *want["db"], "db")
    y, h = ra_spmm.layer_norm(x, w, b, residual=x)
    dx, = torch.autograd.grad((y, h), x, (gy, gh))
    both = exact(h.detach().cpu(), w.detach().cpu(), b.cpu(), 1e-5, gy.cpu(), gh.cpu())["dx"]
    close(dx, 2 * both[0], 2 * both[1] + U * 2 * both[0].abs(), "x twice")


def test_gradients_against_differences():
    """Along a random direction, differences of the 64-bit definition with steps of 1e-4: their own error is of second order,
    1e-8 of third derivatives of order 1 a row."""
    M, D = 7, 50
    x, r, w, b, gy, gh = make(M, D, torch.float32, seed=4)
    gen = torch.Generator().manual_seed(9)
    vx, vr, vw, vb = (torch.randn(s, generator=gen, dtype=torch.float64) for s in ((M, D), (M, D), (D,), (D,)))

    def value(t):
        h = x.double() + r.double() + t * (vx + vr)
        c = h - h.mean(1, keepdim=True)
        n = c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt()
        return ((n * (w.double() + t * vw) + b.double() + t * vb) * gy.double()).sum() + (h * gh.double()).sum()

    want = float(value(1e-4) - value(-1e-4)) / 2e-4
    leaves = [t.cuda().requires_grad_(True) for t in (x, r, w, b)]
    out = ra_spmm.layer_norm(leaves[0], leaves[2], leaves[3], residual=leaves[1])
    grads = torch.autograd.grad(out, leaves, (gy.cuda(), gh.cuda()))
    got = sum(float((g.cpu().double() * v).sum()) for g, v in zip(grads, (vx, vr, vw, vb)))
    size = sum(float((g.cpu().double() * v).abs().sum()) for g, v in zip(grads, (vx, vr, vw, vb)))
    assert abs(got - want) <= 1e-5 * M + 200 * U * size


def test_values_that_are_not_finite_stay_in_their_rows():
    x = torch.randn(6, 40, device="cuda")
    x[1, 3], x[4, 0] = math.inf, math.nan
    y = ra_spmm.layer_norm(x, torch.ones(40, device="cuda"), None)
    assert y[[0, 2, 3, 5]].isfinite().all() and y[1].isnan().any() and y[4].isnan().all()


def test_empty():
    w = torch.ones(24, device="cuda", requires_grad=True)
    b = torch.ones(24, device="cuda", requires_grad=True)
    x = torch.zeros(0, 24, device="cuda", requires_grad=True)
    y, h = ra_spmm.layer_norm(x, w, b, residual=x)
    dx, dw, db = torch.autograd.grad((y, h), (x, w, b), (torch.zeros(0, 24, device="cuda"),) * 2)
    assert y.shape == h.shape == dx.shape == (0, 24) and not dw.any() and not db.any()


def test_offsets_past_32_bits():
    M, D = 150_000, 16_384
    x = torch.zeros(M, D, dtype=torch.bfloat16, device="cuda")
    x[:, ::2] = 2.0
    x[-1, ::2] = 4.0
    y, h = ra_spmm.layer_norm(x, residual=x, eps=0.0)
    assert h[-1, 0] == 8.0 and y[-1, 0] == 1.0 and y[-1, 1] == -1.0 and y[M // 2, 2] == 1.0
    del h
    g = x.zero_()
    g[-1, 5] = 1.0
    dx, dw, db = ra_spmm._C.run_layer_norm_backward(y, None, torch.tensor([[0.0, 1.0]], device="cuda").expand(M, 2).contiguous(),
                                                    g, None, True, True)
    assert db[5] == 1.0 and db.sum() == 1.0 and dw[5] == -1.0 and not dx[:-1].any()
    assert abs(float(dx[-1, 5]) - (1 - 2 / D)) <= 2.0 ** -8  # 1 - 1/D - n^2/D


def test_on_another_stream():
    x, r, w, b, gy, gh = (t.cuda() for t in make(3000, 200, torch.float16))
    for t in (x, r, w, b):
        t.requires_grad_(True)
    want = torch.autograd.grad(ra_spmm.layer_norm(x, w, b, residual=r), (x, r, w, b), (gy, gh))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = torch.autograd.grad(ra_spmm.layer_norm(x, w, b, residual=r), (x, r, w, b), (gy, gh))
    s.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))


@pytest.mark.parametrize("size", [(1, 256), (700, 64), (2000, 147), (50, 5000)], ids=str)
def test_capture_and_replay(size):
    data = [t.cuda() for t in make(*size, torch.bfloat16)]

    def body():
        x, r, w, b = (t.detach().requires_grad_(True) for t in data[:4])
        out = ra_spmm.layer_norm(x, w, b, residual=r)
        return [o.detach() for o in out] + list(torch.autograd.grad(out, (x, r, w, b), data[4:]))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        body()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = body()
    for i in range(4):
        for t in data:
            t.normal_()
        for o in outs:
            o.fill_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        assert all(torch.equal(a, c) for a, c in zip(got, body())), i


def test_refusals():
    x, w = torch.zeros(4, 8, device="cuda"), torch.ones(8, device="cuda")
    for args, kw, match in (((x.cpu(), w), {}, "CUDA"), ((x, w.cpu()), {}, "CUDA"), ((x, w.half()), {}, "float32"), ((x, w[:7]), {}, "shape"),
                            ((x.double(), w), {}, "float32, float16"), ((x, w), {"residual": x.half()}, "dtype"),
                            ((x, w), {"residual": x[:3]}, "shape"), ((torch.zeros(2, 16385, device="cuda"),), {}, "16384"),
                            ((x, w, w[:3]), {}, "shape"), ((x[:, :0],), {}, "no columns"), ((x[0, 0], w), {}, "axis")):
        with pytest.raises(RuntimeError, match=match):
            ra_spmm.layer_norm(*args, **kw)
    with pytest.raises(RuntimeError, match="stats"):
        ra_spmm._C.run_layer_norm_backward(x, w, torch.zeros(3, 2, device="cuda"), x, None, True, True)
