"""Head norms with rotation against their definition in 64 bits.

Tolerances.  The sum of head_dim squares is positive, so r is within (head_dim / 2 + 4) * eps of itself (eps = 2^-24);
products, the rotation's two terms and the weight add a few eps of their magnitudes: (head_dim + 16) * eps of |x r w c| +
|y r w s|.  dx has a second sum of head_dim terms, (2 head_dim + 32) * eps of its magnitudes; the weights' gradients sum
rows * heads terms.  16-bit results add half a unit of their last place (2^-11, 2^-8)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402

EPS = 2.0 ** -24
HALF_UNIT = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def close(got, want, mag, rel, what):
    got, unit = got.detach().cpu(), HALF_UNIT[got.dtype]
    bound = rel * mag + unit * (want.abs() + rel * mag) + (2.0 ** -25 if got.dtype == torch.float16 else 1e-30)
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} beyond; worst {float((err / bound.clamp(min=1e-300)).max()):.3g} bounds"


def matrix(table, pos, D, layout):
    """The rotation of every row as a [rows, D, D] matrix."""
    t = table.double()[pos.long()]
    half = t.shape[1]
    R = torch.eye(D, dtype=torch.float64).repeat(pos.numel(), 1, 1)
    for i in range(half):
        a, b = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
        c, s = t[:, i, 0], t[:, i, 1]
        R[:, a, a], R[:, a, b], R[:, b, a], R[:, b, b] = c, -s, s, c
    return R


def exact(x, w, R, eps, g=None):
    """(y, |y|'s terms) and (dx, its terms, dw, its terms)."""
    x, w = x.double(), w.double()
    D = x.shape[-1]
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x * r
    turn = lambda m, v: (m[:, None] @ v[..., None])[..., 0]  # noqa: E731
    y, ym = turn(R, n * w), turn(R.abs(), (n * w).abs())
    if g is None:
        return y, ym
    gt, gm = turn(R.transpose(1, 2), g.double()), turn(R.abs().transpose(1, 2), g.double().abs())
    dx = r * (w * gt - n * (w * gt * n).mean(-1, keepdim=True))
    dxm = r * (w.abs() * gm + n.abs() * (w.abs() * gm * n.abs()).mean(-1, keepdim=True))
    return y, ym, dx, dxm, (gt * n).sum((0, 1)), (gm * n.abs()).sum((0, 1))


def make(rows, hq, hk, D, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return (r(rows, hq, D).to(dtype), r(rows, hk, D).to(dtype), 1 + 0.3 * r(D), 1 + 0.3 * r(D),
            r(rows, hq, D).to(dtype), r(rows, hk, D).to(dtype))


def check(rows, hq, hk, D, rot, layout, dtype, positions=64, eps=1e-6, strided=False, own_positions=True):
    q, k, wq, wk, gq, gk = make(rows, hq, hk, D, dtype)
    table = ra_spmm.rotation_table(positions, rot)
    pos = torch.arange(rows, dtype=torch.int32) * 7 % positions if own_positions else torch.arange(rows, dtype=torch.int32)
    if strided:  # the columns of one projection
        x = torch.cat([q.flatten(1), k.flatten(1), q.flatten(1)[:, :3]], 1).cuda()
        qd, kd = x[:, :hq * D].unflatten(1, (hq, D)), x[:, hq * D:(hq + hk) * D].unflatten(1, (hk, D))
    else:
        qd, kd = q.cuda(), k.cuda()
    leaves = [t.detach().requires_grad_(True) for t in (qd, kd, wq.cuda(), wk.cuda())]
    args = (table.cuda(), pos.cuda() if own_positions else None)
    yq, yk = ra_spmm.head_norm_rotate(*leaves, *args, eps=eps, layout=layout)
    grads = torch.autograd.grad((yq, yk), leaves, (gq.cuda(), gk.cuda()))
    with torch.no_grad():
        iq, ik = ra_spmm.head_norm_rotate(*leaves, *args, eps=eps, layout=layout)
    assert torch.equal(iq, yq) and torch.equal(ik, yk)
    R = matrix(table, pos, D, layout)
    for x, w, g, y, dx, dw, name in ((q, wq, gq, yq, grads[0], grads[2], "q"), (k, wk, gk, yk, grads[1], grads[3], "k")):
        ye, ym, dxe, dxm, dwe, dwm = exact(x, w, R, eps, g)
        close(y, ye, ym, (D + 16) * EPS, name)
        close(dx, dxe, dxm, (2 * D + 32) * EPS, "d" + name)
        close(dw, dwe, dwm, (D + 32 + x.shape[0] * x.shape[1]) * EPS, "dw" + name)


# head_dim, rotated part
DIMS = [(16, 16), (32, 16), (64, 64), (128, 64), (256, 256), (20, 12), (20, 20), (24, 24), (7, 4), (1, 0), (2, 2), (33, 10),
        (255, 254), (8, 0), (100, 50), (48, 24)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dims", DIMS, ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_dims_layouts_types(dims, layout, dtype):
    print(f"[head_norm] {dims} {layout} {dtype}", flush=True)
    check(37, 5, 2, *dims, layout, dtype)


@pytest.mark.parametrize("rows", [1, 2, 4097])
@pytest.mark.parametrize("heads", [(1, 1), (16, 16), (12, 4), (1, 31)], ids=str)
def test_rows_and_heads(rows, heads):
    print(f"[head_norm] {rows} rows {heads}", flush=True)
    check(rows, *heads, 16, 16, "half", torch.bfloat16)
    check(rows, *heads, 16, 8, "interleaved", torch.float32)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("D", [16, 20])
def test_strided_rows(D, dtype):
    """Columns of one projection, at a row pitch that fits no packet."""
    check(50, 4, 3, D, D // 2, "half", dtype, strided=True)


def test_row_numbers_as_positions():
    check(50, 4, 3, 16, 16, "half", torch.float32, own_positions=False)


def test_middle_dimensions_and_absent_keys():
    """[rows, heads, 2, head_dim] as the attention takes it; one tensor alone; no rotation."""
    q, k, wq, wk, _, _ = (t.cuda() for t in make(30, 8, 6, 16, torch.float32))
    table, pos = ra_spmm.rotation_table(30, 16, device="cuda"), torch.arange(30, dtype=torch.int32, device="cuda")
    both = ra_spmm.head_norm_rotate(q, k, wq, wk, table, pos)
    four = ra_spmm.head_norm_rotate(q.view(30, 4, 2, 16), k.view(30, 3, 2, 16), wq, wk, table, pos)
    alone = ra_spmm.head_norm_rotate(q, None, wq, None, table, pos)
    assert torch.equal(four[0].flatten(1), both[0].flatten(1)) and torch.equal(four[1].flatten(1), both[1].flatten(1))
    assert torch.equal(alone[0], both[0]) and alone[1] is None
    plain, _ = ra_spmm.head_norm_rotate(q, None, wq, None)
    ye, ym = exact(q.cpu(), wq.cpu(), torch.eye(16, dtype=torch.float64).repeat(30, 1, 1), 1e-6)
    close(plain, ye, ym, 32 * EPS, "no rotation")
    x = q.clone().requires_grad_(True)
    ra_spmm.head_norm_rotate(x, None, wq, None, table, pos)[0].sum().backward()
    y = q.clone().requires_grad_(True)
    ra_spmm.head_norm_rotate(y, k, wq, wk, table, pos)[0].sum().backward()  # k's output unused
    assert torch.equal(x.grad, y.grad)


def test_positions_outside_of_the_table():
    q, k, wq, wk, _, _ = (t.cuda() for t in make(6, 2, 2, 16, torch.float32))
    table = ra_spmm.rotation_table(10, 8, device="cuda")
    pos = torch.tensor([0, -1, 9, 10, 2 ** 31 - 1, 3], dtype=torch.int32, device="cuda")
    y, _ = ra_spmm.head_norm_rotate(q, k, wq, wk, table, pos)
    bad = torch.tensor([False, True, False, True, True, False], device="cuda")
    assert y[bad][..., :8].isnan().all() and y[~bad].isfinite().all() and y[bad][..., 8:].isfinite().all()


def test_zeros_and_large_values():
    """A head of zeros stays zero (eps), and its gradient is w g / sqrt(eps); squares of large values do not overflow
    below 2^63 in float32."""
    q = torch.zeros(2, 1, 16, device="cuda")
    q[1] = 2.0 ** 60
    q.requires_grad_(True)
    w = torch.full((16,), 2.0, device="cuda")
    y, _ = ra_spmm.head_norm_rotate(q, None, w, None, eps=1e-4)
    y.sum().backward()
    assert not y[0].any() and torch.allclose(y[1], torch.full_like(y[1], 2.0), rtol=1e-6)
    assert torch.allclose(q.grad[0], torch.full_like(q.grad[0], 200.0), rtol=1e-6)


def test_table():
    t = ra_spmm.rotation_table(1000, 64, base=500.0, scaling=4.0)
    p, i = torch.arange(1000, dtype=torch.float64)[:, None], torch.arange(32, dtype=torch.float64)
    angle = p / 4 * 500.0 ** (-i / 32)
    assert t.shape == (1000, 32, 2) and t.dtype == torch.float32
    assert (t[..., 0].double() - angle.cos()).abs().max() < 2.0 ** -24 + 1e-10
    assert (t[..., 1].double() - angle.sin()).abs().max() < 2.0 ** -24 + 1e-10


def test_gradients_against_differences():
    q, k, wq, wk, gq, gk = make(9, 3, 2, 12, torch.float32)
    table, pos = ra_spmm.rotation_table(64, 8), torch.arange(9, dtype=torch.int32) * 5
    R = matrix(table, pos, 12, "interleaved")
    leaves = [t.cuda().requires_grad_(True) for t in (q, wq)]
    y, _ = ra_spmm.head_norm_rotate(leaves[0], None, leaves[1], None, table.cuda(), pos.cuda(), layout="interleaved")
    grads = torch.autograd.grad(y, leaves, gq.cuda())
    gen = torch.Generator().manual_seed(3)
    for n, x in enumerate((q, wq)):
        d = torch.randn(x.shape, generator=gen, dtype=torch.float64)
        loss = []
        for sign in (1, -1):
            s = [q.double(), wq.double()]
            s[n] = s[n] + sign * 1e-5 * d
            loss.append(float((exact(s[0], s[1], R, 1e-6)[0] * gq.double()).sum()))
        diff, got = (loss[0] - loss[1]) / 2e-5, float((grads[n].cpu().double() * d).sum())
        size = float((grads[n].cpu().double() * d).abs().sum())
        assert abs(got - diff) <= 1e-5 * size, (n, got, diff)


def test_equal_inputs_give_equal_bits():
    q, k, wq, wk, gq, gk = (t.cuda() for t in make(5000, 8, 8, 16, torch.bfloat16))
    table = ra_spmm.rotation_table(5000, 16, device="cuda")
    outs = []
    for _ in range(2):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, wq, wk)]
        outs.append(torch.autograd.grad(ra_spmm.head_norm_rotate(*leaves, table), leaves, (gq, gk)))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_no_rows():
    q = torch.zeros(0, 4, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    y, _ = ra_spmm.head_norm_rotate(q, None, w, None)
    y.sum().backward()
    assert y.shape == (0, 4, 16) and not w.grad.any()


def test_capture_and_replay():
    q, k, wq, wk, gq, gk = (t.cuda() for t in make(3000, 8, 4, 20, torch.bfloat16))
    table = ra_spmm.rotation_table(3000, 20, device="cuda")
    from ra_spmm import _C

    def body():
        a = (q, k, wq, wk, table, None, 1e-6, "half")
        return (*_C.run_head_norm(*a), *_C.run_head_norm_backward(*a, gq, gk))

    eager = body()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        body()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = body()
    for _ in range(3):
        junk = torch.randn(1000, 1000, device="cuda") @ torch.randn(1000, 1000, device="cuda")
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))
        del junk


@pytest.fixture(scope="module")
def case():
    q, k, wq, wk, _, _ = (t.cuda() for t in make(6, 2, 2, 16, torch.float32))
    return dict(q=q, k=k, wq=wq, wk=wk, table=ra_spmm.rotation_table(10, 8, device="cuda"),
                positions=torch.zeros(6, dtype=torch.int32, device="cuda"))


REFUSED = {
    "q on the host": (dict(q=lambda c: c["q"].cpu()), "CUDA"),
    "k on the host": (dict(k=lambda c: c["k"].cpu()), "CUDA"),
    "q float64": (dict(q=lambda c: c["q"].double(), k=lambda c: c["k"].double()), "float32, float16 or"),
    "two dtypes": (dict(k=lambda c: c["k"].half()), "one dtype"),
    "rows of k": (dict(k=lambda c: c["k"][:5]), "same rows"),
    "head_dim of k": (dict(k=lambda c: c["k"][..., :8].contiguous()), "head_dim"),
    "1-D": (dict(q=lambda c: c["q"][0, 0]), "shape"),
    "k without wk": (dict(wk=lambda c: None), "go together"),
    "weight of another length": (dict(wq=lambda c: c["wq"][:8]), "wq"),
    "weight float16": (dict(wq=lambda c: c["wq"].half()), "float32"),
    "table 2-D": (dict(table=lambda c: c["table"][..., 0].contiguous()), "table"),
    "table too wide": (dict(table=lambda c: ra_spmm.rotation_table(10, 18, device="cuda")), "passes head_dim"),
    "positions int64": (dict(positions=lambda c: c["positions"].long()), "int32"),
    "positions of another length": (dict(positions=lambda c: c["positions"][:3]), "positions"),
    "positions without a table": (dict(table=lambda c: None), "need a table"),
    "unknown layout": (dict(layout=lambda c: "quarter"), "layout"),
    "head_dim too large": (dict(q=lambda c: torch.zeros(6, 1, 257, device="cuda"), k=lambda c: None, wk=lambda c: None,
                                wq=lambda c: torch.ones(257, device="cuda")), "at most 256"),
}


@pytest.mark.parametrize("name", list(REFUSED))
def test_refusals(case, name):
    change, match = REFUSED[name]
    with pytest.raises(RuntimeError, match=match):
        ra_spmm.head_norm_rotate(**{**case, **{n: f(case) for n, f in change.items()}})
    torch.cuda.synchronize()
    assert ra_spmm.head_norm_rotate(**case)[0].shape == (6, 2, 16)


def test_table_refusals():
    for bad in (dict(rot_dim=3), dict(rot_dim=8, base=0.0), dict(rot_dim=8, scaling=-1.0)):
        with pytest.raises(RuntimeError):
            ra_spmm.rotation_table(4, **bad)
    assert math.isfinite(float(ra_spmm.rotation_table(4, 0).sum()))
