"""Embedding lookup and its gradient against their definition in 64 bits.

Tolerances, u = 2^-24.  out is one float32 product, u of itself.  A row of the gradient is a sum of the m gradients of its
positions, m * u of the sum of their magnitudes in any order, and one product.  The factor is taken as float32: s' = s (1 + d)
with |d| <= u, so that a product s' t (1 + e) is off by |d + e + d e| <= 2 u + u^2 < (2 + 2^-20) u.  16-bit results add half a unit of their last place (2^-11, 2^-8), or half the smallest fp16 step.  Gradients that are
small whole numbers have exact sums."""
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
    bound = err + unit * (want.abs() + err) + (2.0 ** -25 if unit == 2.0 ** -11 else 1e-37)
    assert got.shape == want.shape, what
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    bad = ~want.isnan() & ~((got - want).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} beyond; first {bad.nonzero()[0].tolist()}"


def exact(ids, table, g, scale, padding):
    """(out, gradient, its magnitudes, positions of every row)."""
    V, D = table.shape
    flat = ids.reshape(-1).long()
    pad = torch.zeros_like(flat, dtype=torch.bool) if padding is None else flat == padding
    inside = (flat >= 0) & (flat < V) & ~pad
    out = torch.full((flat.numel(), D), math.nan, dtype=torch.float64)
    out[inside] = table.double()[flat[inside]] * scale
    out[pad] = 0.0
    grad, mag = torch.zeros(V, D, dtype=torch.float64), torch.zeros(V, D, dtype=torch.float64)
    g = g.double().reshape(-1, D)
    grad.index_add_(0, flat[inside], g[inside] * scale)
    mag.index_add_(0, flat[inside], (g[inside] * scale).abs())
    return out.reshape(*ids.shape, D), grad, mag, torch.bincount(flat[inside], minlength=V)


def make_ids(n, V, kind, seed=1):
    gen = torch.Generator().manual_seed(seed)
    if kind == "one":
        return torch.full((n,), V // 2)
    if kind == "hubs":
        u = torch.rand(n, generator=gen, dtype=torch.float64)
        return (V ** u).long().clamp(max=V) - 1
    if kind == "ascending":
        return torch.arange(n) * V // max(n, 1)
    return torch.randint(0, V, (n,), generator=gen)


def check(ids, V, D, dtype, scale=1.0, padding=None, whole=False, strided=False, seed=2):
    gen = torch.Generator().manual_seed(seed)
    table = torch.randn(V, D, generator=gen).to(dtype)
    g = torch.randint(-3, 4, (ids.numel(), D), generator=gen) if whole else torch.randn(ids.numel(), D, generator=gen)
    g = g.to(dtype).reshape(*ids.shape, D)
    if strided:
        wide = torch.zeros(V, D + 3, dtype=dtype, device="cuda")
        wide[:, :D] = table
        leaf = wide[:, :D].detach().requires_grad_(True)
        wide_g = torch.zeros(ids.numel(), D + 5, dtype=dtype, device="cuda")
        wide_g[:, :D] = g.reshape(-1, D)
        gd = wide_g[:, :D]
        assert ids.dim() == 1
    else:
        leaf, gd = table.cuda().requires_grad_(True), g.cuda()
    out = ra_spmm.embed(ids.cuda(), leaf, scale=scale, padding=padding)
    grad, = torch.autograd.grad(out, leaf, gd, retain_graph=True)
    again, = torch.autograd.grad(out, leaf, gd)
    assert torch.equal(grad, again), "the gradient's bits"
    with torch.no_grad():
        plain = ra_spmm.embed(ids.cuda(), leaf, scale=scale, padding=padding)
    assert torch.equal(plain.nan_to_num(7.0), out.detach().nan_to_num(7.0))
    want, want_g, mag, m = exact(ids, table, g, scale, padding)
    close(out, want, (2 + 2.0 ** -20) * U * want.abs().nan_to_num(0.0), "out")
    err = (m[:, None] + 3) * U * mag
    if whole:
        err = U * want_g.abs() if scale != 1.0 else torch.zeros_like(mag)
        assert float(mag.max()) < 2 ** 24
    close(grad, want_g, err, "gradient")


SIZES = [(1, 1, 1), (1, 5, 256), (3, 7, 2), (63, 64, 16), (64, 64, 17), (65, 1, 40), (257, 300, 33), (1000, 47, 100), (1, 100000, 64),
         (4097, 5000, 8), (5000, 70000, 31), (8192, 20, 64)]


@pytest.mark.parametrize("kind", ["even", "hubs"])
@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_sizes_and_types(size, dtype, kind):
    n, V, D = size
    print(f"[embed] {size} {dtype} {kind}", flush=True)
    check(make_ids(n, V, kind), V, D, dtype, scale=2.5)


@pytest.mark.parametrize("D", [1, 3, 8, 64, 100, 128, 129, 256, 257, 511, 512, 513, 1000, 1024, 1030, 2048, 4096, 5003])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_widths(D, dtype):
    print(f"[embed] width {D} {dtype}", flush=True)
    check(make_ids(301, 40, "hubs"), 40, D, dtype, scale=math.sqrt(2.0))
    check(make_ids(70, 600, "even"), 600, D, dtype)


@pytest.mark.parametrize("kind", ["even", "hubs", "one", "ascending"])
@pytest.mark.parametrize("size", [(200_003, 61, 12), (150_000, 3_000, 32), (300_000, 200_000, 8), (20_000, 2_047, 16), (20_000, 2_048, 16),
                                  (16_384, 4_000_000, 2), (16_385, 4_194_303, 2), (33_000, 4_194_304, 2)], ids=str)
def test_long_runs_have_exact_sums(size, kind):
    """Whole numbers, so that a position that is lost, doubled or added to another row shows."""
    n, V, D = size
    print(f"[embed] {size} {kind}", flush=True)
    check(make_ids(n, V, kind), V, D, torch.float32, whole=True)


def test_more_positions_than_pieces_of_the_sort():
    """2.2e6 positions: pieces of more than 4,096."""
    check(make_ids(2_200_000, 70_000, "hubs"), 70_000, 4, torch.float32, whole=True)


@pytest.mark.parametrize("padding", [0, 5, -1, 100, 1 << 40])
def test_padding(padding):
    ids = make_ids(500, 20, "even")
    ids[::7] = padding if abs(padding) < 1 << 31 else 3
    check(ids, 20, 24, torch.float32, scale=3.0, padding=padding)
    check(torch.full((9,), padding), 20, 24, torch.float32, padding=padding)  # nothing but padding


@pytest.mark.parametrize("n", [40, 20_000])
def test_ids_outside_of_the_table(n):
    ids = make_ids(n, 20, "even")
    ids[1::5], ids[2::11], ids[3::13], ids[5] = 20, -1, 1 << 40, -(1 << 62)
    check(ids, 20, 8, torch.float32)
    check(ids, 20, 8, torch.float32, padding=20)


def test_integer_types_and_shapes():
    ids = make_ids(60, 30, "even")
    table = torch.randn(30, 16, device="cuda", requires_grad=True)
    a, b = ra_spmm.embed(ids.cuda(), table), ra_spmm.embed(ids.int().cuda(), table)
    assert torch.equal(a, b)
    g = torch.randn(60, 16, device="cuda")
    assert torch.equal(*(torch.autograd.grad(o, table, g)[0] for o in (a, b)))
    for shape in ((60,), (5, 12), (3, 1, 20), (60, 1)):
        c = ra_spmm.embed(ids.reshape(shape).cuda(), table)
        assert c.shape == (*shape, 16) and torch.equal(c.reshape(60, 16), a)
    assert torch.equal(ra_spmm.embed(ids.reshape(5, 12).t().cuda(), table), a.reshape(5, 12, 16).transpose(0, 1))
    one = ra_spmm.embed(torch.tensor(3, device="cuda"), table)
    assert one.shape == (16,) and torch.equal(one, table[3])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("D", [8, 20, 64, 301])
def test_strided_rows(D, dtype):
    check(make_ids(333, 50, "hubs"), 50, D, dtype, strided=True, scale=0.5)


def test_broadcast_gradient():
    """The gradient of a sum is one value, expanded."""
    ids = make_ids(333, 10, "even").cuda()
    table = torch.randn(10, 20, device="cuda", requires_grad=True)
    ra_spmm.embed(ids, table).sum().backward()
    assert torch.equal(table.grad, torch.bincount(ids, minlength=10).float()[:, None].expand(10, 20))


def test_empty():
    table = torch.randn(10, 20, device="cuda", requires_grad=True)
    ids = torch.zeros(0, dtype=torch.int64, device="cuda")
    out = ra_spmm.embed(ids, table)
    assert out.shape == (0, 20)
    g, = torch.autograd.grad(out, table, torch.zeros(0, 20, device="cuda"))
    assert torch.equal(g, torch.zeros(10, 20, device="cuda"))
    none = torch.zeros(0, 20, device="cuda", requires_grad=True)  # a table without rows: every id is outside
    out = ra_spmm.embed(torch.zeros(3, dtype=torch.int32, device="cuda"), none)
    assert out.isnan().all()
    assert torch.autograd.grad(out, none, torch.ones(3, 20, device="cuda"))[0].shape == (0, 20)


def test_values_that_are_not_finite():
    """They stay with their rows."""
    table = torch.randn(10, 8, device="cuda")
    table[3, 2], table[4, 1] = math.inf, math.nan
    table.requires_grad_(True)
    out = ra_spmm.embed(torch.tensor([3, 4, 5, 3], device="cuda"), table)
    assert out[0, 2] == math.inf and out[1, 1].isnan() and out[2].isfinite().all()
    g = torch.zeros(4, 8, device="cuda")
    g[2, 5] = math.nan
    grad, = torch.autograd.grad(out, table, g)
    assert grad.isnan().nonzero().tolist() == [[5, 5]]


def test_offsets_past_32_bits():
    """Rows of the table and of out behind 2^31 elements."""
    V, D = 1_200_000, 2048
    table = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda")
    table[-1], table[5] = 3.0, 2.0
    ids = torch.arange(V - 1, -1, -1, device="cuda")
    out = ra_spmm.embed(ids, table)
    assert (out[0] == 3.0).all() and (out[V - 6] == 2.0).all() and not out[-1].any() and not out[1].any()
    table = None
    g = out.zero_()
    g[-1], g[-3], g[0] = 1.0, 2.0, 4.0
    grad = ra_spmm._C.run_embed_backward(ids, g, V, 1.0, None)
    assert (grad[0] == 1.0).all() and (grad[2] == 2.0).all() and (grad[V - 1] == 4.0).all()
    assert not grad[1].any() and not grad[V - 2].any() and not grad[V // 2].any()


def test_on_another_stream():
    ids, table = make_ids(5000, 700, "hubs").cuda(), torch.randn(700, 48, device="cuda", requires_grad=True)
    g = torch.randn(5000, 48, device="cuda")
    want, = torch.autograd.grad(ra_spmm.embed(ids, table), table, g)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        out = ra_spmm.embed(ids, table)
        got, = torch.autograd.grad(out, table, g)
    s.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("n", [300, 40_000])
def test_capture_and_replay(n):
    V, D = 900, 40
    ids, table = make_ids(n, V, "hubs").cuda(), torch.randn(V, D, device="cuda")
    g = torch.randn(n, D, device="cuda")

    def body():
        leaf = table.detach().requires_grad_(True)
        out = ra_spmm.embed(ids, leaf, scale=2.0, padding=3)
        return out.detach(), torch.autograd.grad(out, leaf, g)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        body()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = body()
    for i in range(4):  # new ids, values and gradients each time, eager work between
        ids.copy_(make_ids(n, V, ["hubs", "even", "one", "ascending"][i], seed=i + 5))
        table.normal_()
        g.normal_()
        for o in outs:
            o.fill_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, body())), i


def test_refusals():
    ids, table = torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(5, 8, device="cuda")
    for bad, match in ((dict(ids=ids.cpu()), "CUDA"), (dict(table=table.cpu()), "CUDA"), (dict(ids=ids.float()), "int32 or int64"),
                       (dict(table=table.double()), "float32"), (dict(table=table[0]), "two dimensions"),
                       (dict(table=table[:, :0]), "at least one element"), (dict(table=torch.zeros(1, (1 << 20) + 1, device="cuda")), "2\\^20")):
        args = {"ids": ids, "table": table, **bad}
        with pytest.raises(RuntimeError, match=match):
            ra_spmm.embed(args["ids"], args["table"])
    with pytest.raises(RuntimeError, match="rows"):
        ra_spmm._C.run_embed_backward(ids, torch.zeros(3, 8, device="cuda"), 5, 1.0, None)
