"""Differential attention over neighbour lists against its definition in 64 bits: forward, gradients (formula and
differences), masks, head layouts, strides, plans, refusals.

Tolerances.  Let A be the largest sum of magnitudes in a score, scale * sum |q k| + |finite bias part that varies|, and n
the longest list.  A float32 score is off by at most (head_dim + 2) * eps * A, which moves a weight by that much of itself;
exp and the normalisation add a few eps; a sum of n terms adds n * eps of its magnitudes.  With eps = 2^-24 every float32
result is within (32 + (head_dim + 8) * A + value_dim + n) * eps of the sum of magnitudes that forms it, and 16-bit
results add half a unit of their last place (of 8 bits for bfloat16: 2^-8, of 11 for float16: 2^-11, 2^-25 absolute below its normals)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402

EPS = 2.0 ** -24
HALF_UNIT = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LOWEST = torch.finfo(torch.float32).min


def lists(lengths, K, seed):
    rng = np.random.default_rng(seed)
    rowptr = np.zeros(len(lengths) + 1, np.int32)
    np.cumsum(lengths, out=rowptr[1:])
    cols = [np.sort(rng.choice(K, size=n, replace=n > K)) for n in lengths]
    return torch.from_numpy(rowptr), torch.from_numpy(np.concatenate(cols + [np.zeros(0, int)]).astype(np.int32))


def inputs(M, K, Hq, Hkv, D, Dv, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    return (r(M, Hq, 2, D), r(K, Hkv, 2, D), r(K, Hkv, Dv), 0.2 + 0.6 * torch.rand(Hq, generator=g), r(M, Hq, Dv))


def exact(rowptr, colind, q, k, v, lam, bias=None, g=None, scale=None):
    """Outputs in float64 and, for each, the sum of magnitudes that forms it; A of the module's text."""
    M, Hq, _, D = q.shape
    K, Hkv, Dv = v.shape
    scale = D ** -0.5 if scale is None else scale
    i = torch.repeat_interleave(torch.arange(M), (rowptr[1:] - rowptr[:-1]).long())
    j = colind.long()
    b = torch.zeros(j.numel()) if bias is None else bias
    live = b > -math.inf
    i, j, b = i[live], j[live], b[live].double()
    q, k, v, lam = q.double(), k.double(), v.double(), lam.double()
    out, mag = torch.zeros(M, Hq, Dv, dtype=torch.float64), torch.zeros(M, Hq, Dv, dtype=torch.float64)
    res = {n: (torch.zeros(s, dtype=torch.float64), torch.zeros(s, dtype=torch.float64))
           for n, s in (("dq", q.shape), ("dk", k.shape), ("dv", v.shape), ("dlam", lam.shape))}
    A = 0.0
    for h in range(Hq):
        c = h // (Hq // Hkv)
        p = []
        for a in range(2):
            s = (q[i, h, a] * k[j, c, a]).sum(1) * scale
            A = max(A, float(((q[i, h, a] * k[j, c, a]).abs().sum(1) * scale).max()) if s.numel() else 0.0)
            # Scores next to the type's lowest value are equal in float32.
            s = torch.where(b < -1e30, b, s + b)
            top = torch.full((M,), -math.inf, dtype=torch.float64).scatter_reduce(0, i, s, "amax")
            e = (s - top[i]).exp()
            p.append(e / torch.zeros(M, dtype=torch.float64).index_add_(0, i, e)[i])
        w, wm = p[0] - lam[h] * p[1], p[0] + lam[h].abs() * p[1]
        out[:, h].index_add_(0, i, w[:, None] * v[j, c])
        mag[:, h].index_add_(0, i, wm[:, None] * v[j, c].abs())
        if g is None:
            continue
        go = g[i, h].double()
        dp, dpm = (go * v[j, c]).sum(1), (go * v[j, c]).abs().sum(1)
        res["dv"][0][:, c].index_add_(0, j, w[:, None] * go)
        res["dv"][1][:, c].index_add_(0, j, wm[:, None] * go.abs())
        res["dlam"][0][h] = -(p[1] * dp).sum()
        res["dlam"][1][h] = (p[1] * dpm).sum()
        for a, f in ((0, 1.0), (1, -lam[h])):
            mean = torch.zeros(M, dtype=torch.float64).index_add_(0, i, p[a] * dp)
            meanm = torch.zeros(M, dtype=torch.float64).index_add_(0, i, p[a] * dpm)
            ds, dsm = f * scale * p[a] * (dp - mean[i]), abs(f) * scale * p[a] * (dpm + meanm[i])
            res["dq"][0][:, h, a].index_add_(0, i, ds[:, None] * k[j, c, a])
            res["dq"][1][:, h, a].index_add_(0, i, dsm[:, None] * k[j, c, a].abs())
            res["dk"][0][:, c, a].index_add_(0, j, ds[:, None] * q[i, h, a])
            res["dk"][1][:, c, a].index_add_(0, j, dsm[:, None] * q[i, h, a].abs())
    res["out"] = (out, mag)
    return res, A


def close(got, want, mag, A, D, Dv, n, what):
    got, unit = got.detach().cpu(), HALF_UNIT[got.dtype]
    rel = (32 + (D + 8) * A + Dv + n) * EPS
    bound = rel * mag + unit * (want.abs() + rel * mag) + (2.0 ** -25 if got.dtype == torch.float16 else 1e-30)
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} beyond; worst {float((err / bound.clamp(min=1e-300)).max()):.3g} bounds"


def run_all(rowptr, colind, t, bias=None, scale=None, K=None):
    """Forward, gradients and the plan-free forward on the GPU."""
    q, k, v, lam, g = (x.cuda() for x in t)
    rp, ci = rowptr.cuda(), colind.cuda()
    bd = None if bias is None else bias.cuda()
    plan = ra_spmm.make_attention_plan(rp, ci, q.shape[0], k.shape[0])
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v, lam)]
    out = ra_spmm.diff_attention(plan, *leaves, scale=scale, bias=bd)
    grads = torch.autograd.grad(out, leaves, g)
    free = ra_spmm.diff_attention_csr(rp, ci, q, k, v, lam, scale=scale, bias=bd)
    infer = ra_spmm.run_attention_plan(plan, q, k, v, lam, scale=scale, bias=bd)
    assert torch.equal(infer, out) or not torch.isfinite(out).all()
    return out, dict(zip(("dq", "dk", "dv", "dlam"), grads)), free


def check(rowptr, colind, t, bias=None, scale=None):
    q, k, v, lam, g = t
    res, A = exact(rowptr, colind, q, k, v, lam, bias, g, scale)
    n = max(int((rowptr[1:] - rowptr[:-1]).max()) if rowptr.numel() > 1 else 0,
            int(torch.bincount(colind.long(), minlength=1).max()) if colind.numel() else 0)
    out, grads, free = run_all(rowptr, colind, t, bias, scale)
    D, Dv = q.shape[-1], v.shape[-1]
    close(out, *res["out"], A, D, Dv, n, "out")
    close(free, *res["out"], A, D, Dv, n, "plan-free out")
    for name in ("dq", "dk", "dv"):
        close(grads[name], *res[name], A, D, Dv, n * (q.shape[1] // k.shape[1]), name)
    close(grads["dlam"], *res["dlam"], A, D, Dv, n + q.shape[0], "dlam")


DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# heads, kv heads, head_dim, value_dim
HEADS = [(1, 1, 1, 1), (4, 4, 16, 32), (8, 2, 8, 16), (3, 3, 20, 40), (6, 2, 20, 20), (5, 5, 32, 64), (2, 1, 64, 128),
         (1, 1, 128, 256), (4, 2, 7, 13), (2, 2, 12, 3), (12, 3, 33, 66), (1, 1, 100, 50), (16, 16, 4, 8), (2, 2, 4, 60)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_heads_and_types(heads, dtype):
    print(f"[attention] {heads} {dtype}", flush=True)
    rowptr, colind = lists([0, 1, 2, 17, 40, 0, 5, 64, 3, 31, 1], 70, 3)
    check(rowptr, colind, inputs(11, 70, *heads, dtype, 5))


@pytest.mark.parametrize("lengths,K", [([0], 1), ([1], 1), ([1, 0, 1], 2), ([257], 300), ([256, 255, 512, 513], 600),
                                       ([3000, 0, 2, 777], 3000), ([40] * 300, 7), ([2] * 700, 3), ([0] * 9, 5),
                                       ([127, 128, 129, 130, 15, 16, 17, 64, 65], 200), ([3] * 3000 + [2000], 2500)], ids=lambda x: str(x)[:40])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_lengths_and_hubs(lengths, K, dtype):
    """Rows and columns of no, one and thousands of edges, cut and joined on both sides; duplicate edges."""
    print(f"[attention] lengths {lengths[:4]} K={K} {dtype}", flush=True)
    rowptr, colind = lists(lengths, K, 8)
    check(rowptr, colind, inputs(len(lengths), K, 4, 2, 16, 32, dtype, 6))


def masks(rowptr, kind, seed):
    n, nnz = (rowptr[1:] - rowptr[:-1]).long(), int(rowptr[-1])
    g = torch.Generator().manual_seed(seed)
    rows = torch.repeat_interleave(torch.arange(n.numel()), n)
    drop = torch.rand(nnz, generator=g) < 0.4
    drop |= rows % 3 == 1  # whole rows
    if kind == "-inf":
        return torch.zeros(nnz).masked_fill_(drop, -math.inf)
    if kind == "lowest":
        return torch.zeros(nnz).masked_fill_(drop, LOWEST)
    return torch.randn(nnz, generator=g) * 3  # weights


@pytest.mark.parametrize("kind", ["-inf", "lowest", "weights"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_bias(kind, dtype):
    """Masked edges, rows that lose every edge (zeros for -inf, equal weights for the lowest value), edge weights."""
    print(f"[attention] bias {kind} {dtype}", flush=True)
    rowptr, colind = lists([5, 9, 0, 33, 70, 600, 1, 2, 290], 400, 4)
    check(rowptr, colind, inputs(9, 400, 4, 4, 16, 32, dtype, 2), masks(rowptr, kind, 1))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=str)
def test_masked_edges_do_not_read_their_values(bad, dtype):
    rowptr, colind = lists([5, 9, 0, 33, 70, 300], 90, 4)
    t = list(inputs(6, 90, 4, 2, 16, 32, dtype, 2))
    gone = torch.arange(90) % 4 == 1
    bias = torch.zeros(colind.numel()).masked_fill_(gone[colind.long()], -math.inf)
    want = [x.clone() for x in t]
    for n in (1, 2):
        t[n][gone] = bad
    out, grads, free = run_all(rowptr, colind, t, bias)
    out0, grads0, free0 = run_all(rowptr, colind, want, bias)
    assert torch.equal(out, out0) and torch.equal(free, free0)
    for n in grads:
        assert torch.equal(grads[n], grads0[n]), n
    assert not grads["dk"][gone].any() and not grads["dv"][gone].any()


def test_live_nan_reaches_its_rows_only():
    rowptr, colind = lists([5, 9, 0, 33, 300], 90, 4)
    t = list(inputs(5, 90, 2, 2, 16, 32, torch.float32, 2))
    t[1][int(colind[6])] = math.nan
    out, _, free = run_all(rowptr, colind, t)
    i = torch.repeat_interleave(torch.arange(5), (rowptr[1:] - rowptr[:-1]).long())
    hit = torch.zeros(5, dtype=torch.bool)
    hit[i[colind == colind[6]]] = True
    for o in (out, free):
        assert o.cpu()[hit].isnan().all() and not o.cpu()[~hit].isnan().any()


def test_large_scores_and_scale():
    """Scores far beyond exp's range: one edge takes all of the weight."""
    rowptr, colind = lists([5, 9, 0, 33, 300], 90, 4)
    t = list(inputs(5, 90, 2, 2, 16, 32, torch.float32, 2))
    t[0] = t[0] * 1000
    q, k, v, lam, g = t
    res, A = exact(rowptr, colind, q, k, v, lam, None, g, 0.5)
    out, grads, _ = run_all(rowptr, colind, t, scale=0.5)
    gap = res["out"][0]
    assert torch.isfinite(out).all() and all(torch.isfinite(x).all() for x in grads.values())
    assert (out.cpu().double() - gap).abs().max() < (16 + 2) * A * EPS * 4 * 4  # weights move by the scores' error


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("pad", [0, 8, 3])
def test_rows_of_one_projection(pad, dtype):
    """q, k and v as column slices of one matrix, at odd offsets where pad is odd; gradients of a broadcast lam."""
    H, D, Dv, M = 4, 16, 32, 50
    width = H * 2 * D * 2 + H * Dv + 4 * pad
    x = torch.randn(M, width, generator=torch.Generator().manual_seed(1)).to(dtype)
    cut = lambda t, a, *s: t[:, a:a + math.prod(s)].unflatten(1, s)  # noqa: E731
    a, b, c = pad, H * 2 * D + 2 * pad, H * 4 * D + 3 * pad
    rowptr, colind = lists([n % 23 for n in range(M)], M, 1)
    g = torch.randn(M, H, Dv).to(dtype)
    lam = torch.tensor([0.4])
    xd, ld = x.cuda().requires_grad_(True), lam.cuda().requires_grad_(True)
    plan = ra_spmm.make_attention_plan(rowptr.cuda(), colind.cuda(), M, M)
    out = ra_spmm.diff_attention(plan, cut(xd, a, H, 2, D), cut(xd, b, H, 2, D), cut(xd, c, H, Dv), ld)
    out.backward(g.cuda())
    q, k, v = cut(x, a, H, 2, D), cut(x, b, H, 2, D), cut(x, c, H, Dv)
    res, A = exact(rowptr, colind, q, k, v, lam.expand(H), None, g)
    close(out, *res["out"], A, D, Dv, 50, "out")
    for n, off, s in (("dq", a, (H, 2, D)), ("dk", b, (H, 2, D)), ("dv", c, (H, Dv))):
        close(cut(xd.grad, off, *s), *res[n], A, D, Dv, 50, n)
    close(ld.grad, res["dlam"][0].sum(0, keepdim=True), res["dlam"][1].sum(0, keepdim=True), A, D, Dv, 50 + M, "dlam")


def test_gradients_against_differences():
    """<gradient, direction> against central differences of the loss in 64 bits: with step h the difference is off by
    O(h^2) of the third derivative, far below the float32 gradients' own error."""
    rowptr, colind = lists([5, 9, 0, 33, 300, 1], 90, 4)
    t = inputs(6, 90, 4, 2, 12, 20, torch.float32, 9)
    bias = masks(rowptr, "weights", 3)
    q, k, v, lam, g = t
    _, grads, _ = run_all(rowptr, colind, t, bias)
    res, A = exact(rowptr, colind, q, k, v, lam, bias, g)
    gen = torch.Generator().manual_seed(2)
    for n, name in enumerate(("dq", "dk", "dv", "dlam")):
        for _ in range(3):
            d = torch.randn(t[n].shape, generator=gen, dtype=torch.float64)
            h = 1e-4
            loss = []
            for sign in (1, -1):
                s = [x.double() for x in (q, k, v, lam)]
                s[n] = s[n] + sign * h * d
                loss.append(float((exact(rowptr, colind, *s, bias)[0]["out"][0] * g.double()).sum()))
            diff = (loss[0] - loss[1]) / (2 * h)
            got = float((grads[name].cpu().double() * d).sum())
            rel = (32 + (12 + 8) * A + 20 + 300 * 2) * EPS
            bound = rel * float((res[name][1] * d.abs()).sum()) + 1e-5 * float((res[name][0] * d).abs().sum())
            assert abs(got - diff) <= bound, (name, got, diff, bound)


def test_equal_inputs_give_equal_bits():
    rowptr, colind = lists([3000, 0, 2, 777] + [20] * 400, 900, 3)
    t = inputs(404, 900, 4, 4, 16, 32, torch.float32, 6)
    a, b = run_all(rowptr, colind, t), run_all(rowptr, colind, t)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    assert all(torch.equal(a[1][n], b[1][n]) for n in a[1])


def test_plan_arrays():
    lengths, K = [0, 1, 128, 129, 256, 257, 700, 3], 50
    rowptr, colind = lists(lengths, K, 3)
    plan = ra_spmm.make_attention_plan(rowptr.cuda(), colind.cuda(), 8, K)
    for side, ptr in (("", rowptr.numpy()), ("_t", ra_spmm.export_attention_plan(plan, "rowptr_t").numpy())):
        want, splits, slot = [], [], 0
        for r in range(len(ptr) - 1):
            b, e = int(ptr[r]), int(ptr[r + 1])
            pieces = max(1, -(-(e - b) // 256))
            for c in range(pieces):
                want.append((r, b + 256 * c, min(e, b + 256 * (c + 1)), slot + c if pieces > 1 else -1))
            if pieces > 1:
                splits.append((r, slot, pieces, 0))
                slot += pieces
        assert ra_spmm.export_attention_plan(plan, "items" + side).view(-1, 4).tolist() == [list(x) for x in want]
        assert ra_spmm.export_attention_plan(plan, "splits" + side).view(-1, 4).tolist() == [list(x) for x in splits]
    order = np.argsort(colind.numpy(), kind="stable")
    rows = np.repeat(np.arange(8), lengths)
    assert (ra_spmm.export_attention_plan(plan, "edge_t").numpy() == order).all()
    assert (ra_spmm.export_attention_plan(plan, "row_t").numpy() == rows[order]).all()
    counts = np.bincount(colind.numpy(), minlength=K)
    assert (np.diff(ra_spmm.export_attention_plan(plan, "rowptr_t").numpy()) == counts).all()


def test_no_rows_and_no_columns():
    z = torch.zeros(1, dtype=torch.int32)
    t = inputs(0, 4, 2, 2, 8, 8, torch.float32, 1)
    out, grads, free = run_all(z, torch.zeros(0, dtype=torch.int32), t)
    assert out.shape == (0, 2, 8) and free.shape == (0, 2, 8)
    assert not grads["dk"].any() and not grads["dv"].any() and not grads["dlam"].any()
    t = inputs(3, 0, 2, 2, 8, 8, torch.float32, 1)
    out, grads, free = run_all(torch.zeros(4, dtype=torch.int32), torch.zeros(0, dtype=torch.int32), t)
    assert not out.any() and not free.any() and not grads["dq"].any() and not grads["dlam"].any()


@pytest.mark.parametrize("M,n", [(1, 1), (1, 20_000), (3, 5000), (16, 40)])
def test_new_rows(M, n):
    """The plan-free form at the sizes it is for: few rows, long lists, against the plan's result."""
    print(f"[attention] new rows {M} x {n}", flush=True)
    K = 30_000
    rowptr, colind = lists([n + 7 * i for i in range(M)], K, 5)
    q, k, v, lam, _ = (x.cuda() for x in inputs(M, K, 8, 8, 16, 32, torch.bfloat16, 3))
    free = ra_spmm.diff_attention_csr(rowptr.cuda(), colind.cuda(), q, k, v, lam)
    res, A = exact(rowptr, colind, q.cpu(), k.cpu(), v.cpu(), lam.cpu())
    close(free, *res["out"], A, 16, 32, n, "plan-free out")


def test_rows_past_32_bit_offsets():
    """Rows of k, v, q whose element offsets pass 2^32."""
    H, D, Dv, K, ld = 2, 16, 32, 70_000, 65_536
    need = 3 * K * ld * 2
    if torch.cuda.mem_get_info()[0] < need + (8 << 30):
        pytest.skip("needs 36 GB of free memory")
    q, k, v, lam, g = (x.cuda() for x in inputs(K, K, H, H, D, Dv, torch.bfloat16, 3))
    rowptr, colind = lists([n % 3 for n in range(K)], K, 5)
    plan = ra_spmm.make_attention_plan(rowptr.cuda(), colind.cuda(), K, K)
    wide = []
    for x in (q, k, v):
        w = torch.empty((K, ld), dtype=x.dtype, device="cuda")
        cols = w[:, ld - x[0].numel():]
        cols.copy_(x.flatten(1))
        wide.append(cols.unflatten(1, x.shape[1:]))
    want = ra_spmm.run_attention_plan_train(plan, q, k, v, lam)
    got = ra_spmm.run_attention_plan_train(plan, *wide, lam)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    a = ra_spmm.run_attention_plan_backward(plan, q, k, v, lam, want[1], g)
    b = ra_spmm.run_attention_plan_backward(plan, *wide, lam, want[1], g)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_capture_and_replay():
    rowptr, colind = lists([3000, 0, 2, 777] + [20] * 400, 900, 3)
    q, k, v, lam, g = (x.cuda() for x in inputs(404, 900, 4, 4, 16, 32, torch.bfloat16, 6))
    rp, ci = rowptr.cuda(), colind.cuda()
    plan = ra_spmm.make_attention_plan(rp, ci, 404, 900)

    def body():
        out, stats = ra_spmm.run_attention_plan_train(plan, q, k, v, lam)
        return (out, *ra_spmm.run_attention_plan_backward(plan, q, k, v, lam, stats, g),
                ra_spmm.diff_attention_csr(rp, ci, q, k, v, lam))

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


def test_other_stream_than_the_lists():
    """The plan's lists stay alive for work queued on another stream than their own."""
    rowptr, colind = lists([20] * 4000, 900, 3)
    q, k, v, lam, _ = (x.cuda() for x in inputs(4000, 900, 4, 4, 16, 32, torch.bfloat16, 6))
    plan = ra_spmm.make_attention_plan(rowptr.cuda(), colind.cuda(), 4000, 900)
    want = ra_spmm.run_attention_plan(plan, q, k, v, lam)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        busy = torch.randn(4000, 4000, device="cuda")
        for _ in range(10):
            busy = busy @ busy * 1e-3
        out = ra_spmm.run_attention_plan(plan, q, k, v, lam)
    del plan
    over = [torch.full((80_000,), 2 ** 30, dtype=torch.int32, device="cuda") for _ in range(4)]  # would reuse the lists' memory
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    del over


@pytest.fixture(scope="module")
def case():
    rowptr, colind = lists([5, 9, 0, 33], 40, 4)
    q, k, v, lam, g = (x.cuda() for x in inputs(4, 40, 4, 2, 16, 32, torch.float32, 2))
    rp, ci = rowptr.cuda(), colind.cuda()
    plan = ra_spmm.make_attention_plan(rp, ci, 4, 40)
    stats = ra_spmm.run_attention_plan_train(plan, q, k, v, lam)[1]
    return dict(rp=rp, ci=ci, q=q, k=k, v=v, lam=lam, g=g, plan=plan, stats=stats,
                fwd=ra_spmm.make_attention_plan(rp, ci, 4, 40, backward=False))


def _run(c, **kw):
    a = {**{n: c[n] for n in ("plan", "q", "k", "v", "lam")}, **kw}
    return ra_spmm.run_attention_plan(**a)


REFUSED = {
    "q on the host": (lambda c: _run(c, q=c["q"].cpu()), "CUDA"),
    "q 3-D": (lambda c: _run(c, q=c["q"][:, :, 0]), "shape"),
    "one map": (lambda c: _run(c, q=c["q"][:, :, :1], k=c["k"][:, :, :1]), "shape"),
    "float64": (lambda c: _run(c, q=c["q"].double(), k=c["k"].double(), v=c["v"].double()), "float32, float16 or"),
    "two dtypes": (lambda c: _run(c, v=c["v"].half()), "one dtype"),
    "rows of q": (lambda c: _run(c, q=c["q"][:3]), "rows"),
    "rows of k": (lambda c: _run(c, k=c["k"][:30]), "rows"),
    "head_dim of k": (lambda c: _run(c, k=c["k"][..., :8].contiguous()), "head_dim"),
    "heads not a multiple": (lambda c: _run(c, q=c["q"][:, :3].contiguous(), lam=c["lam"][:3]), "multiple"),
    "heads of v": (lambda c: _run(c, v=c["v"][:, :1].contiguous()), "same heads"),
    "q transposed": (lambda c: _run(c, q=c["q"].transpose(2, 3).contiguous().transpose(2, 3)), "contiguous within"),
    "q broadcast": (lambda c: _run(c, q=c["q"][:1].expand(4, -1, -1, -1)), "overlap"),
    "lam of another length": (lambda c: _run(c, lam=c["lam"][:1]), "lam"),
    "lam float64": (lambda c: _run(c, lam=c["lam"].double()), "float32"),
    "bias of another length": (lambda c: _run(c, bias=torch.zeros(3, device="cuda")), "bias"),
    "bias on the host": (lambda c: _run(c, bias=torch.zeros(47)), "CUDA"),
    "head_dim too large": (lambda c: _run(c, q=c["q"].repeat(1, 1, 1, 9), k=c["k"].repeat(1, 1, 1, 9)), "at most 128"),
    "value_dim too large": (lambda c: _run(c, v=c["v"].repeat(1, 1, 9)), "at most 128|at most 256"),
    "no plan": (lambda c: _run(c, plan=None), "Invalid attention plan"),
    "backward on a plan without it": (lambda c: ra_spmm.run_attention_plan_backward(
        c["fwd"], c["q"], c["k"], c["v"], c["lam"], c["stats"], c["g"]), "backward=False"),
    "grad of another shape": (lambda c: ra_spmm.run_attention_plan_backward(
        c["plan"], c["q"], c["k"], c["v"], c["lam"], c["stats"], c["g"][:3]), "grad_out"),
    "stats of another shape": (lambda c: ra_spmm.run_attention_plan_backward(
        c["plan"], c["q"], c["k"], c["v"], c["lam"], c["stats"][:3], c["g"]), "stats"),
    "bias with a gradient": (lambda c: ra_spmm.diff_attention(
        c["plan"], c["q"], c["k"], c["v"], c["lam"], bias=torch.zeros(47, device="cuda", requires_grad=True)), "bias"),
    "plan: column out of range": (lambda c: ra_spmm.make_attention_plan(c["rp"], c["ci"], 4, 20), "colind"),
    "plan: negative column": (lambda c: ra_spmm.make_attention_plan(c["rp"], c["ci"] - 30, 4, 40), "colind"),
    "plan: rowptr decreases": (lambda c: ra_spmm.make_attention_plan(
        torch.tensor([0, 20, 10, 40, 47], dtype=torch.int32, device="cuda"), c["ci"], 4, 40), "rowptr"),
    "plan: rowptr ends early": (lambda c: ra_spmm.make_attention_plan(
        torch.tensor([0, 5, 14, 14, 40], dtype=torch.int32, device="cuda"), c["ci"], 4, 40), "rowptr"),
    "plan: rowptr does not start at 0": (lambda c: ra_spmm.make_attention_plan(
        torch.tensor([1, 5, 14, 14, 47], dtype=torch.int32, device="cuda"), c["ci"], 4, 40), "rowptr"),
    "plan: M": (lambda c: ra_spmm.make_attention_plan(c["rp"], c["ci"], 5, 40), "M\\+1"),
    "plan: int64": (lambda c: ra_spmm.make_attention_plan(c["rp"].long(), c["ci"], 4, 40), "int32"),
    "csr: int64": (lambda c: ra_spmm.diff_attention_csr(c["rp"], c["ci"].long(), c["q"], c["k"], c["v"], c["lam"]), "int32"),
    "export: unknown array": (lambda c: ra_spmm.export_attention_plan(c["plan"], "vals"), "unknown array"),
}


@pytest.mark.parametrize("name", list(REFUSED))
def test_refusals(case, name):
    fn, match = REFUSED[name]
    print(f"[attention] {name}", flush=True)
    with pytest.raises(RuntimeError, match=match):
        fn(case)
    torch.cuda.synchronize()
    assert _run(case).shape == (4, 4, 32)


@pytest.mark.parametrize("side", ["rows", "columns"])
def test_heads_kept_apart(side):
    """Long lists over gathered rows past the L2s: each XCD takes a part of the heads, on either side."""
    few, many = 300, 70_000
    rng = np.random.default_rng(1)
    if side == "rows":
        rowptr, colind = lists(rng.integers(0, 160, few), many, 5)
        M, K = few, many
    else:
        rowptr, colind = lists(rng.integers(0, 3, many), few, 5)
        M, K = many, few
    check(rowptr, colind, inputs(M, K, 4, 4, 32, 64, torch.bfloat16, 6))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_many_cut_rows(dtype):
    """More joining workgroups than are resident at once; the lists' rows hold 2 and 3 pieces."""
    print(f"[attention] cut rows {dtype}", flush=True)
    rowptr, colind = lists([260, 600] * 300, 500, 12)
    check(rowptr, colind, inputs(600, 500, 4, 4, 16, 32, dtype, 13))
