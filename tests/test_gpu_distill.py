"""Distillation loss and its gradient against their definition in 64 bits.

Tolerances, u = 2^-24.  An exponential exp((x - max) / T) is off by 6 |x - max| / T u + 2 u of itself (the difference, the factor, its
product, the function).  A sum over C classes is of at least min(C, 64) chains: (C / 64 + 80) u and the mean of its terms'
errors; one over k entries (k + 16) u.  Probabilities follow.  A loss sums p ((t - top) - (x - max)) / T + log's difference), in float32:
4 u of the two differences' magnitudes, 3 u of the logarithms', u of the term, and its rounding.  Exponentials below 2^-126 may count as 0: 1e-34 with the
largest factor, 1000.  16-bit gradients add half a unit of their last place (2^-11, 2^-8), or half
the smallest fp16 step."""
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
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), f"{what}: inf in other places"
    bound = err + unit * (want.abs() + err) + (2.0 ** -25 if unit == 2.0 ** -11 else 1e-34)
    bad = ~want.isnan() & ~inf & ~((got - want).abs() <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} beyond; first {bad.nonzero()[0].tolist()}, worst "
                           f"{float(((got - want).abs() / bound)[bad].max()):.3g} bounds")


def softmax(x, T, chain):
    """(softmax, its relative error, log of the sum, that sum's relative error, |x - max| / T, |log of the sum of exp((x - max) / T)|)."""
    m = x.max()
    d = ((x - m) / T).clamp(min=-1e4)
    e = torch.exp(d)
    term = 6 * d.abs() * U + 2 * U
    total = e.sum()
    rel_total = (chain + 2) * U + (e * term).sum() / total
    return e / total, term + rel_total + 2 * U, torch.log(total) + m / T, rel_total, ((x - m) / T).abs(), torch.log(total).abs()


def exact(x, t, ids, T, labels, hard, up):
    """(loss [M], its error, gradient, its error) row by row, from the definition."""
    x, t = x.double(), t.double()
    M, C = x.shape
    loss, lerr = torch.zeros(M, dtype=torch.float64), torch.zeros(M, dtype=torch.float64)
    grad, gerr = torch.zeros(M, C, dtype=torch.float64), torch.zeros(M, C, dtype=torch.float64)
    for i in range(M):
        used = (ids[i] >= 0) & (t[i] != -math.inf)
        if hard < 1 and used.any():
            a = (1 - hard) * T
            at, tt = ids[i][used], t[i][used]
            if (at >= C).any() or not (tt < math.inf).all() or not (x[i] < math.inf).all() or x[i].max() == -math.inf:
                loss[i], grad[i] = math.nan, math.nan
                continue
            p, prel, tl, trel, td, tlog = softmax(tt, T, len(tt) + 16)
            q, qrel, xl, xrel, xd, xlog = softmax(x[i], T, C / 64 + 80)
            # Entries of probability 0 (in float32) add nothing.
            p = torch.where(p < 1e-37, 0.0, p)
            term = torch.where(p > 0, (tt / T - tl) - (x[i][at] / T - xl), 0.0)
            loss[i] += a * T * torch.where(p > 0, p * term, 0.0).sum()
            steps = 4 * U * (td + xd[at]) + 3 * U * (tlog + xlog) + U * term.abs()
            lerr[i] += a * T * (torch.where(p > 0, p * (prel * term.abs() + steps), 0.0).sum() + xrel + trel + 4 * U)
            P = torch.zeros(C, dtype=torch.float64).index_add_(0, at, p)
            Perr = torch.zeros(C, dtype=torch.float64).index_add_(0, at, p * (prel + (len(tt) + 3) * U))
            grad[i] += a * up[i] * (q - P)
            gerr[i] += a * abs(up[i]) * (q * (qrel + 3 * U) + Perr)
        if hard > 0 and labels is not None and labels[i] >= 0:
            y = int(labels[i])
            if y >= C or not (x[i] < math.inf).all() or x[i].max() == -math.inf:
                loss[i], grad[i] = math.nan, math.nan
                continue
            q, qrel, xl, xrel, xd, xlog = softmax(x[i], 1.0, C / 64 + 80)
            loss[i] += hard * (xl - x[i, y])
            lerr[i] += hard * (xrel + U + 3 * U * (xlog + xd[y]))
            h = hard * up[i] * q
            h[y] -= hard * up[i]
            grad[i] += h
            gerr[i] += hard * abs(up[i]) * q * (qrel + 3 * U)
            gerr[i, y] += 2 * U * hard * abs(up[i])
    # The parts are added in float32.
    return loss, lerr + 2 * U * loss.abs(), grad, gerr + 3 * U * grad.abs()


def make(M, C, k, dtype, teacher_dtype=None, seed=1, ragged=True):
    gen = torch.Generator().manual_seed(seed)
    x = (2 * torch.randn(M, C, generator=gen)).to(dtype)
    t = (3 + 2 * torch.randn(M, k, generator=gen)).sort(1, descending=True).values.to(teacher_dtype or dtype)
    ids = torch.stack([torch.randperm(C, generator=gen)[:k] for _ in range(M)]) if M else torch.zeros(0, k, dtype=torch.int64)
    if ragged and k:
        kept = torch.randint(0, k + 1, (M,), generator=gen)
        ids[torch.arange(k)[None] >= kept[:, None]] = -1
    labels = torch.randint(-1, C, (M,), generator=gen)
    return x, t, ids, labels


def check(x, t, ids, labels=None, T=1.0, hard=0.0, ids_type=torch.int64, put=lambda v: v.cuda()):
    M, C = x.shape
    gen = torch.Generator().manual_seed(5)
    xd, td, idd = put(x).detach(), put(t), put(ids.to(ids_type))
    ld = None if labels is None else labels.to(ids_type).cuda()
    kw = {"temperature": T, "labels": ld, "hard": hard}
    up = torch.randn(M, generator=gen).double()
    want, werr, grad, gerr = exact(x, t, ids, T, labels, hard, up.float().double())
    leaf = xd.requires_grad_(True)
    none = ra_spmm.distill_loss(leaf, td, idd, reduction="none", **kw)
    close(none, want, werr, "loss of the rows")
    g, = torch.autograd.grad(none, leaf, up.float().cuda(), retain_graph=True)
    close(g, grad, gerr, "gradient of the rows")
    assert torch.equal(g.nan_to_num(7.0), torch.autograd.grad(none, leaf, up.float().cuda())[0].nan_to_num(7.0))
    with torch.no_grad():
        assert torch.equal(ra_spmm.distill_loss(leaf, td, idd, reduction="none", **kw).nan_to_num(7.0), none.detach().nan_to_num(7.0))
    for reduction, scale in (("mean", 1.0 / M), ("sum", 1.0)):
        ones = torch.full((M,), scale, dtype=torch.float64)
        want, werr, grad, gerr = exact(x, t, ids, T, labels, hard, ones)
        loss = ra_spmm.distill_loss(leaf, td, idd, reduction=reduction, **kw)
        close(loss, (want * scale).sum(), (werr * scale).sum() + U * (want * scale).abs().sum(), reduction)
        g, = torch.autograd.grad(loss, leaf)
        close(g, grad, gerr, f"gradient of the {reduction}")
        both, fused = ra_spmm.distill_loss_grad(leaf, td, idd, reduction=reduction, **kw)
        assert not both.requires_grad and not fused.requires_grad
        close(both, (want * scale).sum(), (werr * scale).sum() + U * (want * scale).abs().sum(), reduction)
        close(fused, grad, gerr, f"gradient of the {reduction} in one call")
    for factor in (8.0, torch.tensor([-0.5], device="cuda")):
        f = float(factor)
        _, fused = ra_spmm.distill_loss_grad(leaf, td, idd, reduction="sum", factor=factor, **kw)
        close(fused, grad * f, gerr * abs(f), "gradient with a factor")


CLASSES = [1, 2, 3, 7, 8, 16, 31, 40, 47, 64, 65, 100, 127, 128, 129, 255, 256, 257, 512, 513, 1000, 1024, 1025, 2047, 2048, 2049, 4099, 8192, 8200,
           16_385, 50_001, 100_003]


@pytest.mark.parametrize("mode", ["soft", "both", "hard"])
@pytest.mark.parametrize("C", CLASSES)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_classes_and_types(C, dtype, mode):
    print(f"[distill] {C} {dtype} {mode}", flush=True)
    x, t, ids, labels = make(5 if C > 5000 else 13, C, min(C, 9), dtype)
    check(x, t, ids, labels, T=2.0, hard={"soft": 0.0, "both": 0.3, "hard": 1.0}[mode])


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 63, 300])
@pytest.mark.parametrize("C", [5, 47, 300, 3000])
def test_rows(M, C):
    print(f"[distill] {M} x {C}", flush=True)
    check(*make(M, C, 4, torch.float32), T=3.0, hard=0.5)


@pytest.mark.parametrize("C", [1, 2, 3, 8, 31, 32, 47, 48, 63, 64, 65])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_many_rows_of_few_classes(C, dtype):
    """Row by row the same as a few rows at a time, to the tolerances of both: the first 150 and the last 83 rows against the
    definition, with every kind of row among them."""
    M = 40_003
    x, t, ids, labels = make(M, C, min(C, 5), dtype, seed=2)
    some = torch.cat([torch.arange(150), torch.arange(M - 83, M)])
    x[7, 0], x[9], ids[11, 0], labels[13], labels[15] = math.nan, -math.inf, C, C, -1
    if C > 2:
        ids[17, 1], ids[18, :], labels[18], x[19, 1] = ids[17, 0], -1, -1, -math.inf
        x[18, 2] = math.nan
    t[21, 0], t[22, 0], t[23, :] = -math.inf, math.inf, -math.inf
    for hard, T in ((0.0, 2.0), (0.4, 2.0), (1.0, 1.0)):
        kw = {"temperature": T, "labels": labels.cuda(), "hard": hard}
        up = torch.randn(M, generator=torch.Generator().manual_seed(5))
        want, werr, grad, gerr = exact(x[some], t[some], ids[some], T, labels[some], hard, up[some].double())
        leaf = x.cuda().requires_grad_(True)
        loss = ra_spmm.distill_loss(leaf, t.cuda(), ids.cuda(), reduction="none", **kw)
        g, = torch.autograd.grad(loss, leaf, up.cuda())
        close(loss[some.cuda()], want, werr, "loss of the rows")
        close(g[some.cuda()], grad, gerr, "gradient of the rows")
        clean = x.clone()
        clean[:150] = 0.5
        good = ids.clone()
        good[:150] = 0
        y = labels.clamp(max=C - 1)
        kw["labels"] = y.cuda()
        rows = ra_spmm.distill_loss(clean.cuda(), t.clamp(-9, 9).cuda(), good.cuda(), reduction="none", **kw)
        both, fused = ra_spmm.distill_loss_grad(clean.cuda(), t.clamp(-9, 9).cuda(), good.cuda(), reduction="sum", factor=-2.0, **kw)
        assert abs(float(both) - float(rows.double().sum())) <= U * float(rows.double().abs().sum())
        minus = torch.full((M,), -2.0, device="cuda")
        leaf = clean.cuda().requires_grad_(True)
        again, = torch.autograd.grad(ra_spmm.distill_loss(leaf, t.clamp(-9, 9).cuda(), good.cuda(), reduction="none", **kw), leaf, minus)
        assert torch.equal(fused, again)


@pytest.mark.parametrize("k", [0, 1, 2, 15, 16, 17, 63, 64, 65, 200, 256, 257, 1000, 1024])
@pytest.mark.parametrize("C", [1024, 20_000])
def test_kept_entries(k, C):
    print(f"[distill] {k} of {C}", flush=True)
    check(*make(4, C, k, torch.bfloat16, ragged=False), T=1.5, hard=0.2)
    check(*make(4, C, k, torch.float32, ragged=True), T=1.5, hard=0.2)


@pytest.mark.parametrize("C", [1, 7, 40, 64])
def test_all_classes_kept(C):
    check(*make(21, C, C, torch.float32, ragged=False), T=1.0)
    check(*make(21, C, C, torch.float16, ragged=False), T=0.7, hard=0.9)


@pytest.mark.parametrize("T", [1e-3, 0.1, 1.0, 8.0, 1000.0])
@pytest.mark.parametrize("C", [30, 5000])
def test_temperatures(T, C):
    check(*make(6, C, 6, torch.float32), T=T, hard=0.25)


@pytest.mark.parametrize("C", [12, 900, 30_000])
def test_one_id_in_several_entries(C):
    """The label among them: their parts of the gradient add up, whatever their order."""
    x, t, ids, labels = make(9, C, 12, torch.float32, ragged=False)
    ids[:, 1::2] = ids[:, :1]
    ids[3] = 5
    ids[4, 2:] = -1
    labels[::2] = ids[::2, 0]
    check(x, t, ids, labels, T=2.0, hard=0.4)


@pytest.mark.parametrize("C", [20, 700, 40_000])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_masked_classes(C, dtype):
    """Logits of -inf and of the type's lowest value: probability 0; as a teacher's entry or a label, a loss of inf."""
    x, t, ids, labels = make(8, C, 5, dtype, ragged=False)
    low = torch.finfo(dtype).min
    x[0, ::2], x[1, 1::2] = -math.inf, low
    x[2, :-1] = -math.inf
    ids[0] = torch.arange(5) * 2 + 1
    ids[1] = torch.arange(5) * 2
    ids[2, 0], ids[2, 1:] = C - 1, -1
    labels[0], labels[1], labels[2] = 3, 4, C - 1
    x[3, int(ids[3, 1])] = -math.inf
    labels[3] = -1
    x[4, int(ids[4, 0])] = -math.inf
    labels[4] = int(ids[4, 0])
    check(x, t, ids, labels, T=2.0, hard=0.5)


@pytest.mark.parametrize("C", [20, 40_000])
def test_teacher_entries_that_take_no_part(C):
    x, t, ids, labels = make(8, C, 6, torch.float32, ragged=False)
    t[0, 2], t[1, :] = -math.inf, -math.inf
    ids[2], ids[3, 1::2] = -1, -7
    t[3, 1::2], t[2] = math.nan, math.inf  # of entries that are not there
    t[4, 1:] = torch.finfo(torch.float32).min
    labels[1], labels[2], labels[5] = -1, 0, -1
    check(x, t, ids, labels, T=2.0, hard=0.5)


@pytest.mark.parametrize("C", [20, 40_000])
def test_rows_that_become_nan(C):
    x, t, ids, labels = make(9, C, 6, torch.float32, ragged=False)
    labels[:] = -1
    labels[0], ids[1, 3], t[2, 0], t[3, 4] = C, C, math.inf, math.nan
    x[4, 3], x[5, 7], x[6] = math.nan, math.inf, -math.inf
    x[7], ids[7] = math.nan, -1  # neither entries nor a label: 0 whatever the logits are
    check(x, t, ids, labels, T=2.0, hard=0.5)


def test_types_of_teacher_and_ids():
    x, t, ids, labels = make(20, 50, 6, torch.bfloat16, torch.float32)
    check(x, t, ids, labels, T=2.0, hard=0.3, ids_type=torch.int32)
    x, t, ids, labels = make(20, 5000, 6, torch.float32, torch.float16)
    check(x, t, ids, labels, T=2.0, hard=0.3, ids_type=torch.int32)


@pytest.mark.parametrize("extra", [1, 3, 8])
@pytest.mark.parametrize("C", [47, 1000, 20_000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_strided_rows(C, extra, dtype):
    """Columns of wider rows, at addresses that fit no packet."""
    def put(v):
        wide = torch.zeros(v.shape[0], v.shape[1] + extra, dtype=v.dtype, device="cuda")
        wide[:, extra // 2:extra // 2 + v.shape[1]] = v.cuda()
        return wide[:, extra // 2:extra // 2 + v.shape[1]]
    x, t, ids, labels = make(6, C, 5, dtype)
    check(x, t, ids, labels, T=2.0, hard=0.3, put=put)


def test_large_values():
    """Far from 0 and from each other."""
    for C in (50, 20_000):
        x, t, ids, labels = make(6, C, 5, torch.float32)
        check(x * 100 + 5e4, t * 50 - 1e4, ids, labels, T=2.0, hard=0.5)
        check(x * 1e30, t * 1e30, ids, labels, T=1.0)


def test_gradients_against_differences():
    """Along a random direction, differences of the 64-bit definition with steps of 1e-4: their own error is of second order."""
    x, t, ids, labels = make(6, 60, 7, torch.float32, seed=3)
    v = torch.randn(6, 60, generator=torch.Generator().manual_seed(4), dtype=torch.float64)
    ones = torch.ones(6, dtype=torch.float64)

    def value(s):
        return float(exact(x.double() + s * v, t, ids, 2.0, labels, 0.4, ones)[0].sum())

    want = (value(1e-4) - value(-1e-4)) / 2e-4
    _, g = ra_spmm.distill_loss_grad(x.cuda(), t.cuda(), ids.cuda(), 2.0, labels.cuda(), 0.4, "sum")
    got = float((g.cpu().double() * v).sum())
    assert abs(got - want) <= 1e-5 + 200 * U * float((g.cpu().double() * v).abs().sum())


def test_a_teacher_that_the_student_equals():
    """No divergence and no gradient, to rounding."""
    x = torch.randn(30, 40, device="cuda")
    t, ids = x.topk(40, dim=1)
    loss, g = ra_spmm.distill_loss_grad(x, t, ids, 2.0, reduction="none")
    assert float(loss.abs().max()) < 4 * 100 * U and float(g.abs().max()) < 2 * 100 * U


def test_empty():
    x = torch.zeros(0, 9, device="cuda", requires_grad=True)
    t, ids = torch.zeros(0, 3, device="cuda"), torch.zeros(0, 3, dtype=torch.int64, device="cuda")
    assert ra_spmm.distill_loss(x, t, ids, reduction="none").shape == (0,)
    assert float(ra_spmm.distill_loss(x, t, ids, reduction="sum")) == 0.0
    loss = ra_spmm.distill_loss(x, t, ids)
    assert loss.isnan() and torch.autograd.grad(loss, x)[0].shape == (0, 9)
    assert ra_spmm.distill_loss_grad(x, t, ids)[1].shape == (0, 9)


def test_offsets_past_32_bits():
    M, C = 1_200_000, 2000
    x = torch.zeros(M, C, dtype=torch.bfloat16, device="cuda")
    x[-1, 7] = 5.0
    t, ids = torch.ones(M, 1, device="cuda"), torch.full((M, 1), 3, device="cuda")
    ids[-1] = 7
    loss, g = ra_spmm.distill_loss_grad(x, t, ids, reduction="none")
    assert abs(float(loss[0]) - math.log(C)) < 1e-4 and torch.equal(loss[:-1], loss[:1].expand(M - 1))
    q = math.exp(5.0) / (math.exp(5.0) + C - 1)
    assert abs(float(loss[-1]) + math.log(q)) < 1e-4 and abs(float(g[-1, 7]) - (q - 1)) < 2.0 ** -8
    assert float(g[-2, 3]) == float(g[0, 3]) and abs(float(g[0, 3]) - (1 / C - 1)) < 2.0 ** -8 and float(g[-1, 3]) > 0


def test_on_another_stream():
    x, t, ids, labels = (v.cuda() for v in make(500, 3000, 8, torch.float32))
    want = ra_spmm.distill_loss_grad(x, t, ids, 2.0, labels, 0.3)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ra_spmm.distill_loss_grad(x, t, ids, 2.0, labels, 0.3)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("size", [(700, 47), (4, 30_000), (600, 9000)], ids=str)
def test_capture_and_replay(size):
    M, C = size
    x, t, ids, labels = (v.cuda() for v in make(M, C, 6, torch.float32))

    def body():
        leaf = x.detach().requires_grad_(True)
        loss = ra_spmm.distill_loss(leaf, t, ids, 2.0, labels, 0.3)
        return (loss.detach(), torch.autograd.grad(loss, leaf)[0], *ra_spmm.distill_loss_grad(x, t, ids, 2.0, labels, 0.3, "sum"))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        body()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = body()
    for i in range(4):
        new = make(M, C, 6, torch.float32, seed=10 + i)
        for a, b in zip((x, t, ids, labels), new):
            a.copy_(b)
        for o in outs:
            o.fill_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, body())), i


def test_refusals():
    x, t, ids = torch.zeros(4, 9, device="cuda"), torch.zeros(4, 3, device="cuda"), torch.zeros(4, 3, dtype=torch.int64, device="cuda")
    labels = torch.zeros(4, dtype=torch.int64, device="cuda")
    for bad, match in ((dict(logits=x.cpu()), "CUDA"), (dict(teacher=t.cpu()), "CUDA"), (dict(ids=ids.cpu()), "CUDA"),
                       (dict(ids=ids.float()), "int32 or int64"), (dict(ids=ids[:, :2]), "one shape"), (dict(teacher=t[:3], ids=ids[:3]), "rows"),
                       (dict(hard=0.5), "labels"), (dict(hard=1.5, labels=labels), "hard"), (dict(hard=math.nan, labels=labels), "hard"),
                       (dict(temperature=0.0), "temperature"), (dict(temperature=math.nan), "temperature"), (dict(temperature=2000.0), "temperature"),
                       (dict(labels=labels[:3], hard=0.5), "labels"), (dict(labels=labels.float(), hard=0.5), "int32 or int64"),
                       (dict(reduction="max"), "reduction"), (dict(logits=x.double()), "float32, float16"),
                       (dict(teacher=torch.zeros(4, 1025, device="cuda"), ids=torch.zeros(4, 1025, dtype=torch.int32, device="cuda")), "1024"),
                       (dict(logits=x[0]), "two dimensions"), (dict(teacher=t.clone().requires_grad_(True)), "teacher takes no gradient")):
        args = {"logits": x, "teacher": t, "ids": ids, **bad}
        with pytest.raises(RuntimeError, match=match):
            ra_spmm.distill_loss(**args)
        with pytest.raises(RuntimeError, match=match):
            ra_spmm.distill_loss_grad(**args)
