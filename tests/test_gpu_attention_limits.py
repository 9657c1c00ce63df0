"""More cut rows and columns than one joining launch holds (2^24 workgroups), against dense attention maps of a few heads
in 64 bits.  Every list is full, so that a head's map is a matrix.

Tolerances: as in test_gpu_attention.py, (32 + (head_dim + 8) * A + value_dim + n) * 2^-24 of the sum of magnitudes, with A
the largest sum of magnitudes in a score and n the longest list, and half a unit of bfloat16's last place."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402

EPS, HALF_UNIT = 2.0 ** -24, {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}


def close(got, want, mag, rel, what):
    err = (got.double() - want).abs()
    bound = rel * mag + HALF_UNIT[got.dtype] * (want.abs() + rel * mag) + 1e-30
    assert (err <= bound).all(), f"{what}: worst {float((err / bound).max()):.3g} bounds"


def check(M, K, H, D, Dv, dtype, heads):
    gen = torch.Generator("cuda").manual_seed(1)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    q, k, v, g = r(M, H, 2, D), r(K, H, 2, D), r(K, H, Dv), r(M, H, Dv)
    lam = 0.2 + 0.6 * torch.rand(H, generator=gen, device="cuda")
    rowptr = torch.arange(M + 1, device="cuda", dtype=torch.int32) * K
    colind = torch.arange(K, device="cuda", dtype=torch.int32).repeat(M)
    plan = ra_spmm.make_attention_plan(rowptr, colind, M, K)
    print(f"[attention] {M} x {K}, {H} heads: {plan.num_splits} cut rows, {plan.num_splits_t} cut columns", flush=True)
    out, stats = ra_spmm.run_attention_plan_train(plan, q, k, v, lam)
    dq, dk, dv, dlam = ra_spmm.run_attention_plan_backward(plan, q, k, v, lam, stats, g)
    n = max(M, K)
    for h in heads:
        qh, kh, vh, gh, l = q[:, h].double(), k[:, h].double(), v[:, h].double(), g[:, h].double(), lam[h].double()
        A = max(float((qh[:, a].abs() @ kh[:, a].abs().t().contiguous()).max()) for a in range(2)) * D ** -0.5
        rel = (32 + (D + 8) * A + Dv + n) * EPS
        p = [(qh[:, a] @ kh[:, a].t().contiguous() * D ** -0.5).softmax(1) for a in range(2)]
        w, wm = p[0] - l * p[1], p[0] + l * p[1]
        close(out[:, h], w @ vh, wm @ vh.abs(), rel, "out")
        close(dv[:, h], w.t().contiguous() @ gh, wm.t().contiguous() @ gh.abs(), rel, "dv")
        dp, dpm = gh @ vh.t().contiguous(), gh.abs() @ vh.abs().t().contiguous()
        close(dlam[h], -(p[1] * dp).sum(), (p[1] * dpm).sum(), rel + M * EPS, "dlam")
        for a, c in ((0, 1.0), (1, -l)):
            ds = c * D ** -0.5 * p[a] * (dp - (p[a] * dp).sum(1, keepdim=True))
            dsm = abs(c) * D ** -0.5 * p[a] * (dpm + (p[a] * dpm).sum(1, keepdim=True))
            close(dq[:, h, a], ds @ kh[:, a], dsm @ kh[:, a].abs(), rel, "dq")
            close(dk[:, h, a], ds.t().contiguous() @ qh[:, a], dsm.t().contiguous() @ qh[:, a].abs(), rel, "dk")
        del p, w, wm, dp, dpm, ds, dsm


def test_columns():
    """65,700 columns of 257 edges, 32 heads of 128 + 256: 256 workgroups join a column."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of free memory")
    check(257, 65_700, 32, 128, 256, torch.bfloat16, (0, 31))


def test_rows():
    """524,500 rows of 257 edges, 32 heads."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of free memory")
    check(524_500, 257, 32, 2, 4, torch.float32, (0, 17, 31))


def test_more_waves_than_a_launch_holds():
    """70e6 rows of one edge: the softmax is 1, so the output is (1 - lam) v and the scores take no gradient."""
    M, K = 70_000_001, 1000
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free memory")
    gen = torch.Generator("cuda").manual_seed(1)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    q, k, v, g, lam = r(M, 1, 2, 1), r(K, 1, 2, 1), r(K, 1, 1), r(M, 1, 1), torch.tensor([0.25], device="cuda")
    colind = torch.randint(0, K, (M,), generator=gen, device="cuda").to(torch.int32)
    plan = ra_spmm.make_attention_plan(torch.arange(M + 1, device="cuda", dtype=torch.int32), colind, M, K)
    assert plan.num_items == M
    out, stats = ra_spmm.run_attention_plan_train(plan, q, k, v, lam)
    j = colind.long()
    assert torch.equal(out, 0.75 * v[j])
    dq, dk, dv, dlam = ra_spmm.run_attention_plan_backward(plan, q, k, v, lam, stats, g)
    assert not dq.any() and not dk.any()
    want, mag = (torch.zeros(K, dtype=torch.float64, device="cuda").index_add_(0, j, 0.75 * x.double().flatten())
                 for x in (g, g.abs()))
    assert ((dv.flatten().double() - want).abs() <= 80_000 * EPS * mag).all()
    terms = (g * v[j]).double()
    assert (dlam.double() + terms.sum()).abs() <= 80_000 * EPS * terms.abs().sum()


def test_rows_without_a_plan():
    """140,000 rows of 300 edges, 128 heads, in two pieces each: more joining workgroups than a launch holds."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of free memory")
    M, K, H, n = 140_000, 300, 128, 300
    gen = torch.Generator("cuda").manual_seed(1)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    q, k, v, lam = r(M, H, 2, 1), r(K, H, 2, 1), r(K, H, 2), torch.rand(H, generator=gen, device="cuda")
    rowptr = torch.arange(M + 1, device="cuda", dtype=torch.int32) * n
    colind = torch.arange(n, device="cuda", dtype=torch.int32).repeat(M)
    free = ra_spmm.diff_attention_csr(rowptr, colind, q, k, v, lam)
    for h in (0, 77, 127):
        p = [(q[:, h, a].double() @ k[:, h, a].double().t().contiguous()).softmax(1) for a in range(2)]
        A = max(float((q[:, h, a].abs().max() * k[:, h, a].abs().max())) for a in range(2))
        l, vh = lam[h].double(), v[:, h].double()
        close(free[:, h], (p[0] - l * p[1]) @ vh, (p[0] + l * p[1]) @ vh.abs(), (32 + 9 * A + 2 + n) * EPS, "out")
