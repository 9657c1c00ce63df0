"""The gradient of the maps' weights sums over all rows, with terms of both signs: what a row's term is off by in one
direction adds up.

Bound: a row's delta is a mean of dot products of value_dim terms of random signs, whose running sum has about the size
of sqrt(value_dim) terms.  Each of its roundings moves it by at most 2^-24 of that, in either direction alike, and so do
about 4 + log2 n others: their root sum of squares, over R rows sqrt(R) of it.  Allowed are 8 times that, and the rounding
of the result."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402


@pytest.mark.parametrize("D,Dv", [(8, 16), (16, 16), (32, 64), (5, 7)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_sum_over_many_rows(D, Dv, dtype):
    M, n, H = 400_000, 8, 2
    gen = torch.Generator("cuda").manual_seed(D)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    q, k, v, g, lam = r(M, H, 2, D), r(M, H, 2, D), r(M, H, Dv), r(M, H, Dv), torch.tensor([0.3, 0.7], device="cuda")
    colind = torch.randint(0, M, (M, n), generator=gen, device="cuda")
    plan = ra_spmm.make_attention_plan(torch.arange(M + 1, device="cuda", dtype=torch.int32) * n,
                                       colind.flatten().to(torch.int32), M, M)
    _, stats = ra_spmm.run_attention_plan_train(plan, q, k, v, lam)
    dlam = ra_spmm.run_attention_plan_backward(plan, q, k, v, lam, stats, g)[3]
    for h in range(H):
        score = (q[:, None, h, 1].double() * k[:, h, 1].double()[colind]).sum(-1) * D ** -0.5
        p = score.softmax(1)
        terms = g[:, None, h].double() * v[:, h].double()[colind]
        want = -(p * terms.sum(-1)).sum()
        size = (p * terms.abs().sum(-1)).sum(1).square().mean().sqrt()
        bound = 8 * math.sqrt(M * (Dv + 4 + math.log2(n))) / Dv * 2.0 ** -24 * size + 2.0 ** -23 * want.abs()
        err = dlam[h].double() - want
        print(f"[attention] {dtype} {D} {Dv}: {float(err):.3g} of {float(want):.6g}, bound {float(bound):.3g}", flush=True)
        assert err.abs() <= bound
