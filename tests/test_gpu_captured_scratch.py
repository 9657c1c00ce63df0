"""A captured run names its plan's scratch: later runs of larger shapes, other plans and their runs leave the replays
right."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402
from ra_spmm import synthetic as S  # noqa: E402


def _capture(body):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        body()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = body()
    return graph, out


def _lists(seed):
    """Rows and columns of up to 3,000 edges, cut on both sides."""
    rng = np.random.default_rng(seed)
    lengths = [3000, 0, 2, 777] + [260] * 60
    rowptr = torch.zeros(len(lengths) + 1, dtype=torch.int32)
    rowptr[1:] = torch.tensor(lengths).cumsum(0)
    colind = np.concatenate([np.sort(rng.integers(0, 50, n)) for n in lengths]).astype(np.int32)
    return rowptr.cuda(), torch.from_numpy(colind).cuda(), len(lengths), 50


def _inputs(M, K, H, D, Dv, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    return r(M, H, 2, D), r(K, H, 2, D), r(K, H, Dv), torch.rand(H, generator=g, device="cuda"), r(M, H, Dv)


@pytest.mark.parametrize("train", [False, True], ids=["forward", "step"])
def test_attention_plan(train):
    rp, ci, M, K = _lists(3)
    plan = ra_spmm.make_attention_plan(rp, ci, M, K)
    q, k, v, lam, g = _inputs(M, K, 2, 16, 32, 1)

    def body():
        out, stats = ra_spmm.run_attention_plan_train(plan, q, k, v, lam)
        return (out, *ra_spmm.run_attention_plan_backward(plan, q, k, v, lam, stats, g)) if train else (out,)

    eager = [x.clone() for x in body()]
    graph, outs = _capture(body)
    larger = _inputs(M, K, 8, 32, 64, 2)
    others = []
    for i in range(3):
        out, stats = ra_spmm.run_attention_plan_train(plan, *larger[:4])
        ra_spmm.run_attention_plan_backward(plan, *larger[:4], stats, larger[4])
        # Plans whose scratch is of the captured sizes, and holds other values.
        others.append(ra_spmm.make_attention_plan(rp, ci, M, K))
        b = _inputs(M, K, 2, 16, 32, 5 + i)
        want, st = ra_spmm.run_attention_plan_train(others[-1], *b[:4])
        ra_spmm.run_attention_plan_backward(others[-1], *b[:4], st, b[4])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(outs, eager)), i
        assert torch.equal(ra_spmm.run_attention_plan(others[-1], *b[:4]), want)


def test_zero_overhead_plan():
    g = S.random_csr(3000, 3000, 20.0, seed=5, skew=1.4)
    rp, ci, vl = g.torch("cuda")
    plan = ra_spmm.make_zero_overhead_plan(rp.cpu(), g.M, g.K)
    B, wide = torch.randn(g.K, 32, device="cuda"), torch.randn(g.K, 512, device="cuda")
    body = lambda: ra_spmm.run_zero_overhead_plan(plan, rp, ci, vl, B)  # noqa: E731
    eager = body().clone()
    graph, out = _capture(body)
    for i in range(3):
        ra_spmm.run_zero_overhead_plan(plan, rp, ci, vl, wide)
        other = ra_spmm.make_zero_overhead_plan(rp.cpu(), g.M, g.K)
        ra_spmm.run_zero_overhead_plan(other, rp, ci, vl, 2 * B)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), i
