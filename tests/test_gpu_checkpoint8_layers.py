"""relu8 and linear8 as layers: under autocast, and what their backward pass allocates."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402
from ra_spmm import transformer as T  # noqa: E402


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("inside", [False, True], ids=["backward outside", "backward inside"])
def test_layers_under_autocast(dtype, inside):
    """float32 weights and inputs, products in 16 bits: the gradients that plain layers give, each to 16-bit rounding, in
    float32."""
    gen = torch.Generator().manual_seed(1)
    x, w1, w2 = (torch.randn(s, generator=gen).cuda() for s in ((300, 64), (96, 64), (40, 96)))
    g = torch.randn(300, 40, generator=gen).cuda()

    def run(plain):
        leaves = [t.clone().requires_grad_(True) for t in (x, w1, w2)]
        a, b, c = leaves
        with torch.autocast("cuda", dtype=dtype):
            if plain:
                y = F.linear(F.linear(a, b).relu(), c)
            else:
                h, kept = ra_spmm.relu8(ra_spmm.linear8(a, b))
                y = ra_spmm.linear8(h, c, kept)
            assert y.dtype == dtype
            if inside:
                y.backward(g.to(dtype))
        if not inside:
            y.backward(g.to(dtype))
        return y.detach(), [t.grad for t in leaves]

    (y0, want), (y, got) = run(True), run(False)
    assert torch.equal(y, y0)
    for a, b in zip(got, want):
        assert a.dtype == torch.float32
        # The plain gradients are rounded to 16 bits (2^-8 at most each); the kept inputs are 1/64 of their group's
        # largest value off at most.
        assert (a - b).norm() <= (2.0 ** -7 + 1 / 64) * b.norm()


def test_model_under_autocast():
    M = 200
    gen = torch.Generator().manual_seed(3)
    dense = torch.rand(M, M, generator=gen) < 0.1
    rowptr = torch.zeros(M + 1, dtype=torch.int32)
    rowptr[1:] = dense.sum(1).cumsum(0)
    plan = ra_spmm.make_attention_plan(rowptr.cuda(), dense.nonzero()[:, 1].to(torch.int32).cuda(), M, M)
    torch.manual_seed(4)
    model = T.DiffTransformer(32, 64, 5, heads=2, positions=M).cuda()
    X, pos = torch.randn(M, 32, generator=gen).cuda().requires_grad_(True), torch.arange(M, dtype=torch.int32, device="cuda")
    g = torch.randn(M, 5, generator=gen).cuda()
    model(X, plan, pos).backward(g)
    want, model_grads = X.grad.clone(), [p.grad.clone() for p in model.parameters()]
    X.grad = None
    model.zero_grad()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = model(X, plan, pos)
    y.backward(g.to(y.dtype))
    assert F.cosine_similarity(X.grad.flatten(), want.flatten(), 0) > 0.99
    for p, b in zip(model.parameters(), model_grads):
        assert p.grad.dtype == torch.float32 and F.cosine_similarity(p.grad.flatten(), b.flatten(), 0) > 0.98


def test_relu_backward_takes_no_memory_of_its_own():
    """The gradient of the input and nothing else; relu8's codes have no gradient, not one of zeros either."""
    rows, cols = 200_000, 128
    x, g = torch.randn(rows, cols, device="cuda", requires_grad=True), torch.randn(rows, cols, device="cuda")
    y, kept = ra_spmm.relu8(x)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    dx, = torch.autograd.grad(y, x, g)
    assert torch.cuda.max_memory_allocated() - before <= rows * cols * 4 + (1 << 20)
    assert torch.equal(dx, g * (x.detach() > 0))


def test_relu_whose_output_takes_no_part():
    x = torch.randn(50, 40, device="cuda", requires_grad=True)
    y, kept = ra_spmm.relu8(x)
    (x * 2 + 0 * y.detach()).sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 2))
    w = torch.randn(7, 40, device="cuda", requires_grad=True)
    h, kept = ra_spmm.relu8(x.detach())  # an input without a gradient
    ra_spmm.linear8(h, w, kept).sum().backward()
    assert w.grad.shape == (7, 40)
