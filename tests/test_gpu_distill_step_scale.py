"""distill_step's loss scale: float16 gradients of a mean over many rows against the formula in 64 bits, and what the scale
leaves as it was."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402
from ra_spmm import transformer as T  # noqa: E402


def ring(M):
    """Every node's neighbours: itself, the one before and the one after."""
    at = torch.arange(M, device="cuda")
    colind = torch.stack([(at - 1) % M, at, (at + 1) % M], 1).sort(1).values.flatten().int()
    return ra_spmm.make_attention_plan(torch.arange(0, 3 * M + 1, 3, dtype=torch.int32, device="cuda"), colind, M, M)


def teacher_of(M, C, k, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    teacher, top = torch.randn(M, k, generator=gen, device="cuda"), torch.randint(0, C, (M, k), generator=gen, device="cuda")
    return teacher, top, torch.randint(-1, C, (M,), generator=gen, device="cuda")


@pytest.mark.parametrize("scale", [None, 4096.0])
def test_float16_gradients_of_many_rows(scale):
    """20,000 rows of 500 nearly even classes at T = 1/4: T q / M = 2.5e-8 is below half of float16's smallest step, so without
    a scale every class that is not the teacher's has the gradient 0.

    The last map's weight gradient is sum_r g_r h_r, of the h that the model formed and g from its logits.  Scaled by s, an
    entry of g is off by half a step, max(2^-25, 2^-11 s |g|), and by what its float32 formula loses: at most 2^-11 |g| with room;
    the product's sums by at most M 2^-24 of the sum of its terms' magnitudes, and its two roundings to float16 (the product, and
    the division by s, below 2^-14 by half of 2^-24) by 2 * 2^-11 of the value and 2^-25 (1 + 1 / s)."""
    M, C, T_ = 20_000, 500, 0.25
    torch.manual_seed(4)
    model = T.DiffTransformer(0, 64, C, layers=1, heads=4, pre_norm=True, nodes=1000)
    model.last_norm.bias.data.fill_(1.0)  # so that what all classes lose does not cancel over the rows
    model.last.weight.data.mul_(0.01)
    model = model.cuda().half()
    ids = torch.randint(0, 1000, (M,), device="cuda")
    teacher, top, labels = teacher_of(M, C, 4, 1)
    seen = {}
    model.last.register_forward_hook(lambda m, i, o: seen.update(h=i[0].detach().double(), s=o.detach().double()))
    whole_sums = torch.backends.cuda.matmul.allow_fp16_reduced_precision_reduction
    torch.backends.cuda.matmul.allow_fp16_reduced_precision_reduction = False
    try:
        T.distill_step(model, ring(M), ids, teacher, top, torch.optim.SGD(model.parameters(), lr=0.0), T_, loss_scale=scale)
    finally:
        torch.backends.cuda.matmul.allow_fp16_reduced_precision_reduction = whole_sums
    p = torch.softmax(teacher.double() / T_, 1)
    g = torch.softmax(seen["s"] / T_, 1).scatter_add_(1, top, -p) * (T_ / M)
    s = scale or 32.0  # 20,000 rows: 2^15 / 1024
    h, want = seen["h"].abs(), g.t() @ seen["h"]
    assert (g[g > 0] < 2.0 ** -25).all() and (g > 0).any(1).all()  # all lost without a scale
    off = torch.maximum(g.abs() * 2.0 ** -11, torch.full_like(g, 2.0 ** -25 / s)) + g.abs() * 2.0 ** -11
    bound = off.t() @ h + M * 2.0 ** -24 * (g.abs().t() @ h) + 2 * 2.0 ** -11 * want.abs() + 2.0 ** -25 * (1 + 1 / s)
    err = (model.last.weight.grad.double() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())
    assert all(w.grad.isfinite().all() for w in model.parameters())


def test_a_scale_changes_nothing_in_float32():
    """Powers of two go through every operation of the backward pass without a rounding.  Gradients are added to what
    a parameter without an optimizer and the features have, and no hook stays behind."""
    M = 600
    plan, (teacher, top, labels) = ring(M), teacher_of(M, 9, 3, 2)
    results = []
    for scale in (None, 1.0, 2.0 ** 20):
        torch.manual_seed(1)
        model = T.DiffTransformer(16, 64, 9, layers=2, heads=4, pre_norm=True).cuda()
        X = torch.randn(M, 16, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).requires_grad_(True)
        X.grad = torch.full_like(X, 0.5)
        model.last.weight.grad = torch.full_like(model.last.weight, 2.0)
        optimizer = torch.optim.SGD([w for w in model.parameters() if w is not model.last.weight], lr=0.1)
        loss = T.distill_step(model, plan, X, teacher, top, optimizer, 2.0, labels, 0.3, loss_scale=scale)
        results.append([loss, X.grad, *(w.grad for w in model.parameters()), *(w.detach() for w in model.parameters())])
        assert not any(w._backward_hooks for w in (*model.parameters(), X))
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(*results))
    assert (results[0][1] != 0.5).any() and abs(float(results[0][1].mean()) - 0.5) < 0.1


@pytest.mark.parametrize("scale", [0.0, -1.0, math.inf, math.nan])
def test_scales_that_are_refused(scale):
    model = T.DiffTransformer(16, 64, 9, layers=1, heads=4)
    with pytest.raises(ValueError, match="loss_scale"):
        T.distill_step(model, None, None, None, None, torch.optim.SGD(model.parameters(), lr=0.1), loss_scale=scale)
