"""The operators under torch's transformations other than reverse-mode autograd, on tensors of the GPU."""
import re

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402


def inputs():
    gen = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(6, 8, generator=gen, device="cuda")
    teacher, top = torch.randn(6, 8, generator=gen, device="cuda").topk(3, dim=1)
    rowptr = torch.arange(7, dtype=torch.int32, device="cuda")
    plan = ra_spmm.make_attention_plan(rowptr, torch.arange(6, dtype=torch.int32, device="cuda").flip(0).contiguous(), 6, 6)
    q, v = torch.randn(6, 2, 2, 8, generator=gen, device="cuda"), torch.randn(6, 2, 8, generator=gen, device="cuda")
    return x, torch.rand(8, generator=gen, device="cuda"), teacher, top, plan, q, v, torch.ones(2, device="cuda")


def operators(x, w, teacher, top, plan, q, v, lam):
    ids = torch.tensor([1, 5, 0], device="cuda")
    return {
        "embed": (x, lambda t: ra_spmm.embed(ids, t)),
        "layer_norm": (x, lambda t: ra_spmm.layer_norm(t, w)),
        "layer_norm weight": (w, lambda t: ra_spmm.layer_norm(x, t)),
        "layer_norm residual": (x, lambda t: ra_spmm.layer_norm(x, w, residual=t)[0]),
        "distill_loss": (x, lambda t: ra_spmm.distill_loss(t, teacher, top)),
        "head_norm_rotate": (q, lambda t: ra_spmm.head_norm_rotate(t, None, w, None)[0]),
        "diff_attention": (q, lambda t: ra_spmm.diff_attention(plan, t, q, v, lam)),
        "diff_attention lam": (lam, lambda t: ra_spmm.diff_attention(plan, q, q, v, t)),
        "relu8": (x, lambda t: ra_spmm.relu8(t)[0]),
    }


NAMES = ["embed", "layer_norm", "layer_norm weight", "layer_norm residual", "distill_loss", "head_norm_rotate", "diff_attention",
         "diff_attention lam", "relu8"]


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name, requires_grad):
    """Whether a gradient is required beside it or not."""
    at, f = operators(*inputs())[name]
    with forward_ad.dual_level():
        leaf = at.clone().requires_grad_(requires_grad)
        dual = forward_ad.make_dual(leaf, torch.ones_like(at))
        with pytest.raises((RuntimeError, NotImplementedError), match="forward-mode tangent|jvp|forward mode"):
            f(dual)
    assert torch.equal(f(at), f(at.clone().requires_grad_(True)).detach())


@pytest.mark.parametrize("name", NAMES)
def test_a_tangent_of_the_incoming_gradient_is_refused(name):
    at, f = operators(*inputs())[name]
    leaf = at.clone().requires_grad_(True)
    y = f(leaf)
    with forward_ad.dual_level():
        g = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(RuntimeError, match="forward-mode tangent"):
            torch.autograd.grad(y, leaf, g)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.filterwarnings("ignore")
def test_traces(name):
    """Refused, or right on other inputs than those of the trace."""
    at, f = operators(*inputs())[name]
    if name.split()[0] in ("embed", "layer_norm", "distill_loss"):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, (at,), check_trace=False)
        return
    traced = torch.jit.trace(f, (at,), check_trace=False)
    for factor in (1.0, -0.5, 2.0):
        other = at * factor
        torch.empty(1 << 20, device="cuda").fill_(float("nan"))  # what unwritten memory would hold
        assert torch.equal(traced(other), f(other)), factor


@pytest.mark.parametrize("name", NAMES)
def test_views_of_negated_values(name):
    """Memory that holds the opposite of the tensor's values, as the imaginary part of a conjugate."""
    at, f = operators(*inputs())[name]
    view = torch.complex(torch.zeros_like(at), at).conj().imag
    for t in (view, torch._neg_view(at)):
        assert t.is_neg() and torch.equal(t, -at)
        try:
            y = f(t)
        except RuntimeError as e:  # weights are taken as they lie
            assert at.dim() == 1 and re.search("negated|contiguous", str(e))
        else:
            assert torch.equal(y, f(-at))
    leaf = at.clone().requires_grad_(True)
    y = f(leaf)
    g = torch.randn(y.shape, generator=torch.Generator("cuda").manual_seed(2), device="cuda")
    want, = torch.autograd.grad(y, leaf, -g, retain_graph=True)
    try:
        got, = torch.autograd.grad(y, leaf, torch._neg_view(g))
    except RuntimeError as e:
        assert "negated" in str(e)
    else:
        assert torch.equal(got, want)


@pytest.mark.parametrize("inside", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_transformations_of_torch_func_are_refused(name, inside):
    """Of an argument, and around a call on tensors from outside, whose outputs would have no memory."""
    at, f = operators(*inputs())[name]

    for transform in (torch.func.functionalize, torch.func.grad, torch.func.vmap):
        def call(x):
            with pytest.raises(RuntimeError, match=None if transform is torch.func.vmap else "functional wrapper|torch.func|functorch|storage"):
                f(at if inside else x)
            return (x * 2).sum()

        transform(call)(at)


def test_products_inside_of_transformations_are_refused():
    rowptr, colind = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    vals, B = torch.ones(2, device="cuda"), torch.ones(2, 4, device="cuda")
    plan = ra_spmm._C.make_zero_overhead_plan(rowptr, 2, 2)

    def call(x):
        for f in (lambda: ra_spmm._C.spmm_csr_direct(rowptr, colind, vals, B), lambda: ra_spmm._C.spmm_cusparse(rowptr, colind, vals, B),
                  lambda: ra_spmm._C.run_zero_overhead_plan(plan, rowptr, colind, vals, B)):
            with pytest.raises(RuntimeError, match="torch.func"):
                f()
        return (x * 2).sum()

    for transform in (torch.func.functionalize, torch.func.grad, torch.func.vmap):
        transform(call)(B)
    assert torch.equal(ra_spmm._C.spmm_csr_direct(rowptr, colind, vals, B), B)
