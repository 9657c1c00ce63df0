"""The operators under torch's transformations other than reverse-mode autograd, on a host without a GPU: what they cannot take
part in is refused before anything else is looked at, where a result without its tangent would be silently wrong."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import ra_spmm
from ra_spmm import _C

X, IDS = torch.ones(4, 8), torch.zeros(4, 2, dtype=torch.int64)
W = torch.ones(8)


def calls(dual):
    """Every operator with one input after the other carrying a tangent."""
    x, w = dual(X), dual(W)
    yield lambda: ra_spmm.embed(IDS, x)
    yield lambda: ra_spmm.layer_norm(x)
    yield lambda: ra_spmm.layer_norm(X, w)
    yield lambda: ra_spmm.layer_norm(X, W, w)
    yield lambda: ra_spmm.layer_norm(X, residual=x)
    yield lambda: ra_spmm.layer_norm(x.view(2, 2, 8), residual=X.view(2, 2, 8))
    yield lambda: ra_spmm.distill_loss(x, X[:, :2], IDS)
    yield lambda: ra_spmm.distill_loss(X, x[:, :2], IDS)
    yield lambda: ra_spmm.distill_loss_grad(x, X[:, :2], IDS)
    yield lambda: ra_spmm.head_norm_rotate(x, None, W, None)
    yield lambda: ra_spmm.pack8(x)
    yield lambda: ra_spmm.relu_pack8(x)


@pytest.mark.parametrize("n", range(12))
def test_forward_mode_is_refused(n):
    with forward_ad.dual_level():
        call = list(calls(lambda t: forward_ad.make_dual(t, torch.ones_like(t))))[n]
        with pytest.raises(RuntimeError, match="forward-mode tangent"):
            call()
    with pytest.raises(RuntimeError, match="CUDA"):  # the same call without tangents
        list(calls(lambda t: t))[n]()


def test_tangents_may_be_switched_off():
    with forward_ad.dual_level():
        x = forward_ad.make_dual(X, X)
        with forward_ad._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="CUDA"):
            _C.embed(IDS, x, 1.0, None)


@pytest.mark.parametrize("n", range(4))
def test_traces_are_refused(n):
    """A tracer would keep the output's allocation and no launch: its replay would return memory that nobody wrote."""
    f = [lambda x: ra_spmm.embed(IDS, x), lambda x: ra_spmm.layer_norm(x, residual=x)[0], lambda x: ra_spmm.distill_loss(x, x[:, :2], IDS),
         lambda x: ra_spmm.distill_loss_grad(x, x[:, :2], IDS)[1]][n]
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(f, (X,), check_trace=False)


@pytest.mark.parametrize("n,mode", [(n, "real") for n in range(12)] + [(n, "fake") for n in (0, 1, 2, 9, 10, 11)])
def test_proxies_are_refused(n, mode):
    def f(x):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            list(calls(lambda t: x if t is X else t))[n]()
        return x + 1

    make_fx(f, tracing_mode=mode)(X.clone())


@pytest.mark.parametrize("n", [0, 1, 5, 6, 8, 9, 10, 11])
def test_functional_wrappers_are_refused(n):
    """Their storage is empty: the address of a view is its offset, which must not reach a launch."""
    def f(x):
        view = torch.cat([x, x])[4:]
        assert 0 < view.data_ptr() < 4096
        with pytest.raises(RuntimeError, match="functional wrapper"):
            list(calls(lambda t: view if t is X else t))[n]()
        return x + 1

    torch.func.functionalize(f)(X.clone())


def test_functional_wrappers_of_a_matrix_are_refused():
    rowptr, colind, vals = torch.tensor([0, 1, 2], dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32), torch.ones(2)

    def f(rowptr, colind, vals, B):
        for call in (lambda: _C.spmm_csr_direct(rowptr, colind, vals, B), lambda: _C.spmm_cusparse(rowptr, colind, vals, B),
                     lambda: _C.make_attention_plan(rowptr, colind, 2, 2), lambda: _C.compute_features(rowptr, 2, 2, 4),
                     lambda: _C.analyze_matrix(rowptr, colind, 2, 2, 4), lambda: _C.make_zero_overhead_plan(rowptr, 2, 2, "host")):
            with pytest.raises(RuntimeError, match="functional wrapper"):
                call()
        return B + 1

    torch.func.functionalize(f)(rowptr, colind, vals, torch.ones(2, 4))


@pytest.mark.parametrize("transform", [torch.func.functionalize, torch.func.grad, torch.func.vmap])
def test_host_calls_inside_of_transformations_are_refused(transform):
    """On tensors from outside of it: what is allocated inside has no memory."""
    rowptr, colind = torch.tensor([0, 1, 2], dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)

    def f(x):
        with pytest.raises(RuntimeError, match="torch.func"):
            _C.analyze_matrix(rowptr, colind, 2, 2, 4)
        return (x + 1).sum()

    transform(f)(torch.ones(3))
    assert _C.analyze_matrix(rowptr, colind, 2, 2, 4)
