"""diff_attention where no gradients are recorded."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_a_learned_bias_without_gradients(mode):
    """A bias that requires a gradient is refused where one would be recorded, and taken as it is where none is."""
    rowptr = torch.tensor([0, 2, 2, 5], dtype=torch.int32, device="cuda")
    colind = torch.tensor([0, 3, 1, 2, 3], dtype=torch.int32, device="cuda")
    plan = ra_spmm.make_attention_plan(rowptr, colind, 3, 4)
    q, k, v = (torch.randn(s, device="cuda", requires_grad=True) for s in ((3, 2, 2, 8), (4, 2, 2, 8), (4, 2, 16)))
    lam = torch.tensor([0.5], device="cuda")
    bias = torch.randn(5, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="bias"):
        ra_spmm.diff_attention(plan, q, k, v, lam, bias=bias)
    with mode():
        out = ra_spmm.diff_attention(plan, q, k, v, lam, bias=bias)
    assert not out.requires_grad
    assert torch.equal(out, ra_spmm.diff_attention(plan, q, k, v, lam, bias=bias.detach()).detach())
