"""A DiffTransformer that keeps its layers' inputs as they are: every gradient against the model in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402
from ra_spmm import transformer as T  # noqa: E402
from test_gpu_transformer import graph, plain  # noqa: E402


@pytest.mark.parametrize("kv_heads", [4, 2])
def test_exact_gradients(kv_heads):
    """float32 throughout: as the logits and the input's gradient of test_gpu_transformer.py, within 1e-3 in norm (lam's
    gradients cancel: 1e-2)."""
    M = 300
    dense, rowptr, colind = graph(M, 1)
    torch.manual_seed(2)
    model = T.DiffTransformer(40, 64, 7, layers=2, heads=4, kv_heads=kv_heads, positions=512, keep8=False).cuda()
    cpu = T.DiffTransformer(40, 64, 7, layers=2, heads=4, kv_heads=kv_heads, positions=512)
    cpu.load_state_dict({n: w.cpu() for n, w in model.state_dict().items()})
    X, g = torch.randn(M, 40), torch.randn(M, 7)
    positions = torch.randint(0, 512, (M,), dtype=torch.int32)
    plan = ra_spmm.make_attention_plan(rowptr.cuda(), colind.cuda(), M, M)
    logits = model(X.cuda(), plan, positions.cuda())
    logits.backward(g.cuda())
    want = plain(cpu, X.double(), dense, positions, torch.zeros(M, M, dtype=torch.float64))
    want.backward(g.double())
    assert (logits.detach().cpu().double() - want).norm() < 1e-4 * want.norm()
    for (n, a), (_, b) in zip(model.named_parameters(), cpu.named_parameters()):
        err = float((a.grad.cpu().double() - b.grad.double()).norm() / b.grad.double().norm())
        assert err < (1e-2 if "lam" in n else 1e-3), (n, err)
    with torch.no_grad():
        assert torch.equal(model(X.cuda(), plan, positions.cuda()), logits)


def test_the_default_keeps_8_bits():
    assert all(m.keep8 for m in T.DiffTransformer(8, 16, 2, heads=2).layers)
