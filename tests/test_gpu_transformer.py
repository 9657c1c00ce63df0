"""The graph transformer runs the operators together: logits and input gradient against the same model in 64 bits from
elementary operations, training lowers the loss.

Weight gradients come from inputs kept in 8 bits, each value within 1/64 of its group's largest magnitude (half a step of
1/128 but for the group's largest): they are held to the direction of the exact ones, cos > 0.999."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402
from ra_spmm import transformer as T  # noqa: E402


def graph(M, seed):
    g = torch.Generator().manual_seed(seed)
    dense = torch.rand(M, M, generator=g) < 0.05
    dense[3] = False  # a node without neighbours
    dense[5] = True   # a hub
    rowptr = torch.zeros(M + 1, dtype=torch.int32)
    rowptr[1:] = dense.sum(1).cumsum(0)
    return dense, rowptr, dense.nonzero()[:, 1].to(torch.int32)


def norm(x, w, eps):
    return x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w


def rotated(x, table, pos):
    half = table.shape[1]
    c, s = table[pos.long(), :, 0][:, None, None], table[pos.long(), :, 1][:, None, None]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * c - b * s, a * s + b * c, x[..., 2 * half:]], -1)


def plain(model, X, dense, positions, bias):
    """The model from elementary float64 operations on dense attention maps."""
    x = X @ model.first.weight.double().t()
    on = dense & (bias > -math.inf)
    for m in model.layers:
        p = {n: w.double() for n, w in m.named_parameters()}
        h, g, d = m.heads, m.kv_heads, m.head_dim
        rows = x @ p["qkv"].t()
        q, k, v = rows.split([2 * h * d, 2 * g * d, 2 * g * d], 1)
        q, k = (rotated(norm(t.unflatten(1, (n, 2, d)), w, m.eps), model.table.double(), positions)
                for t, n, w in ((q, h, p["q_norm"]), (k, g, p["k_norm"])))
        v = v.unflatten(1, (g, 2 * d))
        e = (p["lam_a"] * p["lam_b"]).sum(-1).exp()
        lam = e[0] - e[1] + m.lam0
        out = []
        for i in range(h):
            maps = []
            for a in range(2):
                score = (q[:, i, a] @ k[:, i * g // h, a].t() / math.sqrt(d) + torch.where(on, bias, 0.0)).masked_fill(~on, -1e30)
                w = (score - score.amax(1, keepdim=True).detach()).exp() * on
                maps.append(w / w.sum(1, keepdim=True).clamp_min(1e-300))
            out.append((maps[0] - lam[i] * maps[1]) @ v[:, i * g // h])
        o = norm(torch.stack(out, 1), p["o_norm"], m.eps).flatten(1)
        x = x + (1 - m.lam0) * o @ p["out"].t()
        x = x + (x @ p["up"].t()).relu() @ p["down"].t()
    return x @ model.last.weight.double().t()


@pytest.mark.parametrize("masked", [False, True], ids=["open", "masked"])
@pytest.mark.parametrize("kv_heads", [4, 2])
def test_model_against_64_bits(kv_heads, masked):
    M = 300
    dense, rowptr, colind = graph(M, 1)
    torch.manual_seed(2)
    model = T.DiffTransformer(40, 64, 7, layers=2, heads=4, kv_heads=kv_heads, positions=512).cuda()
    cpu = T.DiffTransformer(40, 64, 7, layers=2, heads=4, kv_heads=kv_heads, positions=512)
    cpu.load_state_dict({n: w.cpu() for n, w in model.state_dict().items()})
    X, g = torch.randn(M, 40), torch.randn(M, 7)
    positions = torch.randint(0, 512, (M,), dtype=torch.int32)
    bias = torch.randn(M, M)
    bias[torch.rand(M, M) < 0.1] = -math.inf
    bias[7] = -math.inf  # a node whose mask leaves nothing
    if not masked:
        bias.zero_()
    plan = ra_spmm.make_attention_plan(rowptr.cuda(), colind.cuda(), M, M)
    Xd, X64 = X.cuda().requires_grad_(True), X.double().requires_grad_(True)
    logits = model(Xd, plan, positions.cuda(), bias[dense].cuda() if masked else None)
    logits.backward(g.cuda())
    want = plain(cpu, X64, dense, positions, bias.double())
    want.backward(g.double())
    assert (logits.detach().cpu().double() - want).norm() < 1e-4 * want.norm()
    assert (Xd.grad.cpu().double() - X64.grad).norm() < 1e-3 * X64.grad.norm()
    for (n, a), (_, b) in zip(model.named_parameters(), cpu.named_parameters()):
        cos = F.cosine_similarity(a.grad.cpu().double().flatten(), b.grad.double().flatten(), 0)
        assert cos > 0.999, (n, float(cos))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_training_lowers_the_loss(dtype):
    M = 400
    dense, rowptr, colind = graph(M, 5)
    torch.manual_seed(6)
    X = torch.randn(M, 32)
    y = (X @ torch.randn(32, 5)).argmax(1).cuda()
    X = X.cuda().to(dtype)
    model = T.DiffTransformer(32, 64, 5, heads=2, positions=M).cuda().to(dtype)
    model.table = model.table.float()
    plan = ra_spmm.make_attention_plan(rowptr.cuda(), colind.cuda(), M, M)
    positions = torch.arange(M, dtype=torch.int32, device="cuda")
    opt = torch.optim.Adam(model.parameters(), lr=1e-2)
    losses = [float(T.train_step(model, plan, X, y, opt, positions)) for _ in range(40)]
    assert all(math.isfinite(x) for x in losses) and losses[-1] < 0.7 * losses[0], losses[::8]


def test_sizes_are_checked():
    with pytest.raises(ValueError, match="multiple"):
        T.DiffTransformerLayer(60, 4)
    with pytest.raises(ValueError, match="multiple"):
        T.DiffTransformerLayer(64, 4, kv_heads=3)
    with pytest.raises(ValueError, match="positions"):
        T.DiffTransformer(8, 16, 2, heads=2)(torch.zeros(1, 8), None, torch.zeros(1, dtype=torch.int32))
