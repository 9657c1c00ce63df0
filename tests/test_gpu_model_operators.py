"""Embedding lookup, layer norm and distillation as a model uses them together: every gradient of one training step against
the same model in 64 bits, and the step captured into a graph."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import ra_spmm  # noqa: E402
from ra_spmm import transformer as T  # noqa: E402
from test_gpu_transformer import graph, norm, rotated  # noqa: E402


def model_of(nodes, **kw):
    torch.manual_seed(2)
    return T.DiffTransformer(0, 64, 9, layers=2, heads=4, kv_heads=2, positions=512, pre_norm=True, nodes=nodes, **kw)


def layer_norm(x, m):
    c = x - x.mean(1, keepdim=True)
    return c / (c.square().mean(1, keepdim=True) + m.eps).sqrt() * m.weight.double() + m.bias.double()


def plain(model, ids, dense, positions):
    """The model from elementary float64 operations on dense attention maps."""
    table = model.nodes.double()
    x = torch.where((ids >= 0)[:, None], table[ids.clamp(min=0)] * math.sqrt(table.shape[1]), 0.0)
    for m in model.layers:
        p = {n: w.double() for n, w in m.named_parameters()}
        h, g, d = m.heads, m.kv_heads, m.head_dim
        q, k, v = (layer_norm(x, m.in_norm) @ p["qkv"].t()).split([2 * h * d, 2 * g * d, 2 * g * d], 1)
        q, k = (rotated(norm(t.unflatten(1, (n, 2, d)), w, m.eps), model.table.double(), positions)
                for t, n, w in ((q, h, p["q_norm"]), (k, g, p["k_norm"])))
        v = v.unflatten(1, (g, 2 * d))
        e = (p["lam_a"] * p["lam_b"]).sum(-1).exp()
        lam = e[0] - e[1] + m.lam0
        out = []
        for i in range(h):
            maps = []
            for a in range(2):
                score = (q[:, i, a] @ k[:, i * g // h, a].t() / math.sqrt(d)).masked_fill(~dense, -1e30)
                w = (score - score.amax(1, keepdim=True).detach()).exp() * dense
                maps.append(w / w.sum(1, keepdim=True).clamp_min(1e-300))
            out.append((maps[0] - lam[i] * maps[1]) @ v[:, i * g // h])
        o = norm(torch.stack(out, 1), p["o_norm"], m.eps).flatten(1)
        x = x + (1 - m.lam0) * o @ p["out"].t()
        x = x + (layer_norm(x, m.mid_norm) @ p["up"].t()).relu() @ p["down"].t()
    return layer_norm(x, model.last_norm) @ model.last.weight.double().t()


def data(M, nodes, seed=1):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, nodes, (M,), generator=g)
    ids[::17] = -1  # nodes that no row of the table belongs to
    labels = torch.randint(-1, 9, (M,), generator=g)
    teacher, top = torch.randn(M, 9, generator=g).mul(3).topk(4, dim=1)
    top[5::11, 2:], top[7] = -1, -1
    return ids, torch.randint(0, 512, (M,), dtype=torch.int32, generator=g), labels, teacher, top


def exact_loss(logits, teacher, top, labels, T_, hard):
    used = top >= 0
    p = torch.where(used, (teacher.double() / T_).exp(), 0.0)
    p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
    log_q = (logits / T_).log_softmax(1).gather(1, top.clamp(min=0))
    kl = torch.where(used, p * (p.clamp_min(1e-300).log() - log_q), 0.0).sum(1)
    ce = torch.where(labels >= 0, -logits.log_softmax(1).gather(1, labels.clamp(min=0)[:, None])[:, 0], 0.0)
    return ((1 - hard) * T_ * T_ * kl + hard * ce).mean()


def test_a_step_against_64_bits():
    """float32 throughout (keep8=False), the tolerances of test_gpu_transformer_exact.py: 1e-4 of the logits and the loss,
    1e-3 of the gradients in norm, 1e-2 of lam's, which cancel."""
    M, nodes = 300, 120
    dense, rowptr, colind = graph(M, 1)
    ids, positions, labels, teacher, top = data(M, nodes)
    model, cpu = model_of(nodes, keep8=False).cuda(), model_of(nodes)
    cpu.load_state_dict({n: w.cpu() for n, w in model.state_dict().items()})
    plan = ra_spmm.make_attention_plan(rowptr.cuda(), colind.cuda(), M, M)
    optimizer = torch.optim.SGD(model.parameters(), lr=0.0)
    loss = T.distill_step(model, plan, ids.cuda(), teacher.cuda(), top.cuda(), optimizer, 2.0, labels.cuda(), 0.3, positions.cuda())
    logits = plain(cpu, ids, dense, positions)
    want = exact_loss(logits, teacher, top, labels, 2.0, 0.3)
    want.backward()
    assert abs(float(loss) - float(want)) < 1e-4 * float(want)
    with torch.no_grad():
        got = model(ids.cuda(), plan, positions.cuda()).cpu().double()
    assert (got - logits).norm() < 1e-4 * logits.norm()
    for (n, a), (_, b) in zip(model.named_parameters(), cpu.named_parameters()):
        err = float((a.grad.cpu().double() - b.grad.double()).norm() / b.grad.double().norm())
        assert err < (1e-2 if "lam" in n else 1e-3), (n, err)
    unused = torch.ones(nodes, dtype=torch.bool)
    unused[ids[ids >= 0]] = False
    assert unused.any() and not model.nodes.grad[unused.cuda()].any()
    # The same through autograd.
    before = [w.grad.clone() for w in model.parameters()]
    model.zero_grad(set_to_none=True)
    loss2 = ra_spmm.distill_loss(model(ids.cuda(), plan, positions.cuda()), teacher.cuda(), top.cuda(), 2.0, labels.cuda(), 0.3)
    loss2.backward()
    assert abs(float(loss2.detach()) - float(loss)) < 1e-6 * float(want)
    for (n, w), b in zip(model.named_parameters(), before):
        assert (w.grad - b).norm() < 1e-5 * b.norm(), n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_types(dtype):
    """A model converted to 16 bits and one under autocast run, with gradients for every parameter."""
    M, nodes = 300, 120
    _, rowptr, colind = graph(M, 1)
    ids, positions, labels, teacher, top = (t.cuda() for t in data(M, nodes))
    plan = ra_spmm.make_attention_plan(rowptr.cuda(), colind.cuda(), M, M)
    model = model_of(nodes).cuda().to(dtype)
    optimizer = torch.optim.SGD(model.parameters(), lr=1e-3)
    assert T.distill_step(model, plan, ids, teacher, top, optimizer, 2.0, labels, 0.3, positions).isfinite()
    assert all(w.grad is not None and w.grad.isfinite().all() for w in model.parameters())
    model = model_of(nodes).cuda()
    optimizer = torch.optim.SGD(model.parameters(), lr=1e-3)
    with torch.autocast("cuda", dtype=dtype):
        logits = model(ids, plan, positions)
        loss, grad = ra_spmm.distill_loss_grad(logits.detach(), teacher, top, 2.0, labels, 0.3, factor=1024.0)
    logits.backward(grad)
    assert logits.dtype == dtype and loss.isfinite()
    assert all(w.grad is not None and w.grad.dtype == torch.float32 and w.grad.isfinite().all() for w in model.parameters())


def test_options_leave_the_default_model_as_it_was():
    a = [n for n, _ in T.DiffTransformer(8, 16, 2, layers=1, heads=2).named_parameters()]
    assert not any("in_norm" in n or "mid_norm" in n or "last_norm" in n or n == "nodes" for n in a) and "first.weight" in a


def test_a_captured_step():
    """Two captured graphs of the operators' step that share a memory pool, replayed in turn with eager work between them."""
    M, V, D, C = 900, 200, 48, 40
    gen = torch.Generator("cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    state = {"ids": torch.randint(0, V, (M,), device="cuda"), "table": r(V, D), "w": r(D), "b": r(D), "out": r(C, D),
             "labels": torch.randint(-1, C, (M,), device="cuda")}
    state["teacher"], state["top"] = r(M, C).topk(5, dim=1)

    def step():
        table, w, b, out = (state[n].detach().requires_grad_(True) for n in ("table", "w", "b", "out"))
        x = ra_spmm.embed(state["ids"], table, 2.0)
        y, h = ra_spmm.layer_norm(x, w, b, residual=x * 0.5)
        logits = y @ out.t() + h[:, :C]
        loss = ra_spmm.distill_loss(logits, state["teacher"], state["top"], 2.0, state["labels"], 0.3)
        return [loss.detach(), *torch.autograd.grad(loss, (table, w, b, out))]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(step())
        graphs.append(g)
    for i in range(6):
        for n in ("table", "w", "b", "out", "teacher"):
            state[n].normal_(generator=gen)
        state["ids"].random_(0, V)
        want = [t.clone() for t in step()]
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        for a, b in zip(outs[i % 2], want):
            assert torch.equal(a, b), i


def test_second_derivatives_are_refused():
    """They raise where they are differentiated; a first derivative with create_graph is the same as without."""
    table, x = torch.randn(9, 16, device="cuda", requires_grad=True), torch.randn(5, 16, device="cuda", requires_grad=True)
    w = torch.rand(16, device="cuda", requires_grad=True)
    ids = torch.tensor([1, 2, 3, 1, 8], device="cuda")
    teacher, top = torch.randn(5, 16, device="cuda").topk(3, dim=1)
    for f, leaf in ((lambda: (ra_spmm.embed(ids, table) * x).sum(), table), (lambda: (ra_spmm.layer_norm(x, w) * table[:5]).sum(), w),
                    (lambda: ra_spmm.layer_norm(x, w, residual=x)[0].square().sum(), x),
                    (lambda: ra_spmm.distill_loss(x * 2.0, teacher, top), x)):
        plain, = torch.autograd.grad(f(), leaf)
        first, = torch.autograd.grad(f(), leaf, create_graph=True)
        assert torch.equal(first.detach(), plain)
        with pytest.raises(RuntimeError, match="twice"):
            first.square().sum().backward()


def test_gradients_that_are_switched_off():
    """No graph under no_grad, nor of inputs without gradients; a frozen table below a trained norm."""
    table, w = torch.randn(9, 16, device="cuda"), torch.ones(16, device="cuda", requires_grad=True)
    ids = torch.tensor([1, 2, 3], device="cuda")
    x = ra_spmm.embed(ids, table)
    assert not x.requires_grad
    y = ra_spmm.layer_norm(x, w)
    assert y.requires_grad and torch.autograd.grad(y.sum(), w)[0].shape == (16,)
    with torch.no_grad():
        assert not ra_spmm.layer_norm(x, w).requires_grad
        assert not ra_spmm.embed(ids, table.requires_grad_(True)).requires_grad
        assert not ra_spmm.distill_loss(w[None], x[:1, :2], ids[None, :2]).requires_grad
    with torch.inference_mode():
        assert not ra_spmm.layer_norm(x, w, residual=x)[1].requires_grad


def test_inputs_changed_after_the_forward_pass():
    """What a backward pass has kept must not have changed."""
    x, w = torch.randn(5, 16, device="cuda"), torch.ones(16, device="cuda", requires_grad=True)
    y = ra_spmm.layer_norm(x, w)
    x.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
