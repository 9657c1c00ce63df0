"""Operators at the two ends of a graph model and between its layers: what their calls cost and what they have to return.

``own`` chooses what ``run`` computes with: elementary torch operations in 32 bits (false), or the operators of
``ra_spmm`` (true).  A case's ``kind`` says what a program does:

  embed         rows of a table by id, times a factor, inference
  embed_step    the same and the table's gradient
  ln            layer norm of every row, inference
  ln_step       layer norm of x, or of h = x + residual (then h is an output too): outputs and all gradients
  distill       loss of a student's logits against a teacher's largest ones, one value per row
  distill_step  mean loss and the gradient of the logits, through autograd
  distill_grad  mean loss and the gradient of the logits in one call

embed: out[i] = scale * table[ids[i]], zeros where ids[i] is the padding id; the gradient of table row v is scale times
the sum of the gradients of v's positions.

layer norm: n = (h - mean(h)) / sqrt(mean((h - mean(h))^2) + eps), y = n * w + b.  h is x + residual in the inputs' type.

distill, for a row of student logits s [C] with kept teacher entries (id_e, t_e): p = softmax(t / T) over the entries with
id_e >= 0, kl = sum_e p_e (log p_e - log softmax(s / T)[id_e]), ce = -log softmax(s)[label] where label >= 0, and the row's
loss is (1 - hard) * T^2 * kl + hard * ce.  A row without an entry (label) has no kl (ce).
"""
import math

import torch

own = False

DEVICE = "cuda"
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


# ------------------------------------------------------------------ the list
def listed():
    return [
        # Serving: the embedding of one node that a request names; latency.
        {"name": "embed_1_bf16", "kind": "embed", "n": 1, "V": 200_000, "D": 256, "ids": "even", "padded": 0.0,
         "dtype": "bf16"},
        # A sampled mini-batch of a node table, popular nodes more often, padded to its size.
        {"name": "embed_step_8k_of_200k_f32", "kind": "embed_step", "n": 8_192, "V": 200_000, "D": 128, "ids": "popular",
         "padded": 0.05, "dtype": "f32"},
        # Types of all nodes: few table rows, each with thousands of positions; an odd width.
        {"name": "embed_step_1m_types_f16", "kind": "embed_step", "n": 1_000_000, "V": 61, "D": 100, "ids": "popular",
         "padded": 0.0, "dtype": "f16"},
        # Largest table: as many positions as rows.
        {"name": "embed_step_1m_of_1m_bf16", "kind": "embed_step", "n": 1_000_000, "V": 1_000_000, "D": 256,
         "ids": "even", "padded": 0.0, "dtype": "bf16"},
        # Serving: the stream of one node.
        {"name": "ln_1x256_bf16", "kind": "ln", "M": 1, "D": 256, "residual": False, "dtype": "bf16"},
        # A width that fits no packet, rows of 294 bytes.
        {"name": "ln_step_150k_147_f16", "kind": "ln_step", "M": 150_000, "D": 147, "residual": False, "dtype": "f16"},
        # Full-batch training, the branch added to the stream and normalised.
        {"name": "ln_step_1m_256_bf16", "kind": "ln_step", "M": 1_000_000, "D": 256, "residual": True, "dtype": "bf16"},
        # Wide rows, fp32.
        {"name": "ln_step_4k_8192_f32", "kind": "ln_step", "M": 4_096, "D": 8_192, "residual": True, "dtype": "f32"},
        # A small graph's validation nodes against all of the teacher's 40 classes.
        {"name": "distill_512x40_f32", "kind": "distill", "M": 512, "C": 40, "k": 40, "T": 1.0, "hard": 0.0,
         "dtype": "f32"},
        # The full-batch graph with 47 classes, half of the nodes labelled.
        {"name": "distill_step_1m_47_f32", "kind": "distill_step", "M": 1_000_000, "C": 47, "k": 8, "T": 2.0, "hard": 0.3,
         "dtype": "f32"},
        # A few rows over many classes (the entities of a link-prediction graph).
        {"name": "distill_step_16x50000_f16", "kind": "distill_step", "M": 16, "C": 50_000, "k": 32, "T": 4.0,
         "hard": 0.5, "dtype": "f16"},
        # A batch over many classes, an odd number of them.
        {"name": "distill_grad_2k_100003_bf16", "kind": "distill_grad", "M": 2_048, "C": 100_003, "k": 64, "T": 2.0,
         "hard": 0.0, "dtype": "bf16"},
    ]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    kind = rng.choice(["embed", "embed_step", "embed_step", "ln", "ln_step", "ln_step", "distill", "distill_step",
                       "distill_step", "distill_grad"])
    c = {"kind": kind, "dtype": rng.choice(["f32", "f16", "bf16"])}
    size = 4 if c["dtype"] == "f32" else 2
    most = 5e8 / size  # elements of one tensor: no more than the largest listed one's
    if kind.startswith("embed"):
        D = rng.choice([16, 64, 128, 256, rng.randint(3, 400), int(_log_uniform(rng, 400, 5_000))])
        V = int(min(_log_uniform(rng, 20, 1_000_000), most / D))
        c.update(n=int(max(1, min(_log_uniform(rng, 1, 1_000_000), most / D))), V=V, D=D,
                 ids=rng.choice(["even", "popular"]), padded=rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.5), 3)]))
        return c
    if kind.startswith("ln"):
        D = rng.choice([16, 64, 100, 256, 512, 1024, rng.randint(2, 1_500), int(_log_uniform(rng, 1_500, 16_384))])
        c.update(M=int(max(1, min(_log_uniform(rng, 1, 1_000_000), most / D))), D=D, residual=rng.random() < 0.5)
        return c
    C = rng.choice([rng.randint(2, 64), int(_log_uniform(rng, 64, 4_000)), int(_log_uniform(rng, 4_000, 120_000))])
    c.update(M=int(max(1, min(_log_uniform(rng, 1, 600_000), most / C))), C=C, k=rng.randint(1, min(C, 64)),
             T=rng.choice([1.0, 2.0, 4.0, round(rng.uniform(0.5, 8.0), 2)]),
             hard=rng.choice([0.0, 0.0, round(rng.uniform(0.05, 0.95), 2)]))
    return c


# ------------------------------------------------------------------ inputs
def _normal(shape, gen, dtype):
    return torch.randn(shape, generator=gen, device=DEVICE).to(dtype)


def _embed_inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed * 2 + 1)
    n, V, D, t = case["n"], case["V"], case["D"], _TYPES[case["dtype"]]
    u = torch.rand(n, generator=gen, device=DEVICE, dtype=torch.float64)
    if case["ids"] == "popular":  # density ~ 1 / rank, over the rows in a random order
        rank = torch.exp(u * math.log(V + 1)).long().clamp(max=V) - 1
        ids = torch.randperm(V, generator=gen, device=DEVICE)[rank]
    else:
        ids = (u * V).long().clamp(max=V - 1)
    s = {"padding": None}
    if case["padded"]:  # the batch's end
        s["padding"] = -1
        ids[n - int(n * case["padded"]):] = -1
    s.update(ids=ids, table=_normal((V, D), gen, t), scale=math.sqrt(D))
    if case["kind"] == "embed_step":
        s["g"] = _normal((n, D), gen, t)
    return s


def _ln_inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed * 2 + 1)
    M, D, t = case["M"], case["D"], _TYPES[case["dtype"]]
    s = {"x": (torch.randn((M, D), generator=gen, device=DEVICE) * 1.5 + 0.3).to(t),
         "w": 1 + 0.2 * torch.randn(D, generator=gen, device=DEVICE),
         "b": 0.2 * torch.randn(D, generator=gen, device=DEVICE), "r": None}
    if case["residual"]:
        s["r"] = _normal((M, D), gen, t)
    if case["kind"] == "ln_step":
        s["gy"] = _normal((M, D), gen, t)
        if case["residual"]:
            s["gh"] = _normal((M, D), gen, t)
    return s


def _distill_inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed * 2 + 1)
    M, C, k, t = case["M"], case["C"], case["k"], _TYPES[case["dtype"]]
    step = 1 + (torch.rand((M, 1), generator=gen, device=DEVICE, dtype=torch.float64) * (C // k)).long().clamp(max=C // k - 1)
    first = (torch.rand((M, 1), generator=gen, device=DEVICE, dtype=torch.float64) * C).long().clamp(max=C - 1)
    ids = (first + torch.arange(k, device=DEVICE) * step) % C  # different ones in a row
    teacher = (4 + 2 * torch.randn((M, k), generator=gen, device=DEVICE)).sort(1, descending=True).values.to(t)
    logits = 1.5 * torch.randn((M, C), generator=gen, device=DEVICE)
    logits = logits.scatter_add_(1, ids, 0.8 * teacher.float()).to(t)  # a student that has learned some of it
    kept = (1 + (torch.rand((M, 1), generator=gen, device=DEVICE) * 2 * k).long()).clamp(max=k)
    kept[5::97] = 0  # rows that the teacher has not seen
    ids = torch.where(torch.arange(k, device=DEVICE) < kept, ids, -1)
    s = {"logits": logits, "teacher": teacher, "ids": ids, "labels": None}
    if case["hard"]:
        labels = torch.randint(0, C, (M,), generator=gen, device=DEVICE)
        s["labels"] = torch.where(torch.rand(M, generator=gen, device=DEVICE) < 0.5, labels, -1)
    return s


def _inputs(case, seed):
    if case["kind"].startswith("embed"):
        return _embed_inputs(case, seed)
    return _ln_inputs(case, seed) if case["kind"].startswith("ln") else _distill_inputs(case, seed)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    return s


# ------------------------------------------------------------------ the plain forms
def _plain_embed(s):
    ids = s["ids"]
    if s["padding"] is None:
        return (s["table"][ids].float() * s["scale"]).to(s["table"].dtype)
    pad = ids == s["padding"]
    rows = s["table"][ids.masked_fill(pad, 0)].float() * s["scale"]
    return rows.masked_fill_(pad[:, None], 0.0).to(s["table"].dtype)


def _plain_embed_step(s):
    ids, g = s["ids"], s["g"].float() * s["scale"]
    if s["padding"] is not None:
        pad = ids == s["padding"]
        ids, g = ids.masked_fill(pad, 0), g.masked_fill_(pad[:, None], 0.0)
    grad = torch.zeros(s["table"].shape, device=DEVICE).index_add_(0, ids, g)
    return _plain_embed(s), grad.to(s["table"].dtype)


def _plain_norm(s):
    """(h, its norm, 1 / deviation, y) with h as it is kept, the others in float32."""
    h = s["x"] if s["r"] is None else (s["x"].float() + s["r"].float()).to(s["x"].dtype)
    d = h.float()
    d = d - d.mean(-1, keepdim=True)
    r = torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS)
    n = d * r
    return h, n, r, (n * s["w"] + s["b"]).to(h.dtype)


def _plain_ln(s):
    h, _, _, y = _plain_norm(s)
    return y if s["r"] is None else (y, h)


def _plain_ln_step(s):
    h, n, r, y = _plain_norm(s)
    g = s["gy"].float()
    dw, db = (g * n).sum(0), g.sum(0)
    g = g * s["w"]
    dx = r * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    if s["r"] is None:
        return y, dx.to(h.dtype), dw, db
    dx = (dx + s["gh"].float()).to(h.dtype)
    return y, h, dx, dx, dw, db


def _plain_softmax(z):
    """(softmax, log of the sum of exponentials) of every row."""
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    return e / total, top + torch.log(total)


def _plain_distill(s, mean, gradient):
    c = s["case"]
    T, hard = c["T"], c["hard"]
    logits, used = s["logits"].float(), s["ids"] >= 0
    any_used, at = used.any(1, keepdim=True), s["ids"].clamp(min=0)
    t = torch.where(used, s["teacher"].float() / T, -math.inf)
    t = torch.where(any_used, t, 0.0)
    p, t_lse = _plain_softmax(t)
    p = torch.where(used, p, 0.0)
    q, lse = _plain_softmax(logits / T)
    log_p, log_q = torch.where(used, t - t_lse, 0.0), logits.gather(1, at) / T - lse
    loss = (1 - hard) * T * T * (p * (log_p - log_q)).sum(1)
    if gradient:
        grad = torch.where(any_used, (1 - hard) * T * q, 0.0).scatter_add_(1, at, p * (-(1 - hard) * T))
    if s["labels"] is not None:
        has, label = (s["labels"] >= 0)[:, None], s["labels"].clamp(min=0)[:, None]
        q, lse = _plain_softmax(logits)
        loss = loss + hard * torch.where(has, lse - logits.gather(1, label), 0.0)[:, 0]
        if gradient:
            grad = grad + torch.where(has, hard * q, 0.0)
            grad = grad.scatter_add_(1, label, torch.where(has, -hard, 0.0))
    if mean:
        loss = loss.mean()
    return (loss, (grad / c["M"]).to(s["logits"].dtype)) if gradient else loss


def run(state):
    s, kind = state, state["case"]["kind"]
    if not own:
        if kind.startswith("distill"):
            return _plain_distill(s, mean=kind != "distill", gradient=kind != "distill")
        return {"embed": _plain_embed, "embed_step": _plain_embed_step, "ln": _plain_ln, "ln_step": _plain_ln_step}[kind](s)
    import ra_spmm
    if kind == "embed":
        return ra_spmm.embed(s["ids"], s["table"], scale=s["scale"], padding=s["padding"])
    if kind == "embed_step":
        table = s["table"].detach().requires_grad_(True)
        out = ra_spmm.embed(s["ids"], table, scale=s["scale"], padding=s["padding"])
        return (out.detach(),) + torch.autograd.grad(out, table, s["g"])
    if kind == "ln":
        return ra_spmm.layer_norm(s["x"], s["w"], s["b"], eps=EPS, residual=s["r"])
    if kind == "ln_step":
        x, w, b = (s[n].detach().requires_grad_(True) for n in ("x", "w", "b"))
        if s["r"] is None:
            y = ra_spmm.layer_norm(x, w, b, eps=EPS)
            return (y.detach(),) + torch.autograd.grad(y, (x, w, b), s["gy"])
        r = s["r"].detach().requires_grad_(True)
        y, h = ra_spmm.layer_norm(x, w, b, eps=EPS, residual=r)
        return (y.detach(), h.detach()) + torch.autograd.grad((y, h), (x, r, w, b), (s["gy"], s["gh"]))
    args = {"temperature": s["case"]["T"], "labels": s["labels"], "hard": s["case"]["hard"]}
    if kind == "distill":
        return ra_spmm.distill_loss(s["logits"], s["teacher"], s["ids"], reduction="none", **args)
    if kind == "distill_grad":
        return ra_spmm.distill_loss_grad(s["logits"], s["teacher"], s["ids"], **args)
    logits = s["logits"].detach().requires_grad_(True)
    loss = ra_spmm.distill_loss(logits, s["teacher"], s["ids"], **args)
    return (loss.detach(),) + torch.autograd.grad(loss, logits)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    """Each input read once and each output written once."""
    size, kind = (4 if case["dtype"] == "f32" else 2), case["kind"]
    if kind.startswith("embed"):
        n, V, D = case["n"], case["V"], case["D"]
        touched = min(V, n)  # table rows that some id names, at most
        out = 8.0 * n + size * D * (touched + n)
        if kind == "embed":
            return {"bytes": out, "flops": float(n * D)}
        return {"bytes": out + size * D * (n + V), "flops": 2.0 * n * D}
    if kind.startswith("ln"):
        n = case["M"] * case["D"]
        passes = 4 if case["residual"] else 2
        if kind == "ln":
            return {"bytes": float(size * n * passes), "flops": 8.0 * n}
        # The incoming gradients are read, those of x and of the residual are one tensor.
        return {"bytes": size * n * (passes + (3.0 if case["residual"] else 2.0)), "flops": 20.0 * n}
    M, C, k = case["M"], case["C"], case["k"]
    once = size * M * C + M * k * (8.0 + size) + (8.0 * M if case["hard"] else 0.0)
    if kind == "distill":
        return {"bytes": once + 4.0 * M, "flops": 6.0 * M * C}
    return {"bytes": once + size * M * C, "flops": 10.0 * M * C}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_embed(case, seed):
    s = _embed_inputs(case, seed)
    ids = s["ids"]
    real = torch.ones_like(ids, dtype=torch.bool) if s["padding"] is None else ids != s["padding"]
    where = real.nonzero()[:, 0]
    out = torch.zeros((case["n"], case["D"]), dtype=torch.float64, device=DEVICE)
    out[where] = s["table"].index_select(0, ids[where]).double() * s["scale"]
    if case["kind"] == "embed":
        return out
    # Runs of equal ids in sorted order, a column of the gradient at a time: differences of a running sum.
    order = torch.argsort(ids[where], stable=True)
    ends = torch.cumsum(torch.bincount(ids[where], minlength=case["V"]), 0)
    starts = torch.nn.functional.pad(ends, (1, 0))[:-1]
    grad = torch.empty((case["V"], case["D"]), dtype=torch.float64, device=DEVICE)
    running = torch.zeros(where.numel() + 1, dtype=torch.float64, device=DEVICE)
    at = where[order]
    for d in range(case["D"]):
        torch.cumsum(s["g"][:, d].contiguous()[at].double(), 0, out=running[1:])
        grad[:, d] = (running[ends] - running[starts]) * s["scale"]
    return out, grad


def _exact_ln(case, seed):
    s = _ln_inputs(case, seed)
    step, D = case["kind"] == "ln_step", case["D"]
    h = s["x"]
    if s["r"] is not None:
        h = (h.double() + s["r"].double()).to(h.dtype)
    var, mean = torch.var_mean(h.double(), dim=1, correction=0, keepdim=True)
    dev = (var + EPS).sqrt()
    n = (h.double() - mean) / dev
    y = torch.addcmul(s["b"].double(), n, s["w"].double())
    head = (y,) if s["r"] is None else (y, h.double())
    if not step:
        return y if s["r"] is None else head
    gy = s["gy"].double()
    gn = gy * s["w"].double()
    along = (gn * n).sum(1, keepdim=True) / D
    dx = (gn - gn.sum(1, keepdim=True) / D - along * n) / dev
    weights = ((gy * n).sum(0), gy.sum(0))
    if s["r"] is None:
        return head + (dx,) + weights
    dx = dx + s["gh"].double()
    return head + (dx, dx) + weights


def _exact_distill(case, seed):
    s = _distill_inputs(case, seed)
    M, C, T, hard, kind = case["M"], case["C"], case["T"], case["hard"], case["kind"]
    rows_at_once = max(1, int(4e8 / (8 * C)))
    losses, grads = [], []
    for lo in range(0, M, rows_at_once):
        part = slice(lo, min(M, lo + rows_at_once))
        x, ids = s["logits"][part].double(), s["ids"][part]
        log_q = torch.log_softmax(x / T, 1)
        soft = torch.zeros_like(x)  # the teacher's distribution over all classes
        e = torch.where(ids >= 0, torch.exp(s["teacher"][part].double() / T), 0.0)
        total = e.sum(1, keepdim=True)
        p = e / torch.where(total > 0, total, 1.0)
        soft.scatter_add_(1, ids.clamp(min=0), p)
        loss = (1 - hard) * T * T * (torch.special.xlogy(soft, soft) - soft * log_q).sum(1)
        grad = (1 - hard) * T * (log_q.exp() * (total > 0) - soft)
        if s["labels"] is not None:
            label = s["labels"][part]
            rows = (label >= 0).nonzero()[:, 0]
            log_q = torch.log_softmax(x[rows], 1)
            loss[rows] -= hard * log_q[torch.arange(rows.numel(), device=DEVICE), label[rows]]
            grad[rows] += hard * log_q.exp()
            grad[rows, label[rows]] -= hard
        losses.append(loss)
        if kind != "distill":
            grads.append(grad / M)
    loss = torch.cat(losses)
    return loss if kind == "distill" else (loss.mean(), torch.cat(grads))


def exact(case, seed):
    if case["kind"].startswith("embed"):
        return _exact_embed(case, seed)
    return _exact_ln(case, seed) if case["kind"].startswith("ln") else _exact_distill(case, seed)
