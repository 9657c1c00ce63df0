"""Operators of graph transformers next to the routed SpMM: what their calls cost and what they have to return.

``own`` chooses what ``run`` computes with: elementary torch operations in 32 bits (false), or the operators of
``ra_spmm`` (true).  A case's ``kind`` says what a program does:

  attend      differential attention over the neighbour lists of a graph, inference on a kept plan
  attend_new  the same for a few new nodes whose lists arrive with the call (no plan)
  attend_step forward and backward on a kept plan: output and the gradients of q, k, v and the maps' weights
  norm        RMS norm of every query and key head with the position rotation, inference
  norm_step   the same forward and backward: outputs, input gradients, gradients of the norms' weights
  pack        an activation kept in 8 bits and read back
  ckpt_step   a linear layer after a ReLU whose input is kept in 8 bits only: activation, its gradient through the
              ReLU from the kept codes, and the weight gradient from the kept codes

Differential attention, for each row i, query head h (key and value head g = h // (Hq / Hkv)) and map a in (1, 2):
s_a[j] = scale * q_a[i, h] . k_a[j, g] + bias[ij] over the row's columns j; p_a = softmax(s_a); the output row is
sum_j (p_1 - lam[h] * p_2)[j] * v[j, g].  An edge with bias -inf takes no part; a row without edges gives zeros.
"""
import math

import torch

own = False

DEVICE = "cuda"
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
GROUP = 32  # columns that share a scale in the 8-bit format


# ------------------------------------------------------------------ the list
def listed():
    return [
        # Serving: a few new nodes of a recommendation graph, thousands of neighbours each; latency.
        {"name": "attend_new_4x6000", "kind": "attend_new", "family": "lists", "M": 4, "K": 200_000, "d": 6000.0,
         "Hq": 8, "Hkv": 8, "D": 16, "Dv": 32, "dtype": "bf16", "mask": 0.0},
        # A 10,000-node graph, fp32, one layer's attention; the launch and the call count.
        {"name": "attend_er_10k_f32", "kind": "attend", "family": "er", "M": 10_000, "K": 10_000, "d": 8.0,
         "Hq": 4, "Hkv": 4, "D": 16, "Dv": 32, "dtype": "f32", "mask": 0.0},
        # Inference on a community graph, hidden width 256.
        {"name": "attend_sbm_512k_f16", "kind": "attend", "family": "sbm", "M": 512_000, "K": 512_000, "d": 32.0,
         "Hq": 4, "Hkv": 4, "D": 32, "Dv": 64, "dtype": "f16", "mask": 0.0},
        # Training with shared key/value heads, an odd head width, edge dropout, skewed rows, fp32.
        {"name": "attend_step_skewed_150k_f32", "kind": "attend_step", "family": "skewed", "M": 150_000, "K": 150_000,
         "d": 20.0, "Hq": 6, "Hkv": 2, "D": 20, "Dv": 20, "dtype": "f32", "mask": 0.1},
        # Training on a social graph with long rows, hidden width 256.
        {"name": "attend_step_social_50k_bf16", "kind": "attend_step", "family": "social", "M": 50_000, "K": 50_000,
         "d": 80.0, "Hq": 4, "Hkv": 4, "D": 32, "Dv": 64, "dtype": "bf16", "mask": 0.0},
        # Largest: the full-batch training graph, power-law rows and columns with hubs, hidden width 128.
        {"name": "attend_step_powerlaw_1m_bf16", "kind": "attend_step", "family": "powerlaw", "M": 1_000_000,
         "K": 1_000_000, "d": 25.0, "Hq": 4, "Hkv": 4, "D": 16, "Dv": 32, "dtype": "bf16", "mask": 0.0},
        # Serving: one new node's heads.
        {"name": "norm_1_bf16", "kind": "norm", "M": 1, "Hq": 16, "Hk": 16, "D": 16, "rot": 16, "layout": "half",
         "positions": 4096, "dtype": "bf16"},
        # Training at an odd head width with part of the head rotated, fewer key heads, fp32.
        {"name": "norm_step_150k_d20_f32", "kind": "norm_step", "M": 150_000, "Hq": 12, "Hk": 4, "D": 20, "rot": 12,
         "layout": "interleaved", "positions": 150_000, "dtype": "f32"},
        # Training on the full-batch graph: heads cut out of one projection's rows.
        {"name": "norm_step_1m_bf16", "kind": "norm_step", "M": 1_000_000, "Hq": 8, "Hk": 8, "D": 16, "rot": 16,
         "layout": "half", "positions": 4096, "dtype": "bf16"},
        # A small graph's class-width activation kept and read back.
        {"name": "pack_10k_c47_f32", "kind": "pack", "M": 10_000, "C": 47, "dtype": "f32"},
        # The full-batch training step's hidden layer, fp32: 256 features to 47 classes.
        {"name": "ckpt_step_1m_256_47_f32", "kind": "ckpt_step", "M": 1_000_000, "C": 256, "out": 47, "dtype": "f32"},
        # A 16-bit feed-forward layer of the community graph.
        {"name": "ckpt_step_512k_128_256_bf16", "kind": "ckpt_step", "M": 512_000, "C": 128, "out": 256,
         "dtype": "bf16"},
    ]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    kind = rng.choice(["attend", "attend_new", "attend_step", "attend_step", "norm", "norm_step", "pack", "ckpt_step"])
    c = {"kind": kind, "dtype": rng.choice(["f32", "f16", "bf16"])}
    if kind.startswith("attend"):
        D = rng.choice([8, 16, 16, 32, 32, 64, rng.randint(4, 64)])
        Hkv = rng.choice([1, 2, 2, 3, 4, 4, 5, 8])
        Hq = Hkv * rng.choice([1, 1, 1, 2, 3, 4])
        Dv = rng.choice([2 * D, 2 * D, D])
        if kind == "attend_new":
            c.update(family="lists", M=rng.randint(1, 16), K=int(_log_uniform(rng, 20_000, 500_000)),
                     d=round(_log_uniform(rng, 50, 12_000), 1))
        else:
            family = rng.choice(["er", "sbm", "social", "skewed", "powerlaw"])
            M = int(_log_uniform(rng, 2_000, 400_000))
            d = round(_log_uniform(rng, 30, 120) if family == "social" else _log_uniform(rng, 3, 32), 2)
            # A drawn case costs no more than the largest listed one (25e6 edges of 4 heads of 2 * 16 + 32).
            most = 25e6 * 4 * 64 / (Hq * (2 * D + Dv)) / 2
            c.update(family=family, M=max(1, min(M, int(most / d))), d=d)
            c["K"] = c["M"]
        c.update(Hq=Hq, Hkv=Hkv, D=D, Dv=Dv, mask=rng.choice([0.0, 0.0, round(rng.uniform(0.05, 0.5), 3)]))
        return c
    if kind.startswith("norm"):
        D = rng.choice([16, 32, 64, 128, rng.randint(8, 128)])
        c.update(M=int(_log_uniform(rng, 1, 400_000)), Hq=rng.randint(1, 16), Hk=rng.randint(1, 16), D=D,
                 rot=rng.choice([D // 2 * 2, D // 4 * 2]), layout=rng.choice(["half", "interleaved"]),
                 positions=int(_log_uniform(rng, 64, 100_000)))
        c["M"] = max(1, min(c["M"], int(1e6 * 256 / ((c["Hq"] + c["Hk"]) * D))))
        return c
    c.update(M=int(_log_uniform(rng, 200, 800_000)), C=rng.choice([16, 64, 128, 256, rng.randint(8, 300)]))
    if kind == "ckpt_step":
        c["out"] = rng.choice([16, 47, 64, 128, 256, rng.randint(3, 256)])
    return c


# ------------------------------------------------------------------ inputs
def _lengths(case, gen):
    """Row lengths: even, log-normal or power-law ones; a few rows are empty."""
    M, d, family = case["M"], case["d"], case["family"]
    if family == "lists":
        n = torch.full((M,), d, device=DEVICE) * (0.5 + torch.rand(M, generator=gen, device=DEVICE))
    elif family in ("er", "sbm"):
        n = torch.poisson(torch.full((M,), d, device=DEVICE), generator=gen)
    elif family in ("social", "skewed"):
        sigma = 0.8 if family == "social" else 1.4
        z = torch.randn(M, generator=gen, device=DEVICE, dtype=torch.float64)
        n = (d * torch.exp(sigma * z - sigma * sigma / 2)).round().clamp(max=50_000)
    else:  # density ~ n^-2.3, hubs of up to 50,000
        u = torch.rand(M, generator=gen, device=DEVICE, dtype=torch.float64).clamp(min=1e-12)
        n = (d * (0.3 / 1.3) * u ** (-1 / 1.3)).round().clamp(max=min(50_000, max(1, case["K"] // 4)))
    return n.long()


def _graph(case, seed):
    """(rowptr, colind) int32 on the GPU; columns ascending without duplicates."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    M, K, family = case["M"], case["K"], case["family"]
    n = _lengths(case, gen)
    rows = torch.repeat_interleave(torch.arange(M, device=DEVICE), n)
    u = torch.rand(rows.numel(), generator=gen, device=DEVICE, dtype=torch.float64)
    if family in ("social", "skewed", "powerlaw"):  # columns by popularity
        cols = torch.randperm(K, generator=gen, device=DEVICE)[(u * u * K).long().clamp(max=K - 1)]
    else:
        cols = (u * K).long().clamp(max=K - 1)
    if family == "sbm":  # communities of 500 consecutive rows, 90 % of the edges inside
        inside = torch.rand(rows.numel(), generator=gen, device=DEVICE) < 0.9
        cols = torch.where(inside, (rows // 500 * 500 + (u * 500).long()).clamp(max=K - 1), cols)
    keys = torch.unique(rows * K + cols, sorted=True)
    rows = torch.div(keys, K, rounding_mode="floor")
    rowptr = torch.zeros(M + 1, dtype=torch.int64, device=DEVICE)
    torch.cumsum(torch.bincount(rows, minlength=M), 0, out=rowptr[1:])
    return rowptr.to(torch.int32), (keys - rows * K).to(torch.int32)


def _normal(shape, gen, dtype):
    return torch.randn(shape, generator=gen, device=DEVICE).to(dtype)


def _attend_inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed * 2 + 1)
    M, K, Hq, Hkv, D, Dv, t = (case["M"], case["K"], case["Hq"], case["Hkv"], case["D"], case["Dv"],
                               _TYPES[case["dtype"]])
    rowptr, colind = _graph(case, seed)
    s = {"rowptr": rowptr, "colind": colind, "q": _normal((M, Hq, 2, D), gen, t), "k": _normal((K, Hkv, 2, D), gen, t),
         "v": _normal((K, Hkv, Dv), gen, t), "lam": 0.2 + 0.6 * torch.rand(Hq, generator=gen, device=DEVICE),
         "bias": None}
    if case["mask"]:  # dropped edges; every 97th row loses all of its edges
        off = torch.rand(colind.numel(), generator=gen, device=DEVICE) < case["mask"]
        rows = torch.repeat_interleave(torch.arange(M, device=DEVICE), (rowptr[1:] - rowptr[:-1]).long())
        s["bias"] = torch.zeros(colind.numel(), device=DEVICE).masked_fill_(off | (rows % 97 == 5), -math.inf)
    if case["kind"] == "attend_step":
        s["g"] = _normal((M, Hq, Dv), gen, t)
    return s


def _table(case):
    """(cos, sin) of the position angles, float32 rounded from 64 bits, [positions, rot / 2, 2]."""
    half = case["rot"] // 2
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEVICE) / max(half, 1))
    angle = torch.arange(case["positions"], dtype=torch.float64, device=DEVICE)[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()


def _norm_inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed * 2 + 1)
    M, Hq, Hk, D, t = case["M"], case["Hq"], case["Hk"], case["D"], _TYPES[case["dtype"]]
    rows = _normal((M, (Hq + 2 * Hk) * D), gen, t)  # a projection's rows: queries, keys, values
    s = {"q": rows[:, :Hq * D].view(M, Hq, D), "k": rows[:, Hq * D:(Hq + Hk) * D].view(M, Hk, D),
         "wq": 1 + 0.2 * torch.randn(D, generator=gen, device=DEVICE),
         "wk": 1 + 0.2 * torch.randn(D, generator=gen, device=DEVICE), "table": _table(case),
         "pos": torch.randint(0, case["positions"], (M,), generator=gen, device=DEVICE).to(torch.int32)}
    if case["kind"] == "norm_step":
        s["gq"], s["gk"] = _normal((M, Hq, D), gen, t), _normal((M, Hk, D), gen, t)
    return s


def _pack_inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed * 2 + 1)
    M, C, t = case["M"], case["C"], _TYPES[case["dtype"]]
    s = {"x": _normal((M, C), gen, t)}
    if case["kind"] == "ckpt_step":
        s["gh"] = _normal((M, C), gen, t)
        s["g"] = _normal((M, case["out"]), gen, t)
    return s


def _inputs(case, seed):
    if case["kind"].startswith("attend"):
        return _attend_inputs(case, seed)
    return _norm_inputs(case, seed) if case["kind"].startswith("norm") else _pack_inputs(case, seed)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] in ("attend", "attend_step"):
        if own:
            import ra_spmm
            s["plan"] = ra_spmm.make_attention_plan(s["rowptr"], s["colind"], case["M"], case["K"],
                                                    backward=case["kind"] == "attend_step")
        else:  # a plain program keeps the row of every edge
            s["rows"] = torch.repeat_interleave(torch.arange(case["M"], device=DEVICE),
                                                (s["rowptr"][1:] - s["rowptr"][:-1]).long())
            s["cols"] = s["colind"].long()
    if own and case["kind"] == "attend_step":
        for n in ("q", "k", "v", "lam"):
            s[n].requires_grad_(True)
    if own and case["kind"] == "norm_step":
        for n in ("q", "k", "wq", "wk"):
            s[n] = s[n].detach().requires_grad_(True)
    return s


# ------------------------------------------------------------------ the plain forms
def _plain_maps(s, scale):
    """Per head: (edges' rows, columns, p_1, p_2) in float32."""
    c = s["case"]
    M, group = c["M"], c["Hq"] // c["Hkv"]
    if "rows" in s:
        rows, cols = s["rows"], s["cols"]
    else:
        cols = s["colind"].long()
        rows = torch.repeat_interleave(torch.arange(M, device=DEVICE), (s["rowptr"][1:] - s["rowptr"][:-1]).long(),
                                       output_size=cols.numel())
    for h in range(c["Hq"]):
        p = []
        for a in range(2):
            score = (s["q"][:, h, a].float()[rows] * s["k"][:, h // group, a].float()[cols]).sum(1) * scale
            if s["bias"] is not None:
                score = score + s["bias"]
            top = torch.full((M,), -math.inf, device=DEVICE).scatter_reduce_(0, rows, score, "amax")
            top = torch.where(top == -math.inf, 0.0, top)  # rows without an edge left
            e = torch.exp(score - top[rows])
            total = torch.zeros(M, device=DEVICE).index_add_(0, rows, e)
            p.append(e / torch.where(total > 0, total, 1.0)[rows])
        yield h, h // group, rows, cols, p


def _plain_attend(s):
    c = s["case"]
    out = torch.zeros((c["M"], c["Hq"], c["Dv"]), device=DEVICE)
    for h, g, rows, cols, p in _plain_maps(s, 1.0 / math.sqrt(c["D"])):
        w = p[0] - s["lam"][h] * p[1]
        out[:, h] = torch.zeros((c["M"], c["Dv"]), device=DEVICE).index_add_(
            0, rows, w[:, None] * s["v"][:, g].float()[cols])
    return out.to(s["v"].dtype)


def _plain_attend_step(s):
    c = s["case"]
    M, K, Dv, scale = c["M"], c["K"], c["Dv"], 1.0 / math.sqrt(c["D"])
    out = torch.zeros((M, c["Hq"], Dv), device=DEVICE)
    dq, dk = (torch.zeros(s[n].shape, device=DEVICE) for n in ("q", "k"))
    dv, dlam = torch.zeros(s["v"].shape, device=DEVICE), torch.zeros(c["Hq"], device=DEVICE)
    for h, g, rows, cols, p in _plain_maps(s, scale):
        lam = s["lam"][h]
        vals, go = s["v"][:, g].float()[cols], s["g"][:, h].float()[rows]
        w = p[0] - lam * p[1]
        out[:, h] = torch.zeros((M, Dv), device=DEVICE).index_add_(0, rows, w[:, None] * vals)
        dp = (vals * go).sum(1)
        dv[:, g] += torch.zeros((K, Dv), device=DEVICE).index_add_(0, cols, w[:, None] * go)
        dlam[h] = -(p[1] * dp).sum()
        del vals, go
        for a in range(2):
            mean = torch.zeros(M, device=DEVICE).index_add_(0, rows, p[a] * dp)
            ds = p[a] * (dp - mean[rows]) * (scale if a == 0 else -lam * scale)
            dq[:, h, a] = torch.zeros((M, c["D"]), device=DEVICE).index_add_(
                0, rows, ds[:, None] * s["k"][:, g, a].float()[cols])
            dk[:, g, a] += torch.zeros((K, c["D"]), device=DEVICE).index_add_(
                0, cols, ds[:, None] * s["q"][:, h, a].float()[rows])
    t = s["q"].dtype
    return out.to(t), dq.to(t), dk.to(t), dv.to(t), dlam


def _pairs(x, rot, layout):
    """The two coordinates of every rotated pair of the last axis."""
    if layout == "half":
        return x[..., :rot // 2], x[..., rot // 2:rot]
    return x[..., 0:rot:2], x[..., 1:rot:2]


def _rotated(x, cos, sin, rot, layout):
    if rot == 0:
        return x
    a, b = _pairs(x, rot, layout)
    y = x.clone()
    ya, yb = _pairs(y, rot, layout)
    ya.copy_(a * cos - b * sin)
    yb.copy_(a * sin + b * cos)
    return y


def _plain_norm(s):
    c = s["case"]
    at = s["table"][s["pos"].long()]
    cos, sin = at[:, None, :, 0], at[:, None, :, 1]
    out = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        x = x.float()
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        out.append(_rotated(y, cos, sin, c["rot"], c["layout"]).to(s["q"].dtype))
    return out


def _plain_norm_step(s):
    c = s["case"]
    at = s["table"][s["pos"].long()]
    cos, sin = at[:, None, :, 0], at[:, None, :, 1]
    grads = []
    for x, w, g in ((s["q"], s["wq"], s["gq"]), (s["k"], s["wk"], s["gk"])):
        x, g = x.float(), _rotated(g.float(), cos, -sin, c["rot"], c["layout"])
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        n, gw = x * r, g * w
        dx = r * (gw - n * (gw * n).mean(-1, keepdim=True))
        grads += [dx.to(s["q"].dtype), (g * n).sum((0, 1))]
    return _plain_norm(s) + grads


def _plain_codes(x, relu):
    """Codes and scales of the 8-bit format (float32 [M, groups, 32], [M, groups, 1]): a group's scale is the power of
    two that puts its largest magnitude into [64, 128), or [128, 256) after a ReLU, where a positive value keeps a
    code of at least 1."""
    M, C = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -C % GROUP)).view(M, -1, GROUP)
    if relu:
        x = x.clamp(min=0)
    top = x.abs().amax(-1, keepdim=True)
    scale = torch.ldexp(torch.ones_like(top), (torch.frexp(top)[1] - (8 if relu else 7)).clamp(min=-126))
    code = torch.round(x / scale).clamp(-127, 255 if relu else 127)
    if relu:
        code = torch.where(x > 0, code.clamp(min=1), torch.zeros_like(code))
    return code, scale


def _plain_pack(s):
    code, scale = _plain_codes(s["x"], False)
    return (code * scale).flatten(1)[:, :s["case"]["C"]].contiguous()


def _plain_ckpt_step(s):
    C = s["case"]["C"]
    code, scale = _plain_codes(s["x"], True)
    kept = (code * scale).flatten(1)[:, :C]
    dx = torch.where(code.flatten(1)[:, :C] > 0, s["gh"].float(), 0.0)
    return s["x"].clamp(min=0), dx.to(s["x"].dtype), s["g"].float().t() @ kept


def run(state):
    s, kind = state, state["case"]["kind"]
    if not own:
        return {"attend": _plain_attend, "attend_new": _plain_attend, "attend_step": _plain_attend_step,
                "norm": _plain_norm, "norm_step": _plain_norm_step, "pack": _plain_pack,
                "ckpt_step": _plain_ckpt_step}[kind](s)
    import ra_spmm
    if kind == "attend":
        return ra_spmm.run_attention_plan(s["plan"], s["q"], s["k"], s["v"], s["lam"], bias=s["bias"])
    if kind == "attend_new":
        return ra_spmm.diff_attention_csr(s["rowptr"], s["colind"], s["q"], s["k"], s["v"], s["lam"], bias=s["bias"])
    if kind == "attend_step":
        out = ra_spmm.diff_attention(s["plan"], s["q"], s["k"], s["v"], s["lam"], bias=s["bias"])
        grads = torch.autograd.grad(out, (s["q"], s["k"], s["v"], s["lam"]), s["g"])
        return (out.detach(),) + grads
    if kind == "norm":
        return ra_spmm.head_norm_rotate(s["q"], s["k"], s["wq"], s["wk"], s["table"], s["pos"], eps=EPS,
                                        layout=s["case"]["layout"])
    if kind == "norm_step":
        q, k = ra_spmm.head_norm_rotate(s["q"], s["k"], s["wq"], s["wk"], s["table"], s["pos"], eps=EPS,
                                        layout=s["case"]["layout"])
        dq, dk, dwq, dwk = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))
        return q.detach(), k.detach(), dq, dwq, dk, dwk
    if kind == "pack":
        return ra_spmm.unpack8(ra_spmm.pack8(s["x"]))
    h, kept = ra_spmm.relu_pack8(s["x"])
    return h, ra_spmm.relu_grad8(s["gh"], kept), ra_spmm.weight_grad8(s["g"], kept)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    """Each input read once and each output written once; the number of edges is the expected one."""
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"].startswith("attend"):
        M, K, Hq, Hkv, D, Dv = (case[n] for n in ("M", "K", "Hq", "Hkv", "D", "Dv"))
        nnz = M * case["d"]
        touched = min(K, nnz)  # rows of k and v that some list names, at most
        rows = size * (M * Hq * (2 * D + Dv) + touched * Hkv * (2 * D + Dv))
        index = 4.0 * (M + 1) + 4.0 * nnz * (2 if case["mask"] else 1)
        flops = nnz * Hq * (4.0 * D + 2 * Dv)
        if case["kind"] != "attend_step":
            return {"bytes": rows + index, "flops": flops}
        # The gradients of q, k and v, and the incoming one; the four further products.
        return {"bytes": rows + index + size * (M * Hq * (2 * D + Dv) + K * Hkv * (2 * D + Dv)),
                "flops": flops + nnz * Hq * (8.0 * D + 4 * Dv)}
    if case["kind"].startswith("norm"):
        n = case["M"] * (case["Hq"] + case["Hk"]) * case["D"]
        table = 4.0 * case["rot"] * min(case["positions"], case["M"]) + 4.0 * case["M"]
        step = case["kind"] == "norm_step"
        return {"bytes": size * n * (4 if step else 2) + table, "flops": n * (20.0 if step else 7.0)}
    M, C = case["M"], case["C"]
    if case["kind"] == "pack":
        return {"bytes": M * C * (size + 4.0), "flops": 4.0 * M * C}
    out = case["out"]
    return {"bytes": M * C * size * 4.0 + M * out * size + 4.0 * out * C, "flops": 2.0 * M * C * out}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_attend(case, seed):
    s = _attend_inputs(case, seed)
    M, K, Hq, Hkv, D, Dv = (case[n] for n in ("M", "K", "Hq", "Hkv", "D", "Dv"))
    step = case["kind"] == "attend_step"
    rowptr, i = s["rowptr"], torch.repeat_interleave(torch.arange(M, device=DEVICE),
                                                     (s["rowptr"][1:] - s["rowptr"][:-1]).long())
    j = s["colind"].long()
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    lam = s["lam"].double()
    gone = torch.zeros_like(j, dtype=torch.bool) if s["bias"] is None else s["bias"] == -math.inf
    out = torch.empty((M, Hq, Dv), dtype=torch.float64, device=DEVICE)
    if step:
        go = s["g"].double()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        dlam = torch.zeros_like(lam)

    def row_sums(x):  # sum over every row's run of edges: differences of a running sum
        running = torch.cat([x.new_zeros(1), x.cumsum(0)])[rowptr.long()]
        return running[1:] - running[:-1]

    def dots(a, b):  # a[i] . b[j] for every edge, a column at a time
        t = torch.zeros(j.numel(), dtype=torch.float64, device=DEVICE)
        for n in range(a.shape[1]):
            t += a[:, n].contiguous()[i] * b[:, n].contiguous()[j]
        return t

    # The edges in column order: (edge, first edge of every column).
    order = torch.argsort(j, stable=True)
    colptr = torch.zeros(K + 1, dtype=torch.int64, device=DEVICE)
    torch.cumsum(torch.bincount(j, minlength=K), 0, out=colptr[1:])
    by_row, by_column = (slice(None), rowptr.long()), (order, colptr)

    def spread(weight, source, at, to):  # sum over every run of edges of weight * source[at]: differences of a running sum
        edges, ptr = to
        weight, at = weight[edges], at[edges]
        r = torch.empty((ptr.numel() - 1, source.shape[1]), dtype=torch.float64, device=DEVICE)
        running = torch.zeros(weight.numel() + 1, dtype=torch.float64, device=DEVICE)
        for n in range(source.shape[1]):
            torch.cumsum(weight * source[:, n].contiguous()[at], 0, out=running[1:])
            r[:, n] = running[ptr[1:]] - running[ptr[:-1]]
        return r

    for h in range(Hq):
        g = h * Hkv // Hq
        maps = []
        for a in range(2):
            t = dots(q[:, h, a], k[:, g, a]) / math.sqrt(D)
            if s["bias"] is not None:
                t = t + s["bias"].double()
            # Each row is shifted by its maximum as float32 holds it: any shift near it does.
            top = torch.full((M,), -math.inf, device=DEVICE).scatter_reduce_(0, i, t.float(), "amax").double()
            top = torch.where(top.isinf(), torch.zeros_like(top), top)
            e = torch.where(gone, torch.zeros_like(t), (t - top[i]).exp())
            total = row_sums(e)
            maps.append(e / torch.where(total > 0, total, torch.ones_like(total))[i])
        w = maps[0] - lam[h] * maps[1]
        out[:, h] = spread(w, v[:, g], j, by_row)
        if not step:
            continue
        dp = dots(go[:, h], v[:, g])
        dv[:, g] += spread(w, go[:, h], i, by_column)
        dlam[h] = -(maps[1] * dp).sum()
        for a, sign in ((0, 1.0), (1, -lam[h])):
            ds = maps[a] * (dp - row_sums(maps[a] * dp)[i]) * sign / math.sqrt(D)
            dq[:, h, a] = spread(ds, k[:, g, a], j, by_row)
            dk[:, g, a] += spread(ds, q[:, h, a], i, by_column)
    return (out, dq, dk, dv, dlam) if step else out


def _exact_norm(case, seed):
    s = _norm_inputs(case, seed)
    D, rot, step = case["D"], case["rot"], case["kind"] == "norm_step"
    at = s["table"].double()[s["pos"].long()]
    # The rotation of a head as first and second indices of its pairs.
    half = torch.arange(rot // 2, device=DEVICE)
    first, second = (half, half + rot // 2) if case["layout"] == "half" else (2 * half, 2 * half + 1)
    z = torch.complex(at[:, None, :, 0].contiguous(), at[:, None, :, 1].contiguous())
    outs, grads = [], []

    def turn(x, by):
        y = x.clone()
        t = torch.complex(x[..., first], x[..., second]) * by
        y[..., first], y[..., second] = t.real, t.imag
        return y

    for n in "qk":
        x, w = s[n].double(), s["w" + n].double()
        rms = (x.square().sum(-1, keepdim=True) / D + EPS).sqrt()
        outs.append(turn(x / rms * w, z))
        if step:
            g = turn(s["g" + n].double(), z.conj())
            inner = (g * w * x).sum(-1, keepdim=True)
            grads += [g * w / rms - x * inner / (D * rms ** 3), (g * x / rms).sum((0, 1))]
    return outs + grads


def _exact_pack(case, seed):
    s = _pack_inputs(case, seed)
    relu = case["kind"] == "ckpt_step"
    x = s["x"].double()
    M, C = x.shape
    kept = torch.zeros_like(x)
    for c in range(0, C, GROUP):
        part = x[:, c:c + GROUP]
        part = part.clamp(min=0) if relu else part
        top = part.abs().max(1, keepdim=True).values
        power = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
        power = power + (2.0 ** (power + 1) <= top).double() - (2.0 ** power > top).double()  # log2 may round
        step = 2.0 ** (power - (7 if relu else 6)).clamp(min=-126)
        code = torch.round(part / step)
        code = torch.minimum(code, torch.full_like(code, 255.0 if relu else 127.0)).clamp(min=-127)
        if relu:
            code = torch.where((part > 0) & (code < 1), torch.ones_like(code), code)
        kept[:, c:c + GROUP] = torch.where(top > 0, code * step, torch.zeros_like(part))
    if not relu:
        return kept
    return x.clamp(min=0), s["gh"].double() * (x > 0), s["g"].double().t() @ kept


def exact(case, seed):
    if case["kind"].startswith("attend"):
        # The largest graphs would take too long in 64 bits.
        if case["M"] * case["d"] * case["Hq"] * (2 * case["D"] + case["Dv"]) > 2e10:
            return None
        return _exact_attend(case, seed)
    return _exact_norm(case, seed) if case["kind"].startswith("norm") else _exact_pack(case, seed)
