"""What the operators of one transformer FFN block are timed on: the calls of a serving or training program.

Three families, each through its public entry points:

* ``moe``: a whole top-k routed SwiGLU mixture-of-experts layer for a handful of tokens (decode), from router logits to
  the gate-weighted sum.
* ``int8``: matrix products with 8-bit integer operands, one scale per token and one per output channel; the tokens are
  quantised within the call.  One matrix (``linear``), or one per expert over ragged groups of rows (``experts``), with or
  without SwiGLU on interleaved gate and up channels.
* ``norm``: the RMS norms behind and in front of a block with the block's gate, the residual scale and the residual sum;
  the forward pass, or both passes.
"""
from __future__ import annotations

import math

import torch

own = False

EXPERT_WEIGHTS = 8 * 4096 * 14336       # experts x hidden x FFN width, at most
INT8_WORK = 16384 * 28672 * 4096        # rows x channels x depth, at most
NORM_ELEMS = 8192 * 4096                # tokens x hidden, at most
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # One decoded token, many small experts: 35 MB of weights, latency counts.
        {"name": "moe_token_64experts", "family": "moe", "tokens": 1, "hidden": 2048, "inter": 1408, "experts": 64, "top_k": 2},
        # One decoded token of the configured layer (hidden 4096, FFN 14336, 8 experts, top-2): 704 MB of weights.
        {"name": "moe_token_8experts", "family": "moe", "tokens": 1, "hidden": 4096, "inter": 14336, "experts": 8, "top_k": 2},
        # A few requests at once (or a speculative draft), more experts per token.
        {"name": "moe_7tokens_top4", "family": "moe", "tokens": 7, "hidden": 1024, "inter": 2816, "experts": 32, "top_k": 4},
        # A decode batch of the configured layer: every expert's weights are read.
        {"name": "moe_32tokens_8experts", "family": "moe", "tokens": 32, "hidden": 4096, "inter": 14336, "experts": 8, "top_k": 2},
        # A square projection for one decoded token.
        {"name": "int8_token", "family": "int8", "kind": "linear", "rows": 1, "groups": 1, "empty": 0, "chan": 4096,
         "depth": 4096, "swiglu": False},
        # A ragged decode batch against a narrower projection.
        {"name": "int8_77rows", "family": "int8", "kind": "linear", "rows": 77, "groups": 1, "empty": 0, "chan": 1000,
         "depth": 2816, "swiglu": False},
        # Down projections of 16 experts on a medium batch, some of them without a row.
        {"name": "int8_16experts", "family": "int8", "kind": "experts", "rows": 2000, "groups": 16, "empty": 3, "chan": 2048,
         "depth": 4096, "swiglu": False},
        # Up projections of the configured layer's prefill: 8192 tokens, top-2.
        {"name": "int8_prefill", "family": "int8", "kind": "experts", "rows": 16384, "groups": 8, "empty": 0, "chan": 28672,
         "depth": 4096, "swiglu": True},
        # Between two blocks while decoding one token.
        {"name": "norm_token", "family": "norm", "tokens": 1, "hidden": 4096, "type": "bf16", "residual": "bf16",
         "weights": "bf16", "gate": "channel", "scale": 0.5, "backward": False},
        # Between two blocks of a prefill.
        {"name": "norm_prefill", "family": "norm", "tokens": 8192, "hidden": 4096, "type": "bf16", "residual": "bf16",
         "weights": "bf16", "gate": "none", "scale": 1.0, "backward": False},
        # A training step with a learned gate per channel and the residual stream in 32 bits.
        {"name": "norm_train", "family": "norm", "tokens": 4096, "hidden": 4096, "type": "bf16", "residual": "fp32",
         "weights": "fp32", "gate": "channel", "scale": 0.5, "backward": True},
        # A training step on a ragged batch of odd width, gated per token.
        {"name": "norm_train_odd", "family": "norm", "tokens": 999, "hidden": 1001, "type": "fp16", "residual": "fp16",
         "weights": "fp32", "gate": "token", "scale": 0.7, "backward": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_moe(rng):
    hidden, inter = rng.choice([(512, 1024), (1024, 2816), (2048, 4096), (2048, 1408), (4096, 14336),
                                (8 * _log(rng, 32, 512), 8 * _log(rng, 32, 1024))])
    experts = rng.choice([e for e in (3, 4, 8, 16, 32, 60, 64, 128) if e * hidden * inter <= EXPERT_WEIGHTS])
    return {"family": "moe", "tokens": _log(rng, 1, 64), "hidden": hidden, "inter": inter, "experts": experts,
            "top_k": rng.choice([k for k in (1, 2, 2, 4, 6, 8) if k <= experts])}


def _draw_int8(rng):
    kind = rng.choice(["linear", "experts"])
    groups = 1 if kind == "linear" else rng.choice([2, 5, 8, 16, 64])
    rows, chan, depth = _log(rng, 1, 16384), 8 * _log(rng, 16, 3500), 16 * _log(rng, 8, 896)
    while rows * chan * depth > INT8_WORK or groups * chan * depth > EXPERT_WEIGHTS:
        rows, chan = max(1, rows // 2), max(128, chan // 16 * 8)
    return {"family": "int8", "kind": kind, "rows": rows, "groups": groups,
            "empty": 0 if kind == "linear" else rng.randrange(groups // 2 + 1), "chan": chan, "depth": depth,
            "swiglu": kind == "experts" and rng.random() < 0.5}


def _draw_norm(rng):
    hidden = _log(rng, 64, 8192)
    if rng.random() < 0.6:
        hidden = max(64, hidden // 64 * 64)
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    return {"family": "norm", "tokens": _log(rng, 1, min(16384, NORM_ELEMS // hidden)), "hidden": hidden, "type": kind,
            "residual": rng.choice([kind, "fp32"]), "weights": rng.choice([kind, "fp32"]),
            "gate": rng.choice(["none", "channel", "token", "full"]), "scale": rng.choice([1.0, 0.5, 0.7]),
            "backward": rng.random() < 0.5}


def draw(rng):
    return rng.choice([_draw_moe, _draw_int8, _draw_norm])(rng)


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _used_experts(case):
    """Experts that some token chooses, on average: the logits are made so that exactly this many are."""
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    return max(k, min(T * k, round(E * (1 - (1 - k / E) ** T))))


def _prepare_moe(case, gen):
    T, H, I, E, k = (case[n] for n in ("tokens", "hidden", "inter", "experts", "top_k"))

    def weight(*shape):
        return torch.randn(*shape, device="cuda", generator=gen, dtype=torch.bfloat16).mul_(0.02)
    w13, w2 = weight(E, 2 * I, H), weight(E, H, I)                  # rows of w13 interleave gate and up
    x = torch.randn(T, H, device="cuda", generator=gen).to(torch.bfloat16)
    # normal logits among the experts in use, each of them the choice of one token at least
    used = torch.randperm(E, device="cuda", generator=gen)[:_used_experts(case)]
    logits = torch.randn(T, E, device="cuda", generator=gen) - 20.0
    logits[:, used] = torch.randn(T, len(used), device="cuda", generator=gen).clamp_(max=2.0)
    slot = torch.arange(len(used), device="cuda")
    logits[slot // k, used] = 2.01 + 0.5 * torch.rand(len(used), device="cuda", generator=gen)
    return {"x": x, "logits": logits, "w13": w13, "w2": w2}


def _group_rows(case, seed):
    """Rows of every group, known to the program that made the groups."""
    g = torch.Generator().manual_seed(77 + seed)
    G, live = case["groups"], case["groups"] - case["empty"]
    share = torch.rand(live, generator=g) + 0.2
    cuts = (share.cumsum(0) / share.sum() * case["rows"]).round().long()
    cuts[-1] = case["rows"]
    rows = torch.zeros(G, dtype=torch.long)
    rows[torch.randperm(G, generator=g)[:live]] = torch.diff(cuts, prepend=torch.zeros(1, dtype=torch.long))
    return rows.tolist()


def _prepare_int8(case, seed, gen):
    G, N, K = case["groups"], case["chan"], case["depth"]
    x = torch.randn(case["rows"], K, device="cuda", generator=gen)
    x *= 0.2 + 2.0 * torch.rand(case["rows"], 1, device="cuda", generator=gen)          # tokens differ in size
    w = torch.empty(G, N, K, dtype=torch.int8, device="cuda")
    for g in range(G):
        w[g] = torch.randn(N, K, device="cuda", generator=gen).mul_(32.0).round_().clamp_(-127, 127)
    scale = (0.5 + torch.rand(G, N, device="cuda", generator=gen)) * (0.02 / 32.0)
    st = {"x": x.to(torch.bfloat16), "w": w, "scale": scale}
    if case["kind"] == "linear":
        st["w"], st["scale"] = w[0], scale[0]
    else:
        rows = _group_rows(case, seed)
        start = [sum(rows[:g]) for g in range(G)]
        st["host_rows"], st["host_start"] = rows, start
        st["group_rows"] = torch.tensor(rows, dtype=torch.int32, device="cuda")
        st["group_start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
    return st


def _prepare_norm(case, gen):
    T, H = case["tokens"], case["hidden"]
    kind, res, wt = TYPES[case["type"]], TYPES[case["residual"]], TYPES[case["weights"]]

    def normal(*shape, mean=0.0, std=1.0):
        return torch.randn(*shape, device="cuda", generator=gen) * std + mean
    st = {"residual": normal(T, H, std=2.0).to(res), "branch": normal(T, H, std=0.5).to(kind),
          "post_weight": normal(H, mean=1.0, std=0.1).to(wt), "pre_weight": normal(H, mean=1.0, std=0.1).to(wt)}
    if case["gate"] == "channel":
        st["gate"] = normal(H, mean=0.5, std=0.2).to(wt)
    elif case["gate"] == "token":
        st["gate"] = normal(T, 1, mean=0.5, std=0.2).to(wt)
    elif case["gate"] == "full":
        st["gate"] = normal(T, H, mean=0.5, std=0.2).to(kind)
    else:
        st["gate"] = None
    if case["backward"]:
        for t in st.values():
            if t is not None:
                t.requires_grad_()
        st["d_residual"], st["d_normed"] = normal(T, H).to(res), normal(T, H).to(kind)
    return st


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1000 + seed)
    if case["family"] == "moe":
        st = _prepare_moe(case, gen)
    elif case["family"] == "int8":
        st = _prepare_int8(case, seed, gen)
    else:
        st = _prepare_norm(case, gen)
    st["case"] = case
    return st


# ---- one pass --------------------------------------------------------------------------------------------------------
EPS = 1e-6


def _plain_moe(st):
    x, logits, k = st["x"].float(), st["logits"], st["case"]["top_k"]
    top, which = torch.sort(logits, dim=-1, descending=True, stable=True)     # stable: ties go to the lowest index
    top, which = top[:, :k], which[:, :k]
    p = torch.exp(top - top[:, :1])
    p = p / p.sum(-1, keepdim=True)
    out = torch.zeros_like(x)
    for e in which.unique().tolist():
        chosen = which == e                                                    # [T, k], one per row at most
        rows = chosen.any(-1).nonzero().squeeze(1)
        gate_up = x[rows] @ st["w13"][e].float().t()
        gate, up = gate_up[:, 0::2], gate_up[:, 1::2]
        mid = gate / (1 + torch.exp(-gate)) * up
        weight = (p * chosen).sum(-1)[rows]
        out[rows] += weight[:, None] * (mid @ st["w2"][e].float().t())
    return out.to(torch.bfloat16)


def _plain_int8(st):
    x = st["x"].float()
    most = x.abs().amax(-1, keepdim=True)
    s = torch.where(most > 0, most / 127.0, torch.ones_like(most))
    q = torch.round(x / s).clamp(-127, 127)
    if st["case"]["kind"] == "linear":
        return (q @ st["w"].float().t() * s * st["scale"]).to(torch.bfloat16)
    outs = []
    for g, (at, n) in enumerate(zip(st["host_start"], st["host_rows"])):
        if n == 0:
            continue
        y = q[at:at + n] @ st["w"][g].float().t() * s[at:at + n] * st["scale"][g]
        if st["case"]["swiglu"]:
            gate, up = y[:, 0::2], y[:, 1::2]
            y = gate / (1 + torch.exp(-gate)) * up
        outs.append(y.to(torch.bfloat16))
    return torch.cat(outs)


def _norm_leaves(st):
    return [n for n in ("residual", "branch", "post_weight", "pre_weight", "gate") if st[n] is not None]


def _plain_norm(st):
    case, names = st["case"], _norm_leaves(st)
    with torch.set_grad_enabled(case["backward"]):
        v = {n: st[n].detach().float().requires_grad_(case["backward"]) for n in names}
        z = v["branch"]
        n = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + EPS) * v["post_weight"]
        r = v["residual"] + case["scale"] * (n * v["gate"] if "gate" in v else n)
        u = r * torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS) * v["pre_weight"]
        out = (r.detach().to(st["residual"].dtype), u.detach().to(st["branch"].dtype))
        if case["backward"]:
            grads = torch.autograd.grad((r, u), [v[n] for n in names], (st["d_residual"].float(), st["d_normed"].float()))
            out += tuple(g.to(st[n].dtype) for n, g in zip(names, grads))
    return out


def run(state):
    case = state["case"]
    if not own:
        return {"moe": _plain_moe, "int8": _plain_int8, "norm": _plain_norm}[case["family"]](state)
    if case["family"] == "moe":
        from rbruck_alltoallv_b200.ops.moe import moe_few_tokens
        return moe_few_tokens(state["x"], state["logits"], state["w13"], state["w2"], top_k=case["top_k"])
    if case["family"] == "int8":
        from rbruck_alltoallv_b200.ops.moe import grouped_gemm_int8, linear_int8, quantize_rows_int8
        if case["kind"] == "linear":
            return linear_int8(state["x"], state["w"], state["scale"])
        q, s = quantize_rows_int8(state["x"])
        return grouped_gemm_int8(q, s, state["w"], state["scale"], state["group_start"], state["group_rows"],
                                 swiglu=case["swiglu"])
    from rbruck_alltoallv_b200.ops.norm import block_norm
    out = block_norm(state["residual"], state["branch"], state["post_weight"], gate=state["gate"], scale=case["scale"],
                     pre_weight=state["pre_weight"], eps=EPS)
    if case["backward"]:
        grads = torch.autograd.grad(out, [state[n] for n in _norm_leaves(state)], (state["d_residual"], state["d_normed"]))
        out = tuple(t.detach() for t in out) + grads
    return out


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    if case["family"] == "moe":
        T, H, I, E, k = (case[n] for n in ("tokens", "hidden", "inter", "experts", "top_k"))
        return {"bytes": _used_experts(case) * 3 * H * I * 2 + T * (2 * 2 * H + 4 * E), "flops": 2 * T * k * 3 * H * I}
    if case["family"] == "int8":
        rows, N, K = case["rows"], case["chan"], case["depth"]
        live = case["groups"] - case["empty"]
        return {"bytes": live * N * (K + 4) + rows * 2 * (K + (N // 2 if case["swiglu"] else N)), "flops": 2 * rows * N * K}
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    T, H = case["tokens"], case["hidden"]
    z, r, w = size[case["type"]], size[case["residual"]], size[case["weights"]]
    gate = {"none": 0, "channel": H * w, "token": T * w, "full": T * H * z}[case["gate"]]
    total = T * H * (2 * r + 2 * z) + 2 * H * w + gate                         # r, z in; r', u out
    flops = 8 * T * H
    if case["backward"]:
        total += T * H * (2 * r + 2 * z) + 2 * H * w + gate                    # dr', du in; dr, dz out; weights' gradients
        flops += 20 * T * H
    return {"bytes": total, "flops": flops}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def _exact_moe(st):
    k = st["case"]["top_k"]
    x, l = st["x"].double(), st["logits"].double()
    out = torch.zeros_like(x)
    per_expert = {}
    for t, row in enumerate(l.tolist()):
        best = sorted(range(len(row)), key=lambda e: (-row[e], e))[:k]
        total = sum(math.exp(row[e] - row[best[0]]) for e in best)
        for e in best:
            per_expert.setdefault(e, []).append((t, math.exp(row[e] - row[best[0]]) / total))
    for e, pairs in per_expert.items():
        rows = torch.tensor([t for t, _ in pairs], device=x.device)
        weight = torch.tensor([p for _, p in pairs], dtype=torch.float64, device=x.device)
        gate_up = x[rows] @ st["w13"][e].double().t()
        mid = torch.nn.functional.silu(gate_up[:, 0::2]) * gate_up[:, 1::2]
        out.index_add_(0, rows, weight[:, None] * (mid @ st["w2"][e].double().t()))
    return out


def _exact_int8(st):
    x = st["x"].double()
    most = x.abs().amax(-1)
    s = torch.where(most > 0, most / 127, 1.0)
    q = torch.round(x / s[:, None])
    if st["case"]["kind"] == "linear":
        return torch.einsum("rk,nk->rn", q, st["w"].double()) * torch.outer(s, st["scale"].double())
    N = st["w"].shape[1]
    y = torch.empty(len(x), N, dtype=torch.float64, device=x.device)
    for g, (at, n) in enumerate(zip(st["host_start"], st["host_rows"])):
        y[at:at + n] = torch.einsum("rk,nk->rn", q[at:at + n], st["w"][g].double()) * torch.outer(s[at:at + n], st["scale"][g].double())
    return torch.nn.functional.silu(y[:, 0::2]) * y[:, 1::2] if st["case"]["swiglu"] else y


def _exact_norm(st):
    case = st["case"]
    v = {n: st[n].detach().double() for n in _norm_leaves(st)}
    z, r, w1, w2 = v["branch"], v["residual"], v["post_weight"], v["pre_weight"]
    g = case["scale"] * v.get("gate", torch.ones((), dtype=torch.float64, device=z.device))
    i1 = 1 / torch.sqrt(z.square().mean(-1, keepdim=True) + EPS)
    zh = z * i1
    r2 = r + g * w1 * zh
    i2 = 1 / torch.sqrt(r2.square().mean(-1, keepdim=True) + EPS)
    xh = r2 * i2
    if not case["backward"]:
        return r2, xh * w2
    dr, du = st["d_residual"].double(), st["d_normed"].double()
    a = du * w2
    d = dr + i2 * (a - xh * (a * xh).mean(-1, keepdim=True))
    b = g * d * w1
    dz = i1 * (b - zh * (b * zh).mean(-1, keepdim=True))
    out = [r2, xh * w2, d, dz, (g * d * zh).sum(0), (du * xh).sum(0)]
    if "gate" in v:
        dg = case["scale"] * w1 * zh * d
        out.append(dg.sum(0) if case["gate"] == "channel" else dg.sum(1, keepdim=True) if case["gate"] == "token" else dg)
    return tuple(out)


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"moe": _exact_moe, "int8": _exact_int8, "norm": _exact_norm}[case["family"]](st)
