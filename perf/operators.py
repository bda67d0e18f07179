"""The serving operators on one GPU, as cases to be timed and compared: a MoE layer for a few
tokens (decoding), and products in 8-bit integers with a scale for each token and channel.

A case is a dict of plain values.  ``kind`` names the operator:

  decode   moe_decode: norm, router, the reached experts, shared expert and combine of a few
           tokens; experts in bf16 as a layer stores them, or in int8 with a scale per channel
  quant    quantize_to_int8 of rows, read back
  linear   int8_linear: rows quantised, times int8 weights, scaled by token and channel
  experts  Int8MoECompute: permute, int8 grouped products, SwiGLU, combine of a routed prompt

Where ``own`` is true, ``run`` makes these calls; else it computes the same in elementary torch
operations.  Routers' inputs are drawn so that every selection is decided by more than rounding.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
GAP = 1e-3     # the K + 1 largest logits of a token lie at least this far apart
EPS = 1e-6     # RMSNorm
FLOOR = 1e-12  # least absolute maximum of a quantised row


# ==================================================================== cases ====
def decode(name=None, **kw):
    case = {"kind": "decode", "tokens": 1, "d_model": 2048, "hidden": 1408, "experts": 8, "top_k": 2, "shared": 0,
            "norm": False, "gating": "softmax", "skew": 0.0, "weights": "bf16"}
    case.update(kw)
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # one sequence's next token through a small layer: launches and latency count
        decode("decode_one"),
        # a few sequences through a fine-grained pre-norm layer with a shared expert: the experts are nearly all distinct
        decode("decode_fine", tokens=5, experts=64, top_k=6, norm=True, shared=2816),
        # a batch of sequences through wide experts, all of them reached: the weights' bytes
        decode("decode_wide", tokens=17, d_model=4096, hidden=14336),
        # the largest batch that is still "a few": a rank's 32 experts in int8, sigmoid router with a score bias
        decode("decode_share", tokens=64, d_model=7168, hidden=2048, experts=32, top_k=8, gating="sigmoid", skew=0.6,
               weights="int8"),
        # a prompt's activations quantised by token
        {"name": "quant_prompt", "kind": "quant", "rows": 8192, "cols": 4096, "dtype": "bf16"},
        # odd sizes and fp32 rows, as of a checkpoint's weight quantised by channel
        {"name": "quant_odd", "kind": "quant", "rows": 1409, "cols": 2817, "dtype": "fp32"},
        # a token through a wide projection: the weights' bytes
        {"name": "linear_one", "kind": "linear", "rows": 1, "cols": 4096, "outs": 14336, "bias": False, "dtype": "bf16"},
        # some tens of tokens, no size a multiple of anything
        {"name": "linear_odd", "kind": "linear", "rows": 77, "cols": 1409, "outs": 2831, "bias": True, "dtype": "fp32"},
        # a short prompt: few tiles of output
        {"name": "linear_short", "kind": "linear", "rows": 512, "cols": 2048, "outs": 5632, "bias": True, "dtype": "bf16"},
        # a long prompt through a wide projection: the matrix cores' rate
        {"name": "linear_long", "kind": "linear", "rows": 8192, "cols": 4096, "outs": 14336, "bias": False,
         "dtype": "bf16"},
        # a prompt through the routed experts of a small layer, balanced
        {"name": "experts_prompt", "kind": "experts", "tokens": 4096, "d_model": 2048, "hidden": 1408, "experts": 8,
         "top_k": 2, "skew": 0.0},
        # a prompt through wide experts of Zipf popularity: ragged groups
        {"name": "experts_wide", "kind": "experts", "tokens": 2048, "d_model": 4096, "hidden": 14336, "experts": 8,
         "top_k": 2, "skew": 1.1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _most():
    every = [work(c) for c in listed()]
    return max(w["bytes"] for w in every), max(w["flops"] for w in every)


def draw(rng):
    most_bytes, most_flops = _most()
    while True:
        kind = rng.choice(("decode", "decode", "decode", "linear", "linear", "linear", "experts", "experts", "quant"))
        if kind == "quant":
            case = {"kind": kind, "rows": _log(rng, 1, 16384), "cols": _log(rng, 64, 16384),
                    "dtype": rng.choice(("bf16", "fp32"))}
        elif kind == "linear":
            case = {"kind": kind, "rows": _log(rng, 1, 8192), "cols": _log(rng, 128, 14336),
                    "outs": _log(rng, 128, 14336), "bias": rng.random() < 0.5, "dtype": rng.choice(("bf16", "bf16", "fp32"))}
            if rng.random() < 0.5:
                case["cols"], case["outs"] = max(1, case["cols"] // 128) * 128, max(1, case["outs"] // 128) * 128
        else:
            experts, top_k = rng.choice(((4, 1), (8, 2), (16, 4), (32, 4), (32, 8), (60, 4), (64, 6), (128, 8)))
            size = {"d_model": 128 * _log(rng, 4, 56), "hidden": 128 * _log(rng, 3, 112), "experts": experts, "top_k": top_k}
            if kind == "experts":
                case = {"kind": kind, "tokens": _log(rng, 65, 8192), **size, "skew": rng.choice((0.0, 0.6, 1.1))}
                if case["tokens"] * experts * size["d_model"] * size["hidden"] > 2.5e12:
                    continue   # the plain form runs every token through every expert
            else:
                case = decode(tokens=_log(rng, 1, 64), **size, shared=rng.choice((0, 0, 1408, 2816)),
                              norm=rng.random() < 0.4, gating=rng.choice(("softmax", "sigmoid")),
                              skew=rng.choice((0.0, 0.6)), weights=rng.choice(("bf16", "int8")))
            if 3 * experts * size["d_model"] * size["hidden"] > 1.5e9:
                continue
        w = work(case)
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops:
            return case


def work(case):
    if case["kind"] == "quant":   # rows in, their int8 values out and back as bf16
        n = case["rows"] * case["cols"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + 2 * n + 4 * case["rows"], "flops": 3 * n}
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["cols"], case["outs"]
        return {"bytes": m * k * (2 if case["dtype"] == "bf16" else 4) + n * (k + 4) + 2 * m * n, "flops": 2 * m * n * k}
    T, D, H, E, K = (case[n] for n in ("tokens", "d_model", "hidden", "experts", "top_k"))
    reached = E * (1 - (1 - K / E) ** T)
    if case["kind"] == "experts":
        return {"bytes": 4 * T * D + 12 * T * K + reached * 3 * H * D, "flops": 6 * T * K * H * D}
    each = 2 if case["weights"] == "bf16" else 1
    return {"bytes": 4 * T * D + 2 * E * D + (reached * H + case["shared"]) * 3 * D * each,
            "flops": 6 * T * D * (K * H + case["shared"]) + 2 * T * D * E}


# =================================================================== inputs ====
def _normal(gen, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=gen, device=DEV) * std).to(dtype)


def _popularity(case, gen):
    """Score bias of a Zipf popularity over a random order of the experts."""
    ranks = torch.randperm(case["experts"], generator=gen, device=DEV) + 1
    return -case["skew"] * torch.log(ranks.float())


def _close(x, norm, gate, bias, k):
    """The tokens whose selection rounding could change."""
    x = x.double()
    if norm is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * norm.double()
    top = (x @ gate.double().t() + bias.double()).topk(k + 1, dim=1).values
    return ((top[:, :-1] - top[:, 1:]).min(dim=1).values < GAP).nonzero().flatten()


def _by_channel(gen, E, H, D, dim):
    """An expert weight [E * H, D] in int8, and its scales: a row's ([E * H]), or an expert's column's ([E, D])."""
    w = torch.randn(E, H, D, generator=gen, device=DEV) * 0.02
    scale = w.abs().amax(dim=dim).clamp_min(FLOOR) / 127
    q = torch.round(w / scale.unsqueeze(dim)).to(torch.int8).view(E * H, D)
    return q, scale.reshape(-1) if dim == 2 else scale


def _expert_weights(gen, kind, E, H, D):
    if kind == "bf16":
        return tuple(_normal(gen, E * H, D, std=0.02) for _ in range(3))
    return tuple(t for dim in (2, 1, 2) for t in _by_channel(gen, E, H, D, dim))


def _held(weights, E):
    """The experts as the framework takes them: bf16 parameters as they are, int8 ones laid out once."""
    import nanopysche_amd as fm

    return weights if len(weights) == 3 else fm.Int8Experts.from_int8(*weights, num_experts=E)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed) + 1)
    state = {"case": dict(case)}
    if case["kind"] in ("quant", "linear"):
        dtype = {"bf16": torch.bfloat16, "fp32": torch.float32}[case["dtype"]]
        x = _normal(gen, case["rows"], case["cols"], dtype=torch.float32)
        x *= torch.where(torch.rand(x.shape, generator=gen, device=DEV) < 1e-3, 20.0, 1.0)   # outlier activations
        state["x"] = x.to(dtype)
        if case["kind"] == "linear":
            q, scale = _by_channel(gen, 1, case["outs"], case["cols"], 2)
            state |= {"q": q, "scale": scale}
            state["bias"] = _normal(gen, case["outs"], dtype=torch.float32) if case["bias"] else None
            if own:
                import nanopysche_amd as fm

                state["weight"] = fm.Int8Tensor.from_int8(q, scale)
        return state
    T, D, H, E, K = (case[n] for n in ("tokens", "d_model", "hidden", "experts", "top_k"))
    bias = _popularity(case, gen)
    if case["kind"] == "experts":
        logits = torch.randn(T, E, generator=gen, device=DEV) + bias
        top = logits.topk(K, dim=1)
        state |= {"x": _normal(gen, T, D), "weights": torch.softmax(top.values, dim=1), "indices": top.indices}
        state["experts"] = _expert_weights(gen, "int8", E, H, D)
        if own:
            import nanopysche_amd as fm

            state["block"] = fm.Int8MoECompute(_held(state["experts"], E))
        return state
    state["gate"] = _normal(gen, E, D, std=0.02)
    state["bias"] = bias
    state["norm"] = 1 + _normal(gen, D, std=0.1, dtype=torch.float32) if case["norm"] else None
    state["experts"] = _expert_weights(gen, case["weights"], E, H, D)
    state["shared"] = _expert_weights(gen, case["weights"], 1, case["shared"], D) if case["shared"] else None
    state["x"] = x = _normal(gen, T, D)
    while (bad := _close(x, state["norm"], state["gate"], bias, K)).numel():
        x[bad] = _normal(gen, bad.numel(), D)
    if own:
        state["held"] = _held(state["experts"], E)
        state["held_shared"] = None if state["shared"] is None else _held(state["shared"], 1)
    return state


# ============================================================ the operators ====
def _run_own(state):
    import nanopysche_amd as fm

    case = state["case"]
    if case["kind"] == "quant":
        t = fm.quantize_to_int8(state["x"])
        return {"values": t.dequantize(), "scale": t.scale}
    if case["kind"] == "linear":
        return fm.int8_linear(state["x"], state["weight"], state["bias"], out_dtype=torch.bfloat16)
    if case["kind"] == "experts":
        return state["block"](state["x"], state["weights"], state["indices"])
    r = fm.moe_decode(state["x"], state["gate"], state["held"], case["top_k"], score_bias=state["bias"],
                      gating=case["gating"], norm_weight=state["norm"], norm_eps=EPS, shared=state["held_shared"])
    return {"out": r.out, "weights": r.weights, "indices": r.indices}


# =============================================================== plain form ====
def _quantised(x):
    """Rows (the last dimension) as whole numbers of their scale, and the scales."""
    scale = x.abs().amax(dim=-1).clamp_min(FLOOR) / 127
    return torch.round(x / scale.unsqueeze(-1)), scale


def _silu(x):
    return x / (1 + torch.exp(-x))


def _widened(weights, E, real):
    """w1, w2, w3 [E * H, D] as the numbers they stand for."""
    if len(weights) == 3:
        return [w.to(real) for w in weights]
    q1, s1, q2, s2, q3, s3 = weights
    EH, D = q2.shape
    w2 = q2.to(real).view(E, EH // E, D) * s2.to(real).view(E, 1, D)
    return [q1.to(real) * s1.to(real).unsqueeze(1), w2.view(EH, D), q3.to(real) * s3.to(real).unsqueeze(1)]


def _share_of(weights, indices, E):
    """[T, E]: the weight with which a token takes an expert (0: not at all)."""
    return torch.zeros(indices.shape[0], E, dtype=weights.dtype, device=weights.device).scatter_add_(1, indices, weights)


def _plain(state, real):
    case = state["case"]
    x = state["x"].to(real)
    if case["kind"] == "quant":
        q, scale = _quantised(x)
        return {"values": q * scale.unsqueeze(1), "scale": scale}
    if case["kind"] == "linear":
        q, scale = _quantised(x)
        out = (q @ state["q"].to(real).t()) * scale.unsqueeze(1) * state["scale"].to(real)
        return out if state["bias"] is None else out + state["bias"].to(real)
    E, T = case["experts"], case["tokens"]
    if case["kind"] == "experts":
        q1, s1, q2, s2, q3, s3 = (t.to(real) for t in state["experts"])
        q, scale = _quantised(x)
        h = _silu((q @ q1.t()) * scale.unsqueeze(1) * s1) * ((q @ q3.t()) * scale.unsqueeze(1) * s3)
        q, scale = _quantised(h.view(T, E, -1))
        scale = scale * _share_of(state["weights"].to(real), state["indices"], E)
        w2 = q2.view(E, -1, q2.shape[1]) * s2.unsqueeze(1)
        return (q * scale.unsqueeze(2)).view(T, -1) @ w2.view(q2.shape)
    if state["norm"] is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * state["norm"].to(real)
    logits = x @ state["gate"].to(real).t() + state["bias"].to(real)
    if case["gating"] == "sigmoid":
        top = (1 / (1 + torch.exp(-logits))).topk(case["top_k"], dim=1)
        weights = top.values / (top.values.sum(dim=1, keepdim=True) + 1e-8)
    else:
        top = logits.topk(case["top_k"], dim=1)
        weights = torch.exp(top.values - top.values[:, :1])
        weights = weights / weights.sum(dim=1, keepdim=True)
    w1, w2, w3 = _widened(state["experts"], E, real)
    h = _silu(x @ w1.t()) * (x @ w3.t())
    h = h.view(T, E, -1) * _share_of(weights, top.indices, E).unsqueeze(2)
    out = h.view(T, -1) @ w2
    if state["shared"] is not None:
        w1, w2, w3 = _widened(state["shared"], 1, real)
        out = out + (_silu(x @ w1.t()) * (x @ w3.t())) @ w2
    return {"out": out, "weights": weights, "indices": top.indices}


def run(state):
    if own:
        return _run_own(state)
    r = _plain(state, torch.float32)
    kind = state["case"]["kind"]
    if kind == "quant":
        return {"values": r["values"].bfloat16(), "scale": r["scale"]}
    if kind == "decode":
        return {"out": r["out"].bfloat16(), "weights": r["weights"], "indices": r["indices"]}
    return r.bfloat16()


# ==================================================================== exact ====
def _exact_rows(x):
    s = torch.clamp(torch.amax(torch.abs(x), -1, keepdim=True), min=FLOOR) / 127.0
    return torch.round(x / s), s


def _exact_ffn(x, up):
    """silu(x w1^T) * (x w3^T) for one expert."""
    g, u = x @ up[0].t(), x @ up[1].t()
    return g * torch.sigmoid(g) * u


def exact(case, seed):
    """The definition in 64 bits, an expert at a time over the tokens that take it."""
    state = prepare(case, seed)
    f64 = torch.float64
    x = state["x"].to(f64)
    kind = case["kind"]
    if kind == "quant":
        q, s = _exact_rows(x)
        return {"values": q * s, "scale": s[:, 0]}
    if kind == "linear":
        q, s = _exact_rows(x)
        w = state["q"].to(f64) * state["scale"].to(f64)[:, None]
        out = (q * s) @ w.t()
        return out if state["bias"] is None else out + state["bias"].to(f64)
    E, K, D, H = case["experts"], case["top_k"], case["d_model"], case["hidden"]
    if kind == "decode":
        if state["norm"] is not None:
            x = x / torch.sqrt((x * x).sum(1, keepdim=True) / D + EPS) * state["norm"].to(f64)
        logits = torch.addmm(state["bias"].to(f64), x, state["gate"].to(f64).t())
        best, indices = torch.sort(logits, dim=1, descending=True)
        best, indices = best[:, :K], indices[:, :K]
        if case["gating"] == "sigmoid":
            best = torch.sigmoid(best)
            weights = best / (best.sum(1, keepdim=True) + 1e-8)
        else:
            weights = torch.softmax(best, dim=1)
    else:
        weights, indices = state["weights"].to(f64), state["indices"]

    def expert(weights, e, h):
        """An expert's matrices [h, D] in 64 bits: gate, down, up."""
        if len(weights) == 3:
            return [w[e * h:(e + 1) * h].to(f64) for w in weights]
        q1, s1, q2, s2, q3, s3 = weights
        rows = slice(e * h, (e + 1) * h)
        return [q1[rows].to(f64) * s1[rows, None].to(f64), q2[rows].to(f64) * s2[e].to(f64),
                q3[rows].to(f64) * s3[rows, None].to(f64)]

    out = torch.zeros_like(x)
    if kind == "experts":
        q, s = _exact_rows(x)
        x = q * s
    for e in range(E):
        token, slot = (indices == e).nonzero(as_tuple=True)
        if token.numel():
            gate, down, up = expert(state["experts"], e, H)
            h = _exact_ffn(x[token], (gate, up))
            if kind == "experts":
                q, s = _exact_rows(h)
                h = q * s
            out.index_add_(0, token, (h @ down) * weights[token, slot, None])
    if kind == "experts":
        return out
    if case["shared"]:
        gate, down, up = expert(state["shared"], 0, case["shared"])
        out += _exact_ffn(x, (gate, up)) @ down
    return {"out": out, "weights": weights, "indices": None}
