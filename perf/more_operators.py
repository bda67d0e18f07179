"""Operators for training a MoE layer in less memory, on one GPU, as cases to be timed and
compared: activations kept in 8 bits between forward and backward, and the balance loss of
packed and padded sequences with its per-expert counts.

A case is a dict of plain values.  ``kind`` names the operator:

  store    compress_activation, then restore (or restore_rows in expert order)
  swiglu   swiglu_compress, then swiglu_backward_8bit: h, and the gradients of gate and up
  norm     rmsnorm_compress, then rmsnorm_backward_8bit: y, and the gradients of x and the weight
  balance  balance_forward, then balance_backward: loss, counts, and the logits' gradient

An activation in 8 bits: blocks of 32 along a row share a power of two s, the largest value's
power of two over 64; a value is the nearest whole multiple of s within +-127 s.

Where ``own`` is true, ``run`` makes the framework's calls; else it computes the same in
elementary torch operations.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6       # RMSNorm
BLOCK = 32       # values that share a scale
SUM_FLOOR = 1e-8  # added to the sum of a token's sigmoid scores
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ==================================================================== cases ====
def store(rows, cols, dtype="bf16", experts=0, top_k=0):
    """``experts``: the rows come back in expert order, ``top_k`` copies of each, groups padded."""
    return {"kind": "store", "rows": rows, "cols": cols, "dtype": dtype, "experts": experts, "top_k": top_k}


def swiglu(rows, hidden, dtype="bf16", packed=True):
    """``packed``: gate and up are the halves of one [rows, 2 hidden] tensor, as the gate|up product leaves them."""
    return {"kind": "swiglu", "rows": rows, "hidden": hidden, "dtype": dtype, "packed": packed}


def norm(rows, cols, dtype="bf16"):
    return {"kind": "norm", "rows": rows, "cols": cols, "dtype": dtype}


def balance(tokens, experts, top_k, sequences=0, scores="softmax", masked=0.0, z=0.0):
    """``sequences`` 0: the tokens are one batch; else packed, some of them empty, a few tokens behind the last."""
    return {"kind": "balance", "tokens": tokens, "experts": experts, "top_k": top_k, "sequences": sequences,
            "scores": scores, "masked": masked, "z": z}


def listed():
    return [
        # a small micro-batch's tokens: launches and latency count
        {"name": "store_small", **store(64, 2048)},
        # an fp32 activation, no size a multiple of anything
        {"name": "store_odd", **store(1409, 2817, "fp32")},
        # tokens kept once, read back in expert order for the weight gradients of top-2 experts
        {"name": "store_experts", **store(16384, 4096, experts=8, top_k=2)},
        # the gate|up rows of one tile of tokens
        {"name": "swiglu_small", **swiglu(128, 1408)},
        # two tensors whose rows start anywhere
        {"name": "swiglu_odd", **swiglu(3001, 1419, packed=False)},
        # a step's tokens through a wide feed-forward layer: the bytes
        {"name": "swiglu_wide", **swiglu(16384, 14336)},
        # a short sequence: latency, and few rows to sum the weight's gradient over
        {"name": "norm_small", **norm(37, 2048)},
        # fp32 residuals of an odd width
        {"name": "norm_odd", **norm(2999, 2831, "fp32")},
        # a long batch of wide tokens: the bytes
        {"name": "norm_wide", **norm(16384, 7168)},
        # a router of 8 experts over a short batch: latency
        {"name": "balance_small", **balance(512, 8, 2)},
        # packed documents with padding, fine-grained experts, a z-loss
        {"name": "balance_packed", **balance(16384, 64, 6, sequences=40, masked=0.1, z=1e-3)},
        # a long step of many short sequences, 256 experts with sigmoid scores
        {"name": "balance_long", **balance(65536, 256, 8, sequences=512, scores="sigmoid")},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(work(c)["bytes"] for c in listed())
    while True:
        kind = rng.choice(("store", "swiglu", "swiglu", "norm", "norm", "balance", "balance"))
        dtype = rng.choice(("bf16", "bf16", "fp32"))
        rows, cols = _log(rng, 1, 32768), _log(rng, 32, 16384)
        if rng.random() < 0.5:
            cols = max(1, cols // 32) * 32
        if kind == "store":
            case = store(rows, cols, dtype)
            if rng.random() < 0.4:
                case["experts"], case["top_k"] = rng.choice(((8, 2), (16, 4), (64, 6)))
        elif kind == "swiglu":
            case = swiglu(rows, cols, dtype, rng.random() < 0.5)
        elif kind == "norm":
            case = norm(rows, cols, dtype)
        else:
            experts, top_k = rng.choice(((4, 1), (8, 2), (16, 4), (60, 4), (64, 6), (128, 8), (160, 6), (256, 8)))
            case = balance(_log(rng, 1, 131072), experts, top_k, scores=rng.choice(("softmax", "softmax", "sigmoid")),
                           masked=rng.choice((0.0, 0.1, 0.5)), z=rng.choice((0.0, 1e-3)))
            if rng.random() < 0.6:
                case["sequences"] = _log(rng, 1, max(1, case["tokens"] // 4))
        if work(case)["bytes"] <= most:
            return case


def _gathered(case):
    """Rows of the expert order, an upper bound known without the routing."""
    return (case["rows"] * case["top_k"] + case["experts"] * 127) // 128 * 128


def work(case):
    if case["kind"] == "balance":   # logits and indices in, the gradient, counts and loss out
        T, E, K = case["tokens"], case["experts"], case["top_k"]
        return {"bytes": 8 * T * E + 8 * T * K + (T if case["masked"] else 0) + 4 * max(1, case["sequences"]) * E,
                "flops": 12 * T * E}
    size = 2 if case["dtype"] == "bf16" else 4
    kept = 1 + 1 / BLOCK   # a value in 8 bits and its share of the scale: written by the forward, read by the backward
    if case["kind"] == "store":
        n = case["rows"] * case["cols"]
        out = _gathered(case) * case["cols"] if case["experts"] else n
        return {"bytes": n * size + 2 * n * kept + out * size, "flops": 3 * n}
    if case["kind"] == "swiglu":   # gate, up, dh in; h, dgate, dup out
        n = case["rows"] * case["hidden"]
        return {"bytes": 6 * n * size + 4 * n * kept, "flops": 20 * n}
    n = case["rows"] * case["cols"]   # x, dy in; y, dx out
    return {"bytes": 4 * n * size + 2 * n * kept + 8 * case["cols"] + 8 * case["rows"], "flops": 16 * n}


# =================================================================== inputs ====
def _normal(gen, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=gen, device=DEV) * std).to(dtype)


def _activation(gen, rows, cols, dtype):
    """Features of different sizes, and a few outliers."""
    x = torch.randn(rows, cols, generator=gen, device=DEV)
    x *= torch.exp(torch.randn(cols, generator=gen, device=DEV))
    x *= torch.where(torch.rand(cols, generator=gen, device=DEV) < 2e-3, 20.0, 1.0)
    return x.to(dtype)


def _expert_order(gen, case):
    """The token of each row of the expert order, -1 on the rows that pad a group to 128."""
    T, E, K = case["rows"], case["experts"], case["top_k"]
    chosen = torch.rand(T, E, generator=gen, device=DEV).topk(K, dim=1).indices.flatten()
    order = torch.argsort(chosen, stable=True)
    sizes = torch.bincount(chosen, minlength=E)
    padded = (sizes + 127) // 128 * 128
    start = torch.cumsum(padded, 0) - padded
    expert = chosen[order]
    place = start[expert] + torch.arange(T * K, device=DEV) - (torch.cumsum(sizes, 0) - sizes)[expert]
    index = torch.full((_gathered(case),), -1, dtype=torch.int32, device=DEV)
    index[place] = (order // K).to(torch.int32)
    return index


def _borders(gen, tokens, sequences):
    """Sequence borders in a packed batch: random ones (equal ones: an empty sequence), a short rest behind the last."""
    end = tokens - tokens // 50
    inner = (torch.rand(sequences - 1, generator=gen, device=DEV) * (end + 1)).long().clamp_max(end).sort().values
    return torch.cat((inner.new_zeros(1), inner, inner.new_full((1,), end))).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed) + 1)
    state = {"case": dict(case)}
    if case["kind"] == "balance":
        T, E = case["tokens"], case["experts"]
        ranks = torch.randperm(E, generator=gen, device=DEV) + 1
        state["logits"] = torch.randn(T, E, generator=gen, device=DEV) - 0.5 * torch.log(ranks.float())
        state["indices"] = state["logits"].topk(case["top_k"], dim=1).indices
        state["mask"] = torch.rand(T, generator=gen, device=DEV) >= case["masked"] if case["masked"] else None
        state["borders"] = _borders(gen, T, case["sequences"]) if case["sequences"] else None
        state["dloss"] = torch.full((), 0.01, device=DEV)
        return state
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "store":
        state["x"] = _activation(gen, case["rows"], case["cols"], dtype)
        state["index"] = _expert_order(gen, case) if case["experts"] else None
    elif case["kind"] == "swiglu":
        M, H = case["rows"], case["hidden"]
        if case["packed"]:
            state["gate"], state["up"] = _activation(gen, M, 2 * H, dtype), None
        else:
            state["gate"], state["up"] = _activation(gen, M, H, dtype), _activation(gen, M, H, dtype)
        state["dh"] = _normal(gen, M, H, std=1e-2, dtype=dtype)
    else:
        state["x"] = _activation(gen, case["rows"], case["cols"], dtype)
        state["weight"] = 1 + _normal(gen, case["cols"], std=0.1, dtype=torch.float32)
        state["dy"] = _normal(gen, case["rows"], case["cols"], std=1e-2, dtype=dtype)
    return state


# ============================================================ the operators ====
def _run_own(state):
    import nanopysche_amd as fm

    case = state["case"]
    if case["kind"] == "store":
        kept = fm.compress_activation(state["x"])
        return kept.restore() if state["index"] is None else kept.restore_rows(state["index"])
    if case["kind"] == "swiglu":
        h, gate, up = fm.swiglu_compress(state["gate"], state["up"])
        grad = fm.swiglu_backward_8bit(state["dh"], gate, up, packed=case["packed"])
        return {"h": h, "grad": grad}
    if case["kind"] == "norm":
        y, kept, rstd = fm.rmsnorm_compress(state["x"], state["weight"], EPS)
        dx, dw = fm.rmsnorm_backward_8bit(state["dy"], kept, state["weight"], rstd)
        return {"y": y, "dx": dx, "dw": dw}
    loss, counts, saved = fm.balance_forward(state["logits"], state["indices"], cu_seqlens=state["borders"],
                                             token_mask=state["mask"], scores=case["scores"],
                                             z_loss_multiplier=case["z"])
    return {"loss": loss, "counts": counts, "dlogits": fm.balance_backward(saved, state["dloss"])}


# =============================================================== plain form ====
def _kept(x):
    """fp32 x [rows, cols] as the values that its 8 bits stand for."""
    rows, cols = x.shape
    blocks = torch.nn.functional.pad(x, (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    top = blocks.abs().amax(dim=2, keepdim=True)
    code = ((top.view(torch.int32) >> 23) - 6).clamp_min(0)   # the scale's exponent, as fp32 stores it
    scale = torch.where(code > 0, code << 23, 1 << 22).view(torch.float32)
    q = torch.round(blocks * ((254 - code) << 23).view(torch.float32)).clamp(-127, 127)
    return (q * scale).view(rows, -1)[:, :cols]


def _plain_balance(state):
    case, logits, indices = state["case"], state["logits"], state["indices"]
    T, E = logits.shape
    borders = torch.tensor([0, T], device=logits.device) if state["borders"] is None else state["borders"].long()
    token = torch.arange(T, device=logits.device)
    S = borders.numel() - 1
    sequence = torch.searchsorted(borders, token, right=True) - 1
    counts_in = (sequence >= 0) & (sequence < S)
    sequence = sequence.clamp(0, S - 1)
    if state["mask"] is not None:
        counts_in = counts_in & state["mask"]
    one = counts_in.double()
    if case["scores"] == "softmax":
        z = torch.exp(logits - logits.amax(dim=1, keepdim=True))
        p = z / z.sum(dim=1, keepdim=True)
    else:
        sigma = 1 / (1 + torch.exp(-logits))
        total = sigma.sum(dim=1, keepdim=True) + SUM_FLOOR
        p = sigma / total
    taken = torch.zeros_like(p).scatter_add_(1, indices, torch.ones_like(indices, dtype=p.dtype))
    every_token = torch.cat((torch.ones_like(p[:, :1]), p, taken), dim=1).double() * one[:, None]
    if S <= 64:   # sums over tokens, long ones: 64 bits, as a product while that is quicker
        sums = (sequence == torch.arange(S, device=logits.device)[:, None]).double() @ every_token
    else:
        sums = torch.zeros(S, 1 + 2 * E, dtype=torch.float64, device=logits.device).index_add_(0, sequence, every_token)
    tokens, sums, slots = sums[:, 0], sums[:, 1:1 + E], sums[:, 1 + E:]
    n = tokens.clamp_min(1)[:, None]
    filled = (tokens > 0).sum().clamp_min(1)
    loss = E * ((slots / n) * (sums / n)).sum() / filled
    f = (E * slots / (n * n) / filled * state["dloss"].double()).float()[sequence]   # the weight of each p of a token
    inner = f - (f * p).sum(dim=1, keepdim=True)
    grad = p * inner if case["scores"] == "softmax" else inner / total * sigma * (1 - sigma)
    if case["z"]:
        top = logits.amax(dim=1)
        lse = top + torch.log(torch.exp(logits - top[:, None]).sum(dim=1))
        every = one.sum().clamp_min(1)
        loss = loss + case["z"] * (lse.double().square() * one).sum() / every
        soft = torch.exp(logits - lse[:, None])
        grad = grad + (2 * case["z"] * state["dloss"].double() / every).float() * lse[:, None] * soft
    counts = slots.to(torch.int32)
    return {"loss": loss.float(), "counts": counts if state["borders"] is not None else counts[0],
            "dlogits": torch.where(counts_in[:, None], grad, 0.0)}


def _run_plain(state):
    case = state["case"]
    if case["kind"] == "balance":
        return _plain_balance(state)
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "store":
        values = _kept(state["x"].float())
        if state["index"] is not None:
            index = state["index"].long()
            values = torch.where((index >= 0)[:, None], values[index.clamp_min(0)], 0.0)
        return values.to(dtype)
    if case["kind"] == "swiglu":
        H = case["hidden"]
        gate, up = (state["gate"][:, :H], state["gate"][:, H:]) if case["packed"] else (state["gate"], state["up"])
        gate, up, dh = gate.float(), up.float(), state["dh"].float()
        h = gate / (1 + torch.exp(-gate)) * up
        gate, up = _kept(gate), _kept(up)
        s = 1 / (1 + torch.exp(-gate))
        dgate = (dh * up * s * (1 + gate * (1 - s))).to(dtype)
        dup = (dh * gate * s).to(dtype)
        return {"h": h.to(dtype), "grad": torch.cat((dgate, dup), dim=1) if case["packed"] else (dgate, dup)}
    x, w, dy = state["x"].float(), state["weight"], state["dy"].float()
    r = 1 / torch.sqrt((x * x).sum(dim=1, keepdim=True) / case["cols"] + EPS)
    y = x * r * w
    x = _kept(x)
    a = dy * w
    dx = r * a - r * r * r * ((a * x).sum(dim=1, keepdim=True) / case["cols"]) * x
    dw = (dy * x * r).sum(dim=0)
    return {"y": y.to(dtype), "dx": dx.to(dtype), "dw": dw}


def run(state):
    with torch.no_grad():
        return _run_own(state) if own else _run_plain(state)


# ============================================================== 64 bits ====
def _exact_kept(x):
    """The same 8 bits from the definition: s = 2^(floor(log2 max) - 6), at least 2^-127."""
    rows, cols = x.shape
    out = torch.empty_like(x)
    whole = cols // BLOCK * BLOCK
    for part in (slice(0, whole), slice(whole, cols)):
        v = x[:, part]
        if v.numel():
            v = v.reshape(rows, -1, min(BLOCK, v.shape[1]))
            power = torch.frexp(v.abs().amax(dim=2, keepdim=True)).exponent - 1   # floor(log2 max)
            s = ((power - 6).clamp_min(-127).long() + 1023 << 52).view(torch.float64)
            out[:, part] = (torch.round(v / s).clamp(-127, 127) * s).reshape(rows, -1)
    return out


def _exact_balance(state):
    case = state["case"]
    logits = state["logits"].double().requires_grad_(True)
    T, E = logits.shape
    borders = [0, T] if state["borders"] is None else state["borders"].tolist()
    S = len(borders) - 1
    lengths = torch.tensor([b - a for a, b in zip(borders, borders[1:])], device=logits.device)
    member = torch.repeat_interleave(torch.arange(S, device=logits.device), lengths)   # tokens 0 .. borders[-1]
    use = torch.ones(T, dtype=torch.bool, device=logits.device) if state["mask"] is None else state["mask"].clone()
    use[borders[-1]:] = False
    rows = use.nonzero().flatten()
    member = member[rows]
    if rows.numel() == 0:
        return {"loss": torch.zeros((), dtype=torch.float64, device=logits.device), "counts": None,
                "dlogits": torch.zeros(T, E, dtype=torch.float64, device=logits.device)}
    with torch.enable_grad():
        if case["scores"] == "softmax":
            p = torch.softmax(logits[rows], dim=1)
        else:
            p = torch.sigmoid(logits[rows])
            p = p / (p.sum(dim=1, keepdim=True) + SUM_FLOOR)
        n = torch.bincount(member, minlength=S).double()
        slots = torch.bincount((member[:, None] * E + state["indices"][rows]).flatten(), minlength=S * E).view(S, E)
        f = slots / n.clamp_min(1)[:, None]
        loss = E * (f[member] * p / n[member, None]).sum() / (n > 0).sum()
        if case["z"]:
            loss = loss + case["z"] * torch.logsumexp(logits[rows], dim=1).square().mean()
        grad, = torch.autograd.grad(loss * state["dloss"].double(), logits)
    counts = slots.to(torch.int32)
    return {"loss": loss.detach(), "counts": counts if state["borders"] is not None else counts[0], "dlogits": grad}


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "balance":
        return _exact_balance(state)
    with torch.no_grad():
        if case["kind"] == "store":
            values = _exact_kept(state["x"].double())
            if state["index"] is None:
                return values
            out = torch.zeros(state["index"].numel(), case["cols"], dtype=torch.float64, device=values.device)
            real = state["index"] >= 0
            out[real] = values[state["index"][real].long()]
            return out
        if case["kind"] == "swiglu":
            gate, up = state["gate"].chunk(2, dim=1) if case["packed"] else (state["gate"], state["up"])
            gate, up, dh = gate.double(), up.double(), state["dh"].double()
            h = gate * torch.sigmoid(gate) * up
            gate, up = _exact_kept(gate), _exact_kept(up)
            s = torch.sigmoid(gate)
            dgate, dup = dh * up * (s + gate * s * (1 - s)), dh * gate * s
            return {"h": h, "grad": torch.cat((dgate, dup), dim=1) if case["packed"] else (dgate, dup)}
        x, w, dy = state["x"].double(), state["weight"].double(), state["dy"].double()
        r = torch.rsqrt(x.square().mean(dim=1) + EPS)[:, None]
        y = x * r * w
        xr = _exact_kept(x) * r
        dx = r * (dy * w - xr * (dy * w * xr).mean(dim=1, keepdim=True))
        return {"y": y, "dx": dx, "dw": (dy * xr).sum(dim=0)}
