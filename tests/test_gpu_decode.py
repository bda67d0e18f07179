"""The few-token MoE layer (moe_decode, expert_decode) against float64, at the edges of its
token passes, slice sizes and expert lists.

Tolerances, per element, from the arithmetic: sums of n products in fp32 are off by at most
n 2^-24 sum |terms|; |silu'| <= 1.1; h (and xn under a norm) enters the second product as two
bf16 pieces, off by at most 2^-16 of its value; the output is rounded once."""

import pytest
import torch

import nanopysche_amd as fm
from tests.helpers import randn_bf16

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def ffn64(x, ex, w1, w2, w3):
    """(y, bound) of one expert's w1, w2, w3 [H, D] for x [n, D], off by at most ex."""
    D, H = w1.shape[1], w1.shape[0]
    g, u = x @ w1.t(), x @ w3.t()
    eg = D * U * (x.abs() @ w1.abs().t()) + ex @ w1.abs().t()
    eu = D * U * (x.abs() @ w3.abs().t()) + ex @ w3.abs().t()
    s = g * torch.sigmoid(g)
    h = s * u
    eh = 1.1 * eg * (u.abs() + eu) + (s.abs() + 1.1 * eg) * eu + (2.0 ** -16 + 16 * U) * h.abs()
    return h @ w2, eh @ w2.abs() + (H + 64) * U * ((h.abs() + eh) @ w2.abs())


def layer64(x, ex, weights, indices, w, E, offset=0, shared=None):
    """(out, bound) [T, D] of the routed experts w = (w1, w2, w3) [E * H, D] in float64."""
    out, bound = torch.zeros_like(x), torch.zeros_like(x)
    w = [t.double().view(E, -1, x.shape[1]) for t in w]
    for e in range(E):
        for t, k in (indices - offset == e).nonzero().tolist():
            y, b = ffn64(x[t:t + 1], ex[t:t + 1], w[0][e], w[1][e], w[2][e])
            c = weights[t, k].double()
            out[t] += c * y[0]
            bound[t] += c.abs() * b[0] + 8 * U * (c * y[0]).abs()
    if shared is not None:
        y, b = ffn64(x, ex, *(t.double() for t in shared))
        out += y
        bound += b + 8 * U * y.abs()
    return out, bound + 1e-30


def check(got, ref, bound):
    half = torch.finfo(got.dtype).eps / 2
    got = got.double()
    assert torch.isfinite(got).all()
    worst = ((got - ref).abs() - half * ref.abs() - (1 + half) * bound).max().item()
    assert worst <= 0, worst


def routing(T, E, K, seed, skew=False):
    g = torch.Generator().manual_seed(seed)
    scores = torch.randn(T, E, generator=g) + (torch.arange(E) == 0) * (10.0 if skew else 0.0)
    top = scores.topk(K, 1)
    return torch.softmax(top.values, 1), top.indices


def expert_weights(E, H, D, seed):
    return [randn_bf16((E * H, D), seed=seed + i, std=0.05) for i in range(3)]


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 33, 64])
@pytest.mark.parametrize("E,K,H,D", [(4, 1, 128, 128), (3, 2, 384, 640), (40, 6, 128, 256)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_experts_match_float64(dev, T, E, K, H, D, dtype):
    x = randn_bf16((T, D), seed=T).to(dev, dtype)
    weights, indices = (t.to(dev) for t in routing(T, E, K, T, skew=True))
    w = [t.to(dev) for t in expert_weights(E, H, D, 5)]
    got = fm.expert_decode(x, weights, indices, w, E)
    assert got.dtype == dtype and got.shape == x.shape
    check(got, *layer64(x.double(), torch.zeros_like(x, dtype=torch.float64), weights, indices, w, E))


@pytest.mark.parametrize("H,E,K,T", [(4096, 16, 8, 20), (2048, 8, 2, 12), (2048, 64, 4, 2), (4096, 32, 6, 2), (1408, 8, 2, 1)])
@pytest.mark.parametrize("norm", [False, True])
def test_every_slice_size(dev, H, E, K, T, norm):
    """Tokens and experts that take 64, 64, 32, 32 and 16 hidden units a workgroup, x in one piece and in two."""
    D = 256
    x = randn_bf16((T, D), seed=T).to(dev)
    gate = randn_bf16((E, D), seed=1, std=0.2).to(dev)
    nw = (1 + 0.1 * torch.randn(D, generator=torch.Generator().manual_seed(4))).to(dev) if norm else None
    w = [t.to(dev) for t in expert_weights(E, H, D, 5)]
    r = fm.moe_decode(x.float(), gate, w, K, norm_weight=nw)
    x64 = x.double()
    ex = torch.zeros_like(x64)
    if norm:
        x64 = x64 * torch.rsqrt(x64.square().mean(1, keepdim=True) + 1e-6) * nw.double()
        ex = 2.0 ** -16 * x64.abs()
    check(r.out, *layer64(x64, ex, r.weights, r.indices, w, E))


def router64(x, gate, bias, score, K, gating, l2):
    logits = x @ gate.double().t()
    for b in (bias, score):
        if b is not None:
            logits = logits + b.double()
    s = torch.sigmoid(logits) if gating == "sigmoid" else logits
    top = s.topk(K, 1)
    w = top.values / (top.values.sum(1, keepdim=True) + 1e-8) if gating == "sigmoid" else torch.softmax(top.values, 1)
    if l2:
        w = w / (w.norm(dim=1, keepdim=True) + 1e-8)
    return w, top.indices


@pytest.mark.parametrize("T", [1, 7, 33])
@pytest.mark.parametrize("E,K", [(1, 1), (8, 2), (65, 6), (256, 8), (1000, 16)])
@pytest.mark.parametrize("gating,norm,shared", [("softmax", False, 0), ("sigmoid", True, 0), ("softmax", True, 256)])
def test_whole_layer_matches_float64(dev, T, E, K, gating, norm, shared):
    D, H = 384, 128
    x = randn_bf16((T, D), seed=T, std=3.0).to(dev)
    gate = randn_bf16((E, D), seed=1, std=0.05).to(dev, torch.float32 if E == 65 else torch.bfloat16)
    gbias = (torch.randn(E, generator=torch.Generator().manual_seed(2)) * 0.1).to(dev) if E != 8 else None
    score = (torch.randn(E, generator=torch.Generator().manual_seed(3)) * 0.1).to(dev) if E != 65 else None
    nw = (1 + 0.1 * torch.randn(D, generator=torch.Generator().manual_seed(4))).to(dev) if norm else None
    w = [t.to(dev) for t in expert_weights(E, H, D, 5)]
    sw = [t.to(dev) for t in expert_weights(1, shared, D, 9)] if shared else None
    r = fm.moe_decode(x, gate, w, K, gate_bias=gbias, score_bias=score, gating=gating, norm_weight=nw, shared=sw,
                      normalize_expert_weights="l2" if E == 8 else None)
    x64 = x.double()
    ex = torch.zeros_like(x64)
    if norm:
        x64 = x64 * torch.rsqrt(x64.square().mean(1, keepdim=True) + 1e-6) * nw.double()
        ex = 2.0 ** -16 * x64.abs()
    weights, indices = router64(x64, gate, gbias, score, K, gating, E == 8)
    # a selection that rounding could turn is no fault: logits are off by at most 1e-4 here
    logits = x64 @ gate.double().t()
    assert r.indices.dtype == torch.int64 and r.weights.dtype == torch.float32
    same = (r.indices == indices).all(1)
    assert same.float().mean() >= 0.9
    assert (r.weights[same].double() - weights[same]).abs().max() <= 1e-4
    assert logits.isfinite().all()
    check(r.out, *layer64(x64, ex, r.weights, r.indices, w, E, shared=sw))
