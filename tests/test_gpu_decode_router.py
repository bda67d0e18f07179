"""moe_decode's router in every form of its kernel (1, 2, 4 or 8 experts a wave, bf16 and fp32
gates, with and without a norm, one launch and two) against float64, and the experts at wide D.

Tolerances.  A logit is summed by 64 lanes in chains of 8 ceil(D / 512) FMAs, then in 6
additions and 2 for the biases: off by at most n U sum |terms|, n = 8 ceil(D / 512) + 8,
U = 2^-24.  Under a norm the terms and the factor rsqrt(mean + eps) are rounded (2 and 4 steps)
and the sum of squares is off by n U, which the root halves: 2 n + 8 in all.  With logits off by
at most b, the k-th pick's logit is within 2 b of the k-th largest.  A softmax weight is then off
by a factor of exp(4 b) (numerator and sum), a sigmoid weight by 1 + 2 b, beside roundings:
expf 2 U, the difference of two logits U of it, K additions, a division."""

import math

import pytest
import torch

import nanopysche_amd as fm
from tests.helpers import randn_bf16
from tests.test_gpu_decode import check, layer64, routing

pytestmark = pytest.mark.gpu
U = 2.0 ** -24

# experts, top_k, D: one launch with 1, 2, 4 and 8 experts a wave, then two launches
FORMS = [(1, 1, 384), (3, 2, 128), (8, 2, 640), (4, 3, 14336), (9, 2, 384), (16, 16, 384), (16, 4, 4096), (17, 4, 384), (32, 8, 2048),
         (33, 4, 384), (60, 4, 1024), (64, 6, 1024), (128, 8, 512), (170, 8, 384),
         (8, 2, 14336), (32, 4, 4096), (64, 6, 2048), (171, 3, 384), (256, 8, 384), (1024, 16, 128)]


def expert_weights(dev, E, H, D, std=0.05):
    g = torch.Generator(device=dev).manual_seed(5)
    return [(torch.randn(E * H, D, generator=g, device=dev) * std).bfloat16() for _ in range(3)]


def logits64(x, gate, bias, score, norm):
    """(xn, logits, b [T]) in float64."""
    D = x.shape[1]
    n = 8 * math.ceil(D / 512) + 8
    x = x.double()
    if norm is not None:
        x = x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-6) * norm.double()
        n = 2 * n + 8
    g = gate.double().t().contiguous()
    logits, size = x @ g, x.abs() @ g.abs()
    for v in (bias, score):
        if v is not None:
            logits, size = logits + v.double(), size + v.double().abs()
    return x, logits, n * U * size.amax(1)


def check_router(r, logits, b, K, gating, l2):
    T, E = logits.shape
    assert r.indices.dtype == torch.int64 and r.weights.dtype == torch.float32 and r.indices.shape == r.weights.shape == (T, K)
    assert all(len(set(row)) == K and 0 <= min(row) and max(row) < E for row in r.indices.tolist())
    score = torch.sigmoid(logits) if gating == "sigmoid" else logits
    off = b / 4 + 6 * U if gating == "sigmoid" else b   # of a score: the sigmoid's slope is at most 1/4
    mine = score.gather(1, r.indices)
    assert ((mine - score.topk(K, 1).values).abs() <= 2 * off[:, None]).all()
    l = logits.gather(1, r.indices)
    if gating == "sigmoid":
        w = torch.sigmoid(l) / (torch.sigmoid(l).sum(1, keepdim=True) + 1e-8)
        rel = (2 * b + (16 + K) * U)[:, None].expand(T, K)
    else:
        w = torch.softmax(l, 1)
        rel = torch.expm1(4 * b)[:, None] + (16 + K + 2 * (l[:, :1] - l).abs().amax(1, keepdim=True)) * U
        rel = rel.expand(T, K)
    if l2:   # the norm's own error adds as much again
        w = w / (w.norm(dim=1, keepdim=True) + 1e-8)
        rel = 2 * rel.amax(1, keepdim=True) + (K + 8) * U
    assert ((r.weights.double() - w).abs() <= rel * w).all()


@pytest.mark.parametrize("E,K,D", FORMS)
@pytest.mark.parametrize("gate_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gating,norm,l2", [("softmax", False, False), ("softmax", True, True), ("sigmoid", False, True),
                                            ("sigmoid", True, False)])
def test_every_router_form(dev, E, K, D, gate_dtype, gating, norm, l2):
    T, H = 5, 128
    g = torch.Generator().manual_seed(E + D)
    x = randn_bf16((T, D), seed=E * K).to(dev)
    gate = (torch.randn(E, D, generator=g) / D ** 0.5).to(gate_dtype).to(dev)
    bias = (torch.randn(E, generator=g) * 0.1).to(dev, torch.bfloat16 if E % 2 else torch.float32) if norm else None
    score = (torch.randn(E, generator=g) * 0.1).to(dev) if gating == "sigmoid" else None
    nw = (1 + 0.1 * torch.randn(D, generator=g)).to(dev, torch.bfloat16 if l2 else torch.float32) if norm else None
    w = expert_weights(dev, E, H, D)
    r = fm.moe_decode(x, gate, w, K, gate_bias=bias, score_bias=score, gating=gating, norm_weight=nw,
                      normalize_expert_weights="l2" if l2 else None)
    xn, logits, b = logits64(x, gate, bias, score, nw)
    check_router(r, logits, b, K, gating, l2)
    ex = 2.0 ** -16 * xn.abs() if norm else torch.zeros_like(xn)
    check(r.out, *layer64(xn, ex, r.weights, r.indices, w, E))


@pytest.mark.parametrize("E,K,D", FORMS)
@pytest.mark.parametrize("gate_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
def test_equal_logits_go_to_the_lowest_indices(dev, E, K, D, gate_dtype, gating):
    """All rows of the gate alike but the last expert's, which is ahead or behind."""
    x = randn_bf16((3, D), seed=1).abs().to(dev)
    gate = torch.full((E, D), 1.0 / D, dtype=gate_dtype, device=dev)
    w = expert_weights(dev, E, 128, D)
    for last in (2.0, -2.0):
        gate[E - 1] = last / D
        r = fm.moe_decode(x, gate, w, K, gating=gating)
        order = [E - 1, *range(E - 1)] if last > 0 else list(range(E))
        assert r.indices.tolist() == [order[:K]] * 3
        _, logits, b = logits64(x, gate, None, None, None)
        check_router(r, logits, b, K, gating, False)


@pytest.mark.parametrize("T", [1, 8, 20, 64])
@pytest.mark.parametrize("E,K,H,D", [(4, 2, 128, 4096), (4, 2, 384, 14336), (2, 1, 128, 14336), (12, 3, 128, 7168)])
@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_wide_tokens(dev, T, E, K, H, D, kind):
    """Many chunks of D in gate|up, whose workgroups start at different ones, and many blocks of down's columns."""
    x = randn_bf16((T, D), seed=T).to(dev)
    weights, indices = (t.to(dev) for t in routing(T, E, K, T, skew=True))
    w = expert_weights(dev, E, H, D, 0.01)
    held, ex = w, torch.zeros(T, D, dtype=torch.float64, device=dev)
    if kind == "int8":
        held = fm.Int8Experts.quantize(*w, E)
        q2 = held.w2.values().double() * held.w2.scale.double()[:, None]
        w = [held.w1.values().double() * held.w1.scale.double()[:, None], q2.view(E, D, H).transpose(1, 2).reshape(E * H, D),
             held.w3.values().double() * held.w3.scale.double()[:, None]]
        ex = 4 * U * x.double().abs()   # the scales' products
    ref, bound = layer64(x.double(), ex, weights, indices, w, E)
    check(fm.expert_decode(x.float(), weights, indices, held, E), ref, bound * 1.01)
    check(fm.expert_decode(x, weights, indices, held, E), ref, bound * 1.01)
