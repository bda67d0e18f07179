"""The expert block, shared expert and layer with ``checkpoint_8bit``: outputs as without it, bit for bit; gradients against
float64 ones of the activations that 8 bits hold; and the layer's loss of masks and sequences.

BF16 products round each operand and result once (2^-8): the block's established bar of 1e-2 of a gradient's largest value."""

import pytest
import torch

import nanopysche_amd as fm
from tests.act8_reference import balance, kept
from tests.helpers import zipf_routing

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
RECIPES = {"none": (False, fm.FP8RecipeType.NONE), "flow_moe": (True, fm.FP8RecipeType.FLOW_MOE),
           "blockwise": (True, fm.FP8RecipeType.BLOCKWISE), "mxfp8": (True, fm.FP8RecipeType.MXFP8)}


def config(recipe):
    on, kind = RECIPES[recipe]
    return fm.FP8FlowMoEConfig(on, fm.FP8RecipeConfig(on, kind))


def rand(gen, *shape, std=1.0):
    return (torch.randn(*shape, generator=gen) * std).to(BF).cuda()


def inputs(T, D, H, E, K, seed=0, skew=0.0):
    g = torch.Generator().manual_seed(seed)
    w, idx = zipf_routing(T, E, K, skew, seed)
    return (rand(g, T, D), w.cuda(), idx.cuda(), *(rand(g, E * H, D, std=0.05) for _ in range(3)), rand(g, T, D, std=1e-2))


def run(recipe, eight, x, w, idx, w1, w2, w3, go, threshold=0, capture=None):
    D = x.shape[1]
    E = int(w1.shape[0] // run.hidden)
    block = fm.FP8FlowMoECompute(config(recipe), D, run.hidden, E, threshold, checkpoint_8bit=eight)
    block.capture_intermediates = capture
    leaves = [t.clone().requires_grad_(True) for t in (x, w, w1, w2, w3)]
    block.set_weights(*leaves[2:])
    out = block(leaves[0], leaves[1], idx, 0, E)
    out.backward(go)
    return out, [t.grad for t in leaves]


def worst(got, ref):
    return ((got.double() - ref).abs().max() / ref.abs().max()).item()


def distance(got, ref):
    return ((got.double() - ref.double()).norm() / ref.double().norm()).item()


def reference(x, w, idx, w1, w2, w3, go, gate_up_rows, plan_rows, H):
    """Gradients in float64 with what 8 bits hold of x, of the device's gate|up and of the expert outputs."""
    T, K = idx.shape
    E = w1.shape[0] // H
    D = x.shape[1]
    w1, w2, w3, go, wd = (t.double() for t in (w1, w2, w3, go, w))
    x8 = kept(x.double())
    dx, dw = torch.zeros(T, D, dtype=torch.float64, device="cuda"), torch.zeros(T, K, dtype=torch.float64, device="cuda")
    dws = [torch.zeros_like(t) for t in (w1, w2, w3)]
    for e in range(E):
        t, k = (idx == e).nonzero(as_tuple=True)
        if len(t) == 0:
            continue
        r = slice(e * H, (e + 1) * H)
        gu = gate_up_rows[plan_rows[t * K + k].long()].double()
        y = ((gu[:, :H] * torch.sigmoid(gu[:, :H]) * gu[:, H:]).to(BF).double() @ w2[r]).to(BF).double()
        g, u = kept(gu).split(H, 1)
        s = torch.sigmoid(g)
        dy = go[t] * wd[t, k, None]
        dh = dy @ w2[r].t()
        dg, du = dh * u * s * (1 + g * (1 - s)), dh * g * s
        dws[1][r] = (g * s * u).t() @ dy
        dws[0][r], dws[2][r] = dg.t() @ x8[t], du.t() @ x8[t]
        dx.index_add_(0, t, dg @ w1[r] + du @ w3[r])
        dw[t, k] = (go[t] * kept(y)).sum(1)
    return [dx, dw, *dws]


# =============================================================== the expert block ====
@pytest.mark.parametrize("T,D,H,E,K,skew", [(1, 128, 128, 4, 2, 0.0), (200, 256, 128, 4, 2, 0.0), (513, 512, 384, 8, 3, 1.2), (900, 1024, 512, 3, 1, 0.0),
                                            (300, 256, 256, 16, 9, 0.5)])
def test_block_against_float64(dev, T, D, H, E, K, skew):
    run.hidden = H
    args = inputs(T, D, H, E, K, seed=T, skew=skew)
    seen = {}
    out, grads = run("none", True, *args, capture=seen)
    plain, _ = run("none", False, *args)
    assert torch.equal(out, plain)
    plan = fm.route_tokens(args[2], E, 1 << 62)
    refs = reference(*args, seen["gate_up"], plan.row_of, H)
    for name, got, ref in zip(("x", "weights", "w1", "w2", "w3"), grads, refs):
        assert worst(got, ref) <= 1e-2, name


@pytest.mark.parametrize("recipe", list(RECIPES))
@pytest.mark.parametrize("T,D,H,E,K,threshold", [(400, 512, 384, 4, 2, 0), (2000, 256, 128, 8, 2, 0), (700, 512, 512, 4, 2, 300), (3000, 512, 384, 1, 1, 0)])
def test_block_of_every_recipe(dev, recipe, T, D, H, E, K, threshold):
    """Beside the same recipe's 16-bit activations: a value moves by a half of its block's 64th at most, uniformly, s / sqrt(12)
    of about 1% of a block's deviation; an FP8 operand made from it then rounds elsewhere with the probability of that share of an
    e4m3 step (an eighth of the value): sqrt(1% * 9%) = 3% of each operand, three to a gradient.  Norms within a tenth."""
    run.hidden = H
    args = inputs(T, D, H, E, K, seed=H + T, skew=0.8)
    out, grads = run(recipe, True, *args, threshold=threshold)
    plain, others = run(recipe, False, *args, threshold=threshold)
    assert torch.equal(out, plain)
    for name, a, b in zip(("x", "weights", "w1", "w2", "w3"), grads, others):
        assert torch.isfinite(a).all() and distance(a, b) <= 0.1, (name, distance(a, b))
    if recipe == "none":   # three operands of 1% to 2%
        assert max(distance(a, b) for a, b in zip(grads, others)) <= 0.05


def test_block_of_no_tokens_and_of_absent_experts(dev):
    run.hidden = 128
    x, w, idx, w1, w2, w3, go = inputs(64, 256, 128, 4, 2, seed=3)
    for recipe in RECIPES:
        out, grads = run(recipe, True, x[:0], w[:0], idx[:0], w1, w2, w3, go[:0])
        assert out.shape == (0, 256) and all(not g.any() for g in grads)
    some = torch.where(idx == 1, -1, idx)   # slots of no expert
    out, grads = run("none", True, x, w, some, w1, w2, w3, go)
    plain, others = run("none", False, x, w, some, w1, w2, w3, go)
    assert torch.equal(out, plain) and not grads[2][128:256].any() and not grads[1][idx == 1].any()
    assert max(distance(a, b) for a, b in zip(grads, others)) <= 0.05


def test_memory_of_the_forward(dev):
    """What the forward holds for the backward, per assignment (2 H + D) 33/32 and D 33/32 per token."""
    run.hidden = H = 1024
    T, D, E, K = 4096, 1024, 8, 4
    x, w, idx, w1, w2, w3, go = inputs(T, D, H, E, K, seed=5)
    held = {}
    for eight in (False, True):
        block = fm.FP8FlowMoECompute(config("none"), D, H, E, 0, checkpoint_8bit=eight)
        leaves = [t.clone().requires_grad_(True) for t in (x, w, w1, w2, w3)]
        block.set_weights(*leaves[2:])
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = block(leaves[0], leaves[1], idx, 0, E)
        held[eight] = torch.cuda.memory_allocated() - before - out.numel() * 2
        del out, leaves, block
    R = fm.route_tokens(idx, E).rows_max
    assert held[True] <= (R * (2 * H + D) + T * D) * 33 / 32 + R * 64 + (1 << 20)
    assert held[False] >= R * (6 * H + 4 * D)


def test_forward_without_gradients_keeps_nothing(dev):
    run.hidden = 128
    x, w, idx, w1, w2, w3, _ = inputs(64, 256, 128, 4, 2, seed=6)
    block = fm.FP8FlowMoECompute(config("flow_moe"), 256, 128, 4, 0, checkpoint_8bit=True)
    block.set_weights(w1, w2, w3)
    plain = fm.FP8FlowMoECompute(config("flow_moe"), 256, 128, 4, 0)
    plain.set_weights(w1, w2, w3)
    assert torch.equal(block(x, w, idx, 0, 4), plain(x, w, idx, 0, 4))


def test_shared_expert(dev):
    g = torch.Generator().manual_seed(8)
    x, w1, w2, w3 = rand(g, 300, 256), *(rand(g, 384, 256, std=0.05) for _ in range(3))
    go = rand(g, 300, 256, std=1e-2)
    res = []
    for eight in (False, True):
        shared = fm.FP8SharedExpertCompute(config("none"), 256, 384, checkpoint_8bit=eight)
        leaves = [t.clone().requires_grad_(True) for t in (x, w1, w2, w3)]
        shared.set_weights(*leaves[1:])
        out = shared(leaves[0])
        out.backward(go)
        res.append((out, [t.grad for t in leaves]))
    assert torch.equal(res[0][0], res[1][0])
    assert max(distance(a, b) for a, b in zip(res[1][1], res[0][1])) <= 0.05


# ======================================================================= the layer ====
def layer_of(recipe, D, H, E, K, seed, eight, **kw):
    g = torch.Generator().manual_seed(seed)
    shared = kw.pop("shared", 0)
    layer = fm.FP8FlowMoELayer(config(recipe), D, H, E, K, shared_hidden_size=shared or None, checkpoint_8bit=eight, **kw)
    p = {"gate": rand(g, E, D, std=0.1).float(), "bias": rand(g, E, std=0.1).float(), **{f"w{i}": rand(g, E * H, D, std=0.05) for i in (1, 2, 3)}}
    if shared:
        p.update({f"s{i}": rand(g, shared, D, std=0.05) for i in (1, 2, 3)})
    if kw.get("pre_norm"):
        p["norm"] = 1 + 0.1 * torch.randn(D, generator=g).cuda()
    p = {k: v.clone().requires_grad_(True) for k, v in p.items()}
    layer.set_weights(p["gate"], p["bias"], p["w1"], p["w2"], p["w3"], shared=tuple(p[f"s{i}"] for i in (1, 2, 3)) if shared else None,
                      norm_weight=p.get("norm"))
    return layer, p


@pytest.mark.parametrize("kw", [dict(), dict(pre_norm=True, shared=256), dict(jitter_eps=0.01), dict(capacity_factor=1.0),
                                dict(pre_norm=True, gating="sigmoid", normalize_expert_weights="l2", z_loss_multiplier=1e-3)])
@pytest.mark.parametrize("E,K", [(8, 2), (16, 4)])
def test_layer(dev, kw, E, K):
    T, D, H = 700, 512, 256
    g = torch.Generator().manual_seed(21)
    x, go = rand(g, T, D), rand(g, T, D, std=1e-2)
    res = []
    for eight in (False, True):
        layer, p = layer_of("none", D, H, E, K, 20, eight, **dict(kw))
        leaf = x.clone().requires_grad_(True)
        torch.manual_seed(7)
        out, aux = layer(leaf)
        torch.autograd.backward([out, aux], [go, torch.ones_like(aux)])
        res.append((out, aux, {"x": leaf.grad, **{k: v.grad for k, v in p.items()}}))
    (o0, a0, g0), (o1, a1, g1) = res
    if not kw.get("pre_norm"):
        assert torch.equal(o0, o1) and torch.equal(a0, a1)
    else:   # the two norms' sums of squares differ in their last bits: a value in some hundred rounds to its neighbour
        assert distance(o1, o0) <= 1e-2 and abs(a0 - a1) <= 1e-3 * abs(a0)
    for k in g0:
        assert distance(g1[k], g0[k]) <= 0.06, (k, distance(g1[k], g0[k]))


def test_step_of_padded_and_packed_tokens(dev):
    """All of it together, as a training step runs it: pre-norm, masked per-sequence loss, experts and shared expert from
    8 bits, the tracker's counts; the loss against float64 of the layer's own logits."""
    T, D, H, E, K = 600, 512, 256, 8, 2
    g = torch.Generator().manual_seed(31)
    x, go = rand(g, 3, 200, D), rand(g, 3, 200, D, std=1e-2)
    mask = torch.ones(3, 200, dtype=torch.bool, device="cuda")
    mask[1, 120:] = False
    mask[2, 5:] = False
    borders = [0, 80, 200, 200, 400, 590]
    cu = torch.tensor(borders, dtype=torch.int32, device="cuda")
    layer, p = layer_of("flow_moe", D, H, E, K, 30, True, pre_norm=True, shared=128, z_loss_multiplier=1e-3, balance_scores="sigmoid")
    tracker = fm.ExpertLoadTracker(E, "cuda")
    leaf = x.clone().requires_grad_(True)
    out, aux = layer(leaf, load_tracker=tracker, token_mask=mask, cu_seqlens=cu)
    y = fm.rmsnorm_compress(x, p["norm"].detach())[0]
    logits = fm.router_logits(y, p["gate"].detach(), p["bias"].detach())
    idx = logits.topk(K, 1).indices
    ref, counts = balance(logits.double(), idx, borders, mask.reshape(-1), "sigmoid", 1e-3)
    assert abs(aux.double() - ref) <= 1e-5 * ref.abs()   # sums of fp32 logits in another order, 600 terms
    assert torch.equal(tracker.tokens_per_expert, counts.sum(0)) and int(tracker.total_tokens) == int(mask.reshape(-1)[:590].sum())
    torch.autograd.backward([out, aux], [go, torch.ones_like(aux)])
    grads = {"x": leaf.grad, **{k: v.grad for k, v in p.items()}}
    assert all(torch.isfinite(v).all() and v.any() for v in grads.values())
    # the loss alone reaches the gate through balance_loss's gradient
    layer.z_loss_multiplier = 0.0
    for t in p.values():
        t.grad = None
    _, aux = layer(x, token_mask=mask, cu_seqlens=cu)
    aux.backward()
    l64 = logits.double().requires_grad_(True)
    loss, _ = balance(l64, idx, borders, mask.reshape(-1), "sigmoid")
    dl = torch.autograd.grad(loss, l64)[0]
    y8 = kept(y.reshape(T, D).double())
    assert worst(p["gate"].grad, dl.t() @ y8) <= 1e-4 and worst(p["bias"].grad, dl.sum(0)) <= 1e-4


@pytest.mark.parametrize("E,K", [(8, 2), (64, 6)])
def test_route_with_masks_and_sequences(dev, E, K):
    g = torch.Generator().manual_seed(41)
    x = rand(g, 4, 100, 256)
    gate = rand(g, E, 256, std=0.1).float().requires_grad_(True)
    mask = (torch.rand(4, 100, generator=g) < 0.7).cuda()
    cu = torch.tensor([0, 150, 380], dtype=torch.int32, device="cuda")
    tracker = fm.ExpertLoadTracker(E, "cuda")
    w, idx, aux = fm.route(x, gate, top_k=K, token_mask=mask, cu_seqlens=cu, load_tracker=tracker, z_loss_multiplier=1e-2)
    wp, idxp, auxp = fm.route(x, gate, top_k=K)
    assert torch.equal(w, wp) and torch.equal(idx, idxp) and not torch.equal(aux, auxp)
    logits = fm.router_logits(x, gate.detach()).requires_grad_(True)
    out = fm.balance_loss(logits.view(4, 100, E), idx, token_mask=mask, cu_seqlens=cu, z_loss_multiplier=1e-2)
    assert abs(out.loss - aux) <= 1e-6 * aux and torch.equal(tracker.tokens_per_expert, out.counts.sum(0))
    dw = torch.randn(w.shape, device="cuda")
    torch.autograd.backward([w, aux], [dw, torch.full_like(aux, 0.5)])
    both, gate.grad = gate.grad, None
    torch.autograd.backward([wp], [dw])
    rest, gate.grad = gate.grad, None
    out.loss.backward(torch.tensor(0.5, device="cuda"))
    want = rest.double() + logits.grad.reshape(400, E).t().double() @ x.reshape(400, 256).double()
    assert worst(both, want) <= 1e-5
    # the loss alone
    _, _, aux = fm.route(x, gate, top_k=K, token_mask=mask, cu_seqlens=cu, z_loss_multiplier=1e-2)
    aux.backward(torch.tensor(0.5, device="cuda"))
    assert worst(gate.grad, logits.grad.reshape(400, E).t().double() @ x.reshape(400, 256).double()) <= 1e-5
    for bad in (dict(token_mask=mask[:3]), dict(token_mask=mask.float()), dict(cu_seqlens=cu.long()), dict(balance_scores="none")):
        with pytest.raises((ValueError, TypeError)):
            fm.route(x, gate, top_k=K, **bad)


def test_layer_graph_replays(dev):
    T, D, H, E, K = 512, 512, 256, 8, 2
    g = torch.Generator().manual_seed(51)
    layer, p = layer_of("flow_moe", D, H, E, K, 50, True, pre_norm=True)
    x = rand(g, T, D).requires_grad_(True)
    go = rand(g, T, D, std=1e-2)
    mask = torch.ones(T, dtype=torch.bool, device="cuda")
    cu = torch.tensor([0, 100, 500], dtype=torch.int32, device="cuda")
    one = torch.ones((), device="cuda")

    def step():
        out, aux = layer(x, token_mask=mask, cu_seqlens=cu)
        torch.autograd.backward([out, aux], [go, one])
        return out, aux

    leaves = [x, *p.values()]
    graphed = fm.GraphedStep(step, leaves=leaves)
    for i in range(3):
        with torch.no_grad():
            x.copy_(rand(g, T, D))
            go.copy_(rand(g, T, D, std=1e-2))
            mask.copy_((torch.rand(T, generator=g) < 0.8).cuda())
            cu.copy_(torch.tensor([i, 200, 512 - i], dtype=torch.int32))
        graphed.replay()
        torch.cuda.synchronize()
        want = [t.clone() for t in (*graphed.outputs, *graphed.grads)]
        held = [t.grad for t in leaves]
        for t in leaves:
            t.grad = None
        out, aux = step()
        torch.cuda.synchronize()
        got = [out, aux, *(t.grad for t in leaves)]
        for t, h in zip(leaves, held):
            t.grad = h
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_mask_changed_in_place_is_noticed(dev):
    layer, p = layer_of("none", 512, 128, 8, 2, 60, False)
    x = rand(torch.Generator().manual_seed(61), 64, 512)
    mask = torch.ones(64, dtype=torch.bool, device="cuda")
    _, aux = layer(x, token_mask=mask)
    mask[3] = False
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        aux.backward()


@pytest.mark.parametrize("kw", [dict(), dict(pre_norm=True, shared=128), dict(capacity_factor=8.0)])
def test_layer_of_one_token_that_does_not_count(dev, kw):
    layer, p = layer_of("flow_moe", 512, 128, 8, 2, 70, True, **dict(kw))
    x = rand(torch.Generator().manual_seed(71), 1, 512).requires_grad_(True)
    out, aux = layer(x, token_mask=torch.zeros(1, dtype=torch.bool, device="cuda"))
    assert out.shape == (1, 512) and out.any() and aux == 0
    torch.autograd.backward([out, aux], [torch.ones_like(out), torch.ones_like(aux)])
    assert torch.isfinite(x.grad).all() and x.grad.any()
    assert all(v.grad is None or torch.isfinite(v.grad).all() for v in p.values())
    with pytest.raises(ValueError, match="at least one token"):
        layer(x[:0], token_mask=torch.zeros(0, dtype=torch.bool, device="cuda"))


@pytest.mark.parametrize("pre_norm", [False, True])
def test_layer_of_fp32_tokens(dev, pre_norm):
    """fp32 tokens are rounded to bf16 where the layer takes them in: its results are those of the rounded ones."""
    res = []
    for x in (rand(torch.Generator().manual_seed(81), 300, 512).float(), rand(torch.Generator().manual_seed(81), 300, 512)):
        layer, p = layer_of("none", 512, 128, 8, 2, 80, True, pre_norm=pre_norm)
        leaf = x.requires_grad_(True)
        out, aux = layer(leaf)
        torch.autograd.backward([out, aux], [torch.ones_like(out), torch.ones_like(aux)])
        res.append((out.bfloat16(), aux, leaf.grad.bfloat16(), *(v.grad for v in p.values())))
    assert all(torch.equal(a, b) for a, b in zip(*res))
