"""The balance loss of packed and padded sequences against float64 and autograd of it.

fp32 throughout: p is within a few ulps (the exponential 2, the sum log2(E) + 2, the quotient 2), a sequence's sum within its
partial sums' depth of 2^-24 of itself; the gradient's terms are p f and p sum f p."""

import pytest
import torch

import nanopysche_amd as fm
from tests.act8_reference import balance

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def inputs(T, E, K, seed, scale=1.0):
    g = gen(seed)
    logits = torch.randn(T, E, generator=g, device="cuda") * scale - 0.5 * torch.log(torch.randperm(E, generator=g, device="cuda") + 1.0)
    return logits, logits.topk(K, dim=1).indices


def check(logits, indices, borders=None, mask=None, scores="softmax", z=0.0, dloss=0.37):
    T, E = logits.shape
    cu = None if borders is None else torch.tensor(borders, dtype=torch.int32, device="cuda")
    ref_in = logits.double().requires_grad_(True)
    loss, counts = balance(ref_in, indices, borders, mask, scores, z)
    grad = torch.autograd.grad(loss * dloss, ref_in)[0] if loss.requires_grad else torch.zeros_like(ref_in)
    leaf = logits.clone().requires_grad_(True)
    out = fm.balance_loss(leaf, indices, cu_seqlens=cu, token_mask=mask, scores=scores, z_loss_multiplier=z)
    out.loss.backward(torch.tensor(dloss, device="cuda"))
    assert out.counts.dtype == torch.int32 and torch.equal(out.counts.long(), counts if borders is not None else counts[0])
    assert abs(out.loss.double() - loss.detach()) <= 64 * U32 * loss.detach().abs()
    # terms of the gradient: dloss E / (S' n) p (f + sum f p), at most E K max f dloss / n of a sequence
    terms = grad_terms(logits.double(), counts.double(), borders or [0, T], mask, scores, z, dloss)
    assert torch.all((leaf.grad.double() - grad).abs() <= 64 * U32 * terms + 1e-30)
    dead = torch.ones(T, dtype=torch.bool, device="cuda")
    for lo, hi in zip(borders or [0, T], (borders or [0, T])[1:]):
        dead[lo:hi] = False
    if mask is not None:
        dead |= ~mask
    assert not leaf.grad[dead].any()
    # through the calls that a step makes itself
    l2, c2, state = fm.balance_forward(logits, indices, cu_seqlens=cu, token_mask=mask, scores=scores, z_loss_multiplier=z)
    d2 = fm.balance_backward(state, torch.tensor(dloss, device="cuda"))
    assert torch.equal(l2, out.loss.detach()) and torch.equal(c2, out.counts) and torch.equal(d2, leaf.grad)
    base = torch.randn(T, E + 3, device="cuda")
    some = base[:, 1:1 + E]
    want = some + d2
    assert fm.balance_backward(state, torch.tensor(dloss, device="cuda"), add_to=some) is some
    assert torch.equal(some, want)
    return out


def grad_terms(l, counts, borders, mask, scores, z, dloss):
    T, E = l.shape
    p = torch.softmax(torch.nan_to_num(l, 0.0, 0.0, 0.0), 1) if scores == "softmax" else torch.sigmoid(l) / torch.sigmoid(l).sum(1, keepdim=True)
    out = torch.zeros_like(l)
    total, live = 0, 0
    for s, (lo, hi) in enumerate(zip(borders, borders[1:])):
        n = int(mask[lo:hi].sum()) if mask is not None else hi - lo
        total, live = total + n, live + (n > 0)
        if n:
            f = counts[s] / n
            out[lo:hi] = E / n * p[lo:hi] * (f + (f * p[lo:hi]).sum(1, keepdim=True))
    out = out / max(live, 1) * dloss
    if z:
        out = out + 2 * z * dloss / max(total, 1) * torch.logsumexp(torch.nan_to_num(l, 0.0, 0.0, 0.0), 1, keepdim=True).abs() * torch.softmax(l, 1)
    return out


EXPERTS = [(1, 1), (2, 1), (3, 2), (4, 1), (5, 2), (8, 2), (15, 4), (16, 4), (31, 3), (60, 4), (64, 6), (65, 2), (100, 8), (128, 8), (160, 6),
           (255, 8), (256, 8), (320, 8), (511, 4), (512, 16), (1000, 8), (1023, 2), (1024, 64)]


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,K", EXPERTS)
def test_widths(dev, E, K, scores):
    logits, idx = inputs(333, E, K, E)
    mask = torch.rand(333, generator=gen(E), device="cuda") < 0.8
    check(logits, idx, [0, 100, 100, 131, 300], mask, scores, z=1e-2)


@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 127, 128, 129, 1000, 4097, 70000])
@pytest.mark.parametrize("E,K", [(8, 2), (60, 4), (7, 1)])
def test_lengths(dev, T, E, K):
    logits, idx = inputs(T, E, K, T)
    check(logits, idx)
    check(logits, idx.int(), scores="sigmoid", z=1e-3)


@pytest.mark.parametrize("T,S,E", [(5000, 1000, 8), (5000, 5000, 16), (3000, 70000, 4), (20000, 40, 64), (20000, 3, 256), (700, 300, 1024), (200000, 2, 4)])
def test_many_sequences(dev, T, S, E):
    """Sequences of every length from nothing to the whole batch, some tokens before the first and behind the last."""
    logits, idx = inputs(T, E, 2, S)
    cuts = (torch.rand(S - 1, generator=gen(S), device="cuda") * (T - 10)).long().sort().values.tolist()
    out = fm.balance_loss(logits, idx, cu_seqlens=torch.tensor([3] + [max(c, 3) for c in cuts] + [T - 5], dtype=torch.int32, device="cuda"))
    if S <= 1000:
        check(logits, idx, [3] + [max(c, 3) for c in cuts] + [T - 5])
    assert int(out.counts.sum()) == 2 * (T - 8) and out.counts.shape == (S, E)


def test_mask_that_leaves_nothing(dev):
    logits, idx = inputs(500, 16, 4, 7)
    logits[200:300] = torch.nan
    mask = torch.ones(500, dtype=torch.bool, device="cuda")
    mask[200:300] = False
    check_nan_free(logits, idx, [0, 200, 300, 300, 500], mask)   # a whole sequence of masked NaNs
    mask[:] = False
    out = check_nan_free(logits, idx, [0, 200, 300, 300, 500], mask)
    assert out.loss == 0 and not out.counts.any()
    out = check_nan_free(logits, idx, None, mask)
    assert out.loss == 0 and out.counts.shape == (16,)


def check_nan_free(logits, idx, borders, mask):
    clean = torch.where(mask[:, None], logits, 0.0)
    cu = None if borders is None else torch.tensor(borders, dtype=torch.int32, device="cuda")
    a, b = logits.clone().requires_grad_(True), clean.clone().requires_grad_(True)
    outs = [fm.balance_loss(t, idx, cu_seqlens=cu, token_mask=mask, z_loss_multiplier=0.1) for t in (a, b)]
    for o in outs:
        o.loss.backward()
    assert torch.equal(outs[0].loss, outs[1].loss) and torch.equal(a.grad, b.grad) and torch.isfinite(a.grad).all()
    return outs[0]


def test_values_in_masked_places(dev):
    logits, idx = inputs(300, 8, 2, 8)
    mask = torch.rand(300, generator=gen(8), device="cuda") < 0.5
    for bad in (torch.inf, -torch.inf, torch.nan, torch.finfo(torch.float32).min, torch.finfo(torch.float32).max):
        check_nan_free(torch.where(mask[:, None], logits, bad), idx, [0, 100, 300], mask)


def test_extreme_logits_that_count(dev):
    logits, idx = inputs(64, 8, 2, 9)
    logits[0] = torch.finfo(torch.float32).min
    logits[1, :7] = -torch.inf
    logits[2] = 1e4
    logits[3, 2] = 500.0
    logits[4] = -300.0
    check(logits, idx)
    nan = logits.clone()
    nan[5, 3] = torch.nan
    leaf = nan.requires_grad_(True)
    out = fm.balance_loss(leaf, idx)
    out.loss.backward()
    assert torch.isnan(out.loss) and torch.isnan(leaf.grad[5]).all() and torch.isfinite(leaf.grad[6]).all()


def test_slots_outside_the_experts(dev):
    logits, idx = inputs(200, 8, 3, 10)
    idx[::3, 1] = -1
    idx[1::5, 0] = 8
    idx[2::7, 2] = 2 ** 40
    idx[3::7] = 5   # the same expert thrice
    check(logits, idx, [0, 50, 200])


def test_shapes_and_strides(dev):
    g = gen(11)
    logits = torch.randn(4, 25, 12, generator=g, device="cuda")
    idx = logits[..., :8].topk(2, dim=-1).indices
    mask = torch.rand(4, 25, generator=g, device="cuda") < 0.7
    ref, counts = balance(logits[..., :8].double().reshape(100, 8), idx.reshape(100, 2), None, mask.reshape(100))
    for l, i, m in ((logits[..., :8], idx, mask), (logits[..., :8].contiguous(), idx.repeat_interleave(2, -1)[..., ::2], mask),
                    (logits[..., :8].transpose(0, 1).contiguous().transpose(0, 1), idx.int(), mask.t().contiguous().t())):
        leaf = l.detach().requires_grad_(True)
        out = fm.balance_loss(leaf, i, token_mask=m)
        out.loss.backward()
        assert abs(out.loss.double() - ref) <= 64 * U32 * ref and torch.equal(out.counts.long(), counts[0])
        assert leaf.grad.shape == l.shape and not leaf.grad[~m].any()
    one = torch.randn(8, generator=g, device="cuda")
    assert fm.balance_loss(one, one.topk(2).indices).counts.sum() == 2


def test_no_tokens_and_no_sequences(dev):
    logits = torch.empty(0, 8, device="cuda", requires_grad=True)
    idx = torch.empty(0, 2, dtype=torch.int64, device="cuda")
    for cu in (None, torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")):
        out = fm.balance_loss(logits, idx, cu_seqlens=cu, z_loss_multiplier=1.0)
        out.loss.backward()
        assert out.loss == 0 and not out.counts.any() and logits.grad.shape == (0, 8)
    leaf, idx = inputs(100, 8, 2, 12)
    leaf.requires_grad_(True)
    out = fm.balance_loss(leaf, idx, cu_seqlens=torch.zeros(1, dtype=torch.int32, device="cuda"))
    out.loss.backward()
    assert out.loss == 0 and out.counts.shape == (0, 8) and not leaf.grad.any()


def test_gradient_by_differences(dev):
    logits, idx = inputs(40, 6, 2, 13)
    borders, mask = [0, 10, 35], torch.rand(40, generator=gen(13), device="cuda") < 0.8
    for scores in ("softmax", "sigmoid"):
        leaf = logits.clone().requires_grad_(True)
        fm.balance_loss(leaf, idx, cu_seqlens=torch.tensor(borders, dtype=torch.int32, device="cuda"), token_mask=mask, scores=scores,
                        z_loss_multiplier=0.1).loss.backward()
        e = 1e-5
        for i in range(0, logits.numel(), 7):
            d = torch.zeros(logits.numel(), dtype=torch.float64, device="cuda")
            d[i] = e
            d = d.view_as(logits)
            up, down = (balance(logits.double() + s * d, idx, borders, mask, scores, 0.1)[0] for s in (1, -1))
            # a loss of about 2 in float64 over 2e, and second-order terms of e^2
            assert abs((up - down) / (2 * e) - leaf.grad.view(-1)[i].double()) <= 1e-9 + 1e-5 * leaf.grad.abs().max()


def test_one_sequence_is_the_routers_loss(dev):
    """Without borders or a mask: the loss, counts and gradients of ``route``."""
    g = gen(14)
    x = torch.randn(1024, 256, generator=g, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(16, 256, generator=g, device="cuda").requires_grad_(True)
    weights, idx, aux = fm.route(x, w, top_k=4, z_loss_multiplier=1e-2)
    aux.backward()
    ref, w.grad = w.grad, None
    logits = fm.router_logits(x, w).requires_grad_(True)
    out = fm.balance_loss(logits, idx, z_loss_multiplier=1e-2)
    assert torch.equal(out.counts, fm.expert_counts(idx, 16))
    assert abs(out.loss.double() - aux.double()) <= 128 * U32 * aux
    out.loss.backward()
    mine = logits.grad.t().double() @ x.double()
    size = logits.grad.t().double().abs() @ x.double().abs()
    assert torch.all((mine - ref.double()).abs() <= 256 * U32 * size + 1e-9 * size.max())


def test_load_tracker(dev):
    logits, idx = inputs(1000, 8, 2, 15)
    mask = torch.rand(1000, generator=gen(15), device="cuda") < 0.6
    cu = torch.tensor([0, 10, 10, 900], dtype=torch.int32, device="cuda")
    tracker = fm.ExpertLoadTracker(8, "cuda")
    for times in (1, 2):
        out = fm.balance_loss(logits, idx, cu_seqlens=cu, token_mask=mask, load_tracker=tracker)
        assert torch.equal(tracker.tokens_per_expert, times * out.counts.sum(0))
        assert int(tracker.total_tokens) == times * int(mask[:900].sum())


def test_graph_replays_and_repeats(dev):
    logits, idx = inputs(3000, 64, 6, 16)
    leaf = logits.clone().requires_grad_(True)
    cu = torch.tensor([0, 700, 701, 2900], dtype=torch.int32, device="cuda")
    mask = torch.ones(3000, dtype=torch.bool, device="cuda")

    def step():
        out = fm.balance_loss(leaf, idx, cu_seqlens=cu, token_mask=mask, z_loss_multiplier=1e-3)
        out.loss.backward()
        return out.loss, out.counts

    graphed = fm.GraphedStep(step, leaves=[leaf])
    for i in range(3):
        l, k = inputs(3000, 64, 6, 20 + i)
        with torch.no_grad():
            leaf.copy_(l)
            idx.copy_(k)
            cu.copy_(torch.tensor([5 * i, 300 + i, 1500, 3000 - i], dtype=torch.int32))
            mask.copy_(torch.rand(3000, generator=gen(i), device="cuda") < 0.9)
        graphed.replay()
        torch.cuda.synchronize()
        again = leaf.detach().clone().requires_grad_(True)
        for _ in range(2):
            again.grad = None
            out = fm.balance_loss(again, idx, cu_seqlens=cu, token_mask=mask, z_loss_multiplier=1e-3)
            out.loss.backward()
            assert torch.equal(graphed.outputs[0], out.loss.detach()) and torch.equal(graphed.outputs[1], out.counts)
            assert torch.equal(graphed.grads[0], again.grad)


def test_logits_changed_in_place_are_noticed(dev):
    leaf, idx = inputs(100, 8, 2, 17)
    leaf.requires_grad_(True)
    logits = leaf * 1.0
    out = fm.balance_loss(logits, idx)
    with torch.no_grad():
        logits += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.loss.backward()


def test_tensors_elsewhere_are_refused(dev):
    logits, idx = inputs(10, 8, 2, 18)
    cu, mask = torch.tensor([0, 10], dtype=torch.int32), torch.ones(10, dtype=torch.bool)
    state = fm.balance_forward(logits, idx)[2]
    for call in (lambda: fm.balance_loss(logits, idx.cpu()), lambda: fm.balance_loss(logits, idx, cu_seqlens=cu),
                 lambda: fm.balance_loss(logits, idx, token_mask=mask), lambda: fm.balance_loss(logits.cpu(), idx),
                 lambda: fm.balance_loss(logits, idx, load_tracker=fm.ExpertLoadTracker(8, "cpu")),
                 lambda: fm.balance_backward(state, torch.ones(())), lambda: fm.balance_backward(state, torch.ones((), device="cuda"), add_to=torch.zeros(10, 8))):
        with pytest.raises((ValueError, RuntimeError), match="is on|device"):
            call()
    with pytest.raises(ValueError, match="load_tracker"):
        fm.balance_loss(logits, idx, load_tracker=fm.ExpertLoadTracker(9, "cuda"))


def test_offsets_past_32_bits(dev):
    """Logits and gradients whose rows lie 2^20 apart: the last ones are past 2^31 elements."""
    T, E, far = 2100, 8, 2 ** 20
    logits, idx = inputs(T, E, 2, 30)
    l = torch.empty(T * far, device="cuda").as_strided((T, E), (far, 1)).copy_(logits)
    d = torch.empty(T * far, device="cuda").as_strided((T, E), (far, 1)).zero_()
    one = torch.ones((), device="cuda")
    loss, counts, state = fm.balance_forward(l, idx)
    near, near_counts, near_state = fm.balance_forward(logits, idx)
    assert torch.equal(loss, near) and torch.equal(counts, near_counts)
    assert torch.equal(fm.balance_backward(state, one, add_to=d), fm.balance_backward(near_state, one))


@pytest.mark.parametrize("S,E", [(3000, 64), (3000, 256), (9000, 20), (200, 24)])
def test_one_long_sequence_among_short_ones(dev, S, E):
    """Sequences of one token, an empty one, and two that hold nearly all."""
    logits, idx = inputs(70000, E, 2, 40)
    half = S // 2
    borders = [*range(half), half - 1, 50000, *range(50001, 50000 + S - half), 70000]
    check(logits, idx, borders, torch.rand(70000, generator=gen(41), device="cuda") < 0.9)
