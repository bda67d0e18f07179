"""The serving operators as a program runs them: a layer's prompt and then its decoding steps,
captured graphs, several streams, routings and rows at the edges."""

import pytest
import torch

import nanopysche_amd as fm
from tests.helpers import randn_bf16, zipf_routing
from tests.test_gpu_decode import check, expert_weights, layer64

pytestmark = pytest.mark.gpu

D, H, E, K = 512, 256, 8, 2


def layer(dev, shared=128, pre_norm=True, gating="softmax"):
    cfg = fm.FP8FlowMoEConfig(True, fm.FP8RecipeConfig(False))
    moe = fm.FP8FlowMoELayer(cfg, D, H, E, K, gating=gating, shared_hidden_size=shared or None, pre_norm=pre_norm).eval()
    w = [t.to(dev) for t in expert_weights(E, H, D, 5)]
    sh = tuple(t.to(dev) for t in expert_weights(1, shared, D, 9)) if shared else None
    nw = (1 + 0.1 * torch.randn(D, generator=torch.Generator().manual_seed(4))).to(dev) if pre_norm else None
    moe.set_weights(randn_bf16((E, D), seed=1, std=0.1).to(dev), randn_bf16((E,), seed=2).to(dev), *w, shared=sh, norm_weight=nw)
    return moe, w, sh


@pytest.mark.parametrize("gating", ["softmax", "sigmoid"])
@pytest.mark.parametrize("pre_norm", [False, True])
@pytest.mark.parametrize("shared", [0, 128])
def test_layer_decode_is_the_layer_within_bf16(dev, gating, pre_norm, shared):
    """The layer rounds to bf16 after the norm, gate|up, SwiGLU, down and the sums: 2^-8 a step of values of their sums' size."""
    moe, _, _ = layer(dev, shared, pre_norm, gating)
    x = randn_bf16((16, D), seed=7).to(dev)
    with torch.no_grad():
        want, _ = moe(x)
        got = moe.decode(x.view(4, 4, D))
    assert got.out.shape == (4, 4, D)
    assert (got.out.view(16, D).double() - want.double()).norm() <= 6 * 2.0 ** -8 * want.double().norm()


def test_a_prompt_then_steps_with_one_set_of_int8_experts(dev):
    """Prefill through Int8MoECompute, decoding through the layer with the same Int8Experts: both near the bf16
    layer, as far as int8 weights (a step of amax / 127 a channel: about 1% of a normal row) and tokens allow."""
    moe, w, sh = layer(dev)
    ex, sx = fm.Int8Experts.quantize(*w, E), fm.Int8Experts.quantize(*sh, 1)
    x = randn_bf16((200, D), seed=7).to(dev)
    with torch.no_grad():
        want, _ = moe(x)
        xn = fm.rmsnorm(x, moe.norm_weight)
        rw, idx, _ = fm.route(xn, moe.gate_weight, moe.gate_bias, top_k=K)
        ones, zeros = torch.ones(200, 1, device=dev), torch.zeros(200, 1, dtype=torch.int64, device=dev)
        got = fm.Int8MoECompute(ex)(xn, rw, idx) + fm.Int8MoECompute(sx)(xn, ones, zeros)
        assert (got.double() - want.double()).norm() <= 0.05 * want.double().norm()
        for at, n in ((0, 1), (5, 64), (100, 33)):
            step = moe.decode(x[at:at + n], ex, sx)
            assert torch.equal(step.indices, idx[at:at + n]) or (step.indices == idx[at:at + n]).float().mean() > 0.95
            part = want[at:at + n].double()
            assert (step.out.double() - part).norm() <= 0.05 * part.norm()


def calls(dev):
    """name -> (inputs that a program rewrites, call)."""
    moe, w, sh = layer(dev)
    ex = fm.Int8Experts.quantize(*w, E)
    x = randn_bf16((17, D), seed=3).to(dev)
    xp = randn_bf16((150, D), seed=4).to(dev)
    rw, idx = (t.to(dev) for t in zipf_routing(150, E, K, 1.0, seed=2, zero_experts=(3,)))
    lin = fm.quantize_to_int8(randn_bf16((384, D), seed=5).to(dev))
    return {
        "decode": (x, lambda: moe.decode(x).out),
        "decode_int8": (x, lambda: fm.moe_decode(x, moe.gate_weight, ex, K).out),
        "experts": (x, lambda: fm.expert_decode(x, rw[:17], idx[:17], w, E)),
        "block_int8": (xp, lambda: fm.Int8MoECompute(ex)(xp, rw, idx)),
        "linear_one": (x, lambda: fm.int8_linear(x[:1], lin)),
        "linear_few": (x, lambda: fm.int8_linear(x, lin)),
        "linear_many": (xp, lambda: fm.int8_linear(xp, lin)),
        "quantise": (xp, lambda: fm.quantize_to_int8(xp).dequantize()),
    }


NAMES = ["decode", "decode_int8", "experts", "block_int8", "linear_one", "linear_few", "linear_many", "quantise"]


@pytest.mark.parametrize("name", NAMES)
def test_captured_and_replayed(dev, name):
    with torch.no_grad():
        x, call = calls(dev)[name]
        first = x.clone()
        step = fm.GraphedStep(call)
        for i in range(4):
            x.copy_(first.roll(i, 1) * (i + 1))
            want = call().clone()
            torch.zeros(1 << 20, device=dev).fill_(float("nan"))   # the program's own work between replays
            step.replay()
            torch.cuda.synchronize()
            assert torch.equal(step.outputs, want), i
        assert torch.equal(call(), want)


def test_two_graphs_and_streams_at_once(dev):
    """Two captured layers and eager calls on two streams, none sharing scratch memory."""
    with torch.no_grad():
        every = {n: c for n, (_, c) in calls(dev).items()}
        want = {n: c().clone() for n, c in every.items()}
        a, b = fm.GraphedStep(every["decode"]), fm.GraphedStep(every["block_int8"])
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        for _ in range(3):
            with torch.cuda.stream(s1):
                a.replay()
                got1 = [every[n]() for n in NAMES]
            with torch.cuda.stream(s2):
                b.replay()
                got2 = [every[n]() for n in reversed(NAMES)]
            torch.cuda.synchronize()
            assert torch.equal(a.outputs, want["decode"]) and torch.equal(b.outputs, want["block_int8"])
            assert all(torch.equal(g, want[n]) for n, g in zip(NAMES, got1))
            assert all(torch.equal(g, want[n]) for n, g in zip(reversed(NAMES), got2))


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_token_that_is_not_finite_stays_alone(dev, bad):
    with torch.no_grad():
        for T, n in ((20, "decode"), (20, "decode_int8"), (150, "block_int8")):
            x, call = calls(dev)[n]
            want = call().clone()
            x[3, 5] = bad
            got = call()
            keep = torch.arange(x.shape[0], device=dev) != 3
            assert torch.equal(got[keep], want[keep]), n
            assert not got[3].isfinite().any(), n


def test_slots_elsewhere_twice_and_offset(dev):
    """The same expert in two slots, experts of other ranks, a token with none, int32 indices, offsets."""
    x = randn_bf16((6, D), seed=3).to(dev)
    w = [t.to(dev) for t in expert_weights(E, H, D, 5)]
    idx = torch.tensor([[2, 2], [7, 8], [-1, 0], [100, -5], [1 << 20, 3], [5, 5]], device=dev)
    rw = torch.rand(6, 2, generator=torch.Generator().manual_seed(1)).to(dev)
    zero = torch.zeros(6, D, dtype=torch.float64, device=dev)
    ref = layer64(x.double(), zero, rw, idx, w, E)
    for ix, off in ((idx, 0), (idx.int(), 0), (idx + 40, 40), ((idx - 3).int(), -3)):
        got = fm.expert_decode(x.float(), rw, ix, w, E, expert_offset=off)
        check(got, *ref)
        assert torch.all(got[3] == 0)
    none = fm.expert_decode(x, rw, torch.full_like(idx, -1), w, E)
    assert torch.all(none == 0)
    ex = fm.Int8Experts.quantize(*w, E)
    many = idx.repeat(20, 1)   # the product path
    a = fm.Int8MoECompute(ex)(x.repeat(20, 1), rw.repeat(20, 1), many)
    b = fm.Int8MoECompute(ex)(x.repeat(20, 1), rw.repeat(20, 1), many + 40, 40)
    assert torch.equal(a, b) and torch.all(a.view(20, 6, D)[:, 3] == 0)
    assert torch.all(fm.Int8MoECompute(ex)(x.repeat(20, 1), rw.repeat(20, 1), torch.full_like(many, -1)) == 0)


def test_strided_rows_and_every_token_to_one_expert(dev):
    w = [t.to(dev) for t in expert_weights(E, H, D, 5)]
    big = randn_bf16((64, D + 40), seed=3).to(dev)
    rw = torch.ones(64, 1, device=dev)
    idx = torch.full((64, 1), 6, dtype=torch.int64, device=dev)
    for x in (big[:, :D], big[:, 8:D + 8], big[:, 3:D + 3], big.t()[:D].t()):   # pitches, offsets, a misaligned base
        got = fm.expert_decode(x, rw, idx, w, E)
        assert torch.equal(got, fm.expert_decode(x.contiguous(), rw, idx, w, E))
        check(got, *layer64(x.double(), torch.zeros(64, D, dtype=torch.float64, device=dev), rw, idx, w, E))


def test_no_expert_is_read_beyond_those_reached(dev):
    """Weights of experts without tokens do not matter, NaN included."""
    w = [t.to(dev) for t in expert_weights(E, H, D, 5)]
    x = randn_bf16((9, D), seed=3).to(dev)
    idx = torch.tensor([[1, 4]] * 9, device=dev)
    rw = torch.rand(9, 2, generator=torch.Generator().manual_seed(1)).to(dev)
    want = fm.expert_decode(x, rw, idx, w, E)
    for t in w:
        t.view(E, H, D)[[0, 2, 3, 5, 6, 7]] = float("nan")
    assert torch.equal(fm.expert_decode(x, rw, idx, w, E), want)


def test_rows_behind_the_groups_are_left(dev):
    """int8_grouped_gemm leaves the rows past the last group as they were."""
    idx = torch.tensor([[0], [2], [2]], device=dev)
    plan = fm.route_tokens(idx, 3)
    q = torch.ones(plan.rows_max, 128, dtype=torch.int8, device=dev)
    t = fm.Int8Tensor.from_int8(q, torch.ones(plan.rows_max, device=dev))
    wq = torch.ones(3 * 64, 128, dtype=torch.int8, device=dev)
    w = fm.Int8Tensor.from_int8(wq, torch.ones(3 * 64, device=dev))
    end = int(plan.offsets[3])
    if end < plan.rows_max:
        out = torch.full((plan.rows_max, 64), 7.0, device=dev)
        from nanopysche_amd import _lib
        _lib.call("fm_int8_grouped_gemm", t.data.data_ptr(), t.scale.data_ptr(), t.rows, plan.offsets.data_ptr(), 3,
                  w.data.data_ptr(), w.scale.data_ptr(), None, None, None, 64, 128, 3, out.data_ptr(), _lib.DTYPE_F32, 64,
                  _lib.stream_of(out))
        assert torch.all(out[end:] == 7.0) and torch.all(out[:end] == 128.0)


@pytest.mark.parametrize("T,D", [(0, 128), (0, 14464), (65, 14464), (66000, 128)])
def test_block_of_no_tokens_wide_ones_and_many(dev, T, D):
    """Beyond the few-token kernels' width, and more tokens than a grid's second dimension holds."""
    E, H = 3, 128
    g = torch.Generator().manual_seed(1)
    q = [torch.randint(-127, 128, (E * H, D), generator=g, dtype=torch.int8).to(dev) for _ in range(3)]
    block = fm.Int8MoECompute(fm.Int8Experts.from_int8(q[0], torch.full((E * H,), 1e-3, device=dev), q[1], torch.full((E, D), 1e-3, device=dev),
                                                       q[2], torch.full((E * H,), 1e-3, device=dev), E))
    x, w = torch.randn(T, D, generator=g).to(dev), torch.rand(T, 1, generator=g).to(dev)
    idx = torch.randint(0, E, (T, 1), generator=g).to(dev)
    out = block(x, w, idx)
    assert out.shape == x.shape and torch.isfinite(out).all()
    if T > 128:   # a token's output does not depend on the others
        assert torch.equal(block(x[-100:], w[-100:], idx[-100:]), out[-100:])
        assert torch.equal(block(x[:100], w[:100], idx[:100]), out[:100])
