"""Int8 quantisation and products against plain forms.

The payload and scales are whole numbers and single fp32 divisions: equal bit for bit.  An
integer sum is exact in float64, so an fp32 output is off by the rounding of the sum to fp32,
two products and the bias's addition (4 steps of 2^-24 of the terms), a bf16 output by half a
step of bf16 more."""

import pytest
import torch

import nanopysche_amd as fm
from nanopysche_amd import _lib
from nanopysche_amd.int8 import MAX_INT8_K, _pack, _quantize
from tests.helpers import randn_bf16, zipf_routing
from tests.test_gpu_decode import check, expert_weights, layer64

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def plain_rows(x):
    """(q fp32, s fp32) of rows, in the definition's fp32 operations."""
    x = x.float()
    s = x.abs().amax(1).clamp_min(1e-12) / torch.tensor(127.0, device=x.device)   # a true division: torch multiplies by a scalar's reciprocal
    return torch.round(x / s[:, None]), s


@pytest.mark.parametrize("rows", [1, 15, 16, 17, 130, 600, 1100])
@pytest.mark.parametrize("cols", [1, 15, 16, 63, 64, 65, 127, 129, 1000, 1025, 2048, 2049, 4097, 8192, 8200, 20001])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantise_is_exact(dev, rows, cols, dtype):
    x = torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows * cols)) * 3
    x = x.to(dtype).to(dev)
    x[0] = 0
    if rows > 1:
        x[1] *= 1e-20
    if rows > 15:
        x[15, -1] = 1e30
    t = fm.quantize_to_int8(x)
    q, s = plain_rows(x)
    assert torch.equal(t.scale, s)
    assert torch.equal(t.values().float(), q)
    assert torch.equal(t.dequantize(torch.float32), q * s[:, None])
    assert torch.equal(t.dequantize(), (q * s[:, None]).bfloat16())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantise_strided_rows_and_leading_dimensions(dev, dtype):
    big = torch.randn(6, 5, 301, generator=torch.Generator().manual_seed(1)).to(dtype).to(dev)
    x = big[1:, :, 1:288]   # odd pitch, misaligned rows
    t = fm.quantize_to_int8(x)
    q, s = plain_rows(x.reshape(-1, 287))
    assert torch.equal(t.values().float(), q) and torch.equal(t.scale, s)
    x = big[:, 2].t()       # columns as rows
    q, s = plain_rows(x)
    t = fm.quantize_to_int8(x)
    assert torch.equal(t.values().float(), q) and torch.equal(t.scale, s)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_row_that_is_not_finite_is_nan(dev, bad, dtype):
    x = torch.randn(20, 300, generator=torch.Generator().manual_seed(1)).to(dtype).to(dev)
    x[3, 299] = bad
    w = fm.quantize_to_int8(torch.randn(40, 300, generator=torch.Generator().manual_seed(2)).to(dev))
    out = fm.int8_linear(x, w)
    assert out[3].isnan().all()
    keep = torch.arange(20, device=dev) != 3
    assert out[keep].isfinite().all()
    assert torch.equal(out[keep], fm.int8_linear(x[keep], w))


def random_int8(dev, rows, cols, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-128, 128, (rows, cols), generator=g, dtype=torch.int8).to(dev)
    s = (torch.rand(rows, generator=g) + 0.5).to(dev) / 100
    return q, s


def check_product(out, qa, sa, qw, sw, bias):
    prod = (qa.double() @ qw.double().t()) * sa.double()[:, None] * sw.double()
    bound = 4 * U * prod.abs()
    if bias is not None:
        bound = bound + 2 * U * bias.abs().double()
        prod = prod + bias.double()
    check(out, prod, bound + 1e-30)


SHAPES = [(1, 1, 1), (1, 17, 64), (3, 100, 130), (16, 48, 128), (17, 33, 1000), (33, 65, 200), (48, 15, 640), (49, 300, 2049),
          (64, 64, 4096), (65, 1, 100), (65, 127, 257), (100, 129, 64), (128, 128, 128), (129, 257, 300), (300, 500, 700),
          (1000, 640, 1409), (4097, 2049, 130), (4300, 2300, 200), (4090, 4300, 200), (1500, 3500, 130), (65, 9001, 300), (129, 6001, 257),
          (300, 3001, 700), (33, 20001, 64), (512, 700, 130), (3000, 5, 300)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_matmul_matches_exact_sums(dev, M, N, K):
    qa, sa = random_int8(dev, M, K, 1)
    qw, sw = random_int8(dev, N, K, 2)
    a, w = fm.Int8Tensor.from_int8(qa, sa), fm.Int8Tensor.from_int8(qw, sw)
    assert torch.equal(a.values(), qa) and torch.equal(w.values(), qw)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(3)).to(dev)
    check_product(fm.int8_matmul(a, w, out_dtype=torch.float32), qa, sa, qw, sw, None)
    check_product(fm.int8_matmul(a, w, bias, out_dtype=torch.float32), qa, sa, qw, sw, bias)
    check_product(fm.int8_matmul(a, w, bias), qa, sa, qw, sw, bias)


@pytest.mark.parametrize("M,N,K", [(1, 40, 129), (1, 17, 20000), (2, 33, 4096), (4, 64, 8192), (4, 20, 8193), (5, 20, 300), (90, 70, 300)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_is_quantise_and_matmul(dev, M, N, K, dtype):
    """A few rows are quantised inside the product: the same bits."""
    x = torch.randn(M + 1, K + 3, generator=torch.Generator().manual_seed(1)).to(dtype).to(dev)[1:, 1:K + 1]
    if M > 1:
        x[1] = 0
    w = fm.quantize_to_int8(torch.randn(N, K, generator=torch.Generator().manual_seed(2)).to(dev))
    bias = torch.randn(N, generator=torch.Generator().manual_seed(3)).to(dev)
    for b in (None, bias):
        for out in (torch.float32, torch.bfloat16):
            got = fm.int8_linear(x, w, b, out_dtype=out)
            assert torch.equal(got, fm.int8_matmul(fm.quantize_to_int8(x), w, b, out_dtype=out))


@pytest.mark.parametrize("M", [5, 200])
def test_longest_sum_does_not_overflow(dev, M):
    q = torch.full((M, MAX_INT8_K), -128, dtype=torch.int8, device=dev)
    one = torch.ones(M, device=dev)
    t = fm.Int8Tensor.from_int8(q, one)
    out = fm.int8_matmul(t, t, out_dtype=torch.float32)
    assert torch.all(out == float(128 * 128 * MAX_INT8_K))


@pytest.mark.parametrize("counts", [(5,), (0, 200, 0, 1), (300, 128, 129, 0, 700), (1,) * 70 + (0, 513), (128,) * 8, (2000, 2200)])
@pytest.mark.parametrize("N,K", [(16, 128), (272, 384), (640, 256), (4096, 128)])
def test_grouped_matches_exact_sums(dev, counts, N, K):
    E = len(counts)
    idx = torch.cat([torch.full((c,), e, dtype=torch.int64) for e, c in enumerate(counts)])
    idx = idx[torch.randperm(idx.numel(), generator=torch.Generator().manual_seed(1))][:, None].to(dev)
    plan = fm.route_tokens(idx, E)
    qa, sa = random_int8(dev, plan.rows_max, K, 1)
    qw, sw = random_int8(dev, E * N, K, 2)
    for dtype in (torch.float32, torch.bfloat16):
        out = fm.int8_grouped_gemm(fm.Int8Tensor.from_int8(qa, sa), fm.Int8Tensor.from_int8(qw, sw), plan, dtype)
        offs = plan.offsets.tolist()
        for e in range(E):
            r, c = slice(offs[e], offs[e + 1]), slice(e * N, (e + 1) * N)
            if offs[e] < offs[e + 1]:
                check_product(out[r], qa[r], sa[r], qw[c], sw[c], None)


def test_quantise_of_a_plan_gathers_and_stops(dev):
    T, E, K, D = 200, 5, 2, 192
    _, idx = zipf_routing(T, E, K, 1.0, seed=3, zero_experts=(2,))
    plan = fm.route_tokens(idx.to(dev), E)
    x = randn_bf16((T, D), seed=1).to(dev)
    end = int(plan.offsets[E])
    t = _quantize(x, plan.rows_max, plan.assign_of_row, K, plan.offsets[E:])
    q, s = plain_rows(x)
    got, a = t.values()[:end].float(), plan.assign_of_row[:end].long()
    assert torch.equal(got[a >= 0], q[a[a >= 0] // K]) and torch.equal(t.scale[:end][a >= 0], s[a[a >= 0] // K])
    assert torch.all(got[a < 0] == 0) and torch.all(t.scale[:end][a < 0] == 0)


def test_padding_of_a_plan_is_left_out_of_swiglu(dev):
    """Its h is not written, its maximum not raised, and a row of maximum 0 is not read."""
    T, E, K, D, H = 100, 6, 2, 256, 384
    _, idx = zipf_routing(T, E, K, 1.0, seed=3, zero_experts=(2,))
    plan = fm.route_tokens(idx.to(dev), E)
    end = int(plan.offsets[E])
    x = randn_bf16((T, D), seed=1).to(dev)
    x[3] = 0
    x[4] *= 1e-30   # below the scale's floor: a row like another
    t = _quantize(x, plan.rows_max, plan.assign_of_row, K, plan.offsets[E:])
    w = [fm.Int8Tensor.from_int8(*random_int8(dev, E * H, D, s)) for s in (2, 3)]
    top = torch.zeros(plan.rows_max, dtype=torch.int32, device=dev)
    h = torch.full((plan.rows_max, H), float("nan"), device=dev)
    _lib.call("fm_int8_grouped_gemm", t.data.data_ptr(), t.scale.data_ptr(), t.rows, plan.offsets.data_ptr(), E, w[0].data.data_ptr(),
              w[0].scale.data_ptr(), w[1].data.data_ptr(), w[1].scale.data_ptr(), top.data_ptr(), H, D, T * K, h.data_ptr(),
              _lib.DTYPE_F32, H, _lib.stream_of(h))
    pad = plan.assign_of_row[:end] < 0
    assert pad.any() and torch.isnan(h[:end][pad]).all() and torch.isfinite(h[:end][~pad]).all()
    assert torch.equal(top[:end].view(torch.float32), torch.where(pad, 0, h[:end].abs().amax(1)))
    q = _quantize(h, plan.rows_max, limit=plan.offsets[E:], top=top)
    got, want = q.values()[:end].float(), plain_rows(h[:end][~pad])
    assert torch.all(got[pad] == 0) and torch.equal(got[~pad], want[0]) and torch.equal(q.scale[:end][~pad], want[1])


@pytest.mark.parametrize("R,C", [(1, 1), (16, 64), (17, 65), (48, 128), (160, 300), (33, 1)])
def test_pack_of_any_strides(dev, R, C):
    """Rows, columns, every second element and repeated rows, from odd addresses; groups too."""
    g = torch.Generator().manual_seed(R * C)
    base = torch.randint(-128, 128, (2 * R * C * 6 + 7,), generator=g, dtype=torch.int8).to(dev)
    one = torch.ones(R, device=dev)
    for q in (base[3:3 + R * C].view(R, C), base[1:1 + R * C].view(C, R).t(), base[:4 * R * C].view(2 * R, 2 * C)[::2, ::2],
              base[5:5 + 2 * R * C].view(C, 2 * R)[:, 1:R + 1].t(), base[2:2 + C].expand(R, C)):
        assert torch.equal(fm.Int8Tensor.from_int8(q, one).values(), q)
    if R % 16 == 0:
        w = base[:2 * R * C].view(2, C, R).transpose(1, 2)
        assert torch.equal(_pack(w, torch.ones(2 * R, device=dev)).values(), w.reshape(2 * R, C))


def block64(x, weights, indices, w, E):
    """The block's definition: x and h quantised by token (h from float64)."""
    q, s = plain_rows(x)
    x = q.double() * s.double()[:, None]
    out = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for e in range(E):
        t, k = (indices == e).nonzero(as_tuple=True)
        if t.numel():
            g, u = x[t] @ w[0][e].t(), x[t] @ w[2][e].t()
            h = g * torch.sigmoid(g) * u
            hs = h.abs().amax(1, keepdim=True).clamp_min(1e-12) / 127
            out.index_add_(0, t, (torch.round(h / hs) * hs) @ w[1][e] * weights[t, k, None].double())
    return out


@pytest.mark.parametrize("T,E,K,H,D", [(65, 4, 1, 128, 128), (200, 8, 2, 384, 256), (700, 3, 2, 256, 640), (130, 64, 6, 128, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_block_matches_its_definition(dev, T, E, K, H, D, dtype):
    """h's payload may turn where h / s lies within fp32 rounding of a half: one step of s in
    about 1e-4 of its elements, far below 1e-3 of the outputs' norm."""
    weights, indices = (t.to(dev) for t in zipf_routing(T, E, K, 0.8, seed=T))
    x = randn_bf16((T, D), seed=1).to(dev, dtype)
    raw = [t.to(dev) for t in expert_weights(E, H, D, 5)]
    ex = fm.Int8Experts.quantize(*raw, E)
    w = [ex.w1.dequantize(torch.float32).double().view(E, H, D), ex.w2.dequantize(torch.float32).double().view(E, D, H).transpose(1, 2),
         ex.w3.dequantize(torch.float32).double().view(E, H, D)]
    out = fm.Int8MoECompute(ex)(x, weights, indices)
    ref = block64(x, weights, indices, w, E)
    assert out.dtype == dtype
    err = (out.double() - ref).norm() / ref.norm()
    assert err <= (1e-3 if dtype == torch.float32 else 1e-3 + 2.0 ** -8), err.item()
    # slots of experts elsewhere add nothing
    part = fm.Int8MoECompute(ex)(x.float(), weights, torch.where(indices == 1, indices, indices + 1000), 0)
    ref = block64(x, weights * (indices == 1), indices, w, E)
    assert (part.double() - ref).norm() <= 1e-3 * ref.norm()


@pytest.mark.parametrize("T", [1, 16, 17, 40, 64])
@pytest.mark.parametrize("E,K,H,D", [(4, 2, 128, 128), (3, 1, 384, 640), (40, 6, 1024, 256), (24, 8, 4096, 128)])
def test_decode_with_int8_experts(dev, T, E, K, H, D):
    x = randn_bf16((T, D), seed=T).to(dev)
    weights, indices = (t.to(dev) for t in zipf_routing(T, E, K, 0.8, seed=T))
    ex = fm.Int8Experts.quantize(*(t.to(dev) for t in expert_weights(E, H, D, 5)), E)
    sh = fm.Int8Experts.quantize(*(t.to(dev) for t in expert_weights(1, 256, D, 9)), 1)

    def real(ex, E, H):
        w2 = ex.w2.dequantize(torch.float32).double().view(E, D, H).transpose(1, 2).reshape(E * H, D)
        s = ex.w2.scale.double().view(E, 1, D).expand(E, H, D).reshape(E * H, D)
        q2 = ex.w2.values().double().view(E, D, H).transpose(1, 2).reshape(E * H, D)
        assert torch.allclose(w2, q2 * s, rtol=1e-6, atol=0)
        return [ex.w1.values().double() * ex.w1.scale.double()[:, None], q2 * s,
                ex.w3.values().double() * ex.w3.scale.double()[:, None]]

    ref, bound = layer64(x.double(), 4 * U * x.double().abs(), weights, indices, real(ex, E, H), E, shared=real(sh, 1, 256))
    check(fm.expert_decode(x.float(), weights, indices, ex, E, shared=sh), ref, bound * 1.01)
    got = fm.Int8MoECompute(ex)(x, weights, indices)
    check(got, *layer64(x.double(), 4 * U * x.double().abs(), weights, indices, real(ex, E, H), E))
