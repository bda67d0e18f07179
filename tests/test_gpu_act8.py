"""Activations in 8 bits against their float64 definition: the format bit for bit, SwiGLU and RMSNorm whose
backward reads it.

A result rounded to t is off by at most eps(t) / 2 of its size (u below: 2^-8 for bf16, 2^-24 for fp32); what was computed
in fp32 before that adds a few 2^-24 of the terms that it summed."""

import pytest
import torch

import nanopysche_amd as fm
from tests.act8_reference import kept, power, step

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
U = {BF: 2.0 ** -8, F32: 2.0 ** -24}
U32 = 2.0 ** -24


def activation(gen, *shape, dtype=BF):
    x = torch.randn(*shape, generator=gen, device="cuda") * torch.exp(torch.randn(shape[-1], generator=gen, device="cuda"))
    return x.to(dtype)


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=123.0), torch.nan_to_num(b, nan=123.0))


SHAPES = [(1, 1), (1, 7), (3, 8), (2, 31), (5, 32), (4, 33), (1, 63), (129, 100), (64, 2048), (37, 2817), (1000, 96), (2, 3, 40), (7,),
          (515, 8200)]


# ================================================================== the format ====
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_values_bit_for_bit(dev, shape, dtype):
    x = activation(gen(len(shape) + shape[-1]), *shape, dtype=dtype)
    t = fm.compress_activation(x)
    ref = kept(x.double())
    assert t.shape == x.shape and t.dtype == dtype and t.data.numel() == t.nbytes
    for out in (BF, F32):
        got = t.restore(out)
        assert got.dtype == out and got.shape == x.shape
        assert torch.equal(got.double(), ref)
    assert t.restore().dtype == dtype
    # half a step, and a bf16 value never lies above 127.5 steps
    bound = step(x.double()) * (0.5 if dtype == BF else 1.0)
    assert torch.all((x.double() - ref).abs() <= bound)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_special_values(dev, dtype):
    big = torch.finfo(dtype).max
    rows = torch.zeros(12, 96, dtype=torch.float64)
    rows[1, :] = -0.0
    rows[2, 5] = 1.0
    rows[3, :] = torch.arange(96) - 48.0                      # whole steps and halves
    rows[4, :32] = (torch.arange(32) + 0.5) * 2.0             # ties to even at s = 1, under a maximum of 127
    rows[4, 31] = 127.0
    rows[5, 0], rows[5, 33], rows[5, 95] = big, -big, big / 2
    rows[6, :] = 2.0 ** -133                                  # subnormal in bf16 and fp32
    rows[7, :] = power(torch.arange(-149, -53)) if dtype == F32 else 2.0 ** -126
    rows[8, 40] = torch.inf
    rows[9, 64] = -torch.inf
    rows[10, 3] = torch.nan
    rows[11, 0], rows[11, 1] = 255.0 / 2, -255.0 / 2
    x = rows.to(dtype).cuda()
    t = fm.compress_activation(x)
    got = t.restore(F32)
    assert same(got.double(), kept(x.double()))
    assert torch.isnan(got[8, 32:64]).all() and torch.isfinite(got[8, :32]).all() and torch.isfinite(got[8, 64:]).all()
    assert torch.isnan(got[9, 64:]).all() and torch.isnan(got[10, :32]).all()
    assert torch.equal(got[0], torch.zeros_like(got[0])) and got[2, 5] == 1.0
    if dtype == F32:   # above 127.5 steps the largest step count is taken
        y = torch.full((1, 32), 127.9, device="cuda")
        assert torch.equal(fm.compress_activation(y).restore(), torch.full_like(y, 127.0))


def test_strides(dev):
    g = gen(3)
    base = activation(g, 50, 301, dtype=BF)
    for x in (base[:, 3:70], base[1::3], base[::2, :64], base.t(), base[:, ::2], base[4].expand(9, 301), base[:, 7:8],
              activation(g, 4, 6, 50).transpose(0, 1), activation(g, 3, 4, 64)[:, 1]):
        assert torch.equal(fm.compress_activation(x).restore(F32).double(), kept(x.double()))


def test_no_rows(dev):
    for shape in ((0, 5), (3, 0, 64)):
        x = torch.empty(shape, dtype=BF, device="cuda")
        assert fm.compress_activation(x).restore().shape == x.shape
    t = fm.compress_activation(torch.empty(0, 5, dtype=BF, device="cuda"))
    out = t.restore_rows(torch.tensor([0, -1], dtype=torch.int32, device="cuda"))
    assert torch.equal(out, torch.zeros(2, 5, dtype=BF, device="cuda"))
    assert t.restore_rows(torch.empty(0, dtype=torch.int32, device="cuda")).shape == (0, 5)


@pytest.mark.parametrize("dtype,cols", [(BF, 64), (BF, 77), (F32, 130)])
def test_rows_of_an_index(dev, dtype, cols):
    x = activation(gen(4), 5, 20, cols, dtype=dtype)
    t = fm.compress_activation(x)
    index = torch.tensor([99, 0, 0, -1, 57, 100, -2 ** 31, 2 ** 31 - 1, 3], dtype=torch.int32, device="cuda")
    ref = kept(x.double()).reshape(100, cols)
    want = torch.stack([ref[i] if 0 <= i < 100 else torch.zeros_like(ref[0]) for i in index.tolist()])
    assert torch.equal(t.restore_rows(index).double(), want)
    assert torch.equal(t.restore_rows(index.repeat_interleave(2)[::2], F32).double(), want)


def test_offsets_past_32_bits(dev):
    """More rows than one launch takes, and more bytes than 2^32."""
    row = activation(gen(5), 1, 32768)
    x = row.expand(300000, 32768)
    t = fm.compress_activation(x)
    assert t.rows * t.cols > 2 ** 33
    index = torch.tensor([0, 1, 131071, 131072, 262143, 262144, 299999], dtype=torch.int32, device="cuda")
    got = t.restore_rows(index)
    assert torch.equal(got.double(), kept(row.double()).expand(len(index), -1))
    q = t.data[:t.rows * t.pitch].view(t.rows, t.pitch)
    assert all(torch.equal(q[i:i + 10000], q[:1].expand(10000, -1)) for i in range(0, t.rows, 10000))


# ====================================================================== SwiGLU ====
def swiglu_ref(gate, up, dh):
    gate, up, dh = gate.double(), up.double(), dh.double()
    h = gate * torch.sigmoid(gate) * up
    g, u = kept(gate), kept(up)
    s = torch.sigmoid(g)
    return h, dh * u * s * (1 + g * (1 - s)), dh * g * s, (dh * u * s).abs() * (1 + g.abs())


def close(got, ref, terms=None, times=8.0, floor=0.0):
    """Rounded once to got's type after fp32 work on terms of this size."""
    terms = ref.abs() if terms is None else terms
    return torch.all((got.double() - ref).abs() <= U[got.dtype] * ref.abs() + times * U32 * terms + floor + 1e-37)


def under(*factors):
    """What SwiGLU loses where 1 / (1 + e^-g) is subnormal (g < -87.3: the hardware's reciprocal is 0 there): up to |g| e^g or (1 + |g|) e^g
    of the other factors' product, at most 89 / 2^126 < 2^-119."""
    product = 1.0
    for f in factors:
        product = product * f.double().abs()
    return 2.0 ** -119 * product


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (3, 32), (5, 33), (2, 3, 100), (128, 1408), (300, 1419), (2000, 4096)])
def test_swiglu(dev, shape, packed, dtype):
    g = gen(shape[-1] + packed)
    gate, up = activation(g, *shape, dtype=dtype) * 2, activation(g, *shape, dtype=dtype)
    dh = activation(g, *shape, dtype=dtype) * 1e-2
    h, dg, du, terms = swiglu_ref(gate, up, dh)
    args = (torch.cat((gate, up), -1),) if packed else (gate, up)
    out, kept_g, kept_u = fm.swiglu_compress(*args)
    assert close(out, h, floor=under(up))
    assert torch.equal(kept_g.restore(F32).double(), kept(gate.double())) and torch.equal(kept_u.restore(F32).double(), kept(up.double()))
    grads = fm.swiglu_backward_8bit(dh, kept_g, kept_u, packed=packed)
    got_g, got_u = grads.chunk(2, -1) if packed else grads
    assert close(got_g, dg, terms, floor=under(dh, kept(up.double()))) and close(got_u, du, floor=under(dh))
    leaves = [a.clone().requires_grad_(True) for a in args]
    y = fm.swiglu_8bit(*leaves)
    y.backward(dh)
    assert torch.equal(y, out)
    auto = leaves[0].grad.chunk(2, -1) if packed else [a.grad for a in leaves]
    assert torch.equal(auto[0], got_g) and torch.equal(auto[1], got_u)


def test_swiglu_extremes(dev):
    gate = torch.tensor([[-200.0, -89.0, -88.0, -30.0, 0.0, -0.0, 30.0, 89.0, 1e30, -1e30, 3e-39, -1.278, 1.0, 2.0, 3.0, 4.0]], device="cuda")
    up = torch.full_like(gate, 1.5)
    h, g8, u8 = fm.swiglu_compress(gate, up)
    assert close(h, (gate.double() * torch.sigmoid(gate.double()) * 1.5), times=16, floor=under(up))
    # one value to a block: each keeps its own size
    wide, wup = (torch.nn.functional.pad(t.t(), (0, 31)) for t in (gate, up))
    dh = torch.full_like(wide, 0.5)
    _, g8, u8 = fm.swiglu_compress(wide, wup)
    dg, du = fm.swiglu_backward_8bit(dh, g8, u8)
    _, rg, ru, terms = swiglu_ref(wide, wup, dh)
    finite = torch.isfinite(rg) & torch.isfinite(terms)
    assert close(dg[finite], rg[finite], terms[finite], 16, under(dh, wup)[finite]) and close(du, ru, times=16, floor=under(dh))


def test_swiglu_gradient_by_differences(dev):
    """Values that 8 bits hold exactly: the gradient is that of the function itself."""
    g = gen(8)
    gate, up, dh = ((torch.randint(-127, 128, (40, 64), generator=g, device="cuda").float() / 32) for _ in range(3))
    gate[:, ::32] = 127 / 32
    up[:, ::32] = 127 / 32
    a, b = gate.clone().requires_grad_(True), up.clone().requires_grad_(True)
    fm.swiglu_8bit(a, b).backward(dh)
    f = lambda x, y: (x * torch.sigmoid(x) * y * dh.double())   # noqa: E731
    x, y, e = gate.double(), up.double(), 1e-5
    # the third derivatives of silu are below 1: differences are off by e^2 |y dh| / 6 and 1e-16 / e of the values
    bound = 1e-9 + 32 * U32 * (dh.double().abs() * (1 + x.abs()) * (1 + y.abs()))
    assert torch.all((a.grad.double() - (f(x + e, y) - f(x - e, y)) / (2 * e)).abs() <= bound)
    assert torch.all((b.grad.double() - (f(x, y + e) - f(x, y - e)) / (2 * e)).abs() <= bound)


def test_swiglu_strides_and_broadcast(dev):
    g = gen(9)
    base, dhb = activation(g, 30, 400), activation(g, 30, 400)
    gate, up, dh = base[:, 1:100], base[::1, 201:300], dhb[:, 5:104]
    h, dg, du, terms = swiglu_ref(gate, up, dh)
    leaves = [base.clone().requires_grad_(True)]
    out = fm.swiglu_8bit(leaves[0][:, 1:100], leaves[0][:, 201:300])
    out.backward(dh)
    assert close(out, h, floor=under(up))
    grad = leaves[0].grad
    assert close(grad[:, 1:100], dg, terms, floor=under(dh, up)) and close(grad[:, 201:300], du, floor=under(dh)) and not grad[:, 100:201].any()
    # one row of gate for all of up's: its gradient is the sum (autograd's, rounded from bf16 terms: compared as such)
    one = gate[:1].clone().requires_grad_(True)
    fm.swiglu_8bit(one.expand(30, 99), up).backward(dh)
    _, dg, _, terms = swiglu_ref(gate[:1].expand(30, 99), up, dh)
    size = dg.abs().sum(0, keepdim=True)
    assert torch.all((one.grad.double() - dg.sum(0, keepdim=True)).abs() <= 2 * U[BF] * size + 1e-30)
    # a gradient that is one number everywhere
    leaf = up.clone().requires_grad_(True)
    fm.swiglu_8bit(gate, leaf).sum().backward()
    _, _, du, _ = swiglu_ref(gate, up, torch.ones_like(up))
    assert close(leaf.grad, du)


def test_swiglu_no_rows_and_nans(dev):
    x = torch.empty(0, 10, dtype=BF, device="cuda", requires_grad=True)
    fm.swiglu_8bit(x).sum().backward()
    assert x.grad.shape == (0, 10)
    gate, up = torch.ones(2, 64, device="cuda"), torch.ones(2, 64, device="cuda")
    gate[0, 40] = torch.nan
    h, g8, u8 = fm.swiglu_compress(gate, up)
    assert torch.isnan(h).sum() == 1
    dg, du = fm.swiglu_backward_8bit(torch.ones_like(gate), g8, u8)
    assert torch.isnan(dg[0, 32:]).all() and torch.isnan(du[0, 32:]).all()
    assert torch.isfinite(dg[0, :32]).all() and torch.isfinite(dg[1]).all()


# ===================================================================== RMSNorm ====
def norm_ref(x, w, dy, eps):
    x, w, dy = x.double(), w.double(), dy.double()
    D = x.shape[-1]
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    k = kept(x)
    a = dy * w
    dot = (a * k).sum(-1, keepdim=True)
    terms = r * a.abs() + r ** 3 / D * (a * k).abs().sum(-1, keepdim=True) * k.abs()
    dims = tuple(range(x.dim() - 1))
    return x * r * w, r * a - r ** 3 / D * dot * k, (dy * k * r).sum(dims), terms, (dy * k * r).abs().sum(dims)


@pytest.mark.parametrize("wdtype", [F32, BF])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 9), (3, 31), (5, 512), (9, 513), (2, 5, 1000), (33, 1024), (37, 1025), (130, 2048), (37, 2831),
                                   (19, 7168), (3, 16384), (2, 16383), (4100, 256), (8200, 40),
                                   (1, 64), (7, 65), (9, 128), (600, 130), (515, 300), (513, 512), (5000, 17), (700, 4096)])
def test_rmsnorm(dev, shape, dtype, wdtype):
    g = gen(shape[0] + shape[-1])
    x, dy = activation(g, *shape, dtype=dtype), activation(g, *shape, dtype=dtype) * 1e-2
    w = (1 + 0.1 * torch.randn(shape[-1], generator=g, device="cuda")).to(wdtype)
    eps = 1e-5
    y, dx, dw, terms, dw_terms = norm_ref(x, w, dy, eps)
    got, kept_x, rstd = fm.rmsnorm_compress(x, w, eps)
    # sums of D squares in fp32, pairwise over lanes and waves: below 32 additions deep each; r, two products
    assert close(got, y, times=48)
    assert torch.equal(kept_x.restore(F32).double(), kept(x.double()))
    gx, gw = fm.rmsnorm_backward_8bit(dy, kept_x, w, rstd)
    assert close(gx, dx, terms, 128)
    # dw: a slice of at most 1024 / 8 rows in order, then 64 shares in order, sixteen sums in order
    assert torch.all((gw.double() - dw).abs() <= U[wdtype] * dw.abs() + 256 * U32 * dw_terms + 1e-37)
    assert gw.dtype == wdtype
    only, none = fm.rmsnorm_backward_8bit(dy, kept_x, w, rstd, need_dw=False)
    assert none is None and torch.equal(only, gx)
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    out = fm.rmsnorm_8bit(a, b, eps)
    out.backward(dy)
    assert torch.equal(out, got) and torch.equal(a.grad, gx) and torch.equal(b.grad, gw)


def test_rmsnorm_gradient_by_differences(dev):
    g = gen(11)
    x = torch.randint(-127, 128, (6, 96), generator=g, device="cuda").float() / 64
    x[:, ::32] = 127 / 64
    w, dy = torch.rand(96, generator=g, device="cuda") + 0.5, torch.randn(6, 96, generator=g, device="cuda")
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    fm.rmsnorm_8bit(a, b, 1e-6).backward(dy)

    def f(x, w):
        return (x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-6) * w * dy.double()).sum()

    e = 1e-6
    for leaf, which in ((a, 0), (b, 1)):
        for i in range(0, leaf.numel(), 37):
            args = [x.double().clone(), w.double().clone()]
            args[which].view(-1)[i] += e
            up = f(*args)
            args[which].view(-1)[i] -= 2 * e
            # values of about 100 in float64 over 2e: 1e-8, and second-order terms of e^2
            assert abs((up - f(*args)) / (2 * e) - leaf.grad.view(-1)[i].double()) <= 1e-5 * (1 + leaf.grad.abs().max())


def test_rmsnorm_strides_and_empty(dev):
    g = gen(12)
    base, dyb = activation(g, 40, 700), activation(g, 40, 700)
    w = torch.rand(1400, generator=g, device="cuda")[::2]
    x, dy = base[::2, 1:], dyb[1::2, :699]
    y, dx, dw, terms, dw_terms = norm_ref(x, w[:699], dy, 1e-6)
    got, k, r = fm.rmsnorm_compress(x, w[:699])
    gx, gw = fm.rmsnorm_backward_8bit(dy, k, w[:699], r)
    assert close(got, y, times=48) and close(gx, dx, terms, 128)
    assert torch.all((gw.double() - dw).abs() <= 256 * U32 * dw_terms + U32 * dw.abs())
    e = torch.empty(0, 64, dtype=BF, device="cuda", requires_grad=True)
    we = torch.ones(64, device="cuda", requires_grad=True)
    fm.rmsnorm_8bit(e, we).sum().backward()
    assert e.grad.shape == (0, 64) and torch.equal(we.grad, torch.zeros_like(we))
    zero = torch.zeros(3, 64, device="cuda")
    y, k, r = fm.rmsnorm_compress(zero, we.detach())
    gx, _ = fm.rmsnorm_backward_8bit(torch.ones_like(zero), k, we.detach(), r)
    assert torch.equal(y, zero) and close(gx, torch.full_like(zero, 1e3).double(), times=16)   # 1 / sqrt(1e-6)


def test_rmsnorm_of_more_rows_than_a_launch_takes(dev):
    """Four rows to a workgroup of 256: 2^25 rows a launch; rows repeat, so a few stand for all."""
    rows = activation(gen(15), 1000, 8)
    T = 2 ** 25 + 4000
    x = rows.repeat((T + 999) // 1000, 1)[:T]
    w = torch.rand(8, generator=gen(16), device="cuda")
    y, k, r = fm.rmsnorm_compress(x, w)
    ys, ks, rs = fm.rmsnorm_compress(rows, w)
    gx, gw = fm.rmsnorm_backward_8bit(x, k, w, r)
    gs, _ = fm.rmsnorm_backward_8bit(rows, ks, w, rs)
    whole = T // 1000
    for got, one in ((y, ys), (gx, gs), (r[:, None], rs[:, None]), (k.restore(), ks.restore())):
        assert torch.equal(got[:whole * 1000].view(whole, 1000, -1), one.expand(whole, 1000, -1))
        assert torch.equal(got[whole * 1000:], one[:T - whole * 1000])
    ref = (rows.double() * kept(rows.double()) * rs.double()[:, None]).sum(0) * (T / 1000)
    assert torch.all((gw.double() - ref).abs() <= 1e-3 * ref.abs().max())   # 65,000 rows a slice, one after the other, in fp32: 2^-24 sqrt of them


def test_rmsnorm_module(dev):
    x = activation(gen(13), 20, 1536)
    a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    plain, eight = fm.RMSNorm(1536).cuda(), fm.RMSNorm(1536, checkpoint_8bit=True).cuda()
    ya, yb = plain(a), eight(b)
    dy = activation(gen(14), 20, 1536)
    ya.backward(dy)
    yb.backward(dy)
    # both round x r once to fp32, times w, to bf16; the sum of squares differs in its last bits
    assert torch.all((ya.double() - yb.double()).abs() <= 2 * U[BF] * ya.double().abs())
    # x within half of a 64th of its block's maximum
    near = step(x.double()) / 2
    y, dx, dw, terms, dw_terms = norm_ref(x, plain.weight, dy, 1e-6)
    r = (1 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-6))
    assert torch.all((plain.weight.grad.double() - eight.weight.grad.double()).abs() <= (dy.double().abs() * near * r).sum(0) + 256 * U32 * dw_terms)
    assert set(eight.state_dict()) == {"weight"}


# =================================================================== in a program ====
def step_fn(gu, w, x, dy):
    y = fm.rmsnorm_8bit(x, w)
    h = fm.swiglu_8bit(gu + y)
    return h, dy


def test_graph_replays(dev):
    """The norm and SwiGLU, forward and backward, captured once and replayed on new inputs."""
    g = gen(20)
    x, gu = activation(g, 100, 1030).requires_grad_(True), activation(g, 100, 1030).requires_grad_(True)
    w = torch.ones(1030, device="cuda", requires_grad=True)
    dh = activation(g, 100, 515)

    def step():
        h = fm.swiglu_8bit(gu + fm.rmsnorm_8bit(x, w))
        h.backward(dh)
        return h

    graphed = fm.GraphedStep(step, leaves=[x, gu, w])
    for i in range(3):
        with torch.no_grad():
            x.copy_(activation(gen(30 + i), 100, 1030))
            gu.copy_(activation(gen(40 + i), 100, 1030))
            dh.copy_(activation(gen(50 + i), 100, 515))
        graphed.replay()
        torch.cuda.synchronize()
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, gu, w)]
        h = fm.swiglu_8bit(leaves[1] + fm.rmsnorm_8bit(leaves[0], leaves[2]))
        h.backward(dh)
        torch.cuda.synchronize()
        assert torch.equal(graphed.outputs, h)
        for got, leaf in zip(graphed.grads, leaves):
            assert torch.equal(got, leaf.grad)


def test_other_stream(dev):
    """On the caller's stream: results of a side stream's inputs, without a synchronisation between."""
    side = torch.cuda.Stream()
    x = activation(gen(60), 3000, 2048)
    w = torch.ones(2048, device="cuda")
    ref, k, r = fm.rmsnorm_compress(x, w)
    gx, gw = fm.rmsnorm_backward_8bit(x, k, w, r)
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.empty_like(x)
        for _ in range(20):
            late.copy_(x * 3)
        late.copy_(x)
        y, k, r = fm.rmsnorm_compress(late, w)
        hx, hw = fm.rmsnorm_backward_8bit(late, k, w, r)
        back = k.restore()
    side.synchronize()
    assert torch.equal(y, ref) and torch.equal(hx, gx) and torch.equal(hw, gw)
    assert torch.equal(back.double(), kept(x.double()))


def test_repeated_calls_agree(dev):
    """dw's sums run in a fixed order."""
    x, dy = activation(gen(61), 5000, 3000), activation(gen(62), 5000, 3000)
    w = torch.ones(3000, device="cuda")
    _, k, r = fm.rmsnorm_compress(x, w)
    first = fm.rmsnorm_backward_8bit(dy, k, w, r)
    for _ in range(3):
        again = fm.rmsnorm_backward_8bit(dy, k, w, r)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_saved_tensor_hooks(dev):
    x = activation(gen(63), 50, 200).requires_grad_(True)
    fm.swiglu_8bit(x).sum().backward()
    ref, x.grad = x.grad, None
    saved = []

    def pack(t):
        saved.append(t.numel())
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()):
        y = fm.swiglu_8bit(x)
    y.sum().backward()
    assert torch.equal(x.grad, ref)
    assert sorted(saved) == [50 * 4 * 33] * 2   # 100 columns: four blocks of 33 bytes


def test_tensors_elsewhere_are_refused(dev):
    x = activation(gen(64), 4, 64)
    t = fm.compress_activation(x)
    host = fm.Activation8(t.data.cpu(), t.shape, BF)
    w, rstd = torch.ones(64, device="cuda"), torch.ones(4, device="cuda")
    for call in (lambda: t.restore_rows(torch.zeros(3, dtype=torch.int32)), lambda: fm.swiglu_compress(x, x.cpu()),
                 lambda: fm.swiglu_backward_8bit(x, t, host), lambda: fm.swiglu_backward_8bit(x.cpu(), t, t),
                 lambda: fm.rmsnorm_compress(x, w.cpu()), lambda: fm.rmsnorm_backward_8bit(x, host, w, rstd),
                 lambda: fm.rmsnorm_backward_8bit(x, t, w, rstd.cpu()), lambda: host.restore()):
        with pytest.raises((ValueError, RuntimeError), match="is on|device"):
            call()
