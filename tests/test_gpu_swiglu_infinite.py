"""SwiGLU of infinite gates: silu(+inf) = +inf, silu(-inf) = NaN, as torch gives both, in every kernel that fuses it."""

import pytest
import torch
import torch.nn.functional as F

import nanopysche_amd as fm
from nanopysche_amd import _lib

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
INF = float("inf")


def rows(dtype, H=128):
    """One infinite gate in some blocks of 32, beside finite ones; every sign of up."""
    gate, up = torch.linspace(-3, 3, 8 * H).reshape(8, H), torch.linspace(2, -2, 8 * H).reshape(8, H)
    gate[0, 0], gate[1, 31], gate[2, 64], gate[3, 127] = INF, INF, -INF, INF
    up[0, 0], up[1, 31], up[3, 127] = 1.5, -1.5, 0.0
    gate[4, 5] = torch.finfo(dtype).max
    up[4, 5] = 0.5
    return gate.to(dtype).cuda(), up.to(dtype).cuda()


def same(got, ref, u):
    """Alike where a value is not finite, else within a rounding and fp32's 16 steps."""
    got, ref = got.double().cpu(), ref.double().cpu()
    odd = ~torch.isfinite(ref)
    assert torch.equal(torch.nan_to_num(got[odd], 7.0, 1e9, -1e9), torch.nan_to_num(ref[odd], 7.0, 1e9, -1e9))
    assert torch.all((got - ref)[~odd].abs() <= u * ref[~odd].abs() + 16 * 2.0 ** -24 * ref[~odd].abs())


@pytest.mark.parametrize("dtype,u", [(BF, 2.0 ** -8), (torch.float32, 2.0 ** -24)])
def test_forward(dev, dtype, u):
    gate, up = rows(dtype)
    want = F.silu(gate.cpu().double()) * up.cpu().double()
    assert want[0, 0] == INF and want[1, 31] == -INF and torch.isnan(want[2, 64]) and torch.isnan(want[3, 127])
    h, g8, _ = fm.swiglu_compress(gate, up)
    same(h, want, u)
    same(fm.swiglu_8bit(torch.cat((gate, up), 1)), want, u)
    assert torch.isnan(g8.restore()[0, :32]).all() and torch.isfinite(g8.restore()[0, 32:]).all()
    if dtype == BF:
        same(fm.fused_silu_multiply_quantize(gate, up, None), want, u)


def test_values_and_gradients(dev):
    """fp32 values of h, and of [dg | du] as torch's autograd of silu gives them."""
    gate, up = rows(BF)
    dh = torch.full_like(gate, 0.25)
    for grad in (None, dh):
        out = torch.empty(8, 128 if grad is None else 256, device="cuda")
        _lib.call("fm_swiglu_values", _lib.ptr(gate), 128, _lib.ptr(up), 128, _lib.ptr(grad), 128, 8, 128, _lib.ptr(out), out.stride(0),
                  _lib.stream_of(gate))
        a, b = gate.cpu().double().requires_grad_(True), up.cpu().double().requires_grad_(True)
        h = F.silu(a) * b
        if grad is None:
            same(out, h.detach(), 0.0)
            continue
        h.backward(dh.cpu().double())
        same(out[:, 128:], b.grad, 0.0)
        odd = ~torch.isfinite(a.grad)
        assert torch.equal(torch.isnan(out[:, :128].cpu()), torch.isnan(a.grad)) and odd.sum() == 4


def test_block_whose_gates_overflow(dev):
    """x w1^T beyond bfloat16: the outputs are infinite, with and without 8-bit activations, and not NaN."""
    D = H = 128
    x = torch.full((64, D), 1e30, dtype=BF, device="cuda")
    w1 = torch.zeros(H, D, dtype=BF, device="cuda")
    w1[:, 0] = 1e30
    w3 = torch.zeros(H, D, dtype=BF, device="cuda")
    w3[:, 0] = 1e-30
    w2 = torch.ones(H, D, dtype=BF, device="cuda")
    idx, w = torch.zeros(64, 1, dtype=torch.int64, device="cuda"), torch.ones(64, 1, device="cuda")
    for eight in (False, True):
        cfg = fm.FP8FlowMoEConfig(False, fm.FP8RecipeConfig(False, fm.FP8RecipeType.NONE))
        block = fm.FP8FlowMoECompute(cfg, D, H, 1, 0, checkpoint_8bit=eight)
        leaves = [t.clone().requires_grad_(True) for t in (w1, w2, w3)]
        block.set_weights(*leaves)
        assert torch.equal(block(x, w, idx, 0, 1), torch.full_like(x, INF))
