"""SwiGLU of gates far beyond any exponential's range, against float64."""

import pytest
import torch

import nanopysche_amd as fm

pytestmark = pytest.mark.gpu


def test_huge_gates(dev):
    """silu(g) is g or 0 there; h is exact but for one rounding to bf16 (2^-8)."""
    sizes = torch.tensor([100.0, 1e4, 2.0 ** 30, 2.0 ** 31, 2.0 ** 32, 1e10, 1e20, 1e30])
    gate = torch.cat((sizes, -sizes)).repeat(8)[None].repeat(4, 1).bfloat16().cuda()
    up = torch.full_like(gate, 1.5)
    h = fm.fused_silu_multiply_quantize(gate, up, None)
    ref = gate.double() * torch.sigmoid(gate.double()) * 1.5
    assert torch.all((h.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-37)
