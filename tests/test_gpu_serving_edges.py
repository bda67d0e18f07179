"""Serving entries at sizes and forms beside those of the other tests, against float64."""

import pytest
import torch

import nanopysche_amd as fm
from tests.test_gpu_int8 import plain_rows

pytestmark = pytest.mark.gpu


def test_few_tokens_of_an_expert_beyond_the_few_token_kernels(dev):
    """A matrix of 2^30 elements and more: up to 64 tokens take the products too, with the bits of a
    longer prompt's.  h's payload may turn where h / s lies within fp32 rounding of a half, as in
    the block's other tests: far below 1e-3 of the outputs' norm."""
    D, H, T = 14336, 75008, 70
    g = torch.Generator(device=dev).manual_seed(1)
    q1, q2, q3 = (torch.randint(-127, 128, (H, D), generator=g, device=dev, dtype=torch.int8) for _ in range(3))
    s1, s2, s3 = ((torch.rand(n, generator=g, device=dev) + 0.5) * 3e-4 for n in (H, D, H))
    block = fm.Int8MoECompute(fm.Int8Experts.from_int8(q1, s1, q2, s2.view(1, D), q3, s3, 1))
    x, w = torch.randn(T, D, generator=g, device=dev), torch.rand(T, 1, generator=g, device=dev)
    idx = torch.zeros(T, 1, dtype=torch.int64, device=dev)
    out = block(x, w, idx)
    for n in (1, 64):
        assert torch.equal(block(x[:n], w[:n], idx[:n]), out[:n]), n
    q, s = plain_rows(x)
    h = torch.empty(T, H, dtype=torch.float64, device=dev)
    for c in range(0, H, 8192):
        r = slice(c, c + 8192)
        gate, up = ((q.double() @ qw[r].double().t().contiguous()) * s.double()[:, None] * sw[r].double() for qw, sw in ((q1, s1), (q3, s3)))
        h[:, r] = gate * torch.sigmoid(gate) * up
    hs = h.abs().amax(1, keepdim=True).clamp_min(1e-12) / 127
    hq = torch.round(h / hs) * hs
    ref = sum(hq[:, c:c + 8192] @ q2[c:c + 8192].double() for c in range(0, H, 8192)) * s2.double() * w.double()
    assert (out.double() - ref).norm() <= 1e-3 * ref.norm()
