"""What the balance loss holds between its forward and its backward: f and its two factors, in autograd's keeping."""

import pytest
import torch

import nanopysche_amd as fm
from tests.test_gpu_balance import gen, inputs
from tests.test_gpu_checkpoint_8bit import layer_of, rand

pytestmark = pytest.mark.gpu

SMALL = (1 << 18) + 512   # a small workspace behind f, and the allocator's rounding


def borders_of(T, S):
    cuts = (torch.rand(S - 1, generator=gen(S), device="cuda") * T).long().sort().values
    return torch.cat((cuts.new_zeros(1), cuts, cuts.new_full((1,), T))).to(torch.int32)


def of_f(seen):
    """Sizes of what could be f: the logits are 2-D, the caller's tensors bool and int32."""
    return [n for dtype, dim, n in seen if dtype == torch.float32 and dim == 1]


@pytest.mark.parametrize("T,E,S", [(512, 8, 1), (65536, 256, 1), (65536, 256, 512), (131072, 64, 30000), (4096, 1024, 9)])
def test_the_workspace_ends_with_the_forward(dev, T, E, S):
    logits, idx = inputs(T, E, 4, T)
    cu = borders_of(T, S) if S > 1 else None
    state = fm.balance_forward(logits, idx, cu_seqlens=cu)[2]
    kept = state.f.untyped_storage().nbytes()   # (a failure would print a storage, value by value)
    del state
    assert kept <= 4 * (S * E + 64) + SMALL
    leaf = logits.requires_grad_(True)
    before = torch.cuda.memory_allocated()
    out = fm.balance_loss(leaf, idx, cu_seqlens=cu)
    held = torch.cuda.memory_allocated() - before - out.counts.numel() * 4
    assert held <= 4 * (S * E + 64) + SMALL + 2048
    out.loss.backward()


def test_hooks_see_what_is_kept(dev):
    """Everything that the backward reads can go to the host and come back."""
    T, E, S = 20000, 64, 40
    logits, idx = inputs(T, E, 6, 3)
    cu = borders_of(T, S)
    mask = torch.rand(T, generator=gen(4), device="cuda") < 0.8
    seen = []

    def pack(t):
        seen.append((t.dtype, t.dim(), t.numel()))
        return t.cpu()

    grads = []
    for hooks in (False, True):
        leaf = logits.clone().requires_grad_(True)
        with torch.autograd.graph.saved_tensors_hooks(pack if hooks else lambda t: t, lambda t: t.cuda()):
            out = fm.balance_loss(leaf, idx, cu_seqlens=cu, token_mask=mask, z_loss_multiplier=1e-3)
        out.loss.backward()
        grads.append(leaf.grad)
    assert torch.equal(*grads)
    f, = of_f(seen)
    assert len(seen) == 4 and S * E + 2 <= f < S * E + 2 + SMALL // 4


@pytest.mark.parametrize("whole", [False, True])
def test_hooks_see_what_route_and_the_layer_keep(dev, whole):
    g = torch.Generator().manual_seed(5)
    x = rand(g, 2000, 512)
    cu = torch.tensor([0, 700, 1900], dtype=torch.int32, device="cuda")
    mask = torch.rand(2000, generator=gen(6), device="cuda") < 0.8
    layer, p = layer_of("none", 512, 128, 64, 4, 7, False)
    gate = p["gate"]
    seen = []

    def pack(t):
        seen.append((t.dtype, t.dim(), t.numel()))
        return t.cpu()

    grads = []
    for hooks in (False, True):
        gate.grad = None
        with torch.autograd.graph.saved_tensors_hooks(pack if hooks else lambda t: t, lambda t: t.cuda()):
            aux = (layer(x, token_mask=mask, cu_seqlens=cu) if whole else fm.route(x, gate, top_k=4, token_mask=mask, cu_seqlens=cu))[-1]
        aux.backward(retain_graph=True)
        first, gate.grad = gate.grad, None
        if not whole:   # the block's backward runs once
            aux.backward()
            assert torch.equal(first, gate.grad)
        grads.append(first)
    assert torch.equal(*grads) and grads[0].any()
    f, = of_f(seen)
    assert 2 * 64 + 2 <= f < 2 * 64 + 2 + SMALL // 4
