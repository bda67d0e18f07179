"""swiglu_8bit and rmsnorm_8bit where no gradient is recorded: the same bits, and nothing kept."""

import pytest
import torch

import nanopysche_amd as fm
from nanopysche_amd import _lib
from tests.test_gpu_act8 import activation, gen
from tests.test_gpu_checkpoint_8bit import layer_of, rand

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture
def calls(monkeypatch):
    """(name, its null arguments' places) of each library call."""
    seen, call = [], _lib.call

    def note(name, *args):
        seen.append((name, [i for i, a in enumerate(args) if a is None]))
        call(name, *args)

    monkeypatch.setattr(_lib, "call", note)
    return seen


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(1, 1), (5, 33), (300, 1419), (700, 40), (37, 2048), (9, 512), (2, 16384), (0, 64)])
def test_the_same_bits_and_nothing_kept(dev, calls, shape, dtype):
    x, up = activation(gen(1), *shape, dtype=dtype), activation(gen(2), *shape, dtype=dtype)
    w = torch.rand(shape[-1], generator=gen(3), device="cuda")
    leaves = [t.clone().requires_grad_(True) for t in (x, up, w)]
    recorded = [fm.swiglu_8bit(leaves[0], leaves[1]), fm.rmsnorm_8bit(leaves[0], leaves[2], 1e-5)]
    assert all(t.requires_grad for t in recorded) and all(not nulls for _, nulls in calls)
    calls.clear()
    plain = [fm.swiglu_8bit(x, up), fm.rmsnorm_8bit(x, w, 1e-5)]
    with torch.no_grad():
        quiet = [fm.swiglu_8bit(leaves[0], leaves[1]), fm.rmsnorm_8bit(leaves[0], leaves[2], 1e-5)]
    for got in (plain, quiet):
        for a, b in zip(got, recorded):
            assert torch.equal(a, b) and not a.requires_grad
    # the payloads' and codes' addresses, and rstd's, are null
    assert calls == ([("fm_act8_swiglu", [9, 10, 11, 12]), ("fm_act8_rmsnorm", [10, 12, 14])] * 2 if shape[0] else [])


def test_memory_of_an_evaluation(dev):
    x = activation(gen(4), 4096, 4096)
    norm = fm.RMSNorm(4096, checkpoint_8bit=True).cuda()
    for f, out in ((lambda: norm(x), x.numel()), (lambda: fm.swiglu_8bit(x), x.numel() // 2)):
        with torch.no_grad():
            f()
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            y = f()
        assert torch.cuda.max_memory_allocated() - before <= 2 * out + 4096
        del y


def test_layer_without_gradients(dev, calls):
    """The layer's pre-norm: outputs of the recorded forward, bit for bit."""
    layer, p = layer_of("none", 512, 128, 8, 2, 5, True, pre_norm=True, shared=128)
    x = rand(torch.Generator().manual_seed(6), 300, 512)
    out, aux = layer(x)
    calls.clear()
    with torch.no_grad():
        again, aux2 = layer(x)
    assert torch.equal(out, again) and torch.equal(aux, aux2)
    norms = [nulls for name, nulls in calls if name == "fm_act8_rmsnorm"]
    assert norms == [[10, 12, 14]] and not any("keep" in name or name == "fm_act8_compress" for name, _ in calls)
