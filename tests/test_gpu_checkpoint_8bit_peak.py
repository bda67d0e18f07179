"""Peak memory with ``checkpoint_8bit``: the forward holds at once what one of its kernels reads and writes and what is kept, and the
backward less than without it."""

import pytest
import torch

from nanopysche_amd.flow_moe import _SLICE_BYTES
from tests.test_gpu_checkpoint_8bit import layer_of, rand

pytestmark = pytest.mark.gpu


def peaks(recipe, eight, T, D, H, E, K):
    layer, p = layer_of(recipe, D, H, E, K, 3, eight, pre_norm=True)
    x, go = rand(torch.Generator().manual_seed(4), T, D).requires_grad_(True), rand(torch.Generator().manual_seed(5), T, D, std=1e-2)
    one = torch.ones((), device="cuda")
    res = None
    for _ in range(2):   # the first step builds the weights' operands
        for t in (x, *p.values()):
            t.grad = None
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out, aux = layer(x)
        forward = torch.cuda.max_memory_allocated() - before
        torch.cuda.reset_peak_memory_stats()
        torch.autograd.backward([out, aux], [go, one])
        res = forward, torch.cuda.max_memory_allocated() - before
        del out, aux
    return res


@pytest.mark.parametrize("recipe", ["none", "flow_moe", "blockwise", "mxfp8"])
@pytest.mark.parametrize("T,D,H,E,K", [(8192, 2048, 1408, 8, 2), (4096, 1024, 3584, 4, 1), (4096, 1024, 512, 16, 4)])
def test_peak_of_a_step(dev, recipe, T, D, H, E, K):
    _, backward = peaks(recipe, False, T, D, H, E, K)
    forward8, backward8 = peaks(recipe, True, T, D, H, E, K)
    assert backward8 < backward
    R = (T * K + E * 127) // 128 * 128 + 128
    kept, op = 33 / 32, 2 if recipe == "none" else 33 / 32   # bytes of a value kept, and of one of a product's operands (with its scales)
    products = (R * (op * D + 4 * H + 2 * D),                              # gate|up of the tokens' rows; the outputs' room is there already
                R * (4 * H + 2 * H * kept + op * H + 2 * D),               # h, and gate|up kept, of gate|up; the outputs
                R * (2 * H * kept + 2 * D + D * kept) + T * D * (2 + kept))   # the outputs' sum and their 8 bits, the tokens' 8 bits
    # a product of fewer tiles than CUs is cut along K, a 256 KiB partial for each CU's slice
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    partials = cus * _SLICE_BYTES if -(-R // 256) * (D // 256) < cus else 0
    norm = T * D * (2 + kept)   # the normalised tokens, and the norm's own
    assert forward8 <= max(products) + partials + norm + T * (16 * E + 64 * K) + (4 << 20)   # the router's, and the allocator's blocks of 2 MiB
