"""The balance loss where the cut of a batch into pieces changes: rows of eight and of sixteen values a lane under pieces of four and
sixteen waves, and batches about the size that one launch takes.  Bounds as in test_gpu_balance.py."""

import pytest
import torch

from tests.test_gpu_balance import check, gen, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E", [255, 256, 257, 260, 511, 512, 513])
@pytest.mark.parametrize("T,borders", [(20000, None), (9000, [0, 4000, 4000, 8990])])
def test_widths_of_long_sequences(dev, T, borders, E):
    logits, idx = inputs(T, E, 4, E)
    mask = torch.rand(T, generator=gen(E), device="cuda") < 0.9 if borders else None
    check(logits, idx, borders, mask, "sigmoid" if borders else "softmax", z=1e-3)


@pytest.mark.parametrize("E,T", [(8, 512), (8, 576), (8, 960), (8, 1024), (8, 1056), (8, 2048), (8, 2049), (4, 1024), (4, 2048), (4, 4096), (4, 4097),
                                 (64, 240), (64, 256), (256, 64), (256, 65), (7, 500), (7, 1000), (7, 1024), (7, 1025), (7, 2340), (60, 273)])
def test_batches_about_one_launch(dev, E, T):
    logits, idx = inputs(T, E, 2, T + E)
    check(logits, idx, z=1e-2)
    check(logits, idx.int(), [1, T // 3, T // 3, T - 1], torch.rand(T, generator=gen(T), device="cuda") < 0.8, "sigmoid")
