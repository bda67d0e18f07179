"""The balance loss where the cut of a batch into pieces changes: rows of eight and of sixteen values a lane under pieces of four and
sixteen waves.  Bounds as in test_gpu_balance.py."""

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
