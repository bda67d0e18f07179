"""What the few-token and int8 entries refuse before a launch, with the launch patched out (no
GPU needed): operands whose fields do not fit, and calls that would lose a gradient."""

import copy

import pytest
import torch

import nanopysche_amd as fm
from nanopysche_amd.int8 import Int8Tensor, _empty
from tests.test_host_decode_int8 import bf, int8_tensor, launched  # noqa: F401

U8 = torch.uint8
FITS = 8 * 2048   # bytes of [64, 256]


def fields(**kw):
    f = dict(data=torch.zeros(FITS, dtype=U8), scale=torch.ones(64), rows=64, cols=256)
    f.update(kw)
    return f


WRONG_FIELDS = [
    (ValueError, "contiguous bytes", dict(data=torch.zeros(10, dtype=U8))),
    (ValueError, "contiguous bytes", dict(data=torch.zeros(FITS - 1, dtype=U8))),
    (ValueError, "contiguous bytes", dict(data=torch.zeros(2 * FITS, dtype=U8)[::2])),
    (ValueError, "contiguous bytes", dict(data=torch.zeros(1, dtype=U8).expand(FITS))),
    (TypeError, "uint8", dict(data=torch.zeros(FITS, dtype=torch.int8))),
    (TypeError, "uint8", dict(data=FITS)),
    (ValueError, "scale must be", dict(scale=torch.ones(1))),
    (ValueError, "scale must be", dict(scale=torch.ones(63))),
    (ValueError, "scale must be", dict(scale=torch.ones(64, 1))),
    (ValueError, "scale must be", dict(scale=torch.ones(128)[::2])),
    (ValueError, "scale must be", dict(scale=torch.ones(64, device="meta"))),
    (TypeError, "float32", dict(scale=torch.ones(64, dtype=torch.float16))),
    (TypeError, "float32", dict(scale=None)),
]


@pytest.mark.parametrize("error,match,wrong", WRONG_FIELDS + [
    (ValueError, "contiguous bytes", dict(rows=65, scale=torch.ones(65))),
    (ValueError, "contiguous bytes", dict(cols=257)),
    (ValueError, "rows", dict(rows=-1)),
    (ValueError, "rows", dict(rows=64.0)),
    (ValueError, "rows", dict(rows=2 ** 31)),
    (ValueError, "columns", dict(cols=0)),
    (ValueError, "columns", dict(cols=131072)),
])
def test_a_tensor_whose_fields_do_not_fit_is_refused(error, match, wrong):
    with pytest.raises(error, match=match):
        Int8Tensor(**fields(**wrong))


@pytest.mark.parametrize("error,match,wrong", WRONG_FIELDS)
def test_a_field_is_replaced_only_by_one_that_fits(error, match, wrong):
    t = Int8Tensor(**fields())
    before = dict(t.__dict__)
    with pytest.raises(error, match=match):
        for name, value in wrong.items():
            setattr(t, name, value)
    assert all(t.__dict__[n] is v for n, v in before.items())


def test_what_fits_is_accepted(launched):  # noqa: F811
    t = Int8Tensor(**fields())
    t.scale = t.scale * 2
    t.scale *= 2
    t.data = torch.zeros(2 * FITS, dtype=U8)   # room behind the payload is not read
    assert torch.all(t.scale == 4) and t.shape == (64, 256)
    for name in ("rows", "cols"):
        with pytest.raises(AttributeError, match="do not change"):
            setattr(t, name, 16)
    for u in (copy.copy(t), copy.deepcopy(t)):
        assert u.shape == t.shape and torch.equal(u.scale, t.scale)
    assert Int8Tensor(torch.empty(0, dtype=U8), torch.empty(0), 0, 5).shape == (0, 5)
    e = _empty(33, 129, "cpu")   # made without the checks, which it passes
    assert Int8Tensor(e.data, e.scale, e.rows, e.cols) is not e and e.data.numel() == 3 * 2 * 2048
    with pytest.raises(ValueError):
        e.scale = torch.ones(32)
    fm.int8_linear(bf(3, 256), t)
    assert launched == ["fm_int8_linear"]


WRONG_EXPERTS = [
    (ValueError, "transposed", dict(w2=int8_tensor(4 * 128, 256))),   # as the expert block stores it
    (ValueError, "transposed", dict(w3=int8_tensor(16, 256))),
    (ValueError, "transposed", dict(w1=int8_tensor(4 * 256, 256))),
    (ValueError, "transposed", dict(w1=int8_tensor(4 * 128, 384))),
    (ValueError, "num_experts", dict(num_experts=0)),
    (ValueError, "num_experts", dict(num_experts=3)),
    (ValueError, "num_experts", dict(num_experts=4.0)),
    (ValueError, "transposed", dict(num_experts=8)),
    (TypeError, "Int8Tensor", dict(w3=torch.zeros(4 * 128, 256))),
    (ValueError, "one device", dict(w2=Int8Tensor(torch.zeros(4 * 256 * 128, dtype=U8, device="meta"),
                                                  torch.ones(4 * 256, device="meta"), 4 * 256, 128))),
]


def experts(**kw):
    f = dict(w1=int8_tensor(4 * 128, 256), w2=int8_tensor(4 * 256, 128), w3=int8_tensor(4 * 128, 256), num_experts=4)
    f.update(kw)
    return f


@pytest.mark.parametrize("error,match,wrong", WRONG_EXPERTS + [
    (ValueError, "multiples of 128", dict(w1=int8_tensor(4 * 64, 256), w2=int8_tensor(4 * 256, 64), w3=int8_tensor(4 * 64, 256))),
    (ValueError, "multiples of 128", dict(w1=int8_tensor(4 * 128, 192), w2=int8_tensor(4 * 192, 128), w3=int8_tensor(4 * 128, 192))),
    (ValueError, "transposed", dict(w1=int8_tensor(0, 256), w3=int8_tensor(0, 256))),
])
def test_experts_that_do_not_fit_each_other_are_refused(error, match, wrong):
    with pytest.raises(error, match=match):
        fm.Int8Experts(**experts(**wrong))


@pytest.mark.parametrize("error,match,wrong", WRONG_EXPERTS)
def test_experts_are_replaced_only_by_ones_that_fit(error, match, wrong):
    e = fm.Int8Experts(**experts())
    before = dict(e.__dict__)
    with pytest.raises(error, match=match):
        for name, value in wrong.items():
            setattr(e, name, value)
    assert all(e.__dict__[n] is v for n, v in before.items())
    e.label = "layer 3"   # a program's own attribute
    e.w1 = int8_tensor(4 * 128, 256)
    assert e.w1 is not before["w1"] and (e.hidden_size, e.d_model) == (128, 256)
