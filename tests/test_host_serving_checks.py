"""What the few-token and int8 entries refuse before a launch, with the launch patched out (no
GPU needed): operands whose fields do not fit, and calls that would lose a gradient."""

import copy

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import nanopysche_amd as fm
from nanopysche_amd import _lib
from nanopysche_amd.decode import MAX_DECODE_DIM, MAX_DECODE_MATRIX, MAX_DECODE_TOKENS, MAX_DECODE_TOP_K
from nanopysche_amd.int8 import Int8Tensor, _empty
from tests.test_host_decode_int8 import IDX, bf, int8_experts, int8_tensor, launched  # noqa: F401

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


def plan_of(rows, E):
    """A plan of one token, as far as the checks read it."""
    i32 = torch.zeros(rows, dtype=torch.int32)
    return fm.RoutingPlan(1, 1, E, rows, i32[:E], torch.zeros(E + 1, dtype=torch.int32), i32[:1], i32, i32[:1], i32[:E])


def learned(t):
    t.scale.requires_grad_()
    return t


def learned_experts(name, E=4, H=128, D=256):
    ex = int8_experts(E, H, D)
    learned(getattr(ex, name))
    return ex


Q = torch.zeros(512, 256, dtype=torch.int8)
USES_OF_SCALES = {
    "from_int8": lambda: Int8Tensor.from_int8(Q[:3], torch.ones(3, requires_grad=True)),
    "experts_from_int8": lambda: fm.Int8Experts.from_int8(Q, torch.ones(512), Q, torch.ones(4, 256, requires_grad=True), Q,
                                                          torch.ones(512), 4),
    "dequantize": lambda: learned(int8_tensor(3, 100)).dequantize(),
    "matmul_a": lambda: fm.int8_matmul(learned(int8_tensor(3, 100)), int8_tensor(4, 100)),
    "matmul_b": lambda: fm.int8_matmul(int8_tensor(3, 100), learned(int8_tensor(4, 100))),
    "linear": lambda: fm.int8_linear(bf(3, 100), learned(int8_tensor(4, 100))),
    "grouped_tokens": lambda: fm.int8_grouped_gemm(learned(int8_tensor(256, 128)), int8_tensor(64, 128), plan_of(256, 2)),
    "grouped_weights": lambda: fm.int8_grouped_gemm(int8_tensor(256, 128), learned(int8_tensor(64, 128)), plan_of(256, 2)),
    **{f"block_{n}_{T}": lambda n=n, T=T: fm.Int8MoECompute(learned_experts(n))(bf(T, 256), torch.ones(T, 1),
                                                                            torch.zeros(T, 1, dtype=torch.int64))
       for n in ("w1", "w2", "w3") for T in (3, 70)},
    "decode": lambda: fm.moe_decode(bf(3, 256), bf(4, 256), learned_experts("w3"), 2),
    "decode_shared": lambda: fm.moe_decode(bf(3, 256), bf(4, 256), int8_experts(4, 128, 256), 2,
                                           shared=learned_experts("w2", 1)),
    "expert_decode": lambda: fm.expert_decode(bf(3, 256), torch.ones(3, 2), IDX, learned_experts("w1"), 4),
}


@pytest.mark.parametrize("name", USES_OF_SCALES)
def test_a_scale_that_requires_a_gradient_is_refused(launched, name):  # noqa: F811
    with pytest.raises(RuntimeError, match="forward only"):
        USES_OF_SCALES[name]()
    assert launched == []
    if not name.startswith("block") or name.endswith("_3"):   # a plan's sizes come from the library, its arrays from the GPU
        with torch.no_grad():
            USES_OF_SCALES[name]()
        assert launched


def test_a_packed_scale_carries_no_gradient(launched):  # noqa: F811
    with torch.no_grad():
        t = Int8Tensor.from_int8(Q[:3], torch.ones(3, requires_grad=True))
    assert not t.scale.requires_grad
    assert fm.int8_linear(bf(3, 256), t).shape == (3, 3) and t.values().shape == (3, 256)


def dual(*shape, dtype=torch.float32):
    return fwAD.make_dual(torch.zeros(*shape, dtype=dtype), torch.ones(*shape, dtype=dtype))


def with_dual_scale(t):
    t.scale = dual(t.rows)
    return t


USES_OF_DUALS = {
    "quantise": lambda: fm.quantize_to_int8(dual(3, 100)),
    "from_int8": lambda: Int8Tensor.from_int8(Q[:3], dual(3)),
    "dequantize": lambda: with_dual_scale(int8_tensor(3, 100)).dequantize(),
    "matmul": lambda: fm.int8_matmul(int8_tensor(3, 100), with_dual_scale(int8_tensor(4, 100))),
    "matmul_bias": lambda: fm.int8_matmul(int8_tensor(3, 100), int8_tensor(4, 100), dual(4)),
    "linear": lambda: fm.int8_linear(dual(3, 100), int8_tensor(4, 100)),
    "linear_view": lambda: fm.int8_linear(dual(6, 100)[::2], int8_tensor(4, 100)),
    "grouped": lambda: fm.int8_grouped_gemm(with_dual_scale(int8_tensor(256, 128)), int8_tensor(64, 128), plan_of(256, 2)),
    "block": lambda: fm.Int8MoECompute(int8_experts(4, 128, 256))(bf(70, 256), dual(70, 1), torch.zeros(70, 1, dtype=torch.int64)),
    "expert_decode": lambda: fm.expert_decode(dual(3, 256, dtype=torch.bfloat16), torch.ones(3, 2), IDX, int8_experts(4, 128, 256), 4),
    "decode_gate": lambda: fm.moe_decode(bf(3, 256), dual(4, 256, dtype=torch.bfloat16), int8_experts(4, 128, 256), 2),
    "decode_norm": lambda: fm.moe_decode(bf(3, 256), bf(4, 256), int8_experts(4, 128, 256), 2, norm_weight=dual(256)),
    "decode_weights": lambda: fm.moe_decode(bf(3, 256), bf(4, 256), [bf(512, 256), dual(512, 256, dtype=torch.bfloat16), bf(512, 256)], 2),
}


@pytest.mark.parametrize("name", USES_OF_DUALS)
@pytest.mark.parametrize("grad", [True, False])
def test_a_forward_mode_tangent_is_refused(launched, name, grad):  # noqa: F811
    """torch.no_grad() does not stop forward-mode differentiation, so it does not silence the refusal."""
    with fwAD.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(RuntimeError, match="forward-mode"):
            USES_OF_DUALS[name]()
        assert launched == []
        fm.int8_linear(torch.zeros(3, 100), int8_tensor(4, 100))   # no tangent
        assert launched == ["fm_int8_linear"]


def test_inference_mode_takes_a_dual(launched):  # noqa: F811
    """It stops both modes, as for torch's own operations."""
    with fwAD.dual_level():
        x = dual(3, 100)
        with torch.inference_mode():
            assert fwAD.unpack_dual(x * 2).tangent is None
            fm.int8_linear(x, int8_tensor(4, 100))
    assert launched == ["fm_int8_linear"]


def unread(rows, cols):
    """An operand whose payload is never touched, so that its pages stay unmapped."""
    return Int8Tensor(torch.empty((rows + 15) // 16 * ((cols + 127) // 128) * 2048, dtype=U8), torch.ones(rows), rows, cols)


@pytest.mark.parametrize("T,D,H,K,few", [
    (64, 14336, 74880, 1, True), (64, 14336, 75008, 1, False), (1, 8320, 130944, 1, False), (64, 14336, 128, 1, True),
    (1, 14464, 128, 1, False), (65, 128, 128, 1, False), (64, 128, 128, 16, True), (64, 128, 128, 17, False)])
def test_any_number_of_tokens_of_any_expert_size(launched, T, D, H, K, few):  # noqa: F811
    """The block's tokens take the few-token kernels wherever those take the sizes, else the products."""
    ex = fm.Int8Experts(unread(H, D), unread(D, H), unread(H, D), 1)
    out = fm.Int8MoECompute(ex)(torch.zeros(T, D), torch.ones(T, K), torch.zeros(T, K, dtype=torch.int64))
    assert out.shape == (T, D)
    products = ["fm_route_sort", "fm_int8_quantize", "fm_int8_grouped_gemm", "fm_int8_quantize", "fm_int8_grouped_gemm", "fm_int8_combine"]
    assert launched == (["fm_decode_experts"] if few else products)
    assert (_lib.load().fm_decode_workspace_bytes(T, D, K, 1, H, 0) >= 0) == few


def test_the_few_token_limits_are_the_librarys():
    size = _lib.load().fm_decode_workspace_bytes
    for T, D, K, H in [(MAX_DECODE_TOKENS, 128, 1, 128), (1, MAX_DECODE_DIM, 1, 128), (1, 128, MAX_DECODE_TOP_K, 128),
                       (1, 1024, 1, MAX_DECODE_MATRIX // 1024 - 128)]:
        assert size(T, D, K, 1, H, 0) >= 0
    for T, D, K, H in [(MAX_DECODE_TOKENS + 1, 128, 1, 128), (1, MAX_DECODE_DIM + 128, 1, 128), (1, 128, MAX_DECODE_TOP_K + 1, 128),
                       (1, 1024, 1, MAX_DECODE_MATRIX // 1024)]:
        assert size(T, D, K, 1, H, 0) == -1
