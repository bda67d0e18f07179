"""What the 8-bit activations and the balance loss refuse before a launch, and the sizes that they compute on the
host, with the launch patched out (no GPU needed)."""

import ctypes as C

import pytest
import torch

import nanopysche_amd as fm
from nanopysche_amd import _lib
from nanopysche_amd.act8 import MAX_ACT8_COLS, MAX_ACT8_NORM, Activation8, _bytes
from nanopysche_amd.balance import MAX_BALANCE_EXPERTS
from tests.test_host_decode_int8 import launched  # noqa: F401

BF, F32, U8 = torch.bfloat16, torch.float32, torch.uint8


def act(*shape, dtype=BF):
    n = 1
    for d in shape[:-1]:
        n *= d
    return Activation8(torch.zeros(_bytes(n, shape[-1]), dtype=U8), shape, dtype)


# ==================================================================== format ====
def test_sizes():
    assert _bytes(3, 32) == 99 and _bytes(3, 33) == 198 and _bytes(0, 7) == 0 and _bytes(2, 1) == 66
    t = act(2, 5, 40)
    assert (t.rows, t.cols, t.pitch, t.nbytes) == (10, 40, 64, 660) and t.shape == (2, 5, 40) and t.dtype == BF
    q, codes, ld_q, ld_c = t.at()
    assert codes - q == 640 and (ld_q, ld_c) == (64, 2)


@pytest.mark.parametrize("error,match,data", [
    (ValueError, "contiguous bytes", torch.zeros(10, dtype=U8)),
    (ValueError, "contiguous bytes", torch.zeros(659, dtype=U8)),
    (ValueError, "contiguous bytes", torch.zeros(1320, dtype=U8)[::2]),
    (ValueError, "contiguous bytes", torch.zeros(1, dtype=U8).expand(660)),
    (ValueError, "8-byte", torch.zeros(700, dtype=U8)[1:]),
    (TypeError, "uint8", torch.zeros(660, dtype=torch.int8)),
    (TypeError, "uint8", None),
])
def test_data_that_does_not_fit_is_refused(error, match, data):
    with pytest.raises(error, match=match):
        Activation8(data, (2, 5, 40))
    t = act(2, 5, 40)
    before = t.data
    with pytest.raises(error, match=match):
        t.data = data
    assert t.data is before
    t.data = torch.zeros(800, dtype=U8)   # room behind is not read


def test_fields_stay():
    t = act(4, 64)
    for name in ("shape", "dtype", "device", "rows", "cols", "pitch"):
        with pytest.raises(AttributeError):
            setattr(t, name, None)
    for shape in ((), (3, 0), (3, MAX_ACT8_COLS + 1)):
        with pytest.raises(ValueError):
            Activation8(torch.zeros(0, dtype=U8), shape)
    with pytest.raises(TypeError):
        Activation8(torch.zeros(33, dtype=U8), (1, 32), torch.float16)


def test_compress_refuses(launched):  # noqa: F811
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        fm.compress_activation(torch.zeros(2, 32, dtype=torch.float16))
    with pytest.raises(ValueError, match="dimension"):
        fm.compress_activation(torch.zeros((), dtype=BF))
    with pytest.raises(ValueError, match="columns"):
        fm.compress_activation(torch.zeros(3, 0, dtype=BF))
    with pytest.raises(ValueError, match="columns"):
        fm.compress_activation(torch.zeros(1, dtype=BF).expand(1, MAX_ACT8_COLS + 1))
    t = act(4, 64)
    with pytest.raises(TypeError, match="int32"):
        t.restore_rows(torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="1-D"):
        t.restore_rows(torch.zeros(3, 1, dtype=torch.int32))
    with pytest.raises(TypeError, match="out_dtype"):
        t.restore(torch.float16)
    assert launched == []


def test_no_gpu_is_an_error():
    if torch.cuda.is_available():
        pytest.skip("for machines without a GPU")
    for call in (lambda: fm.compress_activation(torch.zeros(2, 32, dtype=BF)), lambda: fm.swiglu_8bit(torch.zeros(2, 32, dtype=BF)),
                 lambda: fm.rmsnorm_8bit(torch.zeros(2, 32, dtype=BF), torch.ones(32)),
                 lambda: fm.balance_loss(torch.zeros(2, 4), torch.zeros(2, 1, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()


# ============================================================ SwiGLU, RMSNorm ====
def test_swiglu_refuses(launched):  # noqa: F811
    z = torch.zeros
    with pytest.raises(ValueError, match="even"):
        fm.swiglu_compress(z(2, 33, dtype=BF))
    with pytest.raises(ValueError, match="alike"):
        fm.swiglu_compress(z(2, 32, dtype=BF), z(2, 31, dtype=BF))
    with pytest.raises(ValueError, match="alike"):
        fm.swiglu_compress(z(2, 32, dtype=BF), z(2, 32))
    with pytest.raises(TypeError):
        fm.swiglu_compress(z(2, 32, dtype=torch.float16))
    with pytest.raises(ValueError, match="alike"):
        fm.swiglu_backward_8bit(z(2, 32, dtype=BF), act(2, 32), act(3, 32))
    with pytest.raises(ValueError, match="alike"):
        fm.swiglu_backward_8bit(z(2, 64, dtype=BF), act(2, 32), act(2, 32))
    with pytest.raises(TypeError):
        fm.swiglu_backward_8bit(z(2, 32, dtype=torch.float64), act(2, 32), act(2, 32))
    assert launched == []


def test_rmsnorm_refuses(launched):  # noqa: F811
    z = torch.zeros
    with pytest.raises(ValueError, match="weight must be"):
        fm.rmsnorm_compress(z(2, 32, dtype=BF), z(31))
    with pytest.raises(TypeError, match="weight"):
        fm.rmsnorm_compress(z(2, 32, dtype=BF), z(32, dtype=torch.float16))
    with pytest.raises(ValueError, match="columns"):
        fm.rmsnorm_compress(z(1, MAX_ACT8_NORM + 1, dtype=BF), z(MAX_ACT8_NORM + 1))
    with pytest.raises(ValueError, match="dy must be"):
        fm.rmsnorm_backward_8bit(z(2, 33, dtype=BF), act(2, 32), z(32), z(2))
    for rstd in (z(3), z(2, dtype=BF), z(4)[::2]):
        with pytest.raises(ValueError, match="rstd"):
            fm.rmsnorm_backward_8bit(z(2, 32, dtype=BF), act(2, 32), z(32), rstd)
    assert launched == []
    with pytest.raises(ValueError):
        fm.RMSNorm(100)
    assert fm.RMSNorm(100, checkpoint_8bit=True).weight.shape == (100,)


# ================================================================ balance loss ====
def logits(T=6, E=4):
    return torch.zeros(T, E), torch.zeros(T, 2, dtype=torch.int64)


@pytest.mark.parametrize("error,match,change", [
    (TypeError, "float32", dict(logits=torch.zeros(6, 4, dtype=BF))),
    (ValueError, "E of 1", dict(logits=torch.zeros(6, MAX_BALANCE_EXPERTS + 1))),
    (ValueError, "E of 1", dict(logits=torch.zeros(6, 0))),
    (TypeError, "int64 or int32", dict(indices=torch.zeros(6, 2))),
    (ValueError, "indices must be", dict(indices=torch.zeros(5, 2, dtype=torch.int64))),
    (ValueError, "indices must be", dict(indices=torch.zeros(6, 0, dtype=torch.int64))),
    (ValueError, "indices must be", dict(indices=torch.zeros(6, dtype=torch.int64))),
    (TypeError, "int32", dict(cu_seqlens=torch.zeros(2, dtype=torch.int64))),
    (ValueError, "cu_seqlens must be", dict(cu_seqlens=torch.zeros(2, 1, dtype=torch.int32))),
    (ValueError, "cu_seqlens must be", dict(cu_seqlens=torch.zeros(0, dtype=torch.int32))),
    (ValueError, "cu_seqlens must be", dict(cu_seqlens=torch.zeros(2 ** 20 + 1, dtype=torch.int32))),
    (TypeError, "bool", dict(token_mask=torch.ones(6))),
    (ValueError, "token_mask must be", dict(token_mask=torch.ones(5, dtype=torch.bool))),
    (ValueError, "scores", dict(scores="relu")),
])
def test_balance_refuses(launched, error, match, change):  # noqa: F811
    l, i = logits()
    args = dict(logits=l, indices=i)
    args.update(change)
    with pytest.raises(error, match=match):
        fm.balance_loss(args.pop("logits"), args.pop("indices"), **args)
    assert launched == []


def test_balance_backward_refuses(launched):  # noqa: F811
    l, _ = logits()
    state = fm.BalanceState(l, None, None, torch.zeros(6), False, 0.0, l.shape)
    for bad in (torch.zeros(2), torch.zeros((), dtype=BF)):
        with pytest.raises(TypeError, match="dloss"):
            fm.balance_backward(state, bad)
    for bad in (torch.zeros(6, 5), torch.zeros(6, 4, dtype=BF), torch.zeros(4, 6).t(), torch.zeros(1, 4).expand(6, 4)):
        with pytest.raises(ValueError, match="add_to"):
            fm.balance_backward(state, torch.zeros(()), add_to=bad)
    short = fm.BalanceState(l, None, None, torch.zeros(5), False, 0.0, l.shape)
    masked = fm.BalanceState(l, None, torch.ones(5, dtype=torch.bool), torch.zeros(6), False, 0.0, l.shape)
    borders = fm.BalanceState(l, torch.zeros(3, dtype=torch.int32), None, torch.zeros(6), False, 0.0, l.shape)
    for state in (short, masked, borders):
        with pytest.raises(ValueError, match="do not fit"):
            fm.balance_backward(state, torch.zeros(()))
    assert launched == []


# ======================================================================== C ABI ====
def test_the_library_refuses_before_a_launch():
    lib = _lib.load()
    p, err = C.c_void_p(256), lambda: lib.fm_last_error_string()

    def bad(text, rc):
        assert rc != 0 and text in err(), err()

    bad(b"bad sizes", lib.fm_act8_compress(p, 0, 4, 0, 64, p, 64, p, 2, None, None))
    bad(b"bf16 or fp32", lib.fm_act8_compress(p, 2, 4, 64, 64, p, 64, p, 2, None, None))
    bad(b"pitch", lib.fm_act8_compress(p, 0, 4, 33, 33, p, 32, p, 1, None, None))
    bad(b"null x", lib.fm_act8_compress(None, 0, 4, 64, 64, p, 64, p, 2, None, None))
    bad(b"8 bytes", lib.fm_act8_compress(p, 0, 4, 64, 64, C.c_void_p(260), 64, p, 2, None, None))
    bad(b"more rows", lib.fm_act8_restore(p, 64, p, 2, 3, 64, None, 4, p, 0, 64, None))
    bad(b"pitch below", lib.fm_act8_restore(p, 64, p, 2, 4, 64, None, 4, p, 0, 63, None))
    bad(b"payload", lib.fm_act8_swiglu(p, 64, p, 64, 0, 2, 64, p, 64, p, p, None, p, 64, 2, None))
    bad(b"pitch", lib.fm_act8_swiglu_backward(p, 64, 0, 2, 64, p, p, p, p, 64, 2, p, 63, p, 64, None))
    bad(b"D must be", lib.fm_act8_rmsnorm(p, 0, 64, 2, 16385, p, 1, 1e-6, p, 16385, p, 16416, p, 513, p, None))
    bad(b"workspace", lib.fm_act8_rmsnorm_backward(p, 64, 0, 2, 64, p, 64, p, 2, p, 1, p, p, 64, p, p, 16, None))
    need = lib.fm_balance_workspace_bytes(100, 8, 3)
    assert need > 0 and lib.fm_balance_workspace_bytes(0, 8, 0) > 0 and lib.fm_balance_workspace_bytes(100, 0, 3) == 0
    bad(b"workspace", lib.fm_balance_forward(p, 8, 100, 8, p, 1, 2, p, 3, None, 0, 0.0, p, p, p, p, None, None, p, need - 1, None))
    bad(b"one sequence", lib.fm_balance_forward(p, 8, 100, 8, p, 1, 2, None, 3, None, 0, 0.0, p, p, p, p, None, None, p, need, None))
    bad(b"E must be", lib.fm_balance_forward(p, 8, 100, 1025, p, 1, 2, p, 3, None, 0, 0.0, p, p, p, p, None, None, p, need, None))
    bad(b"sequences", lib.fm_balance_forward(p, 8, 100, 8, p, 1, 2, p, 1 << 20, None, 0, 0.0, p, p, p, p, None, None, p, 1 << 40, None))
    bad(b"multiples of 128", lib.fm_act8_swiglu_keep_quantize(p, 256, 100, 128, p, 256, p, 8, 0, p, 128, None, 0, None, None))
    bad(b"payload", lib.fm_act8_permute(p, 256, None, 8, 4, 256, p, 128, 2, 0, p, 256, None, 0, None, 0, None, 0, None, None))
    bad(b"H must be", lib.fm_act8_swiglu_quantize(p, 64, p, 2, 128, 32, 0, p, 32, None, 0, None, 0, None, 0, None, None))
    bad(b"16 bytes", lib.fm_act8_swiglu_backward_quantize(p, 256, p, 8, C.c_void_p(264), 128, 128, 128, 0, p, 256, None, 0, None, 0, None, 0, None, None))
    bad(b"16 bytes", lib.fm_act8_router_weight_grad(p, 100, p, 128, p, 4, p, 4, 2, 128, p, None))
    bad(b"pitch", lib.fm_balance_backward(p, 8, 100, 8, p, 3, None, 0, 0.0, p, p, p, p, 7, 0, None))


def test_more_slots_than_the_counts_hold_are_refused(launched):  # noqa: F811
    l, i = torch.zeros(1, 4).expand(2 ** 21, 4), torch.zeros(1, 1, dtype=torch.int32).expand(2 ** 21, 1024)
    with pytest.raises(ValueError, match=r"fewer than 2\^31 slots"):
        fm.balance_loss(l, i)
    assert launched == []
    lib, p = _lib.load(), C.c_void_p(256)
    need = lib.fm_balance_workspace_bytes(2 ** 21, 4, 1)
    assert lib.fm_balance_forward(p, 4, 2 ** 21, 4, p, 0, 1024, None, 1, None, 0, 0.0, p, p, p, p, None, None, p, need, None) != 0
    assert b"fewer than 2^31 slots" in lib.fm_last_error_string()


def test_norm_module_checks_its_size():
    for size in (0, MAX_ACT8_NORM + 1):
        with pytest.raises(ValueError, match="columns"):
            fm.RMSNorm(size, checkpoint_8bit=True)
    assert fm.RMSNorm(1000, checkpoint_8bit=True).weight.shape == (1000,)
