"""What the few-token and int8 entries refuse, before any launch (no GPU needed): the Python
checks with the launch patched out, and the library's own checks of pointers and sizes."""

import ctypes as C

import pytest
import torch

import nanopysche_amd as fm
from nanopysche_amd import _lib
from nanopysche_amd.int8 import MAX_INT8_K, Int8Tensor

BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture
def launched(monkeypatch):
    """Tensors pass for device tensors; calls are recorded, not made."""
    names = []
    monkeypatch.setattr(_lib, "call", lambda name, *a: names.append(name))
    monkeypatch.setattr(_lib, "require_device", lambda t, name="tensor": None)
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)
    return names


def bf(*shape):
    return torch.zeros(*shape, dtype=BF)


def int8_tensor(rows, cols):
    return Int8Tensor(torch.zeros((rows + 15) // 16 * ((cols + 127) // 128) * 2048, dtype=torch.uint8), torch.ones(rows),
                      rows, cols)


def int8_experts(E, H, D):
    return fm.Int8Experts(int8_tensor(E * H, D), int8_tensor(E * D, H), int8_tensor(E * H, D), E)


W = [bf(4 * 128, 256) for _ in range(3)]
IDX = torch.zeros(3, 2, dtype=torch.int64)


def decode(x=None, gate=None, experts=None, top_k=2, **kw):
    return fm.moe_decode(bf(3, 256) if x is None else x, bf(4, 256) if gate is None else gate, experts or W, top_k, **kw)


def experts_of(x=None, weights=None, indices=None, experts=None, E=4, **kw):
    return fm.expert_decode(bf(3, 256) if x is None else x, torch.ones(3, 2) if weights is None else weights,
                            IDX if indices is None else indices, experts or W, E, **kw)


def test_what_is_accepted(launched):
    r = decode(bf(1, 3, 256))
    assert r.out.shape == (1, 3, 256) and r.weights.shape == (3, 2) and r.indices.dtype == torch.int64
    decode(torch.zeros(3, 256), gate_bias=bf(4), score_bias=torch.zeros(4), norm_weight=bf(256),
           shared=[bf(128, 256) for _ in range(3)])
    decode(experts=int8_experts(4, 128, 256), shared=int8_experts(1, 384, 256))
    assert experts_of(indices=IDX.int()).dtype == BF
    assert launched == ["fm_moe_decode"] * 3 + ["fm_decode_experts"]
    assert decode(bf(0, 256)).out.shape == (0, 256)
    assert experts_of(bf(0, 256), torch.ones(0, 2), IDX[:0]).shape == (0, 256)
    assert launched == ["fm_moe_decode"] * 3 + ["fm_decode_experts"]


@pytest.mark.parametrize("error,match,call", [
    (ValueError, "at most 64 tokens", lambda: decode(bf(65, 256))),
    (ValueError, "multiple of 128", lambda: decode(bf(3, 192), bf(4, 192))),
    (ValueError, "multiple of 128", lambda: decode(bf(1, 14464), bf(4, 14464))),
    (TypeError, "bfloat16 or float32", lambda: decode(torch.zeros(3, 256, dtype=torch.float16))),
    (ValueError, "gate_weight", lambda: decode(gate=bf(4, 128))),
    (ValueError, "gate_bias", lambda: decode(gate_bias=bf(3))),
    (ValueError, "score_bias", lambda: decode(score_bias=torch.zeros(5))),
    (ValueError, "norm_weight", lambda: decode(norm_weight=bf(128))),
    (ValueError, "top_k", lambda: decode(top_k=0)),
    (ValueError, "top_k", lambda: decode(gate=bf(32, 256), experts=[bf(32 * 128, 256)] * 3, top_k=17)),
    (ValueError, "top_k 5 of 4", lambda: decode(top_k=5)),
    (KeyError, "tanh", lambda: decode(gating="tanh")),
    (ValueError, "normalize", lambda: decode(normalize_expert_weights="l1")),
    (ValueError, r"E \* H", lambda: decode(experts=[bf(4 * 128, 128)] * 3)),
    (ValueError, r"E \* H", lambda: decode(experts=[bf(513, 256)] * 3)),
    (ValueError, r"E \* H", lambda: decode(experts=[W[0], W[0], bf(256, 256)])),
    (ValueError, "hidden size", lambda: decode(experts=[bf(4 * 64, 256)] * 3)),
    (TypeError, "bfloat16", lambda: decode(experts=[torch.zeros(512, 256)] * 3)),
    (TypeError, "Int8Experts", lambda: decode(experts=5)),
    (ValueError, "contiguous", lambda: decode(experts=[bf(256, 512).t()] * 3)),
    (ValueError, "16-byte", lambda: decode(experts=[bf(512 * 256 + 1)[1:].view(512, 256)] * 3)),
    (ValueError, "both", lambda: decode(shared=int8_experts(1, 128, 256))),
    (ValueError, "of width", lambda: decode(experts=int8_experts(4, 128, 128))),
    (ValueError, "int8 weights of 8 experts", lambda: decode(experts=int8_experts(8, 128, 256))),
    (RuntimeError, "forward only", lambda: decode(bf(3, 256).requires_grad_())),
    (RuntimeError, "forward only", lambda: decode(experts=[W[0], W[1], bf(512, 256).requires_grad_()])),
    (ValueError, r"\[T, K\]", lambda: experts_of(weights=torch.ones(2, 2))),
    (ValueError, r"\[T, K\]", lambda: experts_of(weights=torch.ones(2, 3))),
    (ValueError, r"\[T, K\]", lambda: experts_of(indices=IDX[:2])),
    (TypeError, "int64 or int32", lambda: experts_of(indices=IDX.float())),
    (ValueError, "experts", lambda: experts_of(E=0)),
])
def test_decode_refusals(launched, error, match, call):
    with pytest.raises(error, match=match):
        call()
    assert launched == []


@pytest.mark.parametrize("error,match,call", [
    (TypeError, "bfloat16 or float32", lambda: fm.quantize_to_int8(torch.zeros(2, 4, dtype=torch.float16))),
    (ValueError, "columns", lambda: fm.quantize_to_int8(bf(2, 0))),
    (ValueError, "columns", lambda: fm.quantize_to_int8(torch.empty(1, MAX_INT8_K + 1, dtype=BF))),
    (RuntimeError, "forward only", lambda: fm.quantize_to_int8(torch.zeros(2, 4, requires_grad=True))),
    (TypeError, "int8", lambda: Int8Tensor.from_int8(torch.zeros(2, 4), torch.ones(2))),
    (ValueError, "scale", lambda: Int8Tensor.from_int8(torch.zeros(2, 4, dtype=torch.int8), torch.ones(3))),
    (ValueError, "columns", lambda: fm.int8_matmul(int8_tensor(3, 100), int8_tensor(4, 101))),
    (ValueError, "bias", lambda: fm.int8_matmul(int8_tensor(3, 100), int8_tensor(4, 100), torch.zeros(3))),
    (TypeError, "out_dtype", lambda: fm.int8_matmul(int8_tensor(3, 100), int8_tensor(4, 100), out_dtype=torch.float16)),
    (ValueError, "columns", lambda: fm.int8_linear(bf(3, 99), int8_tensor(4, 100))),
    (RuntimeError, "forward only", lambda: fm.int8_linear(bf(3, 100).requires_grad_(), int8_tensor(4, 100))),
    (TypeError, "out_dtype", lambda: int8_tensor(3, 100).dequantize(torch.float64)),
    (ValueError, "multiples of 128", lambda: fm.Int8Experts.quantize(*[bf(4 * 64, 256)] * 3, 4)),
    (ValueError, r"E \* H", lambda: fm.Int8Experts.quantize(bf(512, 256), bf(512, 256), bf(512, 128), 4)),
    (ValueError, "s2", lambda: fm.Int8Experts.from_int8(*[torch.zeros(512, 256, dtype=torch.int8), torch.ones(512)] * 3, 4)),
    (ValueError, "columns", lambda: fm.Int8MoECompute(int8_experts(4, 128, 256))(bf(70, 128), torch.ones(70, 2), IDX)),
    (ValueError, r"\[T, K\]", lambda: fm.Int8MoECompute(int8_experts(4, 128, 256))(bf(70, 256), torch.ones(70, 2), IDX)),
    (ValueError, "num_local_experts", lambda: fm.Int8MoECompute(int8_experts(4, 128, 256))(bf(3, 256), torch.ones(3, 2), IDX, 0, 5)),
    (RuntimeError, "forward only",
     lambda: fm.Int8MoECompute(int8_experts(4, 128, 256))(bf(3, 256), torch.ones(3, 2, requires_grad=True), IDX)),
])
def test_int8_refusals(launched, error, match, call):
    with pytest.raises(error, match=match):
        call()
    assert launched == []


def test_cpu_tensors_are_refused():
    """No CPU path: the first check of every entry."""
    for call in (lambda: decode(), lambda: experts_of(), lambda: fm.quantize_to_int8(bf(2, 4)),
                 lambda: fm.int8_linear(bf(2, 100), int8_tensor(4, 100)),
                 lambda: fm.int8_matmul(int8_tensor(2, 100), int8_tensor(4, 100)),
                 lambda: Int8Tensor.from_int8(torch.zeros(2, 4, dtype=torch.int8), torch.ones(2)),
                 lambda: fm.Int8MoECompute(int8_experts(4, 128, 256))(bf(3, 256), torch.ones(3, 2), IDX)):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()


def test_layer_decode_refusals(launched):
    layer = fm.FP8FlowMoELayer(fm.FP8FlowMoEConfig(), 256, 128, 4, 2, shared_hidden_size=128)
    with pytest.raises(RuntimeError, match="set_weights"):
        layer.decode(bf(3, 256))
    layer.set_weights(bf(4, 256), None, *W, shared=[bf(128, 256)] * 3)
    with pytest.raises(ValueError, match="shared expert's int8"):
        layer.decode(bf(3, 256), experts=int8_experts(4, 128, 256))
    plain = fm.FP8FlowMoELayer(fm.FP8FlowMoEConfig(), 256, 128, 4, 2)
    plain.set_weights(bf(4, 256), None, *W)
    with pytest.raises(ValueError, match="no shared expert"):
        plain.decode(bf(3, 256), shared=int8_experts(1, 128, 256))
    assert launched == []
    layer.decode(bf(3, 256))
    plain.decode(bf(3, 256), experts=int8_experts(4, 128, 256))
    assert launched == ["fm_moe_decode"] * 2


P = C.c_void_p(256)   # passes for an aligned pointer: every call below ends before a launch


def refuses(name, match, *args):
    rc = getattr(_lib.load(), name)(*args)
    assert rc != 0 and match in _lib.load().fm_last_error_string(), _lib.load().fm_last_error_string()


def test_library_refuses_decode_sizes():
    w = _lib.FmDecodeWeights(0, 128, 256, 256, 256)
    size = _lib.load().fm_decode_workspace_bytes
    n = size(3, 256, 2, 4, 128, 0)
    assert n > 0
    for T, D, K, E, H, Hs in [(0, 256, 2, 4, 128, 0), (65, 256, 2, 4, 128, 0), (3, 200, 2, 4, 128, 0), (3, 14464, 2, 4, 128, 0),
                              (3, 256, 0, 4, 128, 0), (3, 256, 17, 40, 128, 0), (3, 256, 2, 1025, 128, 0), (3, 256, 2, 4, 100, 0),
                              (3, 256, 2, 4, 128, 100), (3, 14336, 2, 4, 1 << 20, 0), (3, 8192, 2, 4, 128, 131072)]:
        assert size(T, D, K, E, H, Hs) == -1

    def run(match, x=P, ld=256, T=3, D=256, K=2, E=4, w=w, ws=None, out_dtype=0, ld_out=256, work=P, nbytes=n, idx=P):
        refuses("fm_decode_experts", match, x, None, ld, T, D, P, idx, 1, K, 0, E, C.byref(w), None if ws is None else C.byref(ws),
                P, out_dtype, ld_out, work, nbytes, None)

    run(b"null", idx=None)
    run(b"tokens", T=65)
    run(b"multiples of 128", D=192)
    run(b"16-byte", x=C.c_void_p(264))
    run(b"16-byte", ld=252)
    run(b"workspace of", nbytes=n - 1)
    run(b"output", ld_out=255)
    run(b"output", out_dtype=2)
    run(b"weight kind", w=_lib.FmDecodeWeights(2, 128, 256, 256, 256))
    run(b"scales", w=_lib.FmDecodeWeights(1, 128, 256, 256, 256))
    run(b"weights must be given", w=_lib.FmDecodeWeights(0, 128, 256, None, 256))
    run(b"one kind", ws=_lib.FmDecodeWeights(1, 128, 256, 256, 256, 256, 256, 256), nbytes=1 << 30)


def test_library_refuses_int8_sizes():
    refuses("fm_int8_quantize", b"null", None, 0, 3, 100, 100, None, 1, None, None, None, P, P, None)
    refuses("fm_int8_quantize", b"columns", P, 0, 3, 131072, 131072, None, 1, None, None, None, P, P, None)
    refuses("fm_int8_quantize", b"pitch", P, 0, 3, 100, 99, None, 1, None, None, None, P, P, None)
    refuses("fm_int8_quantize", b"misaligned", C.c_void_p(257), 0, 3, 100, 100, None, 1, None, None, None, P, P, None)
    refuses("fm_int8_quantize", b"bf16 or fp32", P, 2, 3, 100, 100, None, 1, None, None, None, P, P, None)
    refuses("fm_int8_pack", b"groups of a multiple", P, 2, 24, 100, 2400, 100, 1, P, None)
    refuses("fm_int8_unpack", b"bad sizes", P, P, 3, 100, P, 3, 100, None)
    refuses("fm_int8_matmul", b"K < 131072", P, P, 3, P, P, 4, 131072, None, P, 0, 4, None)
    refuses("fm_int8_matmul", b"pitch", P, P, 3, P, P, 4, 100, None, P, 0, 3, None)
    refuses("fm_int8_linear", b"pitch", P, 0, 3, 100, 99, P, P, 4, None, P, 0, 4, P, 1 << 20, None)
    refuses("fm_int8_linear", b"workspace", P, 0, 30, 100, 100, P, P, 4, None, P, 0, 4, P, 100, None)
    assert _lib.load().fm_int8_linear_workspace_bytes(4, 8192) == 0
    assert _lib.load().fm_int8_linear_workspace_bytes(5, 8192) == 16 * 8192 + 64
    assert _lib.load().fm_int8_linear_workspace_bytes(5, 131072) == -1
    refuses("fm_int8_grouped_gemm", b"multiples of 128", P, P, 100, P, 4, P, P, None, None, None, 64, 128, 10, P, 0, 64, None)
    refuses("fm_int8_grouped_gemm", b"multiples of 128", P, P, 128, P, 4, P, P, None, None, None, 64, 100, 10, P, 0, 64, None)
    refuses("fm_int8_grouped_gemm", b"1024 experts", P, P, 128, P, 1025, P, P, None, None, None, 64, 128, 10, P, 0, 64, None)
    refuses("fm_int8_grouped_gemm", b"SwiGLU", P, P, 128, P, 4, P, P, P, P, P, 64, 128, 10, P, 1, 64, None)
    refuses("fm_int8_grouped_gemm", b"SwiGLU", P, P, 128, P, 4, P, P, P, P, None, 128, 128, 10, P, 1, 128, None)
    refuses("fm_int8_combine", b"bad sizes", P, 6, P, P, 3, 2, P, 0, None)
