"""A MoE layer for a few tokens (a decoding step): ``MoEBase.forward`` of the
reference (``model/moe.py:1338-1393``, with the router of ``:133-184`` and the
optional RMSNorm and shared expert around it) at 1 to 64 tokens, forward only.

The layer built for prompts permutes tokens into padded groups and runs about
ten launches; at these sizes the time is reading the reached experts' weights
once.  Here the router is one launch (two for a large gate), the next takes slices
of every reached expert's hidden units through gate, up and SwiGLU, the next
shares of them through the down product, and the last adds the shares per token.

The experts' weights are bf16 as the layer holds them, or int8 with a scale per
output channel (``Int8Experts``), which halves the bytes; activations are not
quantised.  Sums and SwiGLU are fp32, the norm's output and h keep at least 16
bits of mantissa, and the output is rounded once: the results are nearer to the
exact ones than the layer's, which rounds to bf16 between its kernels.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
import torch.autograd.forward_ad as fwAD

from . import _lib
from .norm import DEFAULT_EPS
from .routing import _gating_code, _norm_flags

MAX_DECODE_TOKENS = 64
MAX_DECODE_DIM = 14336
MAX_DECODE_EXPERTS = 1024
MAX_DECODE_TOP_K = 16
MAX_DECODE_MATRIX = 2 ** 30   # elements of an expert's matrix are fewer


class DecodeOutput(NamedTuple):
    """out [..., D]; the router's weights [T, K] fp32 and indices [T, K] int64."""

    out: torch.Tensor
    weights: torch.Tensor
    indices: torch.Tensor


def _no_gradients(*tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("the few-token and int8 kernels are forward only: call them under torch.no_grad(), "
                                   "or use FP8FlowMoELayer / FP8FlowMoECompute to train")
    # tangents live inside a dual level, whether or not gradients are recorded
    if fwAD._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if t is not None and fwAD.unpack_dual(t).tangent is not None:
                raise RuntimeError("the few-token and int8 kernels are forward only: they carry no forward-mode tangents")


def _same_device(x: torch.Tensor, **tensors) -> None:
    index = x.get_device()
    for name, t in tensors.items():
        if t is not None and t.get_device() != index:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as bf16 rows [T, D] that start on 16-byte boundaries."""
    _lib.require_device(x, "x")
    if x.dim() < 1 or x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"x must be a bfloat16 or float32 [..., D], got {x.dtype} {tuple(x.shape)}")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if x2.dtype != torch.bfloat16:
        x2 = x2.to(torch.bfloat16)
    T, D = x2.shape
    if T > MAX_DECODE_TOKENS:
        raise ValueError(f"a decoding step takes at most {MAX_DECODE_TOKENS} tokens, got {T}")
    if D % 128 or not 0 < D <= MAX_DECODE_DIM:
        raise ValueError(f"d_model must be a multiple of 128 up to {MAX_DECODE_DIM}, got {D}")
    ld = x2.stride(0) if T > 1 else D
    if x2.stride(1) != 1 or ld % 8 or not D <= ld <= 1 << 23 or x2.data_ptr() % 16:
        x2 = x2.contiguous()
        x2 = x2 if x2.data_ptr() % 16 == 0 else x2.clone()
    return x2


def _pitch(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]   # a single row's stride says nothing


def _weights_struct(experts, num_experts: int, x: torch.Tensor, what: str) -> _lib.FmDecodeWeights:
    """The kernels' view of (w1, w2, w3) or Int8Experts (the caller keeps the tensors)."""
    from .int8 import Int8Experts

    D = x.shape[1]
    if isinstance(experts, Int8Experts):
        if experts.num_experts != num_experts or experts.d_model != D:
            raise ValueError(f"{what}: int8 weights of {experts.num_experts} experts of width {experts.d_model}, "
                             f"expected {num_experts} of width {D}")
        _same_device(x, **{what: experts.w1.data})
        w1, w2, w3 = experts.w1, experts.w2, experts.w3
        _no_gradients(w1.scale, w2.scale, w3.scale)
        return _lib.FmDecodeWeights(_lib.DECODE_INT8, experts.hidden_size, w1.data.data_ptr(), w2.data.data_ptr(),
                                    w3.data.data_ptr(), w1.scale.data_ptr(), w2.scale.data_ptr(), w3.scale.data_ptr())
    try:
        w1, w2, w3 = experts
    except (TypeError, ValueError):
        raise TypeError(f"{what} must be (w1, w2, w3) or Int8Experts") from None
    _no_gradients(w1, w2, w3)
    shape = w1.shape
    if len(shape) != 2 or shape[1] != D or w2.shape != shape or w3.shape != shape or shape[0] % num_experts:
        raise ValueError(f"{what}: w1, w2, w3 must be [E * H, D] with E = {num_experts} and D = {D}, got {tuple(shape)}, "
                         f"{tuple(w2.shape)}, {tuple(w3.shape)}")
    H = shape[0] // num_experts
    if H % 128 or not H:
        raise ValueError(f"{what}: hidden size must be a multiple of 128, got {H}")
    at = []
    for t in (w1, w2, w3):
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{what}: weights must be bfloat16 (or Int8Experts), got {t.dtype}")
        at.append(t.data_ptr())
        if at[-1] % 16 or not t.is_contiguous():
            raise ValueError(f"{what}: weights must be contiguous, on 16-byte boundaries")
    _same_device(x, w1=w1, w2=w2, w3=w3)
    return _lib.FmDecodeWeights(_lib.DECODE_BF16, H, *at)


def _both(experts, num_experts, shared, x):
    w = _weights_struct(experts, num_experts, x, "experts")
    ws = None if shared is None else _weights_struct(shared, 1, x, "shared")
    if ws is not None and ws.kind != w.kind:
        raise ValueError("experts and shared must both be bf16 or both Int8Experts")
    return w, ws


def _workspace(size: str, x, K, num_experts, w, ws):
    T, D = x.shape
    nbytes = _lib.size_of(size, T, D, K, num_experts, w.H, 0 if ws is None else ws.H)
    if nbytes < 0:
        raise ValueError(f"sizes outside the few-token kernels' range: {T} tokens, D {D}, hidden {w.H}, "
                         f"{num_experts} experts, top {K}")
    return torch.empty(nbytes, dtype=torch.uint8, device=x.device), nbytes


def _dtype_code(dtype: torch.dtype) -> int:
    return _lib.DTYPE_F32 if dtype == torch.float32 else _lib.DTYPE_BF16


def _check_routing(T: int, num_experts: int, top_k: int) -> None:
    if not 1 <= num_experts <= MAX_DECODE_EXPERTS:
        raise ValueError(f"1 to {MAX_DECODE_EXPERTS} experts, got {num_experts}")
    if not 1 <= top_k <= MAX_DECODE_TOP_K:
        raise ValueError(f"top_k must be 1 to {MAX_DECODE_TOP_K}, got {top_k}")


def expert_decode(x: torch.Tensor, weights: torch.Tensor, indices: torch.Tensor, experts, num_experts: int,
                  expert_offset: int = 0, shared=None) -> torch.Tensor:
    """sum_k weights[t, k] expert_{indices[t, k]}(x[t]) (+ shared(x[t])) for 1 to 64
    tokens, as ``FP8FlowMoECompute`` computes it for any number (reference
    ``model/moe.py:1542-1596``), forward only.

    x [..., D] bf16 or fp32 (taken as bf16); weights [..., K] and indices [..., K]
    (int32 or int64) as a router gives them; ``experts`` the (w1, w2, w3)
    [E * H, D] bf16 parameters or ``Int8Experts``; ``shared`` likewise for one
    expert.  Index i means expert i - ``expert_offset`` of the ``num_experts`` held
    here; slots of experts elsewhere add nothing.  Returns x's shape and dtype."""
    x2 = _rows(x)
    T = x2.shape[0]
    _no_gradients(x, weights)
    K = indices.shape[-1] if indices.dim() else 0
    _check_routing(T, num_experts, K)
    if indices.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"indices must be int64 or int32, got {indices.dtype}")
    if indices.numel() != T * K or weights.numel() != T * K or weights.shape[-1] != K:
        raise ValueError(f"weights {tuple(weights.shape)} and indices {tuple(indices.shape)} must be [T, K] for {T} tokens")
    _same_device(x2, weights=weights, indices=indices)
    w = weights.reshape(T, K).to(torch.float32).contiguous()
    idx = indices.reshape(T, K).contiguous()
    if T == 0:
        return torch.empty_like(x)
    with _lib.on_device_of(x2):
        ww, ws = _both(experts, num_experts, shared, x2)
        work, nbytes = _workspace("fm_decode_workspace_bytes", x2, K, num_experts, ww, ws)
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        _lib.call("fm_decode_experts", x2.data_ptr(), None, _pitch(x2), T, x2.shape[1], w.data_ptr(), idx.data_ptr(),
                  int(idx.dtype == torch.int64), K, int(expert_offset), num_experts, ww, ws, out.data_ptr(),
                  _dtype_code(x.dtype), x2.shape[1], work.data_ptr(), nbytes, _lib.stream_of(x2))
    return out


def _gate_rows(gate: torch.Tensor) -> torch.Tensor:
    if gate.dtype not in (torch.bfloat16, torch.float32):
        gate = gate.float()
    unit = 16 // gate.element_size()
    if gate.stride(1) != 1 or gate.stride(0) % unit or gate.stride(0) < gate.shape[1] or gate.data_ptr() % 16:
        gate = gate.clone(memory_format=torch.contiguous_format)
    return gate


def _vector(t: Optional[torch.Tensor], n: int, what: str, only_f32: bool = False) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if tuple(t.shape) != (n,):
        raise ValueError(f"{what} must be [{n}], got {tuple(t.shape)}")
    if t.dtype != torch.float32 and (only_f32 or t.dtype != torch.bfloat16):
        t = t.float()
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _code(t: Optional[torch.Tensor]) -> int:
    return _lib.DTYPE_BF16 if t is not None and t.dtype == torch.bfloat16 else _lib.DTYPE_F32


def moe_decode(x: torch.Tensor, gate_weight: torch.Tensor, experts, top_k: int, *,
               gate_bias: Optional[torch.Tensor] = None, score_bias: Optional[torch.Tensor] = None,
               gating: str = "softmax", normalize_expert_weights: Optional[str] = None,
               norm_weight: Optional[torch.Tensor] = None, norm_eps: float = DEFAULT_EPS,
               shared=None) -> DecodeOutput:
    """A whole MoE layer for 1 to 64 tokens, forward only: RMSNorm of x when
    ``norm_weight`` [D] is given, the router (``route`` without replay, jitter and
    losses: gate_weight [E, D], gate_bias and score_bias [E], softmax or sigmoid
    gating), the reached experts, the shared expert, and their sum.

    x [..., D] bf16 or fp32 (taken as bf16); ``experts`` and ``shared`` as for
    ``expert_decode``.  Returns ``DecodeOutput(out, weights, indices)`` with out in
    x's shape and dtype."""
    x2 = _rows(x)
    T, D = x2.shape
    _no_gradients(x, gate_weight, gate_bias, score_bias, norm_weight)
    if gate_weight.dim() != 2 or gate_weight.shape[1] != D:
        raise ValueError(f"gate_weight must be [E, {D}], got {tuple(gate_weight.shape)}")
    E, K = gate_weight.shape[0], int(top_k)
    _check_routing(T, E, K)
    if K > E:
        raise ValueError(f"top_k {K} of {E} experts")
    _same_device(x2, gate_weight=gate_weight, gate_bias=gate_bias, score_bias=score_bias, norm_weight=norm_weight)
    gate = _gate_rows(gate_weight)
    bias, score = _vector(gate_bias, E, "gate_bias"), _vector(score_bias, E, "score_bias", only_f32=True)
    norm = _vector(norm_weight, D, "norm_weight")
    gating_code, flags = _gating_code(gating), _norm_flags(normalize_expert_weights)
    dev = x2.device
    weights = torch.empty(T, K, dtype=torch.float32, device=dev)
    indices = torch.empty(T, K, dtype=torch.int64, device=dev)
    out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    if T == 0:
        return DecodeOutput(out, weights, indices)
    with _lib.on_device_of(x2):
        w, ws = _both(experts, E, shared, x2)
        work, nbytes = _workspace("fm_moe_decode_workspace_bytes", x2, K, E, w, ws)
        addr = _lib.addr
        _lib.call("fm_moe_decode", x2.data_ptr(), _pitch(x2), T, D, gate.data_ptr(), _dtype_code(gate.dtype),
                  gate.stride(0), addr(bias), _code(bias), addr(score), addr(norm), _code(norm), float(norm_eps), E, K,
                  gating_code, flags, w, ws, weights.data_ptr(), indices.data_ptr(), out.data_ptr(),
                  _dtype_code(x.dtype), D, work.data_ptr(), nbytes, _lib.stream_of(x2))
    return DecodeOutput(out, weights, indices)
