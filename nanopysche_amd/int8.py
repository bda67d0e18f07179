"""Products in 8-bit integers with a scale for each token and each channel, for serving:

    s_r = max(max_k |x_rk|, 1e-12) / 127,   q_rk = rint(x_rk / s_r)
    out[t, n] = (sum_k qx[t, k] qw[n, k]) sx[t] sw[n] (+ bias[n])

``quantize_to_int8`` quantises rows (tokens of an activation, output channels of a
weight), ``int8_matmul`` and ``int8_linear`` are the dense product, ``int8_grouped_gemm``
the product over a ``RoutingPlan``'s groups, and ``Int8MoECompute`` the expert block
(``MoEBase``'s expert compute, reference ``model/moe.py:1542-1596``) with int8 experts.
Integer sums are exact.  A row that holds a NaN or an infinity gives NaN outputs.

Everything here is forward only.  Nothing falls back to torch math.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .decode import (MAX_DECODE_DIM, MAX_DECODE_MATRIX, MAX_DECODE_TOKENS, MAX_DECODE_TOP_K, _no_gradients, _same_device,
                     expert_decode)
from .routing import RoutingPlan, route_tokens

MAX_INT8_K = 131071   # longest product whose int32 sums cannot overflow
MAX_INT8_ROWS = 2 ** 31 - 256   # rows of an operand are fewer


def _payload_bytes(rows: int, cols: int) -> int:
    return (rows + 15) // 16 * ((cols + 127) // 128) * 2048


def _check_cols(cols: int) -> None:
    if not 1 <= cols <= MAX_INT8_K:
        raise ValueError(f"int8 rows hold 1 to {MAX_INT8_K} columns, got {cols}")


def _check_payload(data: torch.Tensor, rows: int, cols: int) -> None:
    if not isinstance(data, torch.Tensor) or data.dtype != torch.uint8:
        raise TypeError(f"data must be a uint8 tensor, got {getattr(data, 'dtype', type(data))}")
    if data.numel() < _payload_bytes(rows, cols) or not data.is_contiguous():
        raise ValueError(f"data must be {_payload_bytes(rows, cols)} contiguous bytes for [{rows}, {cols}], "
                         f"got {tuple(data.shape)} of strides {data.stride()}")


def _check_scale(scale: torch.Tensor, rows: int, data: torch.Tensor) -> None:
    if not isinstance(scale, torch.Tensor) or scale.dtype != torch.float32:
        raise TypeError(f"scale must be a float32 tensor, got {getattr(scale, 'dtype', type(scale))}")
    if scale.shape != (rows,) or not scale.is_contiguous() or scale.device != data.device:
        raise ValueError(f"scale must be [{rows}], contiguous, on {data.device}, got {tuple(scale.shape)} of strides "
                         f"{scale.stride()} on {scale.device}")


@dataclass
class Int8Tensor:
    """An int8 matrix [rows, cols] with an fp32 scale per row.

    data   uint8 buffer: 16 x 64 tiles in the matrix cores' order (``include/fm_hip.h``)
    scale  [rows] fp32, contiguous, on the buffer's device

    The kernels read as far as rows and cols say, so the fields are checked when they are
    set: data and scale may be replaced by tensors that fit, the sizes stay.
    """

    data: torch.Tensor
    scale: torch.Tensor
    rows: int
    cols: int

    def __post_init__(self):
        if not isinstance(self.rows, int) or not isinstance(self.cols, int) or not 0 <= self.rows < MAX_INT8_ROWS:
            raise ValueError(f"rows and cols must be whole numbers, rows 0 to {MAX_INT8_ROWS - 1}, got {self.rows} and {self.cols}")
        _check_cols(self.cols)
        _check_payload(self.data, self.rows, self.cols)
        _check_scale(self.scale, self.rows, self.data)

    def __setattr__(self, name, value):
        if "cols" in self.__dict__:   # the last field that __init__ sets
            if name in ("rows", "cols"):
                raise AttributeError(f"the sizes of an Int8Tensor do not change: {name}")
            if name == "data":
                _check_payload(value, self.rows, self.cols)
                _check_scale(self.scale, self.rows, value)
            elif name == "scale":
                _check_scale(value, self.rows, self.data)
        object.__setattr__(self, name, value)

    @property
    def shape(self):
        return torch.Size((self.rows, self.cols))

    @property
    def device(self):
        return self.data.device

    @staticmethod
    def from_int8(q: torch.Tensor, scale: torch.Tensor) -> "Int8Tensor":
        """Values q [rows, cols] int8 (any strides) and their rows' scales."""
        _lib.require_device(q, "q")
        if q.dim() != 2 or q.dtype != torch.int8:
            raise TypeError(f"q must be a 2-D int8 tensor, got {q.dtype} {tuple(q.shape)}")
        return _pack(q.unsqueeze(0), scale)

    def values(self) -> torch.Tensor:
        """The int8 values as a row-major tensor."""
        return _unpack(self, torch.int8)

    def dequantize(self, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """q * scale, rounded once to ``out_dtype`` (bf16 or fp32)."""
        if out_dtype not in (torch.bfloat16, torch.float32):
            raise TypeError("out_dtype must be bfloat16 or float32")
        _no_gradients(self.scale)
        return _unpack(self, out_dtype)


def _empty(rows: int, cols: int, dev) -> Int8Tensor:
    t = Int8Tensor.__new__(Int8Tensor)   # fits by construction: 2 us of checks less a call
    t.__dict__.update(data=torch.empty(_payload_bytes(rows, cols), dtype=torch.uint8, device=dev),
                      scale=torch.empty(rows, dtype=torch.float32, device=dev), rows=rows, cols=cols)
    return t


def _pack(q: torch.Tensor, scale: torch.Tensor) -> Int8Tensor:
    """Groups q [G, rows, cols] one after the other."""
    G, R, K = q.shape
    _check_cols(K)
    _no_gradients(scale)
    if tuple(scale.shape) != (G * R,) or scale.device != q.device:
        raise ValueError(f"scale must be [{G * R}] on {q.device}, got {tuple(scale.shape)} on {scale.device}")
    t = _empty(G * R, K, q.device)
    t.scale.copy_(scale)
    if G * R:
        with _lib.on_device_of(q):
            _lib.call("fm_int8_pack", q.data_ptr(), G, R, K, *q.stride(), t.data.data_ptr(), _lib.stream_of(q))
    return t


_UNPACK = {torch.bfloat16: 0, torch.float32: 1, torch.int8: 2}


def _unpack(t: Int8Tensor, dtype: torch.dtype) -> torch.Tensor:
    out = torch.empty(t.rows, t.cols, dtype=dtype, device=t.device)
    if t.rows:
        with _lib.on_device_of(out):
            _lib.call("fm_int8_unpack", t.data.data_ptr(), t.scale.data_ptr(), t.rows, t.cols, out.data_ptr(),
                      _UNPACK[dtype], t.cols, _lib.stream_of(out))
    return out


def _quantize(x: torch.Tensor, rows: int, assign=None, top_k: int = 1, limit=None, top=None, clear=None) -> Int8Tensor:
    """Rows of x [R, K] (of the assignments' tokens, with ``assign``) up to ``limit``, by
    their maxima ``top`` where they are known; sets ``clear`` to 0."""
    t = _empty(rows, x.shape[1], x.device)
    ld = x.stride(0) if x.shape[0] > 1 else x.shape[1]
    addr = _lib.addr
    _lib.call("fm_int8_quantize", x.data_ptr(), _lib.DTYPE_BF16 if x.dtype == torch.bfloat16 else _lib.DTYPE_F32, rows,
              x.shape[1], ld, addr(assign), top_k, addr(limit), addr(top), addr(clear), t.data.data_ptr(), t.scale.data_ptr(), _lib.stream_of(x))
    return t


def _float_rows(x: torch.Tensor) -> torch.Tensor:
    _lib.require_device(x, "x")
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"expected bfloat16 or float32 input, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError("expected a tensor with at least 1 dimension")
    _check_cols(x.shape[-1])
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    rows, cols = x2.shape
    ld, one = x2.stride()
    return x2 if one == 1 and (ld >= cols or rows == 1) else x2.contiguous()


def quantize_to_int8(x: torch.Tensor) -> Int8Tensor:
    """x [..., K] (bf16 or fp32) as int8 with a scale per row: the tokens of an
    activation, or the output channels of a weight [N, K]."""
    x2 = _float_rows(x)
    _no_gradients(x)
    if x2.shape[0] == 0:
        return _empty(0, x2.shape[1], x.device)
    with _lib.on_device_of(x2):
        return _quantize(x2, x2.shape[0])


def _out_code(dtype: torch.dtype) -> int:
    if dtype == torch.bfloat16:
        return _lib.DTYPE_BF16
    if dtype == torch.float32:
        return _lib.DTYPE_F32
    raise TypeError("out_dtype must be bfloat16 or float32")


def _bias(bias: Optional[torch.Tensor], N: int) -> Optional[torch.Tensor]:
    if bias is None:
        return None
    if tuple(bias.shape) != (N,):
        raise ValueError(f"bias must be [{N}], got {tuple(bias.shape)}")
    return bias if bias.dtype == torch.float32 and bias.is_contiguous() else bias.to(torch.float32).contiguous()


def int8_matmul(a: Int8Tensor, b: Int8Tensor, bias: Optional[torch.Tensor] = None,
                out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a b^T with both operands' scales: tokens a [M, K] and channels b [N, K] ->
    [M, N] in ``out_dtype`` (bf16 or fp32), plus bias [N] (fp32)."""
    _lib.require_device(a.data, "a")
    if a.cols != b.cols:
        raise ValueError(f"a has {a.cols} columns, b {b.cols}")
    code = _out_code(out_dtype)
    _no_gradients(a.scale, b.scale, bias)
    _same_device(a.data, b=b.data, bias=bias)
    M, N = a.rows, b.rows
    bias = _bias(bias, N)
    out = torch.empty(M, N, dtype=out_dtype, device=a.device)
    if M and N:
        with _lib.on_device_of(out):
            _lib.call("fm_int8_matmul", a.data.data_ptr(), a.scale.data_ptr(), M, b.data.data_ptr(), b.scale.data_ptr(),
                      N, a.cols, _lib.addr(bias), out.data_ptr(), code, N, _lib.stream_of(out))
    return out


def int8_linear(x: torch.Tensor, weight: Int8Tensor, bias: Optional[torch.Tensor] = None,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x [..., K] (bf16 or fp32), quantised by token, times int8 weights [N, K] ->
    [..., N] in ``out_dtype`` (default x's), plus bias [N]: ``int8_matmul`` of
    ``quantize_to_int8(x)``, the same bits."""
    if x.dim() < 1 or x.shape[-1] != weight.cols:
        raise ValueError(f"x {tuple(x.shape)} does not end in the weight's {weight.cols} columns")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    code = _out_code(out_dtype)
    x2 = _float_rows(x)
    _no_gradients(x, weight.scale, bias)
    _same_device(x, weight=weight.data, bias=bias)
    M, K = x2.shape
    N = weight.rows
    bias = _bias(bias, N)
    out = torch.empty(*x.shape[:-1], N, dtype=out_dtype, device=x.device)
    if M and N:
        with _lib.on_device_of(x2):
            nbytes = _lib.size_of("fm_int8_linear_workspace_bytes", M, K)
            work = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
            _lib.call("fm_int8_linear", x2.data_ptr(), _lib.DTYPE_BF16 if x2.dtype == torch.bfloat16 else _lib.DTYPE_F32, M,
                      K, x2.stride(0) if M > 1 else K, weight.data.data_ptr(), weight.scale.data_ptr(), N, _lib.addr(bias),
                      out.data_ptr(), code, N, _lib.addr(work), nbytes, _lib.stream_of(x2))
    return out


def int8_grouped_gemm(tokens: Int8Tensor, weights: Int8Tensor, plan: RoutingPlan,
                      out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Rows [offsets[e], offsets[e + 1]) of the plan's padded buffer ``tokens``
    [rows_max, K] times expert e's channels, ``weights`` [E * N, K] -> [rows_max, N].
    Rows past the last group are left unwritten.  K a multiple of 128, N of 16."""
    _lib.require_device(tokens.data, "tokens")
    E = plan.num_experts
    if tokens.rows != plan.rows_max or tokens.cols != weights.cols or weights.rows % E:
        raise ValueError(f"tokens [{tokens.rows}, {tokens.cols}] and weights [{weights.rows}, {weights.cols}] do not fit "
                         f"a plan of {plan.rows_max} rows and {E} experts")
    _out_code(out_dtype)
    _no_gradients(tokens.scale, weights.scale)
    _same_device(tokens.data, weights=weights.data, plan=plan.offsets)
    with _lib.on_device_of(tokens.data):
        return _grouped(tokens, weights, None, None, plan, weights.rows // E, out_dtype)


def _grouped(tokens, w, up, top, plan, N, out_dtype):
    out = torch.empty(tokens.rows, N, dtype=out_dtype, device=tokens.device)
    _lib.call("fm_int8_grouped_gemm", tokens.data.data_ptr(), tokens.scale.data_ptr(), tokens.rows,
              plan.offsets.data_ptr(), plan.num_experts, w.data.data_ptr(), w.scale.data_ptr(),
              None if up is None else up.data.data_ptr(), None if up is None else up.scale.data_ptr(), _lib.addr(top), N, tokens.cols,
              plan.num_tokens * plan.top_k, out.data_ptr(),
              _lib.DTYPE_F32 if out_dtype == torch.float32 else _lib.DTYPE_BF16, N, _lib.stream_of(out))
    return out


@dataclass
class Int8Experts:
    """SwiGLU experts in int8, laid out once: w1, w3 [E * H, D] with a scale per hidden
    unit, w2 transposed [E * D, H] with a scale per output column; H and D multiples of 128.
    The fields are checked when they are set: one may be replaced by one that fits the others."""

    w1: Int8Tensor
    w2: Int8Tensor
    w3: Int8Tensor
    num_experts: int

    def __post_init__(self):
        self._check(self.w1, self.w2, self.w3, self.num_experts)

    def __setattr__(self, name, value):
        if "num_experts" in self.__dict__:   # the last field that __init__ sets
            self._check(*(value if f == name else getattr(self, f) for f in ("w1", "w2", "w3", "num_experts")))
        object.__setattr__(self, name, value)

    @staticmethod
    def _check(w1, w2, w3, num_experts):
        for name, w in (("w1", w1), ("w2", w2), ("w3", w3)):
            if not isinstance(w, Int8Tensor):
                raise TypeError(f"{name} must be an Int8Tensor, got {type(w)}")
        E = num_experts
        if not isinstance(E, int) or E < 1 or w1.rows % E:
            raise ValueError(f"num_experts must be a positive whole number that divides w1's {w1.rows} rows, got {E}")
        H, D = w1.rows // E, w1.cols
        if w3.shape != (E * H, D) or w2.shape != (E * D, H):
            raise ValueError(f"w1 {tuple(w1.shape)} of {E} experts needs w3 [{E * H}, {D}] and w2, transposed, [{E * D}, {H}], "
                             f"got {tuple(w3.shape)} and {tuple(w2.shape)}")
        if H % 128 or D % 128:
            raise ValueError(f"d_model ({D}) and hidden_size ({H}) must be multiples of 128")
        if w2.device != w1.device or w3.device != w1.device:
            raise ValueError(f"w1, w2 and w3 must be on one device, got {w1.device}, {w2.device} and {w3.device}")

    @property
    def hidden_size(self) -> int:
        return self.w2.cols

    @property
    def d_model(self) -> int:
        return self.w1.cols

    @staticmethod
    def _sizes(w1, w2, w3, num_experts):
        if num_experts < 1 or w1.dim() != 2 or w1.shape != w2.shape or w1.shape != w3.shape or w1.shape[0] % num_experts:
            raise ValueError(f"w1, w2, w3 must be [E * H, D] with E = {num_experts}, got {tuple(w1.shape)}, "
                             f"{tuple(w2.shape)}, {tuple(w3.shape)}")
        H, D = w1.shape[0] // num_experts, w1.shape[1]
        if H % 128 or D % 128 or not H or not D:
            raise ValueError(f"d_model ({D}) and hidden_size ({H}) must be multiples of 128")
        return H, D

    @staticmethod
    def quantize(w1: torch.Tensor, w2: torch.Tensor, w3: torch.Tensor, num_experts: int) -> "Int8Experts":
        """From bf16 or fp32 weights [E * H, D] in the expert block's storage, detached."""
        H, D = Int8Experts._sizes(w1, w2, w3, num_experts)
        _same_device(w1, w2=w2, w3=w3)
        w2t = w2.detach().reshape(num_experts, H, D).transpose(1, 2).reshape(num_experts * D, H)
        return Int8Experts(quantize_to_int8(w1.detach()), quantize_to_int8(w2t), quantize_to_int8(w3.detach()), num_experts)

    @staticmethod
    def from_int8(w1: torch.Tensor, s1: torch.Tensor, w2: torch.Tensor, s2: torch.Tensor, w3: torch.Tensor,
                  s3: torch.Tensor, num_experts: int) -> "Int8Experts":
        """From int8 values [E * H, D] in the expert block's storage and their scales:
        s1, s3 [E * H], s2 [E, D]."""
        H, D = Int8Experts._sizes(w1, w2, w3, num_experts)
        if tuple(s2.shape) != (num_experts, D):
            raise ValueError(f"s2 must be [{num_experts}, {D}], got {tuple(s2.shape)}")
        _lib.require_device(w2, "w2")
        _same_device(w1, w2=w2, w3=w3, s2=s2)
        if w2.dtype != torch.int8:
            raise TypeError(f"w2 must be int8, got {w2.dtype}")
        t2 = _pack(w2.reshape(num_experts, H, D).transpose(1, 2), s2.reshape(-1))
        return Int8Experts(Int8Tensor.from_int8(w1, s1), t2, Int8Tensor.from_int8(w3, s3), num_experts)


class Int8MoECompute:
    """The expert block with int8 experts, forward only, called as ``FP8FlowMoECompute``:
    ``block(x [N, D], weights [N, K], indices [N, K], expert_offset=0) -> [N, D]``.

    Tokens: route (stable counting sort) -> gather and quantise by token -> grouped
    product gate|up with SwiGLU behind it -> quantise h by token -> grouped product
    down -> weighted sum, in fp32 between the products and rounded once.  Up to 64
    tokens (D up to 14336, K up to 16, H D below 2^30) go through ``expert_decode`` instead,
    which does not quantise activations but takes an fp32 x rounded to bf16."""

    def __init__(self, experts: Int8Experts):
        self.experts = experts

    def __call__(self, x: torch.Tensor, weights: torch.Tensor, indices: torch.Tensor, expert_offset: int = 0,
                 num_local_experts: Optional[int] = None) -> torch.Tensor:
        w = self.experts
        E = w.num_experts
        if num_local_experts is not None and int(num_local_experts) != E:
            raise ValueError(f"num_local_experts={num_local_experts} but the block holds {E} experts")
        x2 = _float_rows(x)
        T, D = x2.shape
        if D != w.d_model:
            raise ValueError(f"x has {D} columns, the experts {w.d_model}")
        _no_gradients(x, weights, w.w1.scale, w.w2.scale, w.w3.scale)
        _same_device(x, weights=weights, indices=indices, experts=w.w1.data)
        K = indices.shape[-1] if indices.dim() else 0
        if K < 1 or indices.numel() != T * K or weights.numel() != T * K or weights.shape[-1] != K:
            raise ValueError(f"weights {tuple(weights.shape)} and indices {tuple(indices.shape)} must be [T, K] for {T} tokens")
        if T <= MAX_DECODE_TOKENS and D <= MAX_DECODE_DIM and K <= MAX_DECODE_TOP_K and w.hidden_size * D < MAX_DECODE_MATRIX:
            return expert_decode(x, weights, indices, w, E, expert_offset)
        if T == 0:
            return torch.empty_like(x)
        with _lib.on_device_of(x2):
            if expert_offset:
                indices = indices - int(expert_offset)
            plan = route_tokens(indices.reshape(T, K), E)
            end = plan.offsets[E:]
            top = torch.empty(plan.rows_max, dtype=torch.int32, device=x.device)   # largest |h| of every row, as bits
            q = _quantize(x2, plan.rows_max, plan.assign_of_row, K, end, clear=top)
            h = _grouped(q, w.w1, w.w3, top, plan, w.hidden_size, torch.float32)
            q = _quantize(h, plan.rows_max, limit=end, top=top)
            y = _grouped(q, w.w2, None, None, plan, D, torch.float32)
            rw = weights.reshape(T, K).to(torch.float32).contiguous()
            out = torch.empty(T, D, dtype=x.dtype, device=x.device)
            _lib.call("fm_int8_combine", y.data_ptr(), D, plan.row_of.data_ptr(), rw.data_ptr(), T, K, out.data_ptr(),
                      _lib.DTYPE_F32 if x.dtype == torch.float32 else _lib.DTYPE_BF16, _lib.stream_of(out))
        return out.reshape(x.shape)
