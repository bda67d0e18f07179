"""Activations kept in 8 bits between a forward and its backward.

    k = max(floor(log2 max|x|) - 6, -127) over a block of 32 values of a row,  s = 2^k
    q = min(max(rint(x / s), -127), 127),  the value that it stands for is q s

(an e8m0 code per block, k + 127; 33 bytes hold 32 values.  The values are those of OCP MX int8 down to its
smallest scale, 2^-133; its code of the same block is 6 above this one, its element holding a 2^-6.)  q s is exact in bfloat16 and
float32, so keeping rounds a value once, by at most s / 2 (s for what lies above 127.5 s, which no
bfloat16 value does), s being at most a 64th of its block's largest magnitude.  A block that holds a NaN or an infinity stands for NaNs.

``compress_activation`` keeps any activation; ``swiglu_8bit`` and ``rmsnorm_8bit`` are SwiGLU and
RMSNorm (reference ``model/moe.py:1590``, ``model/norm.py:32-49``) whose backward reads their inputs
from 8 bits.  Their forwards compute from the inputs themselves: only the gradients see the rounding.  SwiGLU's
outputs are those of the layers that keep 16 bits, bit for bit; RMSNorm's differ from ``rmsnorm``'s in the last bits of some, its
sum of squares being added in another order.  The reference keeps activations in the model's type or recomputes them
(``distributed/fsdp.py:80-117``).
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
import torch.autograd.forward_ad as fwAD
from torch.autograd.function import once_differentiable

from . import _lib

DEFAULT_EPS = 1e-6   # of RMSNorm (reference model/norm.py:27)
ACT8_BLOCK = 32
MAX_ACT8_COLS = 2 ** 24 - 1
MAX_ACT8_NORM = 16384   # columns of a normalised row


def _pitch(cols: int) -> int:
    return (cols + ACT8_BLOCK - 1) // ACT8_BLOCK * ACT8_BLOCK


def _bytes(rows: int, cols: int) -> int:
    return rows * _pitch(cols) // ACT8_BLOCK * (ACT8_BLOCK + 1)


def _check_cols(cols: int, most: int = MAX_ACT8_COLS) -> None:
    if not 1 <= cols <= most:
        raise ValueError(f"rows of 1 to {most} columns, got {cols}")


_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}


def _dtype(dtype: torch.dtype, what: str) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"{what} must be bfloat16 or float32, got {dtype}")
    return code


def _no_gradients(name: str, instead: str, *tensors) -> None:
    if not torch.is_grad_enabled() and fwAD._current_level < 0:   # as under no_grad and in a node: nothing is recorded
        return
    carried = _lib.carried(*tensors)
    if carried:
        raise RuntimeError(f"{name} records no {carried}: {instead} is differentiable (once, in reverse mode); call {name} under "
                           "torch.no_grad() or on detached tensors")


class Activation8:
    """An activation [..., cols] in 8 bits.

    data   uint8 buffer: int8 values [rows, cols rounded up to 32], then the blocks' codes, row by row
    shape  the activation's shape
    dtype  its type, which ``restore`` gives back

    The kernels read as far as the shape says, so it does not change; data may be replaced by a tensor of as many bytes.
    """

    __slots__ = ("_data", "_shape", "_dtype", "_sizes")

    def __init__(self, data: torch.Tensor, shape, dtype: torch.dtype = torch.bfloat16):
        shape = torch.Size(shape)
        if not shape:
            raise ValueError("an activation has at least 1 dimension")
        _dtype(dtype, "dtype")
        _check_cols(shape[-1])
        self._shape, self._dtype = shape, dtype
        self._sizes = shape[:-1].numel(), shape[-1], _pitch(shape[-1])
        self.data = data

    @property
    def data(self) -> torch.Tensor:
        return self._data

    @data.setter
    def data(self, data: torch.Tensor) -> None:
        if not isinstance(data, torch.Tensor) or data.dtype != torch.uint8:
            raise TypeError(f"data must be a uint8 tensor, got {getattr(data, 'dtype', type(data))}")
        need = _bytes(self.rows, self.cols)
        if data.numel() < need or not data.is_contiguous() or data.data_ptr() % 8:
            raise ValueError(f"data must be {need} contiguous bytes on an 8-byte boundary for {tuple(self._shape)}, got "
                             f"{tuple(data.shape)} of strides {data.stride()}")
        self._data = data

    @property
    def shape(self) -> torch.Size:
        return self._shape

    @property
    def dtype(self) -> torch.dtype:
        return self._dtype

    @property
    def rows(self) -> int:
        return self._sizes[0]

    @property
    def cols(self) -> int:
        return self._sizes[1]

    @property
    def pitch(self) -> int:
        return self._sizes[2]

    @property
    def device(self) -> torch.device:
        return self._data.device

    @property
    def nbytes(self) -> int:
        return _bytes(self.rows, self.cols)

    def at(self):
        """Addresses of the values and codes, and their pitches."""
        rows, _, pitch = self._sizes
        q = self._data.data_ptr()
        return q, q + rows * pitch, pitch, pitch // ACT8_BLOCK

    def restore(self, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The values that the 8 bits stand for, in ``out_dtype`` (default: the activation's type); they carry no gradient."""
        return _restore(self, None, self.rows, self._shape, out_dtype or self._dtype)

    def restore_rows(self, index: torch.Tensor, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """out[i] = row index[i] of the activation (its leading dimensions flattened), zeros where
        ``index`` (int32) is outside it: ``gather_rows`` of what was kept."""
        if index.dtype != torch.int32:
            raise TypeError(f"index must be int32, got {index.dtype}")
        if index.dim() != 1:
            raise ValueError(f"index must be 1-D, got {tuple(index.shape)}")
        if index.get_device() != self._data.get_device():
            raise ValueError(f"index is on {index.device}, the activation on {self.device}")
        return _restore(self, index.contiguous(), index.numel(), (index.numel(), self.cols), out_dtype or self._dtype)


def _empty(shape: torch.Size, rows: int, dtype, dev) -> Activation8:
    """Room for an activation of this shape; fits by construction."""
    t = Activation8.__new__(Activation8)
    cols = shape[-1]
    pitch = (cols + 31) // 32 * 32
    t._data = torch.empty(rows * pitch // 32 * 33, dtype=torch.uint8, device=dev)
    t._shape, t._dtype, t._sizes = shape, dtype, (rows, cols, pitch)
    return t


def _like(x: torch.Tensor) -> torch.Tensor:
    """An empty contiguous tensor like x."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _here(index: int, what: str, t: torch.Tensor) -> None:
    if t.get_device() != index:
        raise ValueError(f"{what} is on {t.device}, the others on device {index}")


def _rows(x: torch.Tensor, what: str, most: int = MAX_ACT8_COLS) -> torch.Tensor:
    """x [..., cols] as rows whose columns are neighbours."""
    _lib.require_device(x, what)
    _dtype(x.dtype, what)
    if x.dim() < 1:
        raise ValueError(f"{what} must have at least 1 dimension")
    _check_cols(x.shape[-1], most)
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    return x2 if x2.stride(1) == 1 or x2.shape[1] == 1 else x2.contiguous()


def _restore(t: Activation8, index, rows, shape, dtype) -> torch.Tensor:
    code = _dtype(dtype, "out_dtype")
    out = torch.empty(shape, dtype=dtype, device=t.device)
    if out.numel():
        q, codes, ld_q, ld_c = t.at()
        src_rows, cols, _ = t._sizes
        _lib.call_on(out, "fm_act8_restore", q, ld_q, codes, ld_c, src_rows, cols, _lib.addr(index), rows, out.data_ptr(), code, cols)
    return out


def _compress(x2: torch.Tensor, shape, tile_valid=None) -> Activation8:
    rows, cols = x2.shape
    t = _empty(shape, rows, x2.dtype, x2.device)
    if rows:
        q, codes, ld_q, ld_c = t.at()
        _lib.call_on(x2, "fm_act8_compress", x2.data_ptr(), _DTYPES[x2.dtype], rows, cols, x2.stride(0), q, ld_q, codes, ld_c,
                     _lib.addr(tile_valid))
    return t


def compress_activation(x: torch.Tensor) -> Activation8:
    """x [..., cols] (bf16 or fp32) in 8 bits.  Not differentiable (x may require a gradient, which does not reach it through
    what is kept): what a forward keeps of x for its backward."""
    x2 = _rows(x, "x")
    return _compress(x2, x.shape)


# ================================================================== SwiGLU ====
class SwigluKept(NamedTuple):
    """h [..., H], and what the backward needs: gate and up [..., H] in 8 bits."""

    out: torch.Tensor
    gate: Activation8
    up: Activation8


def _halves(gate: torch.Tensor, up: Optional[torch.Tensor]):
    """(gate's and up's tensors of rows, up's address, the shape of h): up's rows may be the second half of gate's."""
    if up is None:
        g2 = _rows(gate, "gate", 2 * MAX_ACT8_COLS)
        H, odd = divmod(g2.shape[1], 2)
        if odd:
            raise ValueError(f"gate|up must have an even number of columns, got {gate.shape[-1]}")
        return g2, g2, g2.data_ptr() + H * g2.element_size(), gate.shape[:-1] + (H,)
    if up.shape != gate.shape or up.dtype != gate.dtype:
        raise ValueError(f"gate and up must be alike, got {tuple(gate.shape)} {gate.dtype} and {tuple(up.shape)} {up.dtype}")
    g2, u2 = _rows(gate, "gate"), _rows(up, "up")
    _here(g2.get_device(), "up", u2)
    return g2, u2, u2.data_ptr(), gate.shape


def swiglu_compress(gate: torch.Tensor, up: Optional[torch.Tensor] = None) -> SwigluKept:
    """h = silu(gate) * up (fp32 arithmetic, rounded once) and gate and up in 8 bits, in one pass.
    gate and up [..., H], bf16 or fp32, or one tensor [..., 2H] of the gate's columns and then up's.  Records no gradient, and
    refuses tensors that want one recorded: ``swiglu_8bit``."""
    _no_gradients("swiglu_compress", "swiglu_8bit", gate, up)
    return _swiglu(gate, up, True)


def _swiglu(gate, up, keep: bool):
    """SwigluKept, or h alone where nothing is kept."""
    g2, u2, at_u, shape = _halves(gate, up)
    H, rows, dtype, dev = shape[-1], g2.shape[0], g2.dtype, g2.device
    h = torch.empty(shape, dtype=dtype, device=dev)
    kept_g = kept_u = qg = cg = qu = cu = None
    ld_q = _pitch(H)
    if keep:
        kept_g, kept_u = _empty(shape, rows, dtype, dev), _empty(shape, rows, dtype, dev)
        qg, cg, _, _ = kept_g.at()
        qu, cu, _, _ = kept_u.at()
    if rows:
        _lib.call_on(g2, "fm_act8_swiglu", g2.data_ptr(), g2.stride(0), at_u, u2.stride(0), _DTYPES[dtype], rows, H, h.data_ptr(), H,
                     qg, cg, qu, cu, ld_q, ld_q // ACT8_BLOCK)
    return SwigluKept(h, kept_g, kept_u) if keep else h


def swiglu_backward_8bit(dh: torch.Tensor, gate: Activation8, up: Activation8, packed: bool = False):
    """(dgate, dup) of ``swiglu_compress`` from dh [..., H] and what it kept, in dh's type; with ``packed`` one
    tensor [..., 2H].  Records no gradient, as its forward."""
    _no_gradients("swiglu_backward_8bit", "swiglu_8bit", dh)
    if dh.shape != gate.shape or up.shape != gate.shape:
        raise ValueError(f"dh, gate and up must be alike, got {tuple(dh.shape)}, {tuple(gate.shape)} and {tuple(up.shape)}")
    d2 = _rows(dh, "dh")
    index = d2.get_device()
    _here(index, "gate", gate._data)
    _here(index, "up", up._data)
    rows, H = d2.shape
    if packed:
        both = torch.empty(dh.shape[:-1] + (2 * H,), dtype=dh.dtype, device=dh.device)
        at_g, at_u, ld = both.data_ptr(), both.data_ptr() + H * both.element_size(), 2 * H
    else:
        dg, du = _like(dh), _like(dh)
        at_g, at_u, ld = dg.data_ptr(), du.data_ptr(), H
    if rows:
        qg, cg, ld_q, ld_c = gate.at()
        qu, cu, _, _ = up.at()
        _lib.call_on(d2, "fm_act8_swiglu_backward", d2.data_ptr(), d2.stride(0), _DTYPES[d2.dtype], rows, H, qg, cg, qu, cu, ld_q, ld_c,
                     at_g, ld, at_u, ld)
    return both if packed else (dg, du)


class _SwigluFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up):
        h, kept_g, kept_u = _swiglu(gate, up, True)
        ctx.save_for_backward(kept_g.data, kept_u.data)
        ctx.packed, ctx.dtype = up is None, gate.dtype
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        gate, up = (Activation8(t, dh.shape, ctx.dtype) for t in ctx.saved_tensors)
        if ctx.packed:
            return swiglu_backward_8bit(dh, gate, up, packed=True), None
        return swiglu_backward_8bit(dh, gate, up)


def swiglu_8bit(gate: torch.Tensor, up: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Differentiable silu(gate) * up that keeps gate and up in 8 bits for its backward (``swiglu_compress``); nothing is kept
    where no gradient is recorded."""
    return _SwigluFunction.apply(gate, up) if _lib.carried(gate, up) else _swiglu(gate, up, False)


# ================================================================= RMSNorm ====
class RMSNormKept(NamedTuple):
    """y [..., D], and what the backward needs: x in 8 bits, rstd [T] fp32."""

    y: torch.Tensor
    x: Activation8
    rstd: torch.Tensor


def _norm_weight(weight: torch.Tensor, D: int) -> torch.Tensor:
    _dtype(weight.dtype, "weight")
    if weight.dim() != 1 or weight.numel() != D:
        raise ValueError(f"weight must be [{D}], got {tuple(weight.shape)}")
    return weight if weight.is_contiguous() else weight.contiguous()


def rmsnorm_compress(x: torch.Tensor, weight: torch.Tensor, eps: float = DEFAULT_EPS) -> RMSNormKept:
    """y = x * rsqrt(mean(x^2) + eps) * weight (fp32 arithmetic, rounded once to x's type) and x in 8 bits,
    in one pass.  x [..., D] and weight [D] bf16 or fp32, D up to 16384.  Records no gradient, and refuses tensors that want one
    recorded: ``rmsnorm_8bit``."""
    _no_gradients("rmsnorm_compress", "rmsnorm_8bit", x, weight)
    return _rmsnorm(x, weight, eps, True)


def _rmsnorm(x, weight, eps, keep: bool):
    """RMSNormKept, or y alone where nothing is kept."""
    x2 = _rows(x, "x", MAX_ACT8_NORM)
    T, D = x2.shape
    w = _norm_weight(weight, D)
    _here(x2.get_device(), "weight", w)
    dev = x2.device
    y = _like(x)
    rstd = kept = q = codes = None
    ld_q = _pitch(D)
    if keep:
        rstd = torch.empty(T, dtype=torch.float32, device=dev)
        kept = _empty(x.shape, T, x.dtype, dev)
        q, codes, _, _ = kept.at()
    if T:
        _lib.call_on(x2, "fm_act8_rmsnorm", x2.data_ptr(), _DTYPES[x2.dtype], x2.stride(0), T, D, w.data_ptr(), _DTYPES[w.dtype], eps,
                     y.data_ptr(), D, q, ld_q, codes, ld_q // ACT8_BLOCK, _lib.addr(rstd))
    return RMSNormKept(y, kept, rstd) if keep else y


def rmsnorm_backward_8bit(dy: torch.Tensor, x: Activation8, weight: torch.Tensor, rstd: torch.Tensor, need_dw: bool = True):
    """(dx in dy's type, dw in weight's or None) of ``rmsnorm_compress`` from dy [..., D] and what it kept.  Records no gradient,
    as its forward."""
    _no_gradients("rmsnorm_backward_8bit", "rmsnorm_8bit", dy, weight)
    if dy.shape != x.shape:
        raise ValueError(f"dy must be {tuple(x.shape)}, got {tuple(dy.shape)}")
    d2 = _rows(dy, "dy", MAX_ACT8_NORM)
    T, D = d2.shape
    w = _norm_weight(weight, D)
    if rstd.dtype != torch.float32 or rstd.numel() != T or not rstd.is_contiguous():
        raise ValueError(f"rstd must be {T} contiguous float32 values, got {rstd.dtype} {tuple(rstd.shape)}")
    index = d2.get_device()
    _here(index, "weight", w)
    _here(index, "rstd", rstd)
    _here(index, "x", x._data)
    dx = _like(dy)
    dw = ws = None
    nbytes = 0
    if need_dw:
        dw = torch.empty(D, dtype=w.dtype, device=dy.device)
        if T == 0:
            return dx, dw.zero_()
        nbytes = _lib.size_of("fm_act8_rmsnorm_backward_workspace_bytes", T, D)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dy.device)
    if T:
        q, codes, ld_q, ld_c = x.at()
        _lib.call_on(d2, "fm_act8_rmsnorm_backward", d2.data_ptr(), d2.stride(0), _DTYPES[d2.dtype], T, D, q, ld_q, codes, ld_c, w.data_ptr(),
                     _DTYPES[w.dtype], rstd.data_ptr(), dx.data_ptr(), D, _lib.addr(dw), _lib.addr(ws), nbytes)
    return dx, dw


class _RMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        y, kept, rstd = _rmsnorm(x, weight, eps, True)
        ctx.save_for_backward(kept.data, weight, rstd)
        ctx.dtype = x.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        data, weight, rstd = ctx.saved_tensors
        dx, dw = rmsnorm_backward_8bit(dy, Activation8(data, dy.shape, ctx.dtype), weight, rstd, need_dw=ctx.needs_input_grad[1])
        return (dx if ctx.needs_input_grad[0] else None), dw, None


def rmsnorm_8bit(x: torch.Tensor, weight: torch.Tensor, eps: float = DEFAULT_EPS) -> torch.Tensor:
    """Differentiable RMSNorm that keeps x in 8 bits for its backward (``rmsnorm_compress``); nothing is kept where no gradient is
    recorded, and y is the same."""
    return _RMSNormFunction.apply(x, weight, float(eps)) if _lib.carried(x, weight) else _rmsnorm(x, weight, float(eps), False)
