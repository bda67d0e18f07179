"""The load-balancing loss of packed and padded sequences, with per-expert counts and gradients.

The reference's loss (``MoERouter._load_balancing_loss``, ``model/moe.py:267-281``) takes every token of the
batch as one sequence.  Here it is taken of each sequence and averaged, over the tokens that count:

    f_se = (slots of sequence s at expert e) / n_s,   P_se = mean over its tokens of p_te
    loss = (E / S') sum_s sum_e f_se P_se  (+ z_loss_multiplier * mean_t logsumexp(l_t)^2)

with n_s the tokens of s that count, S' the sequences that have any, and p the softmax of the logits or,
for sigmoid routers, sigma / (sum sigma + 1e-8).  One sequence without a mask is the
reference's loss.  f carries no gradient, as in the reference.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib

MAX_BALANCE_EXPERTS = 1024
MAX_BALANCE_TOP_K = 1024
MAX_SEQUENCES = 2 ** 20 - 1
_JOINT_BYTES = 1 << 18   # a workspace up to here lies behind f, an allocation (1.4 us) less a call; larger ones are freed with the forward


class BalanceOutput(NamedTuple):
    """loss (0-d fp32) and counts of the slots that counted: [E] int32, [S, E] with sequence borders."""

    loss: torch.Tensor
    counts: torch.Tensor


@dataclass
class BalanceState:
    """What ``balance_backward`` needs of ``balance_forward``."""

    logits: torch.Tensor               # [T, E]
    cu_seqlens: Optional[torch.Tensor]  # [S + 1] int32
    mask: Optional[torch.Tensor]       # [T] bool
    f: torch.Tensor                    # fp32, S * E + 2 and 256 KiB at most behind: E slots / n_s^2, then 1 / S' and 1 / tokens
    sigmoid: bool
    z_mult: float
    shape: torch.Size                  # of the logits as given


def _scores(scores: str) -> bool:
    if scores not in ("softmax", "sigmoid"):
        raise ValueError(f"scores must be 'softmax' or 'sigmoid', got {scores!r}")
    return scores == "sigmoid"


def _check(logits, indices, cu_seqlens, token_mask, load_tracker):
    """Rows of the logits, and the arguments as the kernels read them."""
    _lib.require_device(logits, "logits")
    if logits.dtype != torch.float32:
        raise TypeError(f"logits must be float32 (the router runs the gate in fp32), got {logits.dtype}")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_BALANCE_EXPERTS:
        raise ValueError(f"logits must be [..., E] with E of 1 to {MAX_BALANCE_EXPERTS}, got {tuple(logits.shape)}")
    E = logits.shape[-1]
    l2 = logits if logits.dim() == 2 else logits.reshape(-1, E)
    if l2.stride(1) != 1 or l2.stride(0) < E:
        l2 = l2.contiguous()
    T = l2.shape[0]
    if T >= 2 ** 31:
        raise ValueError(f"fewer than 2^31 tokens, got {T}")
    if indices.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"indices must be int64 or int32, got {indices.dtype}")
    if indices.dim() < 1 or not 1 <= indices.shape[-1] <= MAX_BALANCE_TOP_K or indices.shape[:-1] != logits.shape[:-1]:
        raise ValueError(f"indices must be [..., K] for the logits' {tuple(logits.shape[:-1])} tokens, K of 1 to {MAX_BALANCE_TOP_K}, got "
                         f"{tuple(indices.shape)}")
    if T * indices.shape[-1] >= 2 ** 31:   # the counts are int32
        raise ValueError(f"fewer than 2^31 slots, got {T} tokens of {indices.shape[-1]}")
    idx = indices if indices.dim() == 2 else indices.reshape(T, indices.shape[-1])
    if not idx.is_contiguous():
        idx = idx.contiguous()
    cu = cu_seqlens
    if cu is not None:
        if cu.dtype != torch.int32:
            raise TypeError(f"cu_seqlens must be int32, got {cu.dtype}")
        if cu.dim() != 1 or not 1 <= cu.numel() <= MAX_SEQUENCES + 1:
            raise ValueError(f"cu_seqlens must be [S + 1] with S of 0 to {MAX_SEQUENCES}, got {tuple(cu.shape)}")
        cu = cu.contiguous()
    mask = token_mask
    if mask is not None:
        if mask.dtype != torch.bool:
            raise TypeError(f"token_mask must be bool (True: the token counts), got {mask.dtype}")
        if mask.shape != logits.shape[:-1]:
            raise ValueError(f"token_mask must be {tuple(logits.shape[:-1])}, got {tuple(mask.shape)}")
        mask = mask.reshape(T).contiguous()
    index = l2.get_device()
    for name, t in (("indices", idx), ("cu_seqlens", cu), ("token_mask", mask)):
        if t is not None and t.get_device() != index:
            raise ValueError(f"{name} is on {t.device}, the logits on {l2.device}")
    if load_tracker is not None:
        if load_tracker.num_experts != E:
            raise ValueError(f"load_tracker is for {load_tracker.num_experts} experts, the logits for {E}")
        if load_tracker.tokens_per_expert.get_device() != index:
            raise ValueError(f"load_tracker is on {load_tracker.tokens_per_expert.device}, the logits on {l2.device}")
    return l2, idx, cu, mask


def balance_forward(logits: torch.Tensor, indices: torch.Tensor, *, cu_seqlens: Optional[torch.Tensor] = None,
                    token_mask: Optional[torch.Tensor] = None, scores: str = "softmax",
                    z_loss_multiplier: Optional[float] = None, load_tracker=None):
    """(loss, counts, state) of ``balance_loss``'s arguments, state for ``balance_backward``; records no gradient."""
    sigmoid = _scores(scores)
    l2, idx, cu, mask = _check(logits, indices, cu_seqlens, token_mask, load_tracker)
    if l2.requires_grad:
        l2 = l2.detach()
    T, E = l2.shape
    S = 1 if cu is None else cu.numel() - 1
    dev = l2.device
    z = 0.0 if z_loss_multiplier is None else float(z_loss_multiplier)
    nbytes = _lib.size_of("fm_balance_workspace_bytes", T, E, S)
    if nbytes <= _JOINT_BYTES:
        room = (S * E + 65) // 64 * 64   # f and its two factors, then the workspace, on 256 bytes
        f = torch.empty(room + nbytes // 4, dtype=torch.float32, device=dev)
        workspace = f.data_ptr() + 4 * room
    else:
        f = torch.empty(S * E + 2, dtype=torch.float32, device=dev)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        workspace = scratch.data_ptr()
    loss = torch.empty((), dtype=torch.float32, device=dev)
    counts = torch.empty(E if cu is None else (S, E), dtype=torch.int32, device=dev)
    at = f.data_ptr()
    acc, total = (None, None) if load_tracker is None else (load_tracker.tokens_per_expert, load_tracker.total_tokens)
    _lib.call_on(l2, "fm_balance_forward", l2.data_ptr(), l2.stride(0) if T > 1 else E, T, E, idx.data_ptr(), int(idx.dtype == torch.int64),
                 idx.shape[1], _lib.addr(cu), S, _lib.addr(mask), int(sigmoid), z, at, counts.data_ptr(), at + 4 * S * E, loss.data_ptr(),
                 _lib.addr(acc), _lib.addr(total), workspace, nbytes)
    return loss, counts, BalanceState(l2, cu, mask, f, sigmoid, z, logits.shape)


def balance_backward(state: BalanceState, dloss: torch.Tensor, add_to: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dlogits (fp32, the logits' shape): dloss (0-d fp32) times the loss's gradient, zeros for tokens
    that do not count.  ``add_to`` ([T, E] fp32): added to it in place instead.  Records no gradient."""
    l2, cu = state.logits, state.cu_seqlens
    T, E = l2.shape
    S = 1 if cu is None else cu.numel() - 1
    if state.f.numel() < S * E + 2 or (state.mask is not None and state.mask.numel() != T):
        raise ValueError(f"the state's f and mask do not fit {T} tokens, {E} experts and {S} sequences")
    if dloss.dtype != torch.float32 or dloss.numel() != 1:
        raise TypeError(f"dloss must be one float32 value, got {dloss.dtype} {tuple(dloss.shape)}")
    for name, t in (("dloss", dloss), ("add_to", add_to)):
        if t is not None and t.get_device() != l2.get_device():
            raise ValueError(f"{name} is on {t.device}, the logits on {l2.device}")
    if add_to is None:
        out = torch.empty(state.shape, dtype=torch.float32, device=l2.device)
        ld = E
    else:
        if add_to.dtype != torch.float32 or tuple(add_to.shape) != (T, E) or (T > 0 and add_to.stride(1) != 1 and E > 1) \
                or (T > 1 and add_to.stride(0) < E):
            raise ValueError(f"add_to must be a float32 [{T}, {E}] of rows, got {add_to.dtype} {tuple(add_to.shape)} of strides {add_to.stride()}")
        out, ld = add_to, add_to.stride(0) if T > 1 else E
    if T:
        _lib.call_on(l2, "fm_balance_backward", l2.data_ptr(), l2.stride(0) if T > 1 else E, T, E, _lib.addr(cu), S, _lib.addr(state.mask),
                     int(state.sigmoid), state.z_mult, state.f.data_ptr(), state.f.data_ptr() + 4 * S * E, dloss.data_ptr(), out.data_ptr(),
                     ld, int(add_to is not None))
    return out


class _BalanceFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, indices, cu_seqlens, token_mask, scores, z_mult, load_tracker):
        loss, counts, state = balance_forward(logits, indices, cu_seqlens=cu_seqlens, token_mask=token_mask, scores=scores,
                                              z_loss_multiplier=z_mult, load_tracker=load_tracker)
        ctx.save_for_backward(logits, state.cu_seqlens, state.mask, state.f)
        ctx.state = state
        state.logits = state.cu_seqlens = state.mask = state.f = None   # kept by autograd, which sees changes in place
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        return loss, counts

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _dcounts):
        if dloss is None:
            return (None,) * 7
        logits, cu, mask, f = ctx.saved_tensors
        l2 = logits.reshape(-1, logits.shape[-1])
        if l2.stride(1) != 1 or l2.stride(0) < l2.shape[1]:
            l2 = l2.contiguous()
        s = ctx.state
        state = BalanceState(l2, cu, mask, f, s.sigmoid, s.z_mult, s.shape)
        return balance_backward(state, dloss.float()), None, None, None, None, None, None


def balance_loss(logits: torch.Tensor, indices: torch.Tensor, *, cu_seqlens: Optional[torch.Tensor] = None,
                 token_mask: Optional[torch.Tensor] = None, scores: str = "softmax",
                 z_loss_multiplier: Optional[float] = None, load_tracker=None) -> BalanceOutput:
    """BalanceOutput(loss, counts) of router logits [..., E] (fp32) and the chosen experts [..., K] (int64 or int32;
    those outside [0, E) fill no slot), differentiable in the logits.

    ``cu_seqlens`` [S + 1] (int32, ascending, on the device): sequence s is tokens cu_seqlens[s] up to cu_seqlens[s + 1] of the
    flattened batch; tokens before the first and behind the last do not count.  None: all tokens are one sequence.
    ``token_mask`` [...] (bool): only tokens with True count.  The logits of others may hold anything; their gradient is 0.
    ``scores``: "softmax" or "sigmoid" (normalised over the experts).  ``z_loss_multiplier``: adds it times
    the counting tokens' mean of logsumexp(logits)^2.  ``load_tracker`` (``ExpertLoadTracker``): raised by the slots and tokens that count.
    With no token that counts the loss is 0."""
    loss, counts = _BalanceFunction.apply(logits, indices, cu_seqlens, token_mask, scores, z_loss_multiplier, load_tracker)
    return BalanceOutput(loss, counts)
