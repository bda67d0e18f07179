"""The 8-bit activations' format and the balance loss in float64, for the tests."""

import torch

BLOCK = 32
SUM_FLOOR = 1e-8


def power(k):
    """2^k in float64, by its bits (torch.ldexp multiplies by a power in float32, which is not exact on every device)."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def kept(x):
    """x [..., cols] float64 as the values that its 8 bits stand for: blocks of 32, s = 2^max(floor(log2 max) - 6, -127)."""
    cols = x.shape[-1]
    out = torch.empty_like(x)
    for c in range(0, cols, BLOCK):
        v = x[..., c:c + BLOCK]
        top = v.abs().amax(-1, keepdim=True)
        exponent = (torch.frexp(top).exponent - 1).clamp_min(-121)
        s = power(exponent - 6)
        q = torch.round(v / s).clamp(-127, 127)
        out[..., c:c + BLOCK] = torch.where(torch.isfinite(top), q * s, torch.nan)
    return out


def step(x):
    """s of every value of x, float64."""
    cols = x.shape[-1]
    out = torch.empty_like(x)
    for c in range(0, cols, BLOCK):
        top = x[..., c:c + BLOCK].abs().amax(-1, keepdim=True)
        out[..., c:c + BLOCK] = power((torch.frexp(top).exponent - 1).clamp_min(-121) - 6)
    return out


def balance(logits, indices, borders=None, mask=None, scores="softmax", z=0.0):
    """(loss, counts [S, E]) of float64 logits [T, E], differentiable; borders a list."""
    T, E = logits.shape
    borders = [0, T] if borders is None else borders
    counts, losses, lse = [], [], []
    for lo, hi in zip(borders, borders[1:]):
        rows = torch.arange(lo, hi)
        if mask is not None:
            rows = rows[mask[lo:hi].cpu()]
        rows = rows.to(logits.device)
        idx = indices[rows].flatten()
        c = torch.bincount(idx[(idx >= 0) & (idx < E)].long(), minlength=E)
        counts.append(c)
        if len(rows) == 0:
            continue
        picked = logits[rows]
        if scores == "softmax":
            p = torch.softmax(picked, dim=1)
        else:
            p = torch.sigmoid(picked)
            p = p / (p.sum(1, keepdim=True) + SUM_FLOOR)
        losses.append(E * (c.double() / len(rows) * p.mean(0)).sum())
        lse.append(torch.logsumexp(picked, dim=1))
    counts = torch.stack(counts) if counts else torch.zeros(0, E, dtype=torch.int64, device=logits.device)
    if not losses:
        return logits.new_zeros(()), counts
    loss = torch.stack(losses).mean()
    if z:
        loss = loss + z * torch.cat(lse).square().mean()
    return loss, counts
