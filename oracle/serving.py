"""64-bit restatements of the serving operators (tests only): the 4-bit pages' values,
a step's tables, and attention in which hidden keys take no part."""
from __future__ import annotations

import math

import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in float64 for whole e, from its bits (a device's pow may be a step off)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def stored4(x: torch.Tensor) -> torch.Tensor:
    """float64 values that a 4-bit page keeps of x [..., D], from the definition: the
    exponent by search, the code by distance (ties to the even code)."""
    g = x.double().unflatten(-1, (-1, 32))
    a = g.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(g).all(-1, keepdim=True)
    g = torch.where(fine, g, torch.zeros_like(g))
    e = torch.full_like(a, 125.0)
    for k in range(124, -126, -1):                       # the smallest that holds
        e = torch.where(a <= 7 * 2.0 ** k, torch.full_like(e, float(k)), e)
    step = _pow2(e)
    y = g.abs() / step
    best, val = torch.full_like(y, math.inf), torch.zeros_like(y)
    for i in (0, 2, 4, 6, 1, 3, 5, 7):
        d = (y - GRID[i]).abs()
        val = torch.where(d < best, torch.full_like(val, GRID[i]), val)
        best = torch.minimum(best, d)
    out = val * step * torch.sign(g)
    return torch.where(fine, out, torch.full_like(out, math.nan)).flatten(-2)


def tables(new, cached, table, free, page, max_tokens):
    """(cu_seqlens, positions, slot_map, seq_lens, pages_taken, table) as Python lists;
    `table` is a list of rows, copied."""
    table = [list(r) for r in table]
    new, cached = [max(0, n) for n in new], [max(0, c) for c in cached]
    cu, positions, slots, taken = [0], [], [], 0
    for b, (n, c) in enumerate(zip(new, cached)):
        width, old = len(table[b]), -(-c // page)
        fresh = {}
        for col in range(old, -(-(c + n) // page)):
            s = free[taken] if taken < len(free) else -1
            taken += 1
            fresh[col] = s
            if col < width:
                table[b][col] = s
        for i in range(n):
            p = c + i
            s = (table[b][p // page] if p // page < width else -1)
            positions.append(p)
            slots.append(s * page + p % page if s >= 0 else -1)
        cu.append(cu[-1] + n)
    pad = max_tokens - len(positions)
    positions, slots = (positions + [0] * pad)[:max_tokens], (slots + [-1] * pad)[:max_tokens]
    return cu, positions, slots, [n + c for n, c in zip(new, cached)], taken, table


def attend(q, k, v, scale, cap=0.0, hidden=None, mask=None):
    """float64 attention of q [H, S, D] over k, v [T, D] (one KV head): hidden [S, T] or
    [H, S, T] keys, and those under a mask of -inf, take no part whatever they hold; a row
    that sees nothing is zeros.  Returns (out, mean of |v| under the same weights)."""
    q, k, v = q.double(), k.double(), v.double()
    x = torch.matmul(q, k.t().contiguous()) * scale
    if cap:
        x = torch.tanh(x / cap) * cap
    gone = torch.zeros_like(x, dtype=torch.bool)
    if hidden is not None:
        gone = gone | hidden
    if mask is not None:
        m = mask.double().expand_as(x)
        gone = gone | (m == -math.inf)
        x = x + torch.where(m == -math.inf, torch.zeros_like(m), m)
    x = x.masked_fill(gone, -math.inf)
    top = x.amax(-1, keepdim=True) if x.size(-1) else x.new_full(x.shape[:-1] + (1,), -math.inf)
    w = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    w = torch.where(gone, torch.zeros_like(w), w)
    w = w / torch.where(w.sum(-1, keepdim=True) == 0, torch.ones_like(top), w.sum(-1, keepdim=True))
    if torch.isfinite(v).all():
        return torch.matmul(w, v), torch.matmul(w, v.abs())
    out = torch.zeros(q.shape[:-1] + (v.size(-1),), dtype=torch.float64, device=q.device)
    mag = out
    for t in range(v.size(0)):                       # (a hidden key takes no part)
        wt, no = w[..., t:t + 1], gone[..., t:t + 1]
        out = out + torch.where(no, torch.zeros_like(out), wt * v[t])
        mag = mag + torch.where(no, torch.zeros_like(out), wt * v[t].abs())
    return out, mag


def logit_size(q, k, scale):
    """Largest scale * sum |q| |k| of any row and key: what the rounding of a dot product
    is relative to."""
    return (torch.matmul(q.double().abs(), k.double().abs().t().contiguous())
            .amax().item() * abs(scale)) if k.numel() and q.numel() else 0.0
