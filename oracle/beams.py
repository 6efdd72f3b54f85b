"""Restatements of the beam operators (tests only): the choice in 64 bits, the tables as Python
lists, pages as host tensors."""
from __future__ import annotations

import math

import torch


def select(logits, scores, n):
    """(scores float64, tokens, parents) [B, n] of logits [B, K, V] and scores [B, K]; scores past
    fp32's range are its largest or lowest number."""
    B, K, V = logits.shape
    x, s = logits.double().cpu(), scores.double().cpu()
    ok = (~torch.isnan(x) & (x < math.inf)).all(-1) & torch.isfinite(s)
    ok &= (x > -math.inf).any(-1)
    x = torch.where(ok[..., None], x, torch.zeros_like(x))
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    y = torch.where(ok[..., None], torch.where(ok, s, torch.zeros_like(s))[..., None] + x - lse,
                    torch.full_like(x, -math.inf)).flatten(1)
    y = torch.cat([y, y.new_full((B, n), -math.inf)], 1)
    # a stable sort keeps the lowest index of equals first
    best, at = torch.sort(y, dim=1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    none = best == -math.inf
    most = torch.finfo(torch.float32).max
    return (torch.where(none, best, best.clamp(-most, most)),
            torch.where(none, torch.full_like(at, -1), at % V),
            torch.where(none, torch.full_like(at, -1), at // V))


def tables(parents, table, lens, page, shared=None):
    """(new table, copies, released) of one step; lists of rows."""
    B, K = len(parents), len(parents[0])
    W = len(table[0]) if table else 0
    new, copies, released = [list(r) for r in table], [], []
    for b in range(B):
        rows = table[b * K:(b + 1) * K]
        n = max(0, lens[b * K])
        full, part = n // page, n % page != 0
        first = max(0, shared[b]) if shared is not None else 0
        par = [p if 0 <= p < K else j for j, p in enumerate(parents[b])]
        kids = {i: [j for j in range(K) if par[j] == i] for i in range(K)}
        keeper = {i: (i if i in k else k[0]) for i, k in kids.items() if k}
        spare = [i for i in range(K) if not kids[i]]
        tail = []
        for j in range(K):
            tail.append(par[j] if keeper[par[j]] == j else spare.pop(0))
        assert not spare
        for j in range(K):
            out = new[b * K + j]
            for c in range(min(full, W)):
                out[c] = rows[par[j]][c]
            pair = (-1, -1)
            if part and full < W:
                out[full] = rows[tail[j]][full]
                if tail[j] != par[j]:
                    pair = (rows[par[j]][full], out[full])
            copies.append(pair)
        for c in range(first, min(full, W)):
            held = {new[b * K + j][c] for j in range(K)}
            for i in range(K):
                if rows[i][c] not in held and rows[i][c] >= 0:
                    held.add(rows[i][c])
                    released.append(rows[i][c])
    return new, copies, released


def copy_pages(pool, copies, lens, page, K, unit=1):
    """pool [n_slots, ..., page / unit, bytes] with the copies' used rows moved, as a clone."""
    out = pool.clone()
    for r, (s, d) in enumerate(copies):
        if s == d or not (0 <= s < pool.size(0) and 0 <= d < pool.size(0)):
            continue
        n = -(-(max(0, lens[r // K * K]) % page) // unit)
        out[d, ..., :n, :] = pool[s, ..., :n, :]
    return out
