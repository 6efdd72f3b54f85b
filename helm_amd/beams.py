"""Beam search over a paged cache: the step's choice among the beams' continuations
(``beam_select``) and the block tables that follow from it (``beam_tables``), on the GPU
and without reading anything back.

K beams of a request are K consecutive rows of the step's tables.  They share the pages they
have in common by name (``prefix.prefix_decode_attention`` reads those once for all of
them), and each has a part-filled last page of its own.  A step is

    choice = beam_select(logits, scores)               # [B, K, V] -> K best of each request
    t = beam_tables(choice.parents, table, lens, page_size, pages=store)
    # t.released[:n_released] are free again; batch_tables takes the next token's pages

A request's prompt is cached once: its K rows name the same full pages, and where its last page is
part-filled every row but the first is given a free page there.  With scores of 0, -inf, ...
the first step's choice then comes from row 0, and ``beam_tables`` fills those pages.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Sequence, Union

import torch

from helm_amd import _native
from helm_amd.pool4 import _CODES, Pool4
from helm_amd.runtime import engine as _engine

_MAX = 64                       # HELM_BEAMS_MAX


class BeamChoice(NamedTuple):
    """A step's continuations (``beam_select``), best first, on the device."""
    scores: torch.Tensor        # float32 [B, n] (a sum past its range: the last number), -inf: none
    tokens: torch.Tensor        # int64 [B, n], -1 there
    parents: torch.Tensor       # int32 [B, n], the beam (0 .. K - 1) that it goes on from, -1 there


def beam_select(logits: torch.Tensor, scores: torch.Tensor, n: Optional[int] = None,
                out: Optional[BeamChoice] = None) -> BeamChoice:
    """The n (default K) best continuations of each request's K beams.

    logits: [B, K, V] float16, bfloat16 or float32, rows dense (others are copied first);
    scores: float32 [B, K], the beams' summed log-probabilities.  Token t of beam k scores
    scores[k] + log_softmax(logits[k])[t]; the order is of sums in 64 bits, ties go to the
    lowest k * V + t.  (A beam's log-sum-exp is of 32-bit exponentials, off by some 1e-7, at
    worst 2^-18: as near as that, candidates of different beams may come in either order.)
    A logit of -inf is no candidate, nor is anything of a beam whose score is not finite or
    whose logits hold a NaN or +inf; where fewer than n are left, score -inf, token -1 and
    parent -1 follow.  At most 64 beams and candidates, 65,535 rows.
    out: a former result of the same sizes, written instead of new tensors (it may share no
    memory with an operand; scores may be `out.scores`' copy, not itself)."""
    if logits.dim() != 3 or scores.shape != logits.shape[:2]:
        raise ValueError("logits must be [B, K, V] and scores [B, K]")
    B, K, V = logits.shape
    code = _CODES.get(logits.dtype)
    if code is None:
        raise TypeError("logits are float16, bfloat16 or float32")
    if scores.dtype != torch.float32:
        raise TypeError("scores must be float32")
    if not scores.is_contiguous():
        raise ValueError("scores must be contiguous")
    n = K if n is None else n
    if not (1 <= K <= _MAX and 1 <= n <= _MAX and 1 <= V < 2 ** 31 and B * K <= 65535):
        raise ValueError("beam_select takes 1 to 64 beams and candidates of at most 65535 rows, "
                         "1 to 2^31 - 1 logits each")
    _engine.refuse_grad("beam_select", logits, scores)
    given = out is not None
    if not given:
        out = BeamChoice(scores.new_empty((B, n)), scores.new_empty((B, n), dtype=torch.int64),
                         scores.new_empty((B, n), dtype=torch.int32))
    else:
        for name, t, dt in zip(BeamChoice._fields, out, (torch.float32, torch.int64, torch.int32)):
            if t.shape != (B, n) or t.dtype != dt or not t.is_contiguous():
                raise ValueError(f"out.{name} must be contiguous {dt} [{B}, {n}]")
    idx = _engine.common_device("beam_select", logits, scores, *out)
    if given:
        for i, t in enumerate(out):
            _engine.refuse_shared("beam_select", t, logits, scores, *out[:i])
    sb, sk, sv = logits.stride()
    if sv != 1 and V > 1:
        logits = logits.contiguous()
        sb, sk, _ = logits.stride()
    need = _native.load().helm_beam_select_workspace_bytes(B, K, V, n, code)
    ws = torch.empty(need, dtype=torch.uint8, device=logits.device)
    _engine.launch_on(idx, "helm_beam_select", logits.data_ptr(), sb, sk, code, scores.data_ptr(),
                      B, K, V, n, *(t.data_ptr() for t in out), ws.data_ptr(), need)
    return out


def _overlap(n: int, slot: int, segments: int, step: int, part: int) -> bool:
    """Whether any two of the parts at i * slot + j * step (i < n, j < segments) share memory."""
    if (n > 1 and slot < part) or (segments > 1 and step < part):
        return True
    if n == 1 or slot >= (segments - 1) * step + part:
        return False
    return any(abs(j * step - i * slot) < part for j in range(1, segments)
               for i in (j * step // slot, j * step // slot + 1) if i < n)


class PageStore:
    """The pools of a model's layers, whose pages ``beam_tables`` copies: ``Pool4`` objects, or
    tensors [n_slots, ..., page_size, D] whose pages are made of dense [page_size, D] rows
    (an arena [n_slots, 2, Hkv, page_size, D], or its K and its V as two; slots or heads
    outermost), all of one shape, stride and type and of one slot numbering."""

    def __init__(self, pools: Sequence[Union[torch.Tensor, Pool4]]):
        pools = list(pools)
        if not pools:
            raise ValueError("a PageStore needs a pool")
        tensors = [p.data if isinstance(p, Pool4) else p for p in pools]
        t = tensors[0]
        for p, x in zip(pools, tensors):
            if x.shape != t.shape or x.stride() != t.stride() or x.dtype != t.dtype or \
                    isinstance(p, Pool4) != isinstance(pools[0], Pool4):
                raise ValueError("the pools of a PageStore share shape, strides and type")
        if t.dim() < 3:
            raise ValueError("a pool is [n_slots, ..., page_size, D]")
        es = t.element_size()
        if isinstance(pools[0], Pool4):
            # [n_slots, Hkv, tiles of 16 tokens, bytes]
            self.page_size, tokens, row = pools[0].page_size, 16, t.size(-1)
        else:
            self.page_size, tokens, row = t.size(-2), 1, t.size(-1)
        if t.numel() and ((t.size(-1) > 1 and t.stride(-1) != 1) or
                          (t.size(-2) > 1 and t.stride(-2) != t.size(-1))):
            raise ValueError("a pool's pages need dense [page_size, D] rows")
        segments, step = 1, 0
        for n, s in zip(reversed(t.shape[1:-2]), reversed(t.stride()[1:-2])):
            if n == 1:
                continue
            if segments > 1 and s != segments * step:
                raise ValueError("a page's [page_size, D] parts must lie one stride apart")
            step = step if segments > 1 else s
            segments *= n
        part = t.size(-2) * t.size(-1)
        if segments * part * es >= 2 ** 31:
            raise ValueError("a page holds less than 2^31 bytes")
        # (a slot's parts may lie among other slots': heads outermost)
        if t.numel() and _overlap(t.size(0), t.stride(0), segments, step, part):
            raise ValueError("a pool's pages must not overlap")
        if part == 0 or segments == 0:
            raise ValueError("a pool's pages must hold something")
        self.pools = pools
        self._tensors = tensors
        self._n = len(tensors)
        self._shape = (t.size(0), t.stride(0) * es, segments,
                       (step if segments > 1 else part) * es, tokens, row * es)

    def _addresses(self):
        # (taken at each call: a copied or unpickled store has its own)
        return (ctypes.c_void_p * self._n)(*(t.data_ptr() for t in self._tensors))


class BeamTables(NamedTuple):
    """The tables after a beam step (``beam_tables``), on the device."""
    page_table: torch.Tensor    # int32 [B K, width]
    copies: torch.Tensor        # int32 [B K, 2], the page copied from and to, -1, -1: none
    released: torch.Tensor      # int32 [B K width], full pages that no row names any more, then
    n_released: torch.Tensor    # int32 [1], how many; what lies behind them is left as it is


def beam_tables(parents: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                page_size: int, shared_pages: Optional[torch.Tensor] = None,
                pages: Optional[PageStore] = None,
                out: Optional[BeamTables] = None) -> BeamTables:
    """The block tables after a step in which beam j of each request goes on from beam
    parents[b, j], with the part-filled pages that several go on from copied in every pool.

    parents: int32 [B, K] (``beam_select``'s; a beam outside 0 .. K - 1 goes on from itself);
    page_table: int32 [B * K, width], rows dense; seq_lens: int32 [B * K], the tokens cached (the
    first row's of a request counts: its beams are of one length); shared_pages: int32 [B],
    leading columns in which a request's rows are the same (never released; None: none);
    pages: the pools.

    Full pages are shared by name.  A part-filled page is a row's own: one of a beam's
    children keeps it (the beam itself, else the lowest row), the others take those of the
    beams that none goes on from and get the tokens copied (``copies``; pages outside the
    pool are not copied).  No page comes from a free list; full pages behind the shared ones
    that no row names any more are listed in ``released``.  Columns behind the part-filled page
    are row j's old ones.

    out: a former result of the same sizes, written instead of new tensors; its page_table
    may be page_table itself.  No other output may share memory with an operand, nor any
    operand with the pools' pages."""
    i32 = torch.int32
    if parents.dtype != i32 or page_table.dtype != i32 or seq_lens.dtype != i32:
        raise TypeError("parents, page_table and seq_lens must be int32")
    if parents.dim() != 2 or not parents.is_contiguous():
        raise ValueError("parents must be a contiguous [B, K]")
    B, K = parents.shape
    R = B * K
    if page_table.dim() != 2 or page_table.size(0) != R or seq_lens.shape != (R,):
        raise ValueError("page_table must be [B * K, width] and seq_lens [B * K]")
    if not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be contiguous")
    W = page_table.size(1)
    stride = _table_stride("page_table", page_table)
    if not (1 <= K <= _MAX and R <= 65535 and R * W < 2 ** 31 and 1 <= page_size < 2 ** 31):
        raise ValueError("beam_tables takes 1 to 64 beams of at most 65535 rows, page_size >= 1")
    shared = ()
    if shared_pages is not None:
        if shared_pages.dtype != i32:
            raise TypeError("shared_pages must be int32")
        if shared_pages.shape != (B,) or not shared_pages.is_contiguous():
            raise ValueError("shared_pages must be a contiguous [B]")
        shared = (shared_pages,)
    pools, shape = (), (0, 0, 1, 0, 1, 1)
    if pages is not None:
        if pages.page_size != page_size:
            raise ValueError(f"the pools' pages hold {pages.page_size} tokens, not {page_size}")
        pools, shape = pages._tensors, pages._shape
    if out is None:
        out = BeamTables(page_table.new_empty((R, W)), page_table.new_empty((R, 2)),
                         page_table.new_empty(R * W), page_table.new_empty(1))
    else:
        for name, t, want in zip(BeamTables._fields, out, ((R, W), (R, 2), (R * W,), (1,))):
            if t.shape != want or t.dtype != i32 or (name != "page_table"
                                                     and not t.is_contiguous()):
                raise ValueError(f"out.{name} must be contiguous int32 {list(want)}")
    new, copies, released, count = out
    new_stride = _table_stride("out.page_table", new)
    idx = _engine.common_device("beam_tables", page_table, parents, seq_lens, *shared, *out, *pools)
    need = _native.load().helm_beam_tables_workspace_bytes(B, K, W)
    ws = torch.empty(need, dtype=torch.uint8, device=page_table.device)
    _engine.launch_on(idx, "helm_beam_tables", parents.data_ptr(), B, K, page_table.data_ptr(),
                      stride, W, seq_lens.data_ptr(), page_size,
                      shared_pages.data_ptr() if shared else None, new.data_ptr(), new_stride,
                      copies.data_ptr(), released.data_ptr(), count.data_ptr(),
                      pages._addresses() if pools else None, len(pools), *shape,
                      ws.data_ptr(), need)
    return out


def _table_stride(name: str, t: torch.Tensor) -> int:
    R, W = t.shape
    s0, s1 = t.stride()
    if (s1 != 1 and W > 1) or (s0 < W and R > 1):
        raise ValueError(f"{name} rows must be dense and apart")
    return max(s0, W)
