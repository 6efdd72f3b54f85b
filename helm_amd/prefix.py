"""Decode attention of sequences that share their first pages (``helm_prefix_decode_attn``):
the beams of a prompt (``helm_amd.beams``), requests under one system prompt, questions about one
document.  The pools, page tables and lengths are those of ``paged.paged_decode_attention``;
the pages that a group shares are read once for all of its sequences.

That pays where the sequences' K and V, counted one by one, are more than some 300 MB a call (64,000
to 100,000 tokens of 8 heads of 128): 64 sequences behind 4,096 tokens 35 us for 101, 4 behind 16,384
28 for 32.  Below that ``paged_decode_attention`` over the same tables gets the repeated pages from
the card's last-level cache, and is up to twice as fast (4 behind 1,024: 8.6 us for 17.4)."""
from __future__ import annotations

from typing import Optional

import torch

from helm_amd import _native
from helm_amd.pool4 import _CODES, PreparedPool4Decode, check_scores
from helm_amd.runtime import engine as _engine

_MAX_SEQS, _MAX_GROUPS = 4096, 512      # HELM_PREFIX_MAX_SEQS, _GROUPS


class PreparedPrefixDecode(PreparedPool4Decode):
    """``prefix_decode_attention`` with its arguments checked and its workspace taken once, for
    loops that issue the same shape every step.  ``run`` reads q, pools, page table, lengths
    and groups as they are then, on torch's current stream; runs of one object (its replays
    in graphs among them) share its workspace and `out` and must not overlap.  It may be
    dropped while runs are on their way, on any stream, but not before the last replay
    of a graph that holds one.  It holds addresses: a deep copy or pickle of it is refused."""

    _entry = "helm_prefix_decode_attn"


def prepare_prefix_decode(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                          page_table: torch.Tensor, seq_lens: torch.Tensor,
                          group_starts: torch.Tensor, shared_pages: torch.Tensor,
                          max_pages: Optional[int] = None, scale: Optional[float] = None,
                          softcap: Optional[float] = None, window: Optional[int] = None,
                          out: Optional[torch.Tensor] = None) -> PreparedPrefixDecode:
    """Arguments as ``prefix_decode_attention``; q must be contiguous and 16-byte aligned, so
    that later runs see what is written to it."""
    if not q.is_contiguous():
        raise ValueError("a prepared call reads q in place: it must be contiguous")
    return PreparedPrefixDecode(*_decode_args(q, k_pool, v_pool, page_table, seq_lens,
                                              group_starts, shared_pages, max_pages, scale, softcap,
                                              window, out, in_place=True))


def prefix_decode_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                            page_table: torch.Tensor, seq_lens: torch.Tensor,
                            group_starts: torch.Tensor, shared_pages: torch.Tensor,
                            max_pages: Optional[int] = None, scale: Optional[float] = None,
                            softcap: Optional[float] = None, window: Optional[int] = None,
                            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of q [R, Hq, q_len, D] over pooled pages, the pages that a group's sequences
    share read once for the group.

    k_pool / v_pool: [n_slots, Hkv, page, D] of q's type (float16 or bfloat16), D 64, 128 or
    256, page a multiple of 16, dense [page, D] parts, one pair of strides (an arena's
    ``[:, 0]`` and ``[:, 1]``); page_table: int32 [R, >= max_pages], each sequence's whole
    table, slots outside the pool count as hidden pages; seq_lens: int32 [R] tokens.
    group_starts: int32 [n + 1], ascending: group g is sequences group_starts[g] ..
    group_starts[g + 1], whose first shared_pages[g] (int32 [n]) table columns hold the same
    slots, full pages or not; sequences outside every group share nothing, nor does any where
    the starts do not ascend.  All on the device and read there: one launch shape serves any
    lengths and groups.

    The q_len rows are the sequence's last tokens: row s stands at p = len - q_len + s and
    sees tokens up to p, with `window` only the last `window` of those.  Hidden tokens (those
    past max_pages too) take no part whatever they hold, a visible infinity or NaN in V counts
    at any weight, and a row that sees nothing is zeros.  Weights are held to 2^-16 (bfloat16)
    or 2^-22 of themselves, sums in 32 bits; weights reach 2^8 before the division, so that
    bfloat16 V of about 2^120 and more over the number of tokens may overflow.  At most 4,096
    sequences and 512 groups.  out: contiguous; it may be q itself, but share memory with
    no other operand.  Returns out [R, Hq, q_len, D] in q's dtype."""
    idx, args, out, _ = _decode_args(q, k_pool, v_pool, page_table, seq_lens, group_starts,
                                     shared_pages, max_pages, scale, softcap, window, out)
    _engine.launch_on(idx, "helm_prefix_decode_attn", *args)
    return out


def _decode_args(q, k_pool, v_pool, page_table, seq_lens, group_starts, shared_pages, max_pages,
                 scale, softcap, window, out, in_place=False):
    """Checks the operands; (device, C-ABI arguments up to the stream, out, tensors to keep)."""
    if q.dim() != 4 or k_pool.dim() != 4:
        raise ValueError("q must be [R, Hq, q_len, D], the pools [n_slots, Hkv, page, D]")
    R, Hq, S, D = q.shape
    n_slots, Hkv, P, Dk = k_pool.shape
    if Dk != D or v_pool.shape != k_pool.shape or Hkv < 1 or Hq < 1 or Hq % Hkv or S < 1:
        raise ValueError("the pools do not match q's heads")
    if (q.dtype != torch.float16 and q.dtype != torch.bfloat16) or k_pool.dtype != q.dtype or \
            v_pool.dtype != q.dtype:
        raise TypeError("q and the pools must share float16 or bfloat16")
    if D not in (64, 128, 256):
        raise NotImplementedError(f"shared-prefix decode takes head_dim 64, 128 or 256, not {D}")
    if P < 16 or P % 16:
        raise ValueError("page_size must be a multiple of 16")
    ss, sh, sp, sd = k_pool.stride()
    if v_pool.stride() != k_pool.stride():
        raise ValueError("k_pool and v_pool must share strides")
    if k_pool.numel() and (sd != 1 or sp != D or sh % 8 or ss % 8 or k_pool.data_ptr() % 16
                           or v_pool.data_ptr() % 16):
        raise ValueError("the pools need dense [page, D] parts, 16-byte aligned")
    i32 = torch.int32
    if page_table.dtype != i32 or seq_lens.dtype != i32 or group_starts.dtype != i32 or \
            shared_pages.dtype != i32:
        raise TypeError("page_table, seq_lens, group_starts and shared_pages must be int32")
    n = shared_pages.numel()
    if page_table.dim() != 2 or page_table.size(0) != R or seq_lens.shape != (R,):
        raise ValueError("page_table must be [R, >=max_pages] and seq_lens [R]")
    if shared_pages.shape != (n,) or group_starts.shape != (n + 1,):
        raise ValueError("group_starts must be [n + 1] and shared_pages [n]")
    if (page_table.stride(1) != 1 and page_table.size(1) > 1) or not (
            seq_lens.is_contiguous() and group_starts.is_contiguous()
            and shared_pages.is_contiguous()):
        raise ValueError("page_table rows, seq_lens, group_starts and shared_pages must be dense")
    if max_pages is None:
        max_pages = page_table.size(1)
    if not 0 <= max_pages <= page_table.size(1):
        raise ValueError("max_pages must be 0 to the table's width")
    if max_pages * P > 0x7ffff000:
        raise ValueError("a table's pages hold at most 2^31 - 4096 tokens")
    if R > _MAX_SEQS or n > _MAX_GROUPS:
        raise ValueError(f"at most {_MAX_SEQS} sequences and {_MAX_GROUPS} groups")
    if window is not None and window < 0:
        raise ValueError("window must be positive (None or 0: off)")
    scale, cap = check_scores(scale, softcap, D)
    given = out is not None
    if not given:
        out = torch.empty((R, Hq, S, D), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError("out must be contiguous, of q's shape and dtype")
    _engine.refuse_grad("prefix_decode_attention", q, k_pool, v_pool)
    idx = _engine.common_device("prefix_decode_attention", q, k_pool, v_pool, page_table, seq_lens,
                                group_starts, shared_pages, out)
    q = q.contiguous()
    if q.data_ptr() % 16:
        if in_place:
            raise ValueError("a prepared call reads q in place: it must be 16-byte aligned")
        q = q.clone()
    if given:
        if out.data_ptr() % 16:
            raise ValueError("out must be 16-byte aligned")
        _engine.refuse_overlap("prefix_decode_attention", out, q, k_pool, v_pool, page_table,
                               seq_lens, group_starts, shared_pages)
    need = _native.load().helm_prefix_workspace_bytes(R, Hq, Hkv, S, D, n)
    # (a call of its own takes a workspace of its own: calls on other streams, captured ones)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    args = (q.data_ptr(), out.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), n_slots, ss, sh, P,
            page_table.data_ptr(), page_table.stride(0), max_pages, seq_lens.data_ptr(),
            group_starts.data_ptr(), shared_pages.data_ptr(), n, R, Hq, Hkv, S, D, scale, cap,
            min(window or 0, 0x7fffffff), _CODES[q.dtype], ws.data_ptr(), need)
    return idx, args, out, (q, k_pool, v_pool, page_table, seq_lens, group_starts, shared_pages, ws)
