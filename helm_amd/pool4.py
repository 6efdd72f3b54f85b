"""A slot pool whose pages hold K and V in 4 bits, and decode attention over it.

``Pool4`` is the 4-bit counterpart of the slot pools that ``helm_amd.paged`` reads
(same slots, page tables and lengths, 3.76 times as many tokens in the same memory);
``Pool4.write`` puts a step's K and V rows into it, ``Pool4.read`` gets their values
back, ``pool4_decode_attention`` attends over its pages.

A value is held as an E2M1 code (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives) times
its group's power of two, a group being 32 dims of one token and head: the smallest
2^e, -125 <= e <= 125, that brings the group's largest magnitude to 7 or less; values go
to the nearest code (ties to the even one), those above 6 to 6.  A group that holds an
infinity or NaN stands for NaN.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from helm_amd import _native
from helm_amd.runtime import engine as _engine

_DIMS = (64, 128, 256)
_CODES = {torch.float16: _native.HELM_F16, torch.bfloat16: _native.HELM_BF16,
          torch.float32: _native.HELM_F32}
_SCORE_MAX = 2.0 ** 126


class Pool4:
    """`n_slots` pages of `page_size` tokens (a multiple of 16) of `num_kv_heads` heads
    of `head_dim` 64, 128 or 256, in 4 bits.  ``data`` is the storage, uint8
    ``[n_slots, Hkv, page_size / 16, 17 * head_dim]``; what its bytes mean is the
    library's affair (copying whole slots of it moves pages)."""

    def __init__(self, n_slots: int, num_kv_heads: int, head_dim: int, page_size: int = 16,
                 device="cuda"):
        if head_dim not in _DIMS:
            raise NotImplementedError(f"a 4-bit pool has head_dim 64, 128 or 256, not {head_dim}")
        if n_slots < 0 or n_slots > 0x7fffffff or num_kv_heads < 1:
            raise ValueError("n_slots must be 0 to 2^31 - 1 and num_kv_heads at least 1")
        if page_size < 16 or page_size % 16:
            raise ValueError("page_size must be a multiple of 16")
        self.n_slots, self.num_kv_heads = n_slots, num_kv_heads
        self.head_dim, self.page_size = head_dim, page_size
        self._data = torch.zeros((n_slots, num_kv_heads, page_size // 16, 17 * head_dim),
                                dtype=torch.uint8, device=device)
        # the C-ABI's arguments of a write or read behind the storage's address, which is
        # taken at each call: a copied or unpickled pool has its own
        self._shape = (n_slots, page_size, num_kv_heads, head_dim)

    @property
    def data(self) -> torch.Tensor:
        """The storage (one tensor for the pool's life)."""
        return self._data

    def _slots(self, slot_map: torch.Tensor) -> int:
        if slot_map.dtype != torch.int64:
            raise TypeError("slot_map must be int64")
        if slot_map.dim() != 1 or not slot_map.is_contiguous():
            raise ValueError("slot_map must be a contiguous [n]")
        return slot_map.numel()

    def write(self, k: torch.Tensor, v: torch.Tensor, slot_map: torch.Tensor) -> None:
        """Rows n of k and v ([n, Hkv, D] float16, bfloat16 or float32, any strides) into
        row slot_map[n] (int64, slot * page_size + token; outside the pool, -1 for
        instance: skipped).  Each row needs a slot of its own: what two rows of one call
        leave in one they share is undefined (codes of one under the other's exponents;
        other rows are as they should be)."""
        n = self._slots(slot_map)
        want = (n, self.num_kv_heads, self.head_dim)
        if k.shape != want or v.shape != want:
            raise ValueError(f"Pool4.write: k and v must be {list(want)}, one row a slot")
        code = _CODES.get(k.dtype)
        if code is None or v.dtype != k.dtype:
            raise TypeError("k and v must share float16, bfloat16 or float32")
        _engine.refuse_grad("Pool4.write", k, v)
        idx = _engine.common_device("Pool4.write", self._data, k, v, slot_map)
        unit = 4 if code == _native.HELM_F32 else 8
        k, *k_at = _rows16(k, unit)
        v, *v_at = _rows16(v, unit)
        _engine.launch_on(idx, "helm_pool4_write", self._data.data_ptr(), *self._shape,
                          slot_map.data_ptr(), n, *k_at, *v_at, code)

    def read(self, slot_map: torch.Tensor, dtype: torch.dtype = torch.bfloat16
             ) -> Tuple[torch.Tensor, torch.Tensor]:
        """The values held in rows slot_map, (k, v) [n, Hkv, D] of `dtype` (exact but for
        its rounding); zeros for rows outside the pool."""
        n = self._slots(slot_map)
        code = _CODES.get(dtype)
        if code is None:
            raise TypeError("values are read as float16, bfloat16 or float32")
        idx = _engine.common_device("Pool4.read", self._data, slot_map)
        H, D = self.num_kv_heads, self.head_dim
        k, v = slot_map.new_empty((2, n, H, D), dtype=dtype).unbind(0)
        _engine.launch_on(idx, "helm_pool4_read", self._data.data_ptr(), *self._shape,
                          slot_map.data_ptr(), n, k.data_ptr(), H * D, D, v.data_ptr(), H * D, D,
                          code)
        return k, v


def _rows16(x: torch.Tensor, unit: int) -> tuple:
    """(x, its address, token and head stride): x [n, H, D] itself where its rows are dense,
    16-byte aligned (multiples of `unit` elements) and less than 2^25 elements apart (the
    kernels' addressing), else a copy."""
    s0, s1, s2 = x.stride()
    at = x.data_ptr()
    if s2 != 1 or s0 % unit or s1 % unit or s0 > 1 << 25 or at & 15:
        x = torch.empty(x.shape, dtype=x.dtype, device=x.device).copy_(x)
        (s0, s1, _), at = x.stride(), x.data_ptr()
    return x, at, s0, s1


class PreparedPool4Decode:
    """``pool4_decode_attention`` with its arguments checked and its workspace taken
    once, for loops that issue the same shape every step.  ``run`` reads q, page table,
    lengths, mask and pool as they are then, on torch's current stream; runs of one
    object (its replays in graphs among them) share its workspace and `out` and must
    not overlap.  It may be dropped while runs are on their way, on any stream, but not
    before the last replay of a graph that holds one.  It holds addresses: a deep copy or
    pickle of it is refused."""

    _entry = "helm_pool4_decode_attn"

    def __init__(self, idx, args, out, keep):
        self._idx, self._args, self.out, self._keep = idx, args, out, keep
        self._streams = set()              # those that the workspace and out are recorded on

    def __copy__(self) -> "PreparedPool4Decode":
        return type(self)(self._idx, self._args, self.out, self._keep)

    def __reduce_ex__(self, protocol):
        raise TypeError("a prepared call holds its operands' addresses: prepare the copies' own")

    def run(self) -> torch.Tensor:
        stream = _engine.launch_on(self._idx, self._entry, *self._args)
        if stream not in self._streams:
            for t in (self.out, self._keep[-1]):
                t.record_stream(torch.cuda.current_stream(self._idx))
            self._streams.add(stream)
        return self.out


def prepare_pool4_decode(q: torch.Tensor, pool: Pool4, page_table: torch.Tensor,
                         seq_lens: torch.Tensor, max_pages: Optional[int] = None,
                         scale: Optional[float] = None, softcap: Optional[float] = None,
                         attention_mask: Optional[torch.Tensor] = None, causal: bool = False,
                         out: Optional[torch.Tensor] = None) -> PreparedPool4Decode:
    """Arguments as ``pool4_decode_attention``; q must be contiguous and the mask one that
    is read as given (float32, bfloat16 or float16, dense rows), so that later runs
    see what is written to them."""
    if not q.is_contiguous():
        raise ValueError("a prepared call reads q in place: it must be contiguous")
    m = attention_mask
    if m is not None and (m.dtype not in _CODES or m.stride(-1) != 1):
        raise ValueError("a prepared call reads the mask in place: float32, bfloat16 or "
                         "float16 with dense rows")
    return PreparedPool4Decode(*_decode_args(q, pool, page_table, seq_lens, max_pages, scale,
                                             softcap, attention_mask, causal, out, in_place=True))


def pool4_decode_attention(q: torch.Tensor, pool: Pool4, page_table: torch.Tensor,
                           seq_lens: torch.Tensor, max_pages: Optional[int] = None,
                           scale: Optional[float] = None, softcap: Optional[float] = None,
                           attention_mask: Optional[torch.Tensor] = None, causal: bool = False,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of q [B, Hq, q_len, D] (float16 or bfloat16) over 4-bit pages, the
    arguments of ``paged.paged_decode_attention``; made for single tokens and a few drafts
    (every 16 query rows of a KV head read its pages again).

    page_table: int32 [B, >= max_pages] slots of the pool (others count as hidden
    pages); seq_lens: int32 [B] tokens, on the device; attention_mask: additive
    [B|1, Hq|1, q_len|1, T], tokens from T on are hidden; causal: the q_len rows are
    the sequence's last tokens, each sees those up to its own.  Hidden tokens (-inf in
    the mask among them) take no part whatever they hold, and a row that sees nothing
    is zeros.  out: contiguous; it may be q itself, but share memory with no other
    operand.  Returns out [B, Hq, q_len, D] in q's dtype."""
    idx, args, out, _ = _decode_args(q, pool, page_table, seq_lens, max_pages, scale, softcap,
                                     attention_mask, causal, out)
    _engine.launch_on(idx, "helm_pool4_decode_attn", *args)
    return out


def check_scores(scale: Optional[float], softcap: Optional[float], D: int) -> Tuple[float, float]:
    """(scale, softcap or 0) of an attention call: numbers whose products in the kernels'
    fp32 (by log2 e, by one another's inverse) stay finite."""
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    cap = 0.0 if softcap is None else float(softcap)
    if not abs(scale) <= _SCORE_MAX:
        raise ValueError("scale must be finite, 2^126 at most in magnitude")
    if cap and not 1.0 / _SCORE_MAX <= cap <= _SCORE_MAX:
        raise ValueError("softcap must be a positive number, 2^-126 to 2^126 (None or 0: off)")
    if cap and abs(scale) / cap > _SCORE_MAX:
        raise ValueError("scale / softcap must be 2^126 at most")
    return scale, cap


def _decode_args(q, pool, page_table, seq_lens, max_pages, scale, softcap, mask, causal, out,
                 in_place=False):
    """Checks the operands; (device, C-ABI arguments up to the stream, out, tensors to keep)."""
    if q.dim() != 4:
        raise ValueError("q must be [B, Hq, q_len, D]")
    B, Hq, S, D = q.shape
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("queries over a 4-bit pool are float16 or bfloat16")
    if D != pool.head_dim or Hq < 1 or Hq % pool.num_kv_heads or S < 1:
        raise ValueError("q does not match the pool's heads")
    if page_table.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise TypeError("page_table and seq_lens must be int32")
    if page_table.dim() != 2 or page_table.size(0) != B or seq_lens.shape != (B,):
        raise ValueError("page_table must be [B, >=max_pages] and seq_lens [B]")
    if (page_table.stride(1) != 1 and page_table.size(1) > 1) or not seq_lens.is_contiguous():
        raise ValueError("page_table rows and seq_lens must be dense")
    if max_pages is None:
        max_pages = page_table.size(1)
    if not 0 <= max_pages <= page_table.size(1):
        raise ValueError("max_pages must be 0 to the table's width")
    scale, cap = check_scores(scale, softcap, D)
    m, ms, width = None, (0, 0, 0), 0
    if mask is not None:
        if mask.dim() != 4 or mask.size(0) not in (1, B) or mask.size(1) not in (1, Hq) or \
                mask.size(2) not in (1, S) or mask.size(3) < 1:
            raise ValueError("attention_mask must be [B|1, Hq|1, q_len|1, T]")
        if not mask.is_floating_point():
            raise TypeError("attention_mask is additive: a floating-point tensor")
        m = mask if mask.dtype in _CODES else mask.float()
        if m.stride(3) != 1:
            m = m.contiguous()
        ms = tuple(m.stride(i) if m.size(i) > 1 else 0 for i in range(3))
        width = m.size(3)
    given = out is not None
    if not given:
        out = torch.empty((B, Hq, S, D), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError("out must be contiguous, of q's shape and dtype")
    masks = () if m is None else (m,)
    _engine.refuse_grad("pool4_decode_attention", q, *masks)
    idx = _engine.common_device("pool4_decode_attention", q, pool.data, page_table, seq_lens, out,
                                *masks)
    q = q.contiguous()
    if q.data_ptr() % 16:
        if in_place:
            raise ValueError("a prepared call reads q in place: it must be 16-byte aligned")
        q = q.clone()
    if given:
        _engine.refuse_overlap("pool4_decode_attention", out, q, pool.data, page_table, seq_lens,
                               *masks)
    lib = _native.load()
    need = lib.helm_pool4_workspace_bytes(B, Hq, pool.num_kv_heads, S, D, max_pages,
                                          pool.page_size)
    # (a call of its own takes a workspace of its own: calls on other streams, captured ones)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    args = (q.data_ptr(), out.data_ptr(), pool.data.data_ptr(), pool.n_slots, pool.page_size,
            page_table.data_ptr(), page_table.stride(0), max_pages,
            seq_lens.data_ptr(), B, Hq, pool.num_kv_heads, S, D, scale, cap,
            m.data_ptr() if m is not None else None, *ms, width,
            _CODES[m.dtype] if m is not None else _native.HELM_F32, int(bool(causal)),
            _CODES[q.dtype], ws.data_ptr(), need)
    return idx, args, out, (q, pool, page_table, seq_lens, m, ws)
