"""Causal attention of packed whole prompts (``helm_prompt_attn``): the attention of a
step's prompts over their own tokens, any mix of lengths in one launch.  The pools of
``helm_amd.paged`` and ``helm_amd.pool4`` serve the decode steps that follow."""
from __future__ import annotations

from typing import Optional

import torch

from helm_amd.pool4 import _CODES, _rows16, check_scores
from helm_amd.runtime import engine as _engine


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     scale: Optional[float] = None, softcap: Optional[float] = None,
                     window: Optional[int] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Each sequence's rows attend to its own rows up to their own.

    q: [N, Hq, D], k and v: [N, Hkv, D], float16 or bfloat16, D 64, 128 or 256, any
    strides (rows that are not dense and 16-byte aligned are copied first); sequence
    b is rows cu_seqlens[b] .. cu_seqlens[b + 1] (int32 [B + 1] on the device, ascending
    within 0 .. N, as ``paged.batch_tables`` gives it).  window: a row sees its last
    `window` rows only, itself included.  Rows outside every sequence are left as they
    are in `out`, and zeros where `out` is not given.  out: contiguous; it may be q itself,
    but share memory with no other operand.  Returns [N, Hq, D] in q's dtype."""
    qs, kv = q.shape, k.shape
    if len(qs) != 3 or len(kv) != 3 or v.shape != kv or kv[0] != qs[0] or kv[2] != qs[2]:
        raise ValueError("q must be [N, Hq, D], k and v [N, Hkv, D]")
    (N, Hq, D), Hkv, dt = qs, kv[1], q.dtype
    if (dt != torch.float16 and dt != torch.bfloat16) or k.dtype != dt or v.dtype != dt:
        raise TypeError("q, k and v must share float16 or bfloat16")
    if D != 64 and D != 128 and D != 256:
        raise NotImplementedError(f"prompt attention takes head_dim 64, 128 or 256, not {D}")
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError("Hq must be a multiple of Hkv")
    if cu_seqlens.dtype != torch.int32:
        raise TypeError("cu_seqlens must be int32")
    B = cu_seqlens.numel() - 1
    if B < 0 or cu_seqlens.dim() != 1 or not cu_seqlens.is_contiguous():
        raise ValueError("cu_seqlens must be a contiguous [B + 1]")
    if window is not None and window < 0:
        raise ValueError("window must be positive (None or 0: off)")
    scale, cap = check_scores(scale, softcap, D)
    rest = out is None
    if rest:
        out = q.new_empty(qs)
    elif out.shape != qs or out.dtype != dt or not out.is_contiguous():
        raise ValueError("out must be contiguous, of q's shape and dtype")
    _engine.refuse_grad("prompt_attention", q, k, v)
    idx = _engine.common_device("prompt_attention", q, k, v, cu_seqlens, out)
    q, *q_at = _rows16(q, 8)
    k, *k_at = _rows16(k, 8)
    v, *v_at = _rows16(v, 8)
    if not rest:
        _engine.refuse_overlap("prompt_attention", out, q, k, v, cu_seqlens)
    _engine.launch_on(idx, "helm_prompt_attn", *q_at, *k_at, *v_at, out.data_ptr(), Hq * D, D,
                      cu_seqlens.data_ptr(), B, N, Hq, Hkv, D, scale, cap,
                      min(window or 0, 0x7fffffff), rest, _CODES[dt])
    return out
