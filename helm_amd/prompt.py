"""Causal attention of packed whole prompts (``helm_prompt_attn``): the attention of a
step's prompts over their own tokens, any mix of lengths in one launch.  The pools of
``helm_amd.paged`` and ``helm_amd.pool4`` serve the decode steps that follow."""
from __future__ import annotations

from typing import Optional

import torch

from helm_amd import _native
from helm_amd.pool4 import _aligned_rows, check_scores
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
    are in `out`, and zeros where `out` is not given.  Returns [N, Hq, D] in q's dtype."""
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or k.size(0) != q.size(0) or \
            k.size(2) != q.size(2):
        raise ValueError("q must be [N, Hq, D], k and v [N, Hkv, D]")
    N, Hq, D = q.shape
    Hkv = k.size(1)
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k and v must share float16 or bfloat16")
    if D not in (64, 128, 256):
        raise NotImplementedError(f"prompt attention takes head_dim 64, 128 or 256, not {D}")
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError("Hq must be a multiple of Hkv")
    if cu_seqlens.dtype != torch.int32:
        raise TypeError("cu_seqlens must be int32")
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or not cu_seqlens.is_contiguous():
        raise ValueError("cu_seqlens must be a contiguous [B + 1]")
    if window is not None and window < 0:
        raise ValueError("window must be positive (None or 0: off)")
    scale, cap = check_scores(scale, softcap, D)
    rest = out is None
    if rest:
        out = torch.empty((N, Hq, D), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError("out must be contiguous, of q's shape and dtype")
    _engine.check_operands("prompt_attention", q.device, q, k, v, cu_seqlens, out)
    q, k, v = _aligned_rows(q), _aligned_rows(k), _aligned_rows(v)
    _engine.call_on(q.device, "helm_prompt_attn", q.data_ptr(), q.stride(0), q.stride(1),
                    k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                    out.data_ptr(), out.stride(0), out.stride(1), cu_seqlens.data_ptr(),
                    cu_seqlens.numel() - 1, N, Hq, Hkv, D, scale, cap,
                    min(window or 0, 0x7fffffff), int(rest), _native.dtype_code(q.dtype),
                    _engine.stream_ptr(q.device))
    return out
