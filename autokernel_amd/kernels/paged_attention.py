"""Attention of new tokens over a paged K / V cache: kernel_fn(q, k_cache, v_cache, page_table, q_starts, kv_lens,
sm_scale=None, out=None).

q [T, heads, D] holds the sequences' new tokens one after another, any mix of single tokens and chunks;
k_cache, v_cache, page_table, q_starts and kv_lens are those of kv_append, which has put the new tokens'
keys and values into the cache before. Row t of sequence b stands at position
kv_lens[b] - (q_starts[b + 1] - t) and sees the positions up to its own. heads is a multiple of the
cache's kv_heads (grouped-query attention); sm_scale defaults to D ** -0.5 and must be positive.

Returns [T, heads, D], written into `out` (any row and head strides, q's dtype) when given. Rows outside
every sequence (a padded batch) are left as they were: in a fresh result they hold whatever the allocation
held. A row that sees nothing is zero; what a row does not see has no influence on it, NaN and
infinities among it. A row that sees a position whose page number is outside the cache, or whose
sequence is longer than its page table, is NaN. The index arrays are read by the kernels alone (no
synchronisation; a captured graph may be replayed after they change). Runs ak_paged_attn
(paged_attention.hip), deterministic.
"""
from __future__ import annotations

import torch

from . import _ops, _paged

KERNEL_TYPE = "paged_attention"


def kernel_fn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
              q_starts: torch.Tensor, kv_lens: torch.Tensor, sm_scale: float | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    _paged.check("paged_attention", k_cache, v_cache, page_table, q_starts, kv_lens, "q", q)
    if q.shape[1] % k_cache.shape[1]:
        raise ValueError(f"paged_attention: {q.shape[1]} query heads not a multiple of {k_cache.shape[1]} KV heads")
    scale = float(q.shape[2] ** -0.5 if sm_scale is None else sm_scale)
    if not 0.0 < scale <= 2e38:
        raise ValueError(f"paged_attention: sm_scale {scale} must be above 0, at most 2e38")
    if out is None:
        out = q.new_empty(q.shape)
    elif (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device
          or (out.shape[2] > 1 and out.stride(2) != 1)
          or any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride()))):
        raise ValueError(f"paged_attention: out must be {tuple(q.shape)} {q.dtype} on {q.device}, its last dim "
                         "contiguous and no view that shares elements")
    _ops.paged_attn(out, _paged.row_operand(q), k_cache, v_cache, page_table, q_starts, kv_lens, scale)
    return out
