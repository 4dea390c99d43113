"""Appending to a paged K / V cache: kernel_fn(k, v, k_cache, v_cache, page_table, q_starts, kv_lens, cos=None,
sin=None, q=None, interleaved=True).

One serving step's new tokens, k and v [T, kv_heads, D], go to their slots of k_cache and v_cache
[pages, kv_heads, page_size, D] (any strides with a contiguous last dim: a [pages, page_size, kv_heads, D]
cache is passed as cache.transpose(1, 2)). The T rows are the sequences' tokens one after another:
  q_starts  int32 [B + 1]: sequence b has rows q_starts[b] .. q_starts[b + 1] - 1
  kv_lens   int32 [B]: its cached tokens, the new ones included
  page_table int32 [B, max_pages]: position p is slot p % page_size of page page_table[b, p // page_size]
With fp32 tables cos / sin [positions, rot_dim / 2], k (and q [T, heads, D] when given) is rotated on the
way by its row's own position: the first rot_dim dims, in pairs (2i, 2i + 1) (interleaved, as
rotary_embedding and the LLaMA models here) or (i, i + rot_dim / 2). fp32 arithmetic, one rounding.

Writes the caches in place and returns the rotated q (dense), or None without q. Rows outside every
sequence (a padded batch) are neither read nor written, so their rows of the returned q hold whatever the
allocation held. The index arrays are read by the kernel alone: no synchronisation, and a captured graph
may be replayed after they change. A row whose position is below zero or past the tables writes nothing
and its q is NaN; one whose page number is outside the cache writes no k and v. Runs ak_kv_append
(paged_append.hip).
"""
from __future__ import annotations

import torch

from . import _ops, _paged

KERNEL_TYPE = "kv_append"


def kernel_fn(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              page_table: torch.Tensor, q_starts: torch.Tensor, kv_lens: torch.Tensor,
              cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, q: torch.Tensor | None = None,
              interleaved: bool = True) -> torch.Tensor | None:
    if q is None:
        _paged.check("kv_append", k_cache, v_cache, page_table, q_starts, kv_lens, k=k, v=v)
    else:
        _paged.check("kv_append", k_cache, v_cache, page_table, q_starts, kv_lens, k=k, v=v, q=q)
    if k.shape[1] != k_cache.shape[1] or v.shape[1] != k_cache.shape[1]:
        raise ValueError(f"kv_append: k {tuple(k.shape)} and v {tuple(v.shape)} for {k_cache.shape[1]} KV heads")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if 0 in t.stride() and any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
            raise ValueError(f"kv_append: {name} is an expanded view (strides {t.stride()}): its slots share memory")
    if (cos is None) != (sin is None):
        raise ValueError("kv_append: cos and sin come together")
    if cos is None:
        if q is not None:
            raise ValueError("kv_append: q without cos and sin has nothing done to it")
    else:
        dev = k.get_device()
        if cos.get_device() < 0 or sin.get_device() < 0:
            raise RuntimeError("kv_append: no CPU path (tensors must be on the GPU)")
        if (cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or cos.get_device() != dev
                or sin.get_device() != dev):
            raise ValueError(f"kv_append: cos and sin must be float32 on {k.device}")
        if cos.dim() != 2 or cos.shape != sin.shape or not 0 < 2 * cos.shape[1] <= k.shape[2]:
            raise ValueError(f"kv_append: cos {tuple(cos.shape)} and sin {tuple(sin.shape)} must be "
                             f"[positions, rot_dim / 2] with rot_dim from 2 to {k.shape[2]}")
        cos, sin = cos.contiguous(), sin.contiguous()
    k, v = _paged.row_operand(k), _paged.row_operand(v)
    q_out = None
    if q is not None:
        q = _paged.row_operand(q)
        q_out = q.new_empty(q.shape)
    _ops.kv_append(q_out, k_cache, v_cache, q, k, v, cos, sin, page_table, q_starts, kv_lens, interleaved)
    return q_out
