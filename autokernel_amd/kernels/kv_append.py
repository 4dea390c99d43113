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


def _explain_tables(k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> None:
    if not (cos.is_cuda and sin.is_cuda):
        raise RuntimeError("kv_append: no CPU path (tensors must be on the GPU)")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.device != k.device or sin.device != k.device:
        raise ValueError(f"kv_append: cos and sin must be float32 on {k.device}")
    raise ValueError(f"kv_append: cos {tuple(cos.shape)} and sin {tuple(sin.shape)} must be [positions, rot_dim / 2] "
                     f"with rot_dim from 2 to {k.shape[2]}")


def kernel_fn(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              page_table: torch.Tensor, q_starts: torch.Tensor, kv_lens: torch.Tensor,
              cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, q: torch.Tensor | None = None,
              interleaved: bool = True) -> torch.Tensor | None:
    if q is None:
        _paged.check("kv_append", k_cache, v_cache, page_table, q_starts, kv_lens, "kv", k, v)
    else:
        _paged.check("kv_append", k_cache, v_cache, page_table, q_starts, kv_lens, "kvq", k, v, q)
    heads = k_cache.shape[1]
    if k.shape[1] != heads or v.shape[1] != heads:
        raise ValueError(f"kv_append: k {tuple(k.shape)} and v {tuple(v.shape)} for {heads} KV heads")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if 0 in t.stride() and any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
            raise ValueError(f"kv_append: {name} is an expanded view (strides {t.stride()}): its slots share memory")
    if cos is not None and sin is not None:
        dev, shape = k.get_device(), cos.shape
        if not (cos.get_device() == sin.get_device() == dev and cos.dtype is sin.dtype is torch.float32
                and shape == sin.shape and len(shape) == 2 and 0 < 2 * shape[1] <= k.shape[2]):
            _explain_tables(k, cos, sin)
        cos, sin = cos.contiguous(), sin.contiguous()
    elif cos is not sin:
        raise ValueError("kv_append: cos and sin come together")
    elif q is not None:
        raise ValueError("kv_append: q without cos and sin has nothing done to it")
    k, v = _paged.row_operand(k), _paged.row_operand(v)
    q_out = None
    if q is not None:
        q = _paged.row_operand(q)
        q_out = q.new_empty(q.shape)
    _ops.kv_append(q_out, k_cache, v_cache, q, k, v, cos, sin, page_table, q_starts, kv_lens, interleaved)
    return q_out
