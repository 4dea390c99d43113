"""Argument checks shared by the paged-cache modules (kv_append, paged_attention): what the host can see
without reading device data."""
from __future__ import annotations

import torch

from .host import _DTYPES


_I32 = torch.int32


def check(op: str, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, q_starts: torch.Tensor,
          kv_lens: torch.Tensor, names: str, *rows: torch.Tensor) -> None:
    """ValueError / RuntimeError unless the cache, the index arrays and the row tensors ([T, heads, D], one letter of
    `names` each) fit together on one GPU. One expression for the calls that do (7 us less of CPU than the rules
    one by one); _explain finds what is wrong with the others."""
    ref = rows[0]
    dev, dt, shape, cache, table = ref.get_device(), ref.dtype, ref.shape, k_cache.shape, page_table.shape
    if (dev >= 0 and dt in _DTYPES and len(cache) == 4 and len(shape) == 3 and len(table) == 2
            and cache == v_cache.shape and k_cache.dtype is dt and v_cache.dtype is dt
            and k_cache.get_device() == dev and v_cache.get_device() == dev and page_table.get_device() == dev
            and q_starts.get_device() == dev and kv_lens.get_device() == dev
            and page_table.dtype is _I32 and q_starts.dtype is _I32 and kv_lens.dtype is _I32
            and 1 <= cache[3] <= 256 and cache[1] > 0 and cache[2] > 0 and k_cache.stride(3) == 1
            and v_cache.stride(3) == 1 and kv_lens.shape == table[:1] and q_starts.shape == (table[0] + 1,)
            and q_starts.stride(0) == 1 and (kv_lens.stride(0) == 1 or table[0] <= 1)
            and (page_table.stride(1) == 1 or table[1] <= 1) and (page_table.stride(0) >= table[1] or table[0] <= 1)
            and table[1] * cache[2] < 1 << 31 and shape[2] == cache[3]):
        for t in rows[1:]:
            s = t.shape
            if not (len(s) == 3 and s[0] == shape[0] and s[2] == cache[3] and t.dtype is dt and t.get_device() == dev):
                break
        else:
            return
    _explain(op, k_cache, v_cache, page_table, q_starts, kv_lens, **dict(zip(names, rows)))


def _explain(op: str, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, q_starts: torch.Tensor,
             kv_lens: torch.Tensor, **rows: torch.Tensor) -> None:
    """The error for what does not fit; every rule of check, one by one."""
    ref = next(iter(rows.values()))
    everything = (("k_cache", k_cache), ("v_cache", v_cache), ("page_table", page_table), ("q_starts", q_starts),
                  ("kv_lens", kv_lens), *rows.items())
    for name, t in everything:
        if not t.is_cuda:
            raise RuntimeError(f"{op}: no CPU path (tensors must be on the GPU; {name} is on {t.device})")
    for name, t in everything:
        if t.device != ref.device:
            raise ValueError(f"{op}: {name} is on {t.device}, the rows are on {ref.device}")
    if ref.dtype not in _DTYPES:
        raise ValueError(f"{op}: dtype {ref.dtype} unsupported (float32, float16, bfloat16)")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache), *rows.items()):
        if t.dtype != ref.dtype:
            raise ValueError(f"{op}: {name} has dtype {t.dtype}, the rows have {ref.dtype}")
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError(f"{op}: caches must be [pages, kv_heads, page_size, head_dim] alike, got "
                         f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t.stride(3) != 1 and t.shape[3] > 1:
            raise ValueError(f"{op}: {name}'s last dim must be contiguous (stride {t.stride(3)})")
    if k_cache.shape[1] == 0 or k_cache.shape[2] == 0 or k_cache.shape[3] == 0:
        raise ValueError(f"{op}: empty cache dims {tuple(k_cache.shape)}")
    if k_cache.shape[3] > 256:
        raise ValueError(f"{op}: head_dim {k_cache.shape[3]} unsupported (1 .. 256)")
    for name, t in rows.items():
        if t.dim() != 3 or t.shape[0] != ref.shape[0] or t.shape[2] != k_cache.shape[3]:
            raise ValueError(f"{op}: {name} must be [{ref.shape[0]}, heads, {k_cache.shape[3]}], got {tuple(t.shape)}")
    for name, t, dim in (("page_table", page_table, 2), ("q_starts", q_starts, 1), ("kv_lens", kv_lens, 1)):
        if t.dtype != torch.int32:
            raise ValueError(f"{op}: {name} must be int32, got {t.dtype}")
        if t.dim() != dim or (t.shape[-1] > 1 and t.stride(-1) != 1):
            raise ValueError(f"{op}: {name} must have {dim} dims, the last contiguous, got {tuple(t.shape)}")
    B = kv_lens.shape[0]
    if q_starts.shape[0] != B + 1 or page_table.shape[0] != B:
        raise ValueError(f"{op}: {B} sequences need q_starts [{B + 1}] and page_table [{B}, pages], got "
                         f"{tuple(q_starts.shape)} and {tuple(page_table.shape)}")
    if B > 1 and page_table.stride(0) < page_table.shape[1]:
        raise ValueError(f"{op}: page_table rows overlap (stride {page_table.stride(0)})")
    if page_table.shape[1] * k_cache.shape[2] >= 1 << 31:
        raise ValueError(f"{op}: {page_table.shape[1]} pages of {k_cache.shape[2]} slots pass 2^31 positions")


def row_operand(t: torch.Tensor) -> torch.Tensor:
    """[T, heads, D] with a contiguous last dim (a column slice of a fused projection is read in place)."""
    return t if t.stride(2) == 1 or t.shape[2] <= 1 else t.contiguous()
