"""Sampling from logits: kernel_fn(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0).

logits [.., vocab] (float32, float16 or bfloat16) and one random number u in [0, 1) for each row ([..],
float32) give one token each, int64 [..]. With M a row's maximum and w_i = exp((x_i - M) / temperature), in
falling order (equal logits: lowest index first), each step on what the one before has left:
  min_p  keeps w_i >= min_p (0: all)
  top_k  keeps the first top_k (0: all)
  top_p  keeps the shortest prefix whose mass reaches top_p of theirs (1: all; one element at least)
and the token is the first element whose running mass exceeds u times the mass kept. temperature 0 is
greedy: the maximum, lowest index; others count as 1e-20 at least. Every setting is a number or a tensor with one
value per row (float32; top_k int32), where a value below its range counts as 0, top_p and min_p above 1 as 1.

The random numbers are the caller's, so a seed gives the same tokens whatever the batch; weights and sums
are exact to better than 2^-40 and add up in no particular order, so a row and its number always give the
same token. A row that holds a NaN or nothing but -inf gives -1, as does one whose setting (from a tensor)
is a NaN or, for the temperature, outside 0 .. 1e30; a number like that is refused. +inf counts as the
largest finite float32. u below 0 counts as
0, above 1 - 2^-24 as that. Vocabularies up to 2^20. Runs ak_sample (sample.hip).
"""
from __future__ import annotations

import torch

from . import _ops
from .host import _check

KERNEL_TYPE = "sample"
MAX_VOCAB = 1 << 20


def _setting(name: str, v, dtype: torch.dtype, rows: torch.Size, device: torch.device):
    if torch.is_tensor(v):
        if not v.is_cuda:
            raise RuntimeError(f"sample: no CPU path (tensors must be on the GPU; {name} is on {v.device})")
        if v.dtype != dtype or v.shape != rows or v.device != device:
            raise ValueError(f"sample: {name} must be a number or {dtype} {tuple(rows)} on {device}, got {v.dtype} "
                             f"{tuple(v.shape)} on {v.device}")
        return v.reshape(-1).contiguous()
    if isinstance(v, bool) or not isinstance(v, (int, float)):
        raise ValueError(f"sample: {name} must be a number or a tensor, got {type(v).__name__}")
    return v


def kernel_fn(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
    _check("sample", logits, u)
    if logits.dim() == 0 or not 1 <= logits.shape[-1] <= MAX_VOCAB:
        raise ValueError(f"sample: logits must be [.., 1 .. {MAX_VOCAB}], got {tuple(logits.shape)}")
    rows = logits.shape[:-1]
    if u.dtype != torch.float32 or u.shape != rows or u.device != logits.device:
        raise ValueError(f"sample: u must be float32 {tuple(rows)} on {logits.device}, got {u.dtype} {tuple(u.shape)} on "
                         f"{u.device}")
    t = _setting("temperature", temperature, torch.float32, rows, logits.device)
    k = _setting("top_k", top_k, torch.int32, rows, logits.device)
    p = _setting("top_p", top_p, torch.float32, rows, logits.device)
    m = _setting("min_p", min_p, torch.float32, rows, logits.device)
    if not torch.is_tensor(t) and not 0.0 <= t <= 1e30:
        raise ValueError(f"sample: temperature {t} must be from 0 to 1e30")
    for name, v in (("top_p", p), ("min_p", m)):
        if not torch.is_tensor(v) and not 0.0 <= v <= 1.0:
            raise ValueError(f"sample: {name} {v} must be from 0 to 1")
    if not torch.is_tensor(k) and (not isinstance(k, int) or k < 0):
        raise ValueError(f"sample: top_k {k} must be a whole number, 0 or more")
    x = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    if (x.shape[1] > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    out = torch.empty(rows, device=logits.device, dtype=torch.int64)
    _ops.sample(out, x, u.reshape(-1).contiguous(), t, k if torch.is_tensor(k) else min(k, MAX_VOCAB), p, m)
    return out
