"""The nine AutoKernel ops as drop-in kernel_fn modules backed by libak355 (gfx950 HIP).

Each module exposes KERNEL_TYPE and kernel_fn with the signature of the matching reference.py
function, like the reference's kernels/*.py slot modules. The kernel_fns themselves live in
kernels/host.py (the shape layer shared with the HuggingFace Kernels export), bound here to the
ctypes-backed ops of kernels/_ops.py.

Beside the nine stand the operators of serving from a paged K / V cache, which the reference does not have:
kv_append, paged_attention and sample.
"""
from __future__ import annotations

from . import _ops, host

host.bind(_ops)

from . import (cross_entropy, flash_attention, fused_mlp, kv_append, layernorm, matmul,  # noqa: E402
               paged_attention, reduce, rmsnorm, rotary_embedding, sample, softmax)

MODULES = {m.KERNEL_TYPE: m for m in (matmul, softmax, layernorm, rmsnorm, flash_attention,
                                      fused_mlp, cross_entropy, rotary_embedding, reduce,
                                      kv_append, paged_attention, sample)}
KERNELS = {name: m.kernel_fn for name, m in MODULES.items()}


def get(kernel_type: str):
    """kernel_fn for a KERNEL_TYPE name (bench.py KERNEL_CONFIGS keys, and the serving operators)."""
    try:
        return KERNELS[kernel_type]
    except KeyError:
        raise KeyError(f"unknown kernel type {kernel_type!r}; known: {sorted(KERNELS)}") from None
