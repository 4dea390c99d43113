"""64-bit restatement of the paged-cache operators for their tests: plain loops over sequences on the CPU."""
from __future__ import annotations

import math

import torch

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


class Batch:
    """A paged cache and one step's rows, on the CPU. chunks / lens: new and cached tokens of each sequence;
    pad: rows behind the last sequence; lead: rows before the first."""

    def __init__(self, chunks, lens, heads, kv_heads, D, page, dtype, seed=0, pad=0, lead=0, slack=1, layout="hnd",
                 shift=0, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.chunks, self.lens, self.page, self.dtype = list(chunks), list(lens), page, dtype
        B = len(chunks)
        self.width = max([max(0, -(-n // page)) for n in lens] + [0]) + slack
        need = sum(max(0, -(-n // page)) for n in lens)
        self.pages = need + 2
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        self.table = torch.full((B, self.width), -7, dtype=torch.int32)  # unused entries are never read
        at = 0
        for b, n in enumerate(lens):
            c = max(0, -(-n // page))
            self.table[b, :c] = order[at:at + c]
            at += c
        starts = [lead]
        for n in chunks:
            starts.append(starts[-1] + n)
        self.T = starts[-1] + pad
        self.starts = torch.tensor(starts, dtype=torch.int32)
        self.lens_t = torch.tensor(self.lens, dtype=torch.int32)

        def rows(h):  # heads inside wider rows, `shift` elements off the row's start
            wide = (torch.randn(self.T, (h + 2) * D + shift, generator=g) * spread).to(dtype)
            return wide[:, shift + D:shift + (h + 1) * D].view(self.T, h, D) if self.T else wide.new_empty(0, h, D)
        self.q, self.k, self.v = rows(heads), rows(kv_heads), rows(kv_heads)

        def cache():
            if layout == "hnd":
                return torch.randn(self.pages, kv_heads, page, D, generator=g).to(dtype)
            if layout == "nhd":
                return torch.randn(self.pages, page, kv_heads, D, generator=g).to(dtype).transpose(1, 2)
            wide = torch.randn(self.pages, kv_heads, page, D + 3, generator=g).to(dtype)  # "odd": rows of odd stride
            return wide[..., 1:1 + D]
        self.kc, self.vc = cache(), cache()

    def dev(self, t):
        """t on the GPU with the strides it has here."""
        if t.numel() == 0:
            return t.to("cuda")
        base = torch.as_strided(t, (t.untyped_storage().nbytes() // t.element_size(),), (1,), 0)
        return torch.as_strided(base.to("cuda"), t.shape, t.stride(), t.storage_offset())

    def index(self):
        return self.table.cuda(), self.starts.cuda(), self.lens_t.cuda()


def visible(b: Batch, s: int, i: int) -> int:
    """How many positions row i of sequence s sees."""
    return max(0, b.lens[s] - b.chunks[s] + i + 1)


def attention(b: Batch, scale=None):
    """(o, tolerance factor per row) in 64 bits; rows outside every sequence NaN in both."""
    T, H, D = b.q.shape
    Hk = b.kc.shape[1]
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    o = torch.full((T, H, D), math.nan, dtype=torch.float64)
    tol = torch.full((T, H, D), math.nan, dtype=torch.float64)
    half = HALF[b.dtype]
    for s in range(len(b.chunks)):
        L = max(0, b.lens[s])
        ids = b.table[s, :-(-L // b.page)].long()
        for hk in range(Hk):
            K = b.kc[ids, hk].reshape(-1, D)[:L].double()
            V = b.vc[ids, hk].reshape(-1, D)[:L].double()
            for i in range(b.chunks[s]):
                row = int(b.starts[s]) + i
                n = visible(b, s, i)
                q = b.q[row, hk * G:(hk + 1) * G].double()
                if n == 0:
                    o[row, hk * G:(hk + 1) * G] = 0.0
                    tol[row, hk * G:(hk + 1) * G] = 0.0
                    continue
                x = q @ K[:n].T * scale
                p = torch.softmax(x, -1)
                out = p @ V[:n]
                # Scores: D products and sums in fp32, each off by 2^-24 of the running absolute sum, one
                # scaling, one exp2 argument (another 2^-24 of its size) and an exp2 of 2^-22. A relative
                # error d of every weight moves the mean of V by at most 2 d max |V|. f16 / bf16 weights
                # are rounded too (half a step), fp32 sums of n weighted values add n 2^-24 at most.
                mag = (q.abs() @ K[:n].abs().T * scale).amax(-1, keepdim=True) if n else 0.0
                d = (D + 6) * 2.0 ** -24 * mag + 2.0 ** -21 + n * 2.0 ** -24 + (half if b.dtype != torch.float32 else 0)
                vmax = V[:n].abs().amax(0, keepdim=True)
                o[row, hk * G:(hk + 1) * G] = out
                tol[row, hk * G:(hk + 1) * G] = 2 * d * vmax + half * out.abs() + TINY[b.dtype]
    return o, tol


def append(b: Batch, cos, sin, interleaved=True):
    """(q', its tolerance, k cache, v cache, k cache tolerance) in 64 bits; q' of untouched rows NaN."""
    T, H, D = b.q.shape
    half_step = HALF[b.dtype]
    q = torch.full((T, H, D), math.nan, dtype=torch.float64)
    qt = torch.zeros_like(q)
    kc, vc = b.kc.double().clone(), b.vc.double().clone()
    kt = torch.zeros_like(kc)

    def turn(x, pos):
        x = x.double()
        y, t = x.clone(), torch.zeros_like(x)
        if cos is None:
            return y, t
        r = 2 * cos.shape[1]
        e0 = torch.arange(0, r, 2) if interleaved else torch.arange(r // 2)
        e1 = e0 + 1 if interleaved else e0 + r // 2
        c, s = cos[pos].double(), sin[pos].double()
        y[:, e0] = x[:, e0] * c - x[:, e1] * s
        y[:, e1] = x[:, e0] * s + x[:, e1] * c
        # two products and a sum, each off by 2^-24 of its value, then the rounding to the type
        m0 = (x[:, e0] * c).abs() + (x[:, e1] * s).abs()
        m1 = (x[:, e0] * s).abs() + (x[:, e1] * c).abs()
        t[:, e0] = 2.0 ** -23 * m0 + half_step * y[:, e0].abs() * (1 + 2.0 ** -20) + half_step * 2.0 ** -22 * m0
        t[:, e1] = 2.0 ** -23 * m1 + half_step * y[:, e1].abs() * (1 + 2.0 ** -20) + half_step * 2.0 ** -22 * m1
        return y, t + TINY[b.dtype] * (t > 0)

    for s in range(len(b.chunks)):
        for i in range(b.chunks[s]):
            row = int(b.starts[s]) + i
            pos = b.lens[s] - b.chunks[s] + i
            if pos < 0 or (cos is not None and pos >= cos.shape[0]):
                continue
            if cos is not None:
                q[row], qt[row] = turn(b.q[row], pos)
            pg = int(b.table[s, pos // b.page]) if pos // b.page < b.width else -1
            if 0 <= pg < b.pages:
                kc[pg, :, pos % b.page], kt[pg, :, pos % b.page] = turn(b.k[row], pos)
                vc[pg, :, pos % b.page] = b.v[row].double()
    return q, qt, kc, vc, kt


def tables(rows, half):
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    return ang.cos().float(), ang.sin().float()
