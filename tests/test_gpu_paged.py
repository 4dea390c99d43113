"""kv_append and paged_attention against a 64-bit restatement (paged_oracle.py), on the GPU."""
from __future__ import annotations

import math

import pytest
import torch

import paged_oracle as po
from autokernel_amd import kernels
from autokernel_amd._lib import AkError

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
append, attn = kernels.get("kv_append"), kernels.get("paged_attention")


def _bits(t):
    return t.contiguous().view(torch.int32 if t.element_size() == 4 else torch.int16)


def _check_attn(b, what="", scale=None, **kw):
    print(f"paged_attention {what} chunks={b.chunks[:8]} lens={b.lens[:8]} {b.dtype} q={tuple(b.q.shape)} "
          f"cache={tuple(b.kc.shape)}", flush=True)
    want, tol = po.attention(b, scale)
    mark = torch.full(b.q.shape, 7.0, dtype=b.dtype, device="cuda")  # untouched rows keep this
    out = attn(b.dev(b.q), b.dev(b.kc), b.dev(b.vc), *b.index(), sm_scale=scale, out=mark, **kw)
    torch.cuda.synchronize()
    got = out.double().cpu()
    outside = torch.isnan(tol)
    assert (got[outside] == 7.0).all()
    diff = (got - want).abs()[~outside]
    assert (diff <= tol[~outside]).all(), (what, diff.max(), (diff / tol[~outside].clamp(min=1e-30)).max())
    return out


# Page tables for more than 1536 tokens (whatever the sequences hold): keys are sliced, and sequences of more than 16 rows
# per KV head take the large tiles.
LONG = pytest.mark.parametrize("long", [False, True])


def _slack(long, page):
    return 1600 // page + 1 if long else 1


SHAPES = [(8, 2, 128), (40, 1, 64), (4, 4, 64), (6, 2, 64), (32, 2, 128), (3, 1, 80), (5, 5, 17), (4, 2, 256), (16, 1, 128), (2, 1, 1)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,D", SHAPES)
@LONG
def test_attention_shapes(gpu, dtype, heads, kv_heads, D, long):
    # single tokens, chunks, an empty sequence, one whose tokens are all new, a length of one
    b = po.Batch([1, 5, 0, 37, 1, 2], [1, 70, 0, 37, 300, 3], heads, kv_heads, D, 16, dtype, seed=D, pad=3,
                 slack=_slack(long, 16))
    _check_attn(b, "shapes")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 48, 64, 100, 1024])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@LONG
def test_attention_page_sizes(gpu, dtype, page, layout, long):
    b = po.Batch([70, 1, 9], [129, 257, 64], 4, 2, 64, page, dtype, seed=page, layout=layout, slack=_slack(long, page))
    _check_attn(b, f"page {page} {layout}")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shift,layout", [(0, "odd"), (1, "hnd"), (1, "odd"), (4, "nhd")])
def test_attention_unaligned(gpu, dtype, shift, layout):
    b = po.Batch([40, 1], [100, 65], 4, 2, 64, 16, dtype, seed=5, shift=shift, layout=layout)
    _check_attn(b, f"shift {shift} {layout}")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,L", [(1, 1), (1, 2), (1, 63), (1, 64), (1, 65), (2, 64), (63, 63), (64, 64), (65, 65), (33, 127),
                                 (17, 128), (129, 129), (130, 400), (1, 255), (1, 256), (1, 257), (1, 511), (3, 513)])
@LONG
def test_attention_lengths(gpu, dtype, n, L, long):
    _check_attn(po.Batch([n], [L], 8, 2, 128, 16, dtype, seed=L, slack=_slack(long, 16)), "lengths")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,D,page", [(32, 4, 128, 16), (16, 16, 64, 48)])
def test_attention_large_tiles_unsliced(gpu, dtype, heads, kv_heads, D, page):
    """Rows enough for the large tiles over short tables; among them rows whose masked values are not finite, and a page
    outside the cache."""
    b = po.Batch([600, 1, 17, 130], [900, 40, 33, 129], heads, kv_heads, D, page, dtype, seed=D, lead=1, pad=2)
    _check_attn(b, "large tiles")
    last = int(b.table[0, 899 // page])
    b.vc[last, :, 899 % page] = float("nan")
    b.kc[last, :, 899 % page] = float("inf")
    b.table[3, 0] = b.pages
    want, tol = po.attention(po.Batch([600, 1, 17, 130], [900, 40, 33, 129], heads, kv_heads, D, page, dtype, seed=D, lead=1,
                                      pad=2))
    out = attn(b.dev(b.q), b.dev(b.kc), b.dev(b.vc), *b.index()).double().cpu()
    bad = torch.zeros(b.T, dtype=torch.bool)
    bad[600] = True   # the row of the last position
    bad[620:749] = True  # (the first of the 130 rows sees nothing)
    assert torch.isnan(out[bad]).all()
    good = ~bad
    good[0] = good[749:] = False
    assert ((out - want).abs()[good] <= tol[good]).all() and (out[619] == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,D", [(8, 2, 128), (4, 4, 64), (3, 1, 48)])
def test_attention_sliced(gpu, dtype, heads, kv_heads, D):
    """Long caches: keys sliced over blocks, slices of very different sequences, rows that see none of some."""
    b = po.Batch([1, 1, 20, 1], [9001, 3, 2500, 700], heads, kv_heads, D, 16, dtype, seed=1, pad=2)
    _check_attn(b, "sliced")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,D,page", [(8, 2, 128, 16), (12, 4, 64, 24), (2, 2, 64, 8), (32, 2, 128, 32), (4, 2, 96, 16)])
@pytest.mark.parametrize("B", [6, 40])
def test_attention_single_tokens_sliced(gpu, dtype, heads, kv_heads, D, page, B):
    """Decode steps over long and short caches, a sequence without a new token among them, with few rows and with many."""
    g = torch.Generator().manual_seed(B + D)
    lens = [2600, 1, 257, 0, 513, 1537] + torch.randint(1, 1200, (B - 6,), generator=g).tolist()
    b = po.Batch([1, 1, 1, 0, 1, 1] + [1] * (B - 6), lens, heads, kv_heads, D, page, dtype, seed=B, pad=1)
    _check_attn(b, "single tokens")


@pytest.mark.parametrize("B", [63, 64, 65, 130, 300])
def test_attention_many_sequences(gpu, B):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 40, (B,), generator=g).tolist()
    chunks = [min(n, int(c)) for n, c in zip(lens, torch.randint(0, 4, (B,), generator=g))]
    _check_attn(po.Batch(chunks, lens, 4, 2, 64, 8, BF16, seed=B, pad=1), f"{B} sequences")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@LONG
def test_attention_rows_that_see_nothing(gpu, dtype, long):
    """Fewer cached tokens than rows: the first rows' positions are below zero."""
    b = po.Batch([5, 150, 1, 40], [2, 30, 0, -3], 8, 2, 128, 16, dtype, seed=3, lead=2, pad=2, slack=_slack(long, 16))
    out = _check_attn(b, "empty rows")
    assert (out[2:5] == 0).all() and (out[5] != 0).any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,D,page", [(8, 2, 128, 16), (4, 4, 64, 64), (2, 1, 40, 8)])
@pytest.mark.parametrize("chunks,lens", [([50, 1], [200, 700]), ([300], [1300])])
@LONG
def test_attention_garbage_beside_the_keys(gpu, dtype, heads, kv_heads, D, page, chunks, lens, long):
    """NaN and infinities in later tokens' keys and values, in slots past the end and in unused pages."""
    b = po.Batch(chunks, lens, heads, kv_heads, D, page, dtype, seed=11, slack=_slack(long, page))
    # the last new token of the first sequence is NaN / inf: rows before it must not see it
    pos = lens[0] - 1
    b.kc[int(b.table[0, pos // page]), :, pos % page] = float("nan")
    b.vc[int(b.table[0, pos // page]), :, pos % page, ::2] = float("inf")
    b.vc[int(b.table[0, pos // page]), :, pos % page, 1::2] = float("nan")
    used = torch.zeros(b.pages, page, dtype=torch.bool)
    for s, L in enumerate(lens):
        for p in range(L):
            used[int(b.table[s, p // page]), p % page] = True
    for c in (b.kc, b.vc):
        c.transpose(1, 2)[~used] = float("nan")
    want, tol = po.attention(b)
    out = attn(b.dev(b.q), b.dev(b.kc), b.dev(b.vc), *b.index()).double().cpu()
    last = chunks[0] - 1
    assert torch.isnan(out[last]).all()
    ok = [t for t in range(b.T) if t != last]
    assert ((out - want).abs()[ok] <= tol[ok]).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [64, 128, 24])
@LONG
def test_attention_infinite_values(gpu, dtype, D, long):
    """An infinite V entry that a row sees makes that dim infinite, and no other dim or row."""
    b = po.Batch([40, 1], [100, 300], 4, 2, D, 16, dtype, seed=2, spread=0.5, slack=_slack(long, 16))
    b.vc[int(b.table[0, 80 // 16]), 1, 80 % 16, 3] = float("inf")
    out = attn(b.dev(b.q), b.dev(b.kc), b.dev(b.vc), *b.index()).double().cpu()
    b.vc[int(b.table[0, 80 // 16]), 1, 80 % 16, 3] = 0.0
    want, tol = po.attention(b)
    inf = torch.zeros(out.shape, dtype=torch.bool)
    inf[20:40, 2:, 3] = True  # rows at positions 80 .. 99, the second KV head's query heads
    assert (out[inf] == float("inf")).all()
    assert ((out - want).abs()[~inf] <= tol[~inf]).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D,page", [(128, 16), (64, 32), (20, 8)])
@pytest.mark.parametrize("entry", [-1, 1 << 30, -(1 << 31), "pages"])
@LONG
def test_attention_pages_outside_the_cache(gpu, dtype, D, page, entry, long):
    """Rows that see such a page are NaN, the others are not."""
    b = po.Batch([90, 1, 1], [200, 200, 600], 4, 2, D, page, dtype, seed=4, slack=_slack(long, page))
    want, tol = po.attention(b)
    at = 160 // page * page
    b.table[0, at // page] = b.pages if entry == "pages" else entry
    b.table[2, 0] = b.pages if entry == "pages" else entry
    out = attn(b.dev(b.q), b.dev(b.kc), b.dev(b.vc), *b.index()).double().cpu()
    bad = torch.zeros(b.T, dtype=torch.bool)
    bad[at - 110:90] = True  # position t + 110 of sequence 0
    bad[91] = True
    assert torch.isnan(out[bad]).all()
    assert ((out - want).abs()[~bad] <= tol[~bad]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_longer_than_the_table(gpu, dtype):
    b = po.Batch([3, 40, 2], [50, 90, 20], 4, 2, 64, 16, dtype, seed=6, slack=0)
    want, tol = po.attention(b)
    for n in (97, 1 << 20, (1 << 31) - 1):
        lens = b.lens_t.clone()
        lens[1] = n
        out = attn(b.dev(b.q), b.dev(b.kc), b.dev(b.vc), b.table.cuda(), b.starts.cuda(), lens.cuda()).double().cpu()
        assert torch.isnan(out[3:43]).all()
        for r in (slice(0, 3), slice(43, 45)):
            assert ((out - want).abs()[r] <= tol[r]).all()


@pytest.mark.parametrize("starts", [[0, 9, 4, 20], [5, 3, 2, 1], [-4, 2, 1 << 30, 7], [20, 20, 20, 20]])
@LONG
def test_attention_starts_that_do_not_rise(gpu, starts, long):
    """Refused by no check (the host does not read them): any result, but no access outside the buffers."""
    b = po.Batch([5, 5, 10], [50, 90, 20], 4, 2, 64, 16, BF16, seed=6, slack=_slack(long, 16))
    attn(b.dev(b.q), b.dev(b.kc), b.dev(b.vc), b.table.cuda(), torch.tensor(starts, dtype=torch.int32).cuda(),
         b.lens_t.cuda())
    torch.cuda.synchronize()


def test_attention_empty(gpu):
    b = po.Batch([], [], 4, 2, 64, 16, BF16)
    assert attn(b.dev(b.q), b.dev(b.kc), b.dev(b.vc), *b.index()).shape == (0, 4, 64)
    b = po.Batch([0, 0], [30, 0], 4, 2, 64, 16, BF16, pad=2)
    _check_attn(b, "no rows")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_scale_and_large_scores(gpu, dtype):
    """Scores of several thousand: one key takes all the weight; no overflow in f16 either."""
    b = po.Batch([30, 1], [90, 400], 4, 2, 64, 16, dtype, seed=8, spread=20.0)
    b.kc.mul_(8.0)
    _check_attn(b, "large scores")
    b = po.Batch([30, 1], [90, 400], 4, 2, 64, 16, dtype, seed=9)
    _check_attn(b, "small scale", scale=1e-3)


def test_attention_cache_past_32_bits(gpu):
    """Pages whose element offsets pass 2^31 and byte offsets 2^32."""
    page, D, Hk = 1024, 128, 8
    pages = 2200  # 2200 * 2^20 elements
    kc = torch.zeros(pages, Hk, page, D, dtype=BF16, device="cuda")
    vc = torch.zeros_like(kc)
    b = po.Batch([3, 1], [1500, 900], 16, 8, D, page, BF16, seed=12)
    far = torch.tensor([2199, 2050, 1, 2049], dtype=torch.int32)
    table = torch.full_like(b.table, -1)
    i = 0
    for s in range(2):
        for p in range(-(-b.lens[s] // page)):
            kc[far[i]], vc[far[i]] = b.kc[b.table[s, p]].cuda(), b.vc[b.table[s, p]].cuda()
            table[s, p] = far[i]
            i += 1
    want, tol = po.attention(b)
    out = attn(b.dev(b.q), kc, vc, table.cuda(), b.starts.cuda(), b.lens_t.cuda()).double().cpu()
    assert ((out - want).abs() <= tol).all()


@pytest.mark.parametrize("width", [524256, 524287])  # of 2^31 / 4096: the tiled kernel's longest cache; beyond, the general one's
def test_attention_positions_up_to_2_31(gpu, width):
    """Nearly 2^31 cached tokens: one page over and over (scores 0, values 1) and a last one with scores of 13.125 and
    values of -1, which carries half of the weight. Sums of ones are exact to 2^24, and what is added up of slices
    and exponentials rounds a few thousand times at 2^-24: below 1e-3 / 4 with the share of bf16 weights (2^-8 of
    the last slice's 1 / 1000)."""
    page, D = 4096, 64
    kc = torch.zeros(2, 1, page, D, dtype=BF16, device="cuda")
    vc = torch.ones_like(kc)
    kc[1], vc[1] = 1.640625, -1.0
    table = torch.zeros(1, width, dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    n = width * page
    starts, lens = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, 1], [n]))
    out = attn(torch.ones(1, 1, D, dtype=BF16, device="cuda"), kc, vc, table, starts, lens).double().cpu()
    last = page * math.exp(8 * 1.640625)
    want = (n - page - last) / (n - page + last)
    assert (out - want).abs().max() <= 2.0 ** -8 * abs(want) + 2.5e-4, (out.flatten()[0], want)


def test_attention_streams_and_repeats(gpu):
    """Two streams at once, each with its own call: the same bits as alone."""
    bs = [po.Batch([1] * 5, [3000, 10, 700, 4000, 64], 8, 2, 128, 16, BF16, seed=s) for s in (1, 2)]
    args = [(b.dev(b.q), b.dev(b.kc), b.dev(b.vc), *b.index()) for b in bs]
    alone = [attn(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in bs]
    for _ in range(3):
        outs = []
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                outs.append([attn(*a) for _ in range(4)])
        torch.cuda.synchronize()
        for o, w in zip(outs, alone):
            assert all(torch.equal(_bits(x), _bits(w)) for x in o)


# ------------------------------------------------------------------------------ append
def _check_append(b, cos, sin, interleaved, with_q=True):
    print(f"kv_append chunks={b.chunks[:8]} lens={b.lens[:8]} {b.dtype} k={tuple(b.k.shape)} rot="
          f"{None if cos is None else 2 * cos.shape[1]} {interleaved}", flush=True)
    q, qt, kc, vc, kt = po.append(b, cos, sin, interleaved)
    gk, gv = b.dev(b.kc), b.dev(b.vc)
    got = append(b.dev(b.k), b.dev(b.v), gk, gv, *b.index(), *(None if t is None else t.cuda() for t in (cos, sin)),
                 q=b.dev(b.q) if with_q else None, interleaved=interleaved)
    torch.cuda.synchronize()
    assert torch.equal(gv.double().cpu(), vc)
    d = (gk.double().cpu() - kc).abs()
    assert (d <= kt).all(), (d.max(), (d - kt).max())
    if with_q:
        rows = ~torch.isnan(q[:, 0, 0]) if q.numel() else torch.zeros(0, dtype=torch.bool)
        d = (got.double().cpu() - q).abs()[rows]
        assert (d <= qt[rows]).all()
    else:
        assert got is None
    return got


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("heads,kv_heads,D,rot,page,layout,shift", [
    (8, 2, 128, 128, 16, "hnd", 0), (4, 4, 64, 64, 16, "nhd", 0), (6, 2, 64, 32, 24, "hnd", 0), (3, 1, 80, 80, 1, "hnd", 0),
    (5, 5, 18, 18, 7, "hnd", 0), (4, 2, 256, 256, 32, "nhd", 0), (4, 2, 64, 64, 16, "odd", 1), (4, 2, 64, 20, 16, "hnd", 0),
    (2, 1, 17, 2, 16, "hnd", 3), (32, 8, 128, 64, 64, "hnd", 0), (7, 7, 96, 96, 16, "hnd", 0)])
def test_append_shapes(gpu, dtype, interleaved, heads, kv_heads, D, rot, page, layout, shift):
    cos, sin = po.tables(400, rot // 2)
    b = po.Batch([1, 5, 0, 37, 1, 2], [1, 70, 0, 37, 300, 3], heads, kv_heads, D, page, dtype, seed=D, pad=3, lead=1,
                 layout=layout, shift=shift)
    _check_append(b, cos, sin, interleaved)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("layout,shift", [("hnd", 0), ("odd", 1)])
def test_append_without_rotation(gpu, dtype, layout, shift):
    b = po.Batch([1, 5, 90], [1, 70, 200], 4, 2, 64, 16, dtype, seed=1, layout=layout, shift=shift)
    _check_append(b, None, None, True, with_q=False)
    cos, sin = po.tables(200, 32)
    _check_append(b, cos, sin, True, with_q=False)


@pytest.mark.parametrize("B", [1, 64, 65, 200])
def test_append_many_sequences(gpu, B):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 40, (B,), generator=g).tolist()
    chunks = [min(n, int(c)) for n, c in zip(lens, torch.randint(0, 4, (B,), generator=g))]
    cos, sin = po.tables(64, 32)
    _check_append(po.Batch(chunks, lens, 4, 2, 64, 8, BF16, seed=B, pad=2), cos, sin, True)


def test_append_prompt(gpu):
    """Enough rows for one wave per token."""
    cos, sin = po.tables(3500, 32)
    b = po.Batch([3001, 1, 1500], [3400, 5, 1500], 4, 2, 64, 16, F16, seed=3)
    _check_append(b, cos, sin, False)


@pytest.mark.parametrize("layout,shift", [("hnd", 0), ("odd", 1)])
@pytest.mark.parametrize("interleaved", [True, False])
def test_append_rows_without_a_place(gpu, layout, shift, interleaved):
    """Positions below zero or past the tables, pages outside the cache: nothing written, q NaN without a position."""
    b = po.Batch([4, 6, 3, 2], [2, 53, 20, 30], 4, 2, 64, 8, F16, seed=7, pad=2, layout=layout, shift=shift)
    b.table[2, 2] = b.pages          # positions 17, 18, 19 of sequence 2: slots of page 2
    b.table[3, 28 // 8] = -1         # positions 28, 29
    cos, sin = po.tables(50, 32)     # sequence 1 stands at 47 .. 52
    got = _check_append(b, cos, sin, interleaved).cpu()
    nan = torch.isnan(got).all(-1).all(-1)
    assert nan.tolist()[:15] == [True, True, False, False, False, False, False, True, True, True] + [False] * 5
    lens = b.lens_t.clone()
    lens[0] = (1 << 31) - 1
    lens[1] = -(1 << 31)
    kc, vc = b.dev(b.kc), b.dev(b.vc)
    append(b.dev(b.k), b.dev(b.v), kc, vc, b.table.cuda(), b.starts.cuda(), lens.cuda(), cos.cuda(), sin.cuda(),
           q=b.dev(b.q), interleaved=interleaved)
    torch.cuda.synchronize()
    assert torch.equal(vc.cpu().nan_to_num(), b.vc.nan_to_num())


def test_append_untouched_rows_of_q(gpu):
    from autokernel_amd.kernels import _ops
    b = po.Batch([2, 3], [20, 9], 4, 2, 64, 8, BF16, seed=7, pad=4, lead=3)
    cos, sin = (t.cuda() for t in po.tables(50, 32))
    q_out = torch.full(b.q.shape, 5.0, dtype=BF16, device="cuda")
    _ops.kv_append(q_out, b.dev(b.kc), b.dev(b.vc), b.dev(b.q), b.dev(b.k), b.dev(b.v), cos, sin, *b.index(), True)
    assert (q_out[:3] == 5).all() and (q_out[8:] == 5).all() and (q_out[3:8] != 5).any()


def test_append_matches_rotary_embedding_of_the_models(gpu):
    """A prompt from position 0: the bits of the LLaMA block's RoPE (fp32 tables)."""
    from autokernel_amd.kernels import rotary_embedding
    cos, sin = (t.cuda() for t in po.tables(300, 64))
    b = po.Batch([300], [300], 8, 2, 128, 16, F16, seed=1)
    q, k = b.dev(b.q), b.dev(b.k)
    kc, vc = b.dev(b.kc), b.dev(b.vc)
    got = append(k, b.dev(b.v), kc, vc, *b.index(), cos, sin, q=q)
    want = rotary_embedding.apply_fp32_tables(q[None], cos, sin)[0]
    assert torch.equal(_bits(got), _bits(want))
    want = rotary_embedding.apply_fp32_tables(k[None], cos, sin)[0]
    flat = kc[b.table[0, :19].long().cuda()].transpose(1, 2).reshape(-1, 2, 128)[:300]
    assert torch.equal(_bits(flat), _bits(want))


# ------------------------------------------------------------------------------ together, graphs, refusals
def test_append_then_attend_in_chunks_equals_flash_attention(gpu):
    """A prompt fed in uneven chunks, then single tokens, through both operators: causal attention of the whole."""
    g = torch.Generator().manual_seed(0)
    T, H, Hk, D, P = 200, 8, 2, 64, 16
    q, k, v = ((torch.randn(T, h, D, generator=g)).to(F16).cuda() for h in (H, Hk, Hk))
    cos, sin = (t.cuda() for t in po.tables(T, D // 2))
    kc = torch.full((20, Hk, P, D), float("nan"), dtype=F16, device="cuda")
    vc = kc.clone()
    table = torch.randperm(20, generator=g)[:14].to(torch.int32).cuda()[None]
    outs, at = [], 0
    for n in [1, 63, 64, 1, 50, 17] + [1] * 4:
        starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        lens = torch.tensor([at + n], dtype=torch.int32, device="cuda")
        s = slice(at, at + n)
        qr = append(k[s], v[s], kc, vc, table, starts, lens, cos, sin, q=q[s])
        outs.append(attn(qr, kc, vc, table, starts, lens))
        at += n
    assert at == T
    from autokernel_amd.kernels import rotary_embedding as rope
    b = po.Batch([T], [T], H, Hk, D, P, F16)
    b.q, k_ = rope.apply_fp32_tables(q[None], cos, sin)[0].cpu(), rope.apply_fp32_tables(k[None], cos, sin)[0]
    for p in range(13):
        pg, n = int(b.table[0, p]), min(P, T - p * P)
        b.kc[pg, :, :n] = k_[p * P:p * P + n].transpose(0, 1).cpu()
        b.vc[pg, :, :n] = v[p * P:p * P + n].transpose(0, 1).cpu()
    want, tol = po.attention(b)
    assert ((torch.cat(outs).double().cpu() - want).abs() <= tol).all()


def test_graph_replayed_as_the_sequences_grow(gpu):
    """One decode step captured once, replayed with the index arrays rewritten in between."""
    g = torch.Generator().manual_seed(5)
    B, H, Hk, D, P, W = 3, 8, 2, 128, 16, 40
    kc = torch.randn(130, Hk, P, D, generator=g).to(BF16).cuda()
    vc = torch.randn(130, Hk, P, D, generator=g).to(BF16).cuda()
    table = torch.randperm(130, generator=g)[:B * W].to(torch.int32).view(B, W).cuda()
    starts = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    lens = torch.tensor([1, 300, 16], dtype=torch.int32, device="cuda")
    cos, sin = (t.cuda() for t in po.tables(W * P, D // 2))
    q, k, v = ((torch.randn(5, h, D, generator=g)).to(BF16).cuda() for h in (H, Hk, Hk))

    def step():
        return attn(append(k, v, kc, vc, table, starts, lens, cos, sin, q=q), kc, vc, table, starts, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for r, new in enumerate(([2, 301, 17], [1, 640, 1], [600, 0, 333], [640, 640, 640])):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        starts.copy_(torch.tensor([0, 1, 2, 3] if r != 2 else [0, 1, 1, 4], dtype=torch.int32))
        q.copy_(torch.randn(q.shape, generator=g).to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        got = out[:int(starts[-1])].clone()
        other = torch.randn(64, 64, device="cuda") @ torch.randn(64, 64, device="cuda")
        want = step()[:int(starts[-1])]
        torch.cuda.synchronize()
        assert other.shape == (64, 64) and torch.equal(_bits(got), _bits(want)), r


def test_refusals(gpu):
    b = po.Batch([2, 1], [20, 9], 4, 2, 64, 8, BF16)
    q, k, v, kc, vc = (b.dev(t) for t in (b.q, b.k, b.v, b.kc, b.vc))
    table, starts, lens = b.index()
    cos, sin = (t.cuda() for t in po.tables(50, 32))

    def no(match, fn, *a, err=ValueError, **kw):
        with pytest.raises(err, match=match):
            fn(*a, **kw)
    no("no CPU path", attn, q.cpu(), kc, vc, table, starts, lens, err=RuntimeError)
    no("no CPU path", attn, q, kc, vc, table.cpu(), starts, lens, err=RuntimeError)
    no("int32", attn, q, kc, vc, table.long(), starts, lens)
    no("int32", attn, q, kc, vc, table, starts.long(), lens)
    no("dtype", attn, q, kc.half(), vc, table, starts, lens)
    no("dtype", attn, q.double(), kc.double(), vc.double(), table, starts, lens)
    no("alike", attn, q, kc, vc[:, :1], table, starts, lens)
    no("alike", attn, q, kc[0], vc[0], table, starts, lens)
    no("must be", attn, q[:, :, :32], kc, vc, table, starts, lens)
    no("must be", attn, q[0], kc, vc, table, starts, lens)
    no("not a multiple", attn, q[:, :3], kc, vc, table, starts, lens)
    no("sequences need", attn, q, kc, vc, table, starts[:2], lens)
    no("sequences need", attn, q, kc, vc, table[:1], starts, lens)
    no("last dim must be contiguous", attn, q, kc.transpose(2, 3).contiguous().transpose(2, 3), vc, table, starts, lens)
    no("contiguous", attn, q, kc, vc, table.t().contiguous().t(), starts, lens)
    no("overlap", attn, q, kc, vc, table[:1].expand(2, -1), starts, lens)
    for s in (0.0, -1.0, float("nan"), float("inf")):
        no("sm_scale", attn, q, kc, vc, table, starts, lens, sm_scale=s)
    no("out must be", attn, q, kc, vc, table, starts, lens, out=torch.empty(3, 4, 64, device="cuda"))
    no("out must be", attn, q, kc, vc, table, starts, lens, out=torch.empty(3, 1, 64, device="cuda", dtype=BF16).expand(3, 4, 64))
    no("head_dim", attn, q.repeat(1, 1, 5), kc.repeat(1, 1, 1, 5), vc.repeat(1, 1, 1, 5), table, starts, lens)
    no("pass 2\\^31", attn, q, kc, vc, torch.empty_strided((2, 1 << 28), (1 << 28, 1), dtype=torch.int32, device="cuda"),
       starts, lens)
    args = (k, v, kc, vc, table, starts, lens)
    no("come together", append, *args, cos)
    no("nothing done", append, *args, q=q)
    no("float32", append, *args, cos.half(), sin.half())
    no("rot_dim", append, *args, *(t.cuda() for t in po.tables(50, 33)))
    no("rot_dim", append, *args, cos, sin[:10])
    no("KV heads", append, k[:, :1], *args[1:], cos, sin)
    no("expanded view", append, k, v, kc[:1].expand(6, -1, -1, -1), vc[:6], *args[4:], cos, sin)
    no("no CPU path", append, *args, cos.cpu(), sin.cpu(), err=RuntimeError)


def test_workspace_too_small_is_refused(gpu):
    from autokernel_amd import _lib
    from autokernel_amd.kernels import _ops
    b = po.Batch([1], [2000], 4, 2, 64, 8, BF16)
    q, kc, vc = (b.dev(t) for t in (b.q, b.kc, b.vc))
    need = _lib.load().ak_paged_attn_workspace_bytes(_lib.AK_BF16, 1, 1, 4, 2, 64, 8, b.width)
    assert need > 0
    o = torch.empty_like(q)
    st2, st3 = _ops._strides(q.stride()), _ops._strides(kc.stride())
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    for ptr, n in ((ws.data_ptr(), need - 1), (None, need), (ws.data_ptr() + 8, need)):
        with pytest.raises(AkError, match="invalid argument"):
            _ops._run("ak_paged_attn", q, None, _lib.AK_BF16, q.data_ptr(), kc.data_ptr(), vc.data_ptr(), o.data_ptr(),
                      *(t.data_ptr() for t in b.index()), 1, 1, 4, 2, 64, b.pages, 8, b.width, b.width, st2, st3, st3, st2,
                      0.125, ptr, n)


def _check_rows(q, kc, vc, table, starts, lens, out, rows, dtype):
    """Some rows of a large call against 64-bit attention on the GPU (the bound of paged_oracle.attention)."""
    H, D = q.shape[1:]
    Hk, P = kc.shape[1:3]
    G = H // Hk
    st, ln = starts.tolist(), lens.tolist()
    half = po.HALF[dtype]
    for t in rows:
        b = max(i for i in range(len(ln)) if st[i] <= t)
        n = ln[b] - (st[b + 1] - t) + 1
        ids = table[b, :-(-n // P)].long()
        for hk in range(Hk):
            K = kc[ids, hk].reshape(-1, D)[:n].double()
            V = vc[ids, hk].reshape(-1, D)[:n].double()
            x = q[t, hk * G:(hk + 1) * G].double()
            s = x @ K.T.contiguous() * D ** -0.5
            want = torch.softmax(s, -1) @ V
            mag = (x.abs() @ K.abs().T.contiguous() * D ** -0.5).amax(-1, keepdim=True)
            d = (D + 6) * 2.0 ** -24 * mag + 2.0 ** -21 + n * 2.0 ** -24 + (half if dtype != F32 else 0)
            tol = 2 * d * V.abs().amax(0, keepdim=True) + half * want.abs() + po.TINY[dtype]
            got = out[t, hk * G:(hk + 1) * G].double()
            assert ((got - want).abs() <= tol).all(), (t, hk, (got - want).abs().max())


@pytest.mark.parametrize("heads,kv_heads,D,page,chunks,lens", [
    (32, 2, 64, 8, [1024], [40000]),            # page numbers of a slice past the ring that holds them
    (8, 8, 128, 16, [2100, 1, 130], [2100, 5000, 9000]),
    (32, 8, 128, 32, [512], [16513]),
    (16, 1, 128, 8, [700, 3], [30000, 70]),
])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_large_chunks(gpu, dtype, heads, kv_heads, D, page, chunks, lens):
    print(f"paged_attention large {heads}/{kv_heads} {D} page {page} {chunks} {lens} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 1
    kc, vc = ((torch.randn(pages, kv_heads, page, D, generator=g, device="cuda")).to(dtype) for _ in range(2))
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b, c in enumerate(need):
        table[b, :c] = order[at:at + c]
        at += c
    starts = torch.tensor([0] + torch.tensor(chunks).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    T = int(starts[-1])
    q = torch.randn(T, heads, D, generator=g, device="cuda").to(dtype)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = attn(q, kc, vc, table, starts, ln)
    picks = {0, 1, 31, 32, T // 2, T - 2, T - 1} | set(torch.randint(0, T, (12,)).tolist()) | {int(x) for x in starts[:-1]}
    _check_rows(q, kc, vc, table, starts, ln, out, sorted(picks), dtype)
    assert torch.equal(_bits(out), _bits(attn(q, kc, vc, table, starts, ln)))


@LONG
def test_attention_a_sequence_alone_or_in_a_batch(gpu, long):
    """Chunks beside single tokens (both tile sizes in one launch): each sequence within its own bound."""
    b = po.Batch([1, 200, 16, 17, 1, 65, 64, 1], [700, 1000, 16, 300, 1, 65, 2000, 64], 8, 2, 128, 16, BF16, seed=2, pad=5,
                 slack=_slack(long, 16))
    _check_attn(b, "mixed")
    b = po.Batch([1, 200, 64, 65, 1, 130, 1], [700, 1000, 64, 300, 1, 130, 64], 4, 4, 64, 8, F16, seed=3, pad=1, slack=_slack(long, 8))
    _check_attn(b, "mixed")
