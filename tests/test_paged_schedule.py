"""paged_attention's work split, restated: items found from the lengths alone (pa_chunk, pa_find) and the items that
pa_merge reads, over ordinary, extreme and nonsensical batches. Every (KV head, tile, slice) is an item exactly once,
no item or partial lies past what the host planned for, and nothing indexes past the page table (CPU only)."""
from __future__ import annotations

import ctypes
import random

import pytest

SLICE, STEP, MIN_SLICED, SPLIT_ROWS, TILED_ROWS, ONE_EACH = 256, 128, 1536, 16, 64, 256


def plan(T, B, Hq, Hk, page, width, fast, tiles_ok):
    """(rows a tile, items, target) of both classes, as pa_plan."""
    G, rows, seqs = Hq // Hk, T * (Hq // Hk), min(B, T)
    sliced = page * width > MIN_SLICED
    tiles = fast and tiles_ok and page % 16 == 0 and rows > SPLIT_ROWS and (
        T > B or rows > TILED_ROWS if sliced else (rows // 16 + seqs // 2) * Hk > 2 * ONE_EACH)
    bm = [16 if fast else 4, 128]
    items, target = [(rows // bm[0] + seqs) * Hk, 0], [0, 0]
    if tiles:
        items[0] = min(items[0], seqs * -(-SPLIT_ROWS // bm[0]) * Hk)
        items[1] = (rows // 128 + min(seqs, rows // (SPLIT_ROWS + 1))) * Hk
    if sliced:
        target[0] = 1536
        if tiles and rows // 128 * Hk < 4 * 512:
            target[1] = 512
    return bm, [i + t for i, t in zip(items, target)], target, (SPLIT_ROWS if items[1] else 1 << 31)


def workspace(bm, items, target, D):
    return sum(4 * items[c] * bm[c] * ((D + 3) // 4 * 4 + 2) for c in range(2) if target[c])


class Seq:
    def __init__(self, starts, lens, b, T, cap):
        self.t0 = min(max(starts[b], 0), T)
        self.n = min(max(starts[b + 1], self.t0), T) - self.t0
        self.len = 0 if lens[b] > cap else max(lens[b], 0)


def f32(x):
    return ctypes.c_float(x).value


def chunk(seqs, G, Hk, bm, mine, target):
    if target == 0:
        return None
    w = f32(sum(f32(-(-s.n * G // bm)) * f32(s.len) for s in seqs if mine(s)))
    if bm < 128 and max([s.len for s in seqs if mine(s)] + [0]) * sum(-(-s.n * G // bm) for s in seqs if mine(s)) < 1.5 * w:
        target = f32(target * 2 / 3)  # sequences of about one length
    w = f32(w * Hk * 1.001)
    c = -(-int(w / target) // SLICE) * SLICE if w / target == int(w / target) else (int(w / target) // SLICE + 1) * SLICE
    return max(c, SLICE)


def splits(n, c):
    return 1 if c is None else max(1, -(-n // c))


def items_of(seqs, G, Hk, bm, mine, target):
    """[(sequence, KV head, tile, slice)] in item order, the slice length, and each sequence's first item."""
    c = chunk(seqs, G, Hk, bm, mine, target)
    out, first = [], {}
    for b, s in enumerate(seqs):
        if not mine(s):
            continue
        tiles = -(-s.n * G // bm)
        first[b] = len(out)
        for sp in range(splits(s.len, c)):
            for t in range(tiles):
                out += [(b, hk, tiles - 1 - t, sp) for hk in range(Hk)]
    return out, c, first


def check(chunks, lens, Hq, Hk, D, page, width, fast, tiles_ok=True, starts=None, extra=0):
    if starts is None:
        starts = [0]
        for n in chunks:
            starts.append(starts[-1] + n)
    T, B, G = max(max(starts), 0) + extra, len(lens), Hq // Hk
    bm, planned, target, split_rows = plan(T, B, Hq, Hk, page, width, fast, tiles_ok)
    seqs = [Seq(starts, lens, b, T, page * width) for b in range(B)]
    rising = all(a <= b for a, b in zip(starts, starts[1:])) and starts[0] >= 0
    for cls in range(2):
        def mine(s):
            return s.n > 0 and (cls == 0) == (s.n * G <= split_rows)
        items, c, first = items_of(seqs, G, Hk, bm[cls], mine, target[cls])
        if rising:
            assert len(items) <= planned[cls], (cls, len(items), planned)
            assert len(set(items)) == len(items)
        for b, hk, tile, sp in items[:planned[cls]]:
            s = seqs[b]
            n = splits(s.len, c)
            each = -(-(-(-s.len // n)) // STEP) * STEP if n > 1 else s.len  # keys of this sequence's slices
            lo = sp * each
            hi = min(max(0, s.len - s.n + min(s.n * G - 1, tile * bm[cls] + bm[cls] - 1) // G + 1), lo + each)
            assert n * each >= s.len and lo < 2 ** 31 and (n == 1 or each <= c)
            assert 0 <= tile * bm[cls] < s.n * G and hi <= s.len <= page * width
            if hi > lo:
                assert (hi - 1) // page < width
        # the merge's items of a row: all its slices, each the item that computed it
        for b, s in enumerate(seqs):
            if not mine(s) or splits(s.len, c) == 1 or not rising:
                continue
            for r in {0, s.n * G // 2, s.n * G - 1}:
                tiles, tile = -(-s.n * G // bm[cls]), r // bm[cls]
                for hk in (0, Hk - 1):
                    got = [items[first[b] + (sp * tiles + tiles - 1 - tile) * Hk + hk] for sp in range(splits(s.len, c))]
                    assert got == [(b, hk, tile, sp) for sp in range(splits(s.len, c))]
    return workspace(bm, planned, target, D)


BATCHES = [
    ([1], [1001]), ([1] * 64, list(range(100, 6500, 100))), ([512], [16513]), ([2048] * 4, [2048] * 4), ([1], [200000]),
    ([333, 1, 1, 129, 1, 0, 16, 17, 64, 65], [333, 901, 18, 529, 1024, 0, 16, 300, 64, 9000]), ([5, 150], [2, 30]),
    ([1] * 300, [50] * 299 + [60000]), ([0, 0, 3], [10, 0, 5]), ([1500, 1], [1500, 32000]),
]


@pytest.mark.parametrize("chunks,lens", BATCHES)
@pytest.mark.parametrize("Hq,Hk", [(32, 8), (12, 12), (16, 1), (3, 1)])
@pytest.mark.parametrize("page", [1, 8, 16, 128])
def test_items_cover_the_batch(chunks, lens, Hq, Hk, page):
    from autokernel_amd import _lib
    lib = _lib.load()
    width = max(1, -(-max(lens) // page)) + 1
    for dtype, D, fast, tiles_ok in ((1, 128, True, True), (0, 64, True, False), (1, 80, False, False)):
        ws = check(chunks, lens, Hq, Hk, D, page, width, fast, tiles_ok)
        need = lib.ak_paged_attn_workspace_bytes(dtype, sum(chunks), len(lens), Hq, Hk, D, page, width)
        assert need >= ws  # what the library asks for holds the plan restated here


def test_items_of_random_batches():
    rng = random.Random(0)
    for _ in range(300):
        B = rng.choice([1, 2, 7, 63, 64, 65, 200])
        chunks = [rng.choice([0, 1, 1, 1, rng.randint(1, 700)]) for _ in range(B)]
        lens = [c + int(rng.expovariate(1 / 2000)) for c in chunks]
        Hk = rng.choice([1, 2, 8])
        page = rng.choice([1, 16, 24, 64])
        check(chunks, lens, Hk * rng.choice([1, 3, 8]), Hk, 64, page, max(1, -(-max(lens) // page)) + rng.randint(0, 500),
              True, extra=rng.randint(0, 9))


@pytest.mark.parametrize("starts", [[0, 9, 4, 20], [5, 3, 2, 1], [-4, 2, 1 << 30, 7], [20, 20, 20, 20], [0, 1 << 30, 0, 9]])
def test_nonsensical_arrays_stay_inside(starts):
    """Starts that do not rise, lengths past the table or negative: whatever is found stays inside the buffers."""
    for lens in ([50, 90, 20], [-5, 1 << 30, (1 << 31) - 1], [0, 0, 0]):
        T = 20
        fixed = [min(max(s, -(1 << 31)), (1 << 31) - 1) for s in starts]
        seqs = [Seq(fixed, lens, b, T, 16 * 8) for b in range(3)]
        for s in seqs:
            assert 0 <= s.t0 <= s.t0 + s.n <= T and 0 <= s.len <= 16 * 8
