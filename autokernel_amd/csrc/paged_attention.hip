// paged_attention.hip -- attention of new tokens over a paged cache.
//
//   o_i = softmax_j(q_i . K_j sm_scale) V_j over the cached keys j <= pos(i) of the token's sequence
// (paged_common.h: rows, positions, pages), grouped-query heads, one softmax pass with fp32 statistics.
// A row that sees no key (a position below zero) is zero; rows outside every sequence are not written; a
// row that sees a key in a page outside the cache is NaN, and so is every row of a sequence longer than
// its page table.
//
// Work split. The rows of a (sequence, KV head) are its group's query heads of each new token, token by
// token (row r: token r / group, head r % group), cut into tiles: of 128 rows for sequences of more than
// kPaSplitRows of them (pa_tiles), of 16 for the others (pa_rows). A tile's keys are cut into slices of C
// keys, and a block takes one (tile, slice). The lengths are device data, so every block finds its item
// itself: it adds up its class's work, derives C (about `target` items in all) and walks the sequences'
// item counts. The grid covers the most items there can be; blocks past the last one end at once. Sliced
// rows leave fp32 partials (max, sum, weighted values) that pa_merge combines in slice order, so results
// do not depend on the order in which blocks run.
#include <limits.h>

#include <algorithm>

#include "attention_common.h"
#include "mfma.h"
#include "paged_common.h"

namespace ak {

constexpr int kPaWaves = 4;
constexpr int kPaThreads = kPaWaves * kWave;

// Sequences with few rows, or with many: their tiles of BM rows.
struct PaClass {
  float *part, *stat;  // [items][BM][Dp], [items][BM][2] (exp2 base, sum)
  float target;        // items aimed at; 0: keys are not sliced
  uint32_t items;      // the most items there can be
};
struct PaArgs {
  const void *q, *kc, *vc;
  void* o;
  PaClass c[2];    // few rows, many rows
  int split_rows;  // most rows (new tokens times group) of a sequence of class 0
  FastDiv f_units;  // pa_merge's units of a token
  int64_t qst, qsh, ost, osh;            // row and head strides (elements)
  int64_t kcp, kch, kct, vcp, vch, vct;  // cache: page, head, slot strides
  int Hq, Hk, G, D, Dp, vec;  // Dp: floats of a partial row, D rounded up to 4
  float c_log2;
  FastDiv f_g, f_hk;
  PagedSeqs s;
};

__device__ __forceinline__ int pa_uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

struct PaSeq {
  int t0, n, len;   // first row, rows, cached tokens (new ones among them)
  bool overlong;    // longer than its page table: NaN rows
};
__device__ __forceinline__ PaSeq pa_seq(const PagedSeqs& s, int b) {
  PaSeq q;
  q.t0 = min(max(s.starts[b], 0), s.T);
  q.n = min(max(s.starts[b + 1], q.t0), s.T) - q.t0;
  const int len = s.lens[b];
  q.overlong = len > s.width * s.page_size;
  q.len = q.overlong ? 0 : max(len, 0);
  return q;
}

struct PaItem {
  int b, hk, tile, split, nsplit;
  int chunk;      // keys of a slice of this sequence
  uint32_t slot;  // the item's place among its class's partials
  PaSeq seq;
};

// Inclusive sum over the lanes: within rows of 16 lanes by row_shr, then each row's last lane to the rows after
// it by row_bcast (six VALU instructions; __shfl_up goes through LDS six times).
__device__ __forceinline__ int pa_wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// Keys per slice, at most: all of them when the class's work fills the chip without slicing, else the work over
// `target`, in multiples of kPaSlice. A sequence's slices are alike, in multiples of kPaStep.
constexpr int kPaSlice = 256, kPaStep = 128;
template <int BM, int CLS>
__device__ __forceinline__ int pa_tiles_of(const PaArgs& a, const PaSeq& q) {
  const int rows = q.n * a.G;
  return (CLS == 0) == (rows <= a.split_rows) ? (rows + BM - 1) / BM : 0;
}
// The batch, one sequence a lane: a call of up to 64 sequences reads its lengths once.
struct PaBatch {
  PaSeq q;  // sequence lane_id() (no rows past the last)
};
__device__ __forceinline__ PaSeq pa_lane_seq(const PagedSeqs& s, int b) {
  return b < s.B ? pa_seq(s, b) : PaSeq{0, 0, 0, false};
}
// f(first sequence of 64, this lane's sequence) until it returns true
template <typename F>
__device__ __forceinline__ void pa_each(const PaArgs& a, const PaBatch& x, F f) {
  if (f(0, x.q)) return;
  for (int i = kWave; i < a.s.B; i += kWave)
    if (f(i, pa_lane_seq(a.s, i + lane_id()))) return;
}
template <int BM, int CLS>
__device__ __forceinline__ int pa_chunk(const PaArgs& a, const PaBatch& x) {
  float target = a.c[CLS].target;
  if (target <= 0.f) return INT_MAX;
  float w = 0.f, tiles = 0.f, longest = 0.f;
  pa_each(a, x, [&](int, const PaSeq& q) {
    const float n = (float)pa_tiles_of<BM, CLS>(a, q), len = (float)q.len;
    w += n * len;
    if constexpr (CLS == 0) {
      tiles += n;
      longest = n > 0.f ? fmaxf(longest, len) : longest;
    }
    return false;
  });
  w = wave_sum(w);
  // Sequences of about one length balance by themselves, and two rounds of items are enough (128 of 2000 tokens 180 us in
  // three, 170 in two; 24 of 3000 65, 61); ragged ones not (64 of 200 to 8000 120.4 in three, 123.2 in two).
  if constexpr (CLS == 0)
    if (wave_max(longest) * wave_sum(tiles) < 1.5f * w) target *= 2.f / 3.f;
  w *= (float)a.Hk * 1.001f;
  const float c = ceilf(w / target / (float)kPaSlice) * (float)kPaSlice;
  return pa_uniform(c >= 1e9f ? INT_MAX : max((int)c, kPaSlice));
}
__device__ __forceinline__ int pa_splits(int len, int chunk) { return len > 0 ? (len - 1) / chunk + 1 : 1; }

// Item `it` of a class; false when there are fewer. Within a sequence the KV heads run fastest (one
// per XCD, whose L2 then serves the tiles that share a head's keys), then tiles, last rows first (they see
// the most keys), then slices.
template <int BM, int CLS>
__device__ __forceinline__ bool pa_find(const PaArgs& a, uint32_t it, PaItem& o) {
  const PaBatch x{pa_lane_seq(a.s, lane_id())};
  o.chunk = pa_chunk<BM, CLS>(a, x);
  o.slot = it;
  o.split = o.nsplit = 0;
  uint32_t base = 0;
  pa_each(a, x, [&](int i, const PaSeq& q) {
    int tiles = pa_tiles_of<BM, CLS>(a, q);
    const int splits = pa_splits(q.len, o.chunk), cnt = tiles * a.Hk * splits;
    const int inc = pa_wave_scan(cnt);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(it - base < (uint32_t)inc && cnt > 0);
    if (!hit) {
      base += (uint32_t)__builtin_amdgcn_readlane(inc, kWave - 1);
      return false;
    }
    // one sequence for the whole block: what is made from it belongs in scalar registers
    const int l = __builtin_ctzll(hit);
    o.b = i + l;
    tiles = __builtin_amdgcn_readlane(tiles, l);
    o.seq.t0 = __builtin_amdgcn_readlane(q.t0, l);
    o.seq.n = __builtin_amdgcn_readlane(q.n, l);
    o.seq.len = __builtin_amdgcn_readlane(q.len, l);
    o.seq.overlong = __builtin_amdgcn_readlane((int)q.overlong, l) != 0;
    o.nsplit = __builtin_amdgcn_readlane(splits, l);
    // equal slices: 2000 keys are two of 1024, not 1536 and 464 (128 such sequences:
    // 228 us, 180 in equal ones)
    if (o.nsplit > 1) o.chunk = pa_uniform((((o.seq.len - 1) / o.nsplit + 1) + kPaStep - 1) / kPaStep * kPaStep);
    const uint32_t rel = it - base - (uint32_t)__builtin_amdgcn_readlane(inc - cnt, l);
    const uint32_t y = fdiv(rel, a.f_hk);
    o.hk = pa_uniform((int)(rel - y * a.Hk));
    o.split = pa_uniform((int)(y / (uint32_t)tiles));
    o.tile = pa_uniform(tiles - 1 - (int)(y - (uint32_t)o.split * tiles));
    return true;
  });
  return o.split < o.nsplit;
}

// Keys [lo, hi) of one row, by one wave: exact about what a row sees, whatever the rest of its pages hold.
// m: exp2 base (max), l: sum, acc[r]: dim lane + 64 r.
template <typename T>
__device__ void pa_row(const PaArgs& a, int b, int hk, const typename T::S* qrow, int64_t lo, int64_t hi, float& m,
                       float& l, float (&acc)[4]) {
  using S = typename T::S;
  const int lane = lane_id(), D = a.D;
  const S* kc = (const S*)a.kc + hk * a.kch;
  const S* vc = (const S*)a.vc + hk * a.vch;
  float q[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    acc[r] = 0.f;
    q[r] = lane + 64 * r < D ? T::to_f(qrow[lane + 64 * r]) : 0.f;
  }
  m = -INFINITY;
  l = 0.f;
  for (int64_t k0 = lo; k0 < hi; k0 += kWave) {
    const int64_t key = k0 + lane;
    const int cnt = (int)min((int64_t)kWave, hi - k0);
    int64_t page = -1;
    int slot = 0;
    if (lane < cnt) {
      page = paged_page_of(a.s, b, key);
      slot = (int)((uint32_t)key - fdiv((uint32_t)key, a.s.page_div) * a.s.page_size);
    }
    float s = 0.f;
    const S* kr = kc + (page < 0 ? 0 : page * a.kcp + slot * a.kct);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (64 * r >= D) break;
      asm volatile("" : "+v"(q[r]));  // or the broadcasts below move out of the loop, into 256 registers
#pragma unroll 1
      for (int d = 0; d < 64 && 64 * r + d < D; d += T::kVec) {
        float x[T::kVec];
        if (page >= 0 && a.vec) {
          const u32x4 v = ld16(kr + 64 * r + d);
#pragma unroll
          for (int e = 0; e < T::kVec; ++e) x[e] = T::lane_elem(v, e);
        } else {
#pragma unroll
          for (int e = 0; e < T::kVec; ++e)
            x[e] = page >= 0 && 64 * r + d + e < D ? T::to_f(kr[64 * r + d + e]) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < T::kVec; ++e)
          s = __builtin_fmaf(x[e], __int_as_float(__builtin_amdgcn_readlane(__float_as_int(q[r]), d + e)), s);
      }
    }
    s = lane >= cnt ? -INFINITY : page < 0 ? __builtin_nanf("") : s * a.c_log2;
    const float m_new = nan_max(m, wave_nan_max(s));
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = m_new == m ? 1.0f : __builtin_amdgcn_exp2f(m - base);
    const float p = lane >= cnt ? 0.f : __builtin_amdgcn_exp2f(s - base);
    m = m_new;
    l = l * alpha + wave_sum(p);
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] *= alpha;
    const int64_t voff = page < 0 ? -1 : page * a.vcp + slot * a.vct;
    for (int j = 0; j < cnt; ++j) {
      const float pj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(p), j));
      const int64_t off = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)voff, j) |
                          (int64_t)__builtin_amdgcn_readlane((int)(voff >> 32), j) << 32;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = lane + 64 * r;
        if (d < D) acc[r] = __builtin_fmaf(pj, off < 0 ? 1.0f : T::to_f(vc[off + d]), acc[r]);
      }
    }
  }
}

// Where an item's keys begin, and where those of them end that lie below `seen` (without passing 2^31 on the way).
__device__ __forceinline__ int pa_begin(const PaItem& it) { return pa_uniform(it.split ? it.split * it.chunk : 0); }
__device__ __forceinline__ int pa_end(const PaItem& it, int seen) {
  const int lo = pa_begin(it);
  return pa_uniform(lo + min(seen - lo, it.chunk));
}
// Row r of a tile: the end of the keys that it sees.
__device__ __forceinline__ int pa_seen(const PaItem& it, int r, FastDiv f_g) {
  return max(0, it.seq.len - it.seq.n + (int)fdiv((uint32_t)r, f_g) + 1);
}

// What a row's weighted values are multiplied with: 1 / sum, 0 for a row that sees no key.
__device__ __forceinline__ float pa_inv(const PaSeq& q, bool sees, float l) {
  return q.overlong ? __builtin_nanf("") : sees ? 1.0f / l : 0.f;
}

// Rows r_begin .. r_end - 1 of an item's tile over keys [lo, hi), one wave per row: results, or partials when
// the keys are sliced.
template <typename T, int BM, int CLS, int NW = kPaWaves>
__device__ void pa_one_by_one(const PaArgs& a, const PaItem& it, int r_begin, int r_end, int lo, int hi) {
  using S = typename T::S;
  const int lane = lane_id();
  for (int r = r_begin + wave_id(); r < r_end; r += NW) {
    const int tk = (int)fdiv((uint32_t)r, a.f_g);
    const int tok = it.seq.t0 + tk, h = it.hk * a.G + r - tk * a.G;
    const int seen = pa_seen(it, r, a.f_g);
    float m, l, acc[4];
    pa_row<T>(a, it.b, it.hk, (const S*)a.q + tok * a.qst + h * a.qsh, lo, min(seen, hi), m, l, acc);
    if (it.nsplit > 1) {
      const int64_t slot = (int64_t)it.slot * BM + (r - r_begin);
      float* p = a.c[CLS].part + slot * a.Dp;
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (lane + 64 * x < a.D) p[lane + 64 * x] = acc[x];
      if (lane == 0) {
        a.c[CLS].stat[slot * 2] = m;
        a.c[CLS].stat[slot * 2 + 1] = l;
      }
      continue;
    }
    S* o = (S*)a.o + tok * a.ost + h * a.osh;
    const float inv = pa_inv(it.seq, seen > 0, l);
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (lane + 64 * x < a.D) o[lane + 64 * x] = T::from_f(it.seq.overlong ? inv : acc[x] * inv);
  }
}

// Any type, head_dim and alignment: one wave per row, four rows per block. Each row reads its keys for itself, from the
// L2 where rows share them (64 ragged sequences of 200 to 8000 tokens: 1391 us, 120 by pa_rows).
constexpr int kPaRowTile = kPaWaves;
template <typename T>
__global__ __launch_bounds__(kPaThreads) void pa_general(const PaArgs a) {
  PaItem it;
  if (!pa_find<kPaRowTile, 0>(a, blockIdx.x, it)) return;
  const int r0 = it.tile * kPaRowTile;
  pa_one_by_one<T, kPaRowTile, 0>(a, it, r0, min(it.seq.n * a.G, r0 + kPaRowTile), pa_begin(it), pa_end(it, it.seq.len));
}

// Sliced rows: the partials of each (row, query head), added in slice order by groups of 16 lanes (lane c: dims
// 4 c .. 4 c + 3 of each 64; JN: 64s of head_dim), four slices in flight. With many rows a group has a row to
// itself (WIDE false: a wave takes four heads of one token); with few, the block's sixteen groups share a row,
// so that 64 slices' partials are in flight at once, and combine in group order. The grid is bounded and walks the
// rows: in most calls with many rows nothing is sliced and it ends at once.
// Bound by reading the partials where there are many: 512 tokens of 32 heads in 4 slices, 35 MB, 9.5 us (a wave per
// row 16); by latency otherwise, 4.4 to 8 us.
template <int JN>
struct PaSum {
  float m, l, acc[JN][4];  // exp2 base, sum, weighted values
};
// acc = acc, then x, to the common base
template <int JN>
__device__ __forceinline__ void pa_add(PaSum<JN>& s, float m, float l, const f32x4 (&v)[JN]) {
  if (m == -INFINITY && l == 0.f) return;  // a slice without a key that the row sees
  const float m_new = nan_max(s.m, m);
  const float f0 = s.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s.m - m_new);
  const float f1 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
  s.m = m_new;
  s.l = s.l * f0 + l * f1;
#pragma unroll
  for (int j = 0; j < JN; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) s.acc[j][e] = s.acc[j][e] * f0 + v[j][e] * f1;
}
template <typename T, int BM0, int BM1, int JN, bool WIDE>
__global__ __launch_bounds__(kPaThreads) void pa_merge(const PaArgs a) {
  using S = typename T::S;
  constexpr int NG = WIDE ? 4 * kPaWaves : 1;  // groups of a row
  __shared__ float so[WIDE ? NG : 1][64 * JN + 4], sm[NG], sl[NG];
  const int lane = lane_id(), c = lane & 15, grp = threadIdx.x >> 4;
  const PaBatch x{pa_lane_seq(a.s, lane)};
  const int chunk0 = pa_chunk<BM0, 0>(a, x), chunk1 = pa_chunk<BM1, 1>(a, x);
  bool sliced = false;
  pa_each(a, x, [&](int, const PaSeq& q) {
    const int rows = q.n * a.G;
    sliced = __builtin_amdgcn_ballot_w64(rows > 0 && pa_splits(q.len, rows <= a.split_rows ? chunk0 : chunk1) > 1) != 0;
    return sliced;
  });
  if (!sliced) return;
  // items of each class up to and with a lane's sequence
  auto items = [&](const PaSeq& s, int (&n)[2], int (&upto)[2]) {
    n[0] = pa_tiles_of<BM0, 0>(a, s) * a.Hk * pa_splits(s.len, chunk0);
    n[1] = pa_tiles_of<BM1, 1>(a, s) * a.Hk * pa_splits(s.len, chunk1);
    upto[0] = pa_wave_scan(n[0]);
    upto[1] = pa_wave_scan(n[1]);
  };
  int n64[2], upto64[2];
  items(x.q, n64, upto64);
  // a unit: one (token, head) for the block, or four heads of a token for the wave
  const int64_t units = (int64_t)a.s.T * (WIDE ? a.Hq : (a.Hq + 3) / 4);
  const int64_t step = (int64_t)gridDim.x * (WIDE ? 1 : kPaWaves);
  for (int64_t unit = WIDE ? blockIdx.x : (int64_t)blockIdx.x * kPaWaves + pa_uniform(wave_id()); unit < units;
       unit += step) {
    const int tok = pa_uniform((int)fdiv((uint32_t)unit, a.f_units));
    const int h = WIDE ? (int)unit - tok * a.Hq : 4 * ((int)unit - tok * ((a.Hq + 3) / 4)) + lane / 16;
    // the token's sequence, and the items of its class before it
    PaSeq q{0, 0, 0, false};
    int cls = 0, nsplit = 1;
    uint32_t first = 0, before[2] = {0, 0};
    pa_each(a, x, [&](int i, const PaSeq& s) {
      const uint64_t hit = __builtin_amdgcn_ballot_w64(tok >= s.t0 && tok < s.t0 + s.n);
      int n[2] = {n64[0], n64[1]}, upto[2] = {upto64[0], upto64[1]};
      if (i > 0) items(s, n, upto);
      if (!hit) {
        before[0] += (uint32_t)__builtin_amdgcn_readlane(upto[0], kWave - 1);
        before[1] += (uint32_t)__builtin_amdgcn_readlane(upto[1], kWave - 1);
        return false;
      }
      const int l = __builtin_ctzll(hit);
      q.t0 = __builtin_amdgcn_readlane(s.t0, l);
      q.n = __builtin_amdgcn_readlane(s.n, l);
      q.len = __builtin_amdgcn_readlane(s.len, l);
      q.overlong = __builtin_amdgcn_readlane((int)s.overlong, l) != 0;
      cls = q.n * a.G <= a.split_rows ? 0 : 1;
      nsplit = pa_splits(q.len, cls ? chunk1 : chunk0);
      first = before[cls] + (uint32_t)__builtin_amdgcn_readlane(cls ? upto[1] - n[1] : upto[0] - n[0], l);
      return true;
    });
    if (nsplit == 1) continue;  // (the same for the whole block where it shares a unit)
    const int bm = cls ? BM1 : BM0, tiles = (q.n * a.G + bm - 1) / bm;
    const PaClass& cl = a.c[cls];
    const int hk = (int)fdiv((uint32_t)h, a.f_g), r = (tok - q.t0) * a.G + h - hk * a.G;
    const uint32_t it0 = first + (uint32_t)(tiles - 1 - r / bm) * a.Hk + hk;
    PaSum<JN> sum{-INFINITY, 0.f, {}};
    for (int sp = WIDE ? grp : 0; sp < nsplit; sp += 4 * NG) {
      float ms[4], ls[4];
      f32x4 v[4][JN];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t it = it0 + (uint32_t)(sp + u * NG) * tiles * a.Hk;
        const bool in = sp + u * NG < nsplit && it < cl.items && h < a.Hq;
        const int64_t slot = in ? (int64_t)it * bm + r % bm : 0;
        ms[u] = in ? cl.stat[slot * 2] : -INFINITY;
        ls[u] = in ? cl.stat[slot * 2 + 1] : 0.f;
#pragma unroll
        for (int j = 0; j < JN; ++j)
          v[u][j] = in && 64 * j + 4 * c < a.D ? *reinterpret_cast<const f32x4*>(cl.part + slot * a.Dp + 64 * j + 4 * c)
                                               : f32x4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) pa_add(sum, ms[u], ls[u], v[u]);
    }
    const bool sees = q.len - (q.t0 + q.n - tok) >= 0;  // its position
    S* o = (S*)a.o + (int64_t)tok * a.ost + (int64_t)h * a.osh;
    if constexpr (!WIDE) {
      if (h >= a.Hq) continue;
      const float inv = pa_inv(q, sees, sum.l);
#pragma unroll
      for (int j = 0; j < JN; ++j) {
        const int d = 64 * j + 4 * c;
        float* y = sum.acc[j];
        if constexpr (JN <= 2) {  // head_dim 64 JN, aligned rows
          if constexpr (T::kCode == AK_F32)
            *reinterpret_cast<f32x4*>(o + d) = f32x4{y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv};
          else
            *reinterpret_cast<u32x2*>(o + d) =
                u32x2{fa2_pack<T>(y[0] * inv, y[1] * inv), fa2_pack<T>(y[2] * inv, y[3] * inv)};
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (d + e < a.D) o[d + e] = T::from_f(y[e] * inv);
        }
      }
    } else {
      __syncthreads();  // the unit before this one has been read
#pragma unroll
      for (int j = 0; j < JN; ++j)
        *reinterpret_cast<f32x4*>(&so[grp][64 * j + 4 * c]) =
            f32x4{sum.acc[j][0], sum.acc[j][1], sum.acc[j][2], sum.acc[j][3]};
      if (c == 0) {
        sm[grp] = sum.m;
        sl[grp] = sum.l;
      }
      __syncthreads();
      float mb = -INFINITY, lb = 0.f, f[NG];
      for (int y = 0; y < NG; ++y) mb = nan_max(mb, sm[y]);
#pragma unroll
      for (int y = 0; y < NG; ++y) {
        f[y] = sm[y] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[y] - mb);
        lb += sl[y] * f[y];
      }
      const float inv = pa_inv(q, sees, lb);
      for (int d = threadIdx.x; d < a.D; d += kPaThreads) {
        float v = 0.f;
#pragma unroll
        for (int y = 0; y < NG; ++y) v += so[y][d] * f[y];
        o[d] = T::from_f(v * inv);
      }
    }
  }
}

// Few rows per KV head, f16 / bf16, head_dim 64 or 128, 16-byte aligned rows. What bounds it is reading K and
// V once from HBM. 16 rows are the columns of one MFMA tile; a wave takes 32 keys per step straight from
// the pages into registers (no LDS, no barrier), the next step's loads and the page numbers of the one after
// in flight while it computes, and the block's four waves take every fourth step.
//   * S^T = K Q^T on v_mfma_f32_16x16x32: two 16-key tiles whose row i of tile t is key 8 (i / 4) + 4 t +
//     i % 4, so lane group g ends up with the scores of keys 8 g .. 8 g + 7 of one query: in order, the B
//     operand of the next product. A lane reads keys of one aligned group of 8 for K and of one for V, so
//     pages of a multiple of 8 slots cost one page number each; others one per key (PG = 1).
//   * O^T += V^T P^T: a lane loads D / 16 consecutive dims of eight keys and transposes them in registers.
//   * Weights are rounded to the element type for the product; the sum adds the rounded ones.
// Keys past a row's position weigh nothing as long as their V is finite. Where a result is NaN, or a page
// lies outside the cache, the rows are computed again by pa_row.
// 64 sequences of 200 to 8000 cached tokens, one new one each, 8 KV heads of 128 in bf16: 613 MB in 110 us, 5.6 TB/s (a
// large copy moves 5.1, a large read 6.1), and 7 for the merge. One sequence of 1000: 14.4 us, eight CUs' latency: 1 us to find
// the item, 2 to its page numbers and 3 per two steps of keys.
constexpr int kPrRows = 16, kPrKeys = 32;
struct PrMaximum {
  __device__ __forceinline__ float operator()(float a, float b) const { return fa2_max(a, b); }
};
template <typename Op>
__device__ __forceinline__ float pr_groups(float v, Op op) {  // over the four 16-lane groups of a wave
  return wave_step<5>(wave_step<4>(v, op), op);
}
template <int D>
struct PrVec;  // D / 16 16-bit values of one V row
template <>
struct PrVec<128> {
  typedef u32x4 type;
};
template <>
struct PrVec<64> {
  typedef u32x2 type;
};

template <int D, int NW>
struct PrShared {
  float so[NW][kPrRows][D + 4];
  float st[NW][kPrRows][2];
  int again;
};

// The end of a few-row item: the waves' results (lane (i16, g) holds of row i16, in o[e][v], dim VW (4 g + v) + e)
// merged and stored, or the rows computed again.
template <typename T, int D, int NW>
__device__ __forceinline__ void pr_finish(const PaArgs& a, const PaItem& it, PrShared<D, NW>& sh,
                                          const f32x4 (&o)[D / 16], float m_run, float l_run, bool bad, int rows, int r0,
                                          int kbeg, int kend) {
  constexpr int VW = D / 16;
  const int lane = lane_id(), w = wave_id(), i16 = lane & 15, g = lane >> 4;
  l_run = pr_groups(l_run, OpAdd());
  bad |= l_run != l_run;
#pragma unroll
  for (int e = 0; e < VW; ++e)
#pragma unroll
    for (int v = 0; v < 4; ++v) bad |= o[e][v] != o[e][v];
#pragma unroll
  for (int v = 0; v < 4; ++v)
#pragma unroll
    for (int e = 0; e < VW; ++e) sh.so[w][i16][VW * (4 * g + v) + e] = o[e][v];
  if (g == 0) {
    sh.st[w][i16][0] = m_run;
    sh.st[w][i16][1] = l_run;
  }
  __syncthreads();  // (the flag is cleared by now)
  if (__builtin_amdgcn_ballot_w64(bad) && lane == 0) atomicOr(&sh.again, 1);
  __syncthreads();
  if (sh.again) {
    pa_one_by_one<T, kPrRows, 0, NW>(a, it, r0, min(rows, r0 + kPrRows), kbeg, kend);
    return;
  }
  const int q = threadIdx.x >> 4, c = threadIdx.x & 15;  // row of the tile, VW dims at c * VW
  if (q >= kPrRows || r0 + q >= rows) return;
  float mb = -INFINITY, l = 0.f, acc[VW];
#pragma unroll
  for (int x = 0; x < NW; ++x) mb = fmaxf(mb, sh.st[x][q][0]);
#pragma unroll
  for (int e = 0; e < VW; ++e) acc[e] = 0.f;
#pragma unroll
  for (int x = 0; x < NW; ++x) {
    const float f = sh.st[x][q][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sh.st[x][q][0] - mb);
    l += sh.st[x][q][1] * f;
#pragma unroll
    for (int e = 0; e < VW; ++e) acc[e] += sh.so[x][q][c * VW + e] * f;
  }
  if (it.nsplit > 1) {
    const int64_t slot = (int64_t)it.slot * kPrRows + q;
    float* p = a.c[0].part + slot * a.Dp + c * VW;
#pragma unroll
    for (int e = 0; e < VW; e += 4) *reinterpret_cast<f32x4*>(p + e) = f32x4{acc[e], acc[e + 1], acc[e + 2], acc[e + 3]};
    if (c == 0) {
      a.c[0].stat[slot * 2] = mb;
      a.c[0].stat[slot * 2 + 1] = l;
    }
    return;
  }
  const float inv = pa_inv(it.seq, pa_seen(it, r0 + q, a.f_g) > 0, l);
  const int tk = (int)fdiv((uint32_t)(r0 + q), a.f_g);
  typename T::S* dst = (typename T::S*)a.o + (int64_t)(it.seq.t0 + tk) * a.ost +
                       (int64_t)(it.hk * a.G + r0 + q - tk * a.G) * a.osh + c * VW;
  if constexpr (T::kCode == AK_F32) {
#pragma unroll
    for (int e = 0; e < VW; e += 4)
      *reinterpret_cast<f32x4*>(dst + e) = f32x4{acc[e] * inv, acc[e + 1] * inv, acc[e + 2] * inv, acc[e + 3] * inv};
  } else {
    typename PrVec<D>::type pk;
#pragma unroll
    for (int e = 0; e < VW / 2; ++e) pk[e] = fa2_pack<T>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
    *reinterpret_cast<typename PrVec<D>::type*>(dst) = pk;
  }
}

// A piece of a K or V row. STREAM: nontemporal, for keys that no other block reads (64 ragged sequences 129.5 ->
// 120.6 us a call; 256 x 4000 tokens 711 -> 649; 40 x 1600 after a flush of the caches 72 -> 68, but 56 -> 63 where the
// last call's keys are still in them).
template <bool STREAM, typename V>
__device__ __forceinline__ V pr_load(const uint16_t* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
  else return *reinterpret_cast<const V*>(p);
}

template <typename T, int D, int PG, int NW, bool STREAM>
__device__ __forceinline__ void pa_rows_item(const PaArgs& a, uint32_t item, PrShared<D, NW>& sh) {
  constexpr int NS = D / 32, VW = D / 16;
  constexpr int NK = PG == 8 ? 1 : 2, NV = PG == 8 ? 1 : 8;  // page numbers of a lane and step
  using VV = typename PrVec<D>::type;
  PaItem it;
  if (!pa_find<kPrRows, 0>(a, item, it)) return;
  if (threadIdx.x == 0) sh.again = 0;
  const int lane = lane_id(), w = wave_id();
  const int i16 = lane & 15, g = lane >> 4;
  const uint16_t* Kb = (const uint16_t*)a.kc + it.hk * a.kch + g * 8;
  const uint16_t* Vb = (const uint16_t*)a.vc + it.hk * a.vch + i16 * VW;
  const int rows = it.seq.n * a.G, r0 = it.tile * kPrRows, r = r0 + i16;
  const int lim = r < rows ? pa_seen(it, r, a.f_g) : 0;  // keys that this lane's row sees
  u32x4 qf[NS];
  {
    const int tk = (int)fdiv((uint32_t)min(r, rows - 1), a.f_g);
    const uint16_t* q = (const uint16_t*)a.q + (int64_t)(it.seq.t0 + tk) * a.qst +
                        (int64_t)(it.hk * a.G + min(r, rows - 1) - tk * a.G) * a.qsh;
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] = r < rows ? ld16(q + s * 32 + g * 8) : u32x4{0u, 0u, 0u, 0u};
  }
  const int rl = min(rows, r0 + kPrRows) - 1;  // the tile's last row sees the most
  const int kbeg = pa_begin(it), kend = pa_end(it, pa_seen(it, rl, a.f_g));
  const int full = pa_uniform(pa_seen(it, r0, a.f_g));  // every row sees the keys below

  struct Pages {
    int k[NK], v[NV];
  };
  const int32_t* tab = a.s.table + it.b * a.s.table_stride;
  bool bad = false;
  auto pages = [&](int k0, Pages& p) {
    // keys past the end take the last one's page
#pragma unroll
    for (int x = 0; x < NK; ++x)
      p.k[x] = tab[fdiv((uint32_t)min(k0 + 8 * (i16 >> 2) + (PG == 8 ? 0 : 4 * x + (i16 & 3)), kend - 1), a.s.page_div)];
#pragma unroll
    for (int x = 0; x < NV; ++x) p.v[x] = tab[fdiv((uint32_t)min(k0 + 8 * g + x, kend - 1), a.s.page_div)];
  };
  struct Step {
    u32x4 k[2][NS];
    VV v[8];
  };
  auto load = [&](int k0, const Pages& p, Step& st) {
    const bool tail = k0 + kPrKeys > kend;  // uniform
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int key = min(k0 + 8 * (i16 >> 2) + 4 * t + (i16 & 3), kend - 1);
      const int pg = p.k[PG == 8 ? 0 : t];
      const bool in = (uint32_t)pg < a.s.num_pages;
      const uint32_t slot = (uint32_t)key - fdiv((uint32_t)key, a.s.page_div) * a.s.page_size;
      bad |= !in;
      const uint16_t* src = Kb + (in ? pg * a.kcp + slot * a.kct : 0);
#pragma unroll
      for (int s = 0; s < NS; ++s) st.k[t][s] = in ? pr_load<STREAM, u32x4>(src + s * 32) : u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int key = k0 + 8 * g + e;
      const int pg = p.v[PG == 8 ? 0 : e];
      const bool in = (uint32_t)pg < a.s.num_pages && (!tail || key < kend);
      const uint32_t slot = (uint32_t)key - fdiv((uint32_t)key, a.s.page_div) * a.s.page_size;
      if (in) {
        st.v[e] = pr_load<STREAM, VV>(Vb + pg * a.vcp + slot * a.vct);
      } else {
#pragma unroll
        for (int x = 0; x < VW / 2; ++x) st.v[e][x] = 0u;
      }
    }
  };

  f32x4 o[VW];
#pragma unroll
  for (int e = 0; e < VW; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;  // l_run: this lane's keys only
  auto compute = [&](int k0, const Step& st) {
    f32x4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < NS; ++x)
#pragma unroll
      for (int t = 0; t < 2; ++t) s[t] = mfma16x16x32<T>(st.k[t][x], qf[x], s[t]);
    if (k0 + kPrKeys > full) {
      const int left = min(lim, kend) - (k0 + 8 * g);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          if (4 * t + v >= left) s[t][v] = -INFINITY;
    }
    float mt = fa2_max(fa2_max(s[0][0], s[0][1]), fa2_max(s[0][2], s[0][3]));
    mt = fa2_max(mt, fa2_max(fa2_max(s[1][0], s[1][1]), fa2_max(s[1][2], s[1][3])));
    mt = pr_groups(mt, PrMaximum());
    const float m_new = fa2_max(m_run, mt * a.c_log2);
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = m_new == m_run ? 1.0f : __builtin_amdgcn_exp2f(m_run - base);
    m_run = m_new;
    u32x4 pf;
    float ps = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 1][2 * (e & 1)], a.c_log2, -base));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 1][2 * (e & 1) + 1], a.c_log2, -base));
      pf[e] = fa2_pack<T>(p0, p1);
      ps = fa2_sum2<T>(pf[e], ps);
    }
    l_run = l_run * alpha + ps;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
      for (int e = 0; e < VW; ++e)
#pragma unroll
        for (int v = 0; v < 4; ++v) o[e][v] *= alpha;
    }
#pragma unroll
    for (int e = 0; e < VW; ++e) {
      const uint32_t sel = (e & 1) ? 0x07060302u : 0x05040100u;
      u32x4 vt;
#pragma unroll
      for (int p = 0; p < 4; ++p) vt[p] = __builtin_amdgcn_perm(st.v[2 * p + 1][e >> 1], st.v[2 * p][e >> 1], sel);
      o[e] = mfma16x16x32<T>(vt, pf, o[e]);
    }
  };

  constexpr int kStride = NW * kPrKeys;
  int k0 = kbeg + pa_uniform(w) * kPrKeys;
  if (k0 < kend) {
    Step s0, s1;
    Pages p0, p1;
    pages(k0, p0);
    if (k0 + kStride < kend) pages(k0 + kStride, p1);
    load(k0, p0, s0);
    while (true) {
      const bool more1 = k0 + kStride < kend;
      if (k0 + 2 * kStride < kend) pages(k0 + 2 * kStride, p0);
      if (more1) load(k0 + kStride, p1, s1);
      compute(k0, s0);
      if (!more1) break;
      k0 += kStride;
      const bool more0 = k0 + kStride < kend;
      if (k0 + 2 * kStride < kend) pages(k0 + 2 * kStride, p1);
      if (more0) load(k0 + kStride, p0, s0);
      compute(k0, s1);
      if (!more0) break;
      k0 += kStride;
    }
  }
  pr_finish<T, D, NW>(a, it, sh, o, m_run, l_run, bad, rows, r0, kbeg, kend);
}

// The same in fp32 (v_mfma_f32_16x16x4, whose products and sums are fp32), 16 keys a step. A lane's K operand is
// a quarter of one key's row: the contraction's order is free, so k index g of step s is dim g D / 4 + s and K
// and Q load as whole vectors. S^T leaves lane group g with the scores of keys 4 g .. 4 g + 3, so step t of
// O^T += V^T P^T takes keys 4 g + t: weight t as it stands, and the V rows of four consecutive keys.
// 43 tokens of four sequences over 4000 cached ones, 12 heads of 64 on 4 KV heads: 16.5 us a call, 84 by pa_general.
template <int D, int PG, int NW>
__device__ __forceinline__ void pa_rows_f32_item(const PaArgs& a, uint32_t item, PrShared<D, NW>& sh) {
  constexpr int NS = D / 4, VW = D / 16;
  constexpr int kKeys = 16, NV = PG == 4 ? 1 : 4;
  PaItem it;
  if (!pa_find<kPrRows, 0>(a, item, it)) return;
  if (threadIdx.x == 0) sh.again = 0;
  const int lane = lane_id(), w = wave_id();
  const int i16 = lane & 15, g = lane >> 4;
  const float* Kb = (const float*)a.kc + it.hk * a.kch + g * NS;
  const float* Vb = (const float*)a.vc + it.hk * a.vch + i16 * VW;
  const int rows = it.seq.n * a.G, r0 = it.tile * kPrRows, r = r0 + i16;
  const int lim = r < rows ? pa_seen(it, r, a.f_g) : 0;
  f32x4 qf[NS / 4];
  {
    const int tk = (int)fdiv((uint32_t)min(r, rows - 1), a.f_g);
    const float* q = (const float*)a.q + (int64_t)(it.seq.t0 + tk) * a.qst +
                     (int64_t)(it.hk * a.G + min(r, rows - 1) - tk * a.G) * a.qsh + g * NS;
#pragma unroll
    for (int s = 0; s < NS / 4; ++s)
      qf[s] = r < rows ? *reinterpret_cast<const f32x4*>(q + 4 * s) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int rl = min(rows, r0 + kPrRows) - 1;
  const int kbeg = pa_begin(it), kend = pa_end(it, pa_seen(it, rl, a.f_g));
  const int full = pa_uniform(pa_seen(it, r0, a.f_g));
  struct Pages {
    int k, v[NV];
  };
  const int32_t* tab = a.s.table + it.b * a.s.table_stride;
  bool bad = false;
  auto pages = [&](int k0, Pages& p) {
    p.k = tab[fdiv((uint32_t)min(k0 + i16, kend - 1), a.s.page_div)];
#pragma unroll
    for (int x = 0; x < NV; ++x) p.v[x] = tab[fdiv((uint32_t)min(k0 + 4 * g + x, kend - 1), a.s.page_div)];
  };
  struct Step {
    f32x4 k[NS / 4], v[4][VW / 4];
  };
  auto load = [&](int k0, const Pages& p, Step& st) {
    {
      const int key = min(k0 + i16, kend - 1);
      const bool in = (uint32_t)p.k < a.s.num_pages;
      bad |= !in;
      const uint32_t slot = (uint32_t)key - fdiv((uint32_t)key, a.s.page_div) * a.s.page_size;
      const float* src = Kb + (in ? p.k * a.kcp + slot * a.kct : 0);
#pragma unroll
      for (int s = 0; s < NS / 4; ++s)
        st.k[s] = in ? *reinterpret_cast<const f32x4*>(src + 4 * s) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int key = k0 + 4 * g + t, pg = p.v[PG == 4 ? 0 : t];
      const bool in = (uint32_t)pg < a.s.num_pages && key < kend;
      const uint32_t slot = (uint32_t)key - fdiv((uint32_t)key, a.s.page_div) * a.s.page_size;
      const float* src = Vb + (in ? pg * a.vcp + slot * a.vct : 0);
#pragma unroll
      for (int e = 0; e < VW / 4; ++e)
        st.v[t][e] = in ? *reinterpret_cast<const f32x4*>(src + 4 * e) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
  };
  f32x4 o[VW];
#pragma unroll
  for (int e = 0; e < VW; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;
  auto compute = [&](int k0, const Step& st) {
    f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};  // even and odd steps: two chains
#pragma unroll
    for (int x = 0; x < NS; ++x)
      s[x & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(st.k[x / 4][x % 4], qf[x / 4][x % 4], s[x & 1], 0, 0, 0);
    f32x4 z = s[0] + s[1];
    if (k0 + kKeys > full) {
      const int left = min(lim, kend) - (k0 + 4 * g);
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (v >= left) z[v] = -INFINITY;
    }
    float mt = fa2_max(fa2_max(z[0], z[1]), fa2_max(z[2], z[3]));
    mt = pr_groups(mt, PrMaximum());
    const float m_new = fa2_max(m_run, mt * a.c_log2);
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = m_new == m_run ? 1.0f : __builtin_amdgcn_exp2f(m_run - base);
    m_run = m_new;
    float p[4], ps = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      p[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[v], a.c_log2, -base));
      ps += p[v];
    }
    l_run = l_run * alpha + ps;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
      for (int e = 0; e < VW; ++e)
#pragma unroll
        for (int v = 0; v < 4; ++v) o[e][v] *= alpha;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < VW; ++e) o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(st.v[t][e / 4][e % 4], p[t], o[e], 0, 0, 0);
  };
  constexpr int kStride = NW * kKeys;
  int k0 = kbeg + pa_uniform(w) * kKeys;
  if (k0 < kend) {
    Step s0, s1;
    Pages p0, p1;
    pages(k0, p0);
    if (k0 + kStride < kend) pages(k0 + kStride, p1);
    load(k0, p0, s0);
    while (true) {
      const bool more1 = k0 + kStride < kend;
      if (k0 + 2 * kStride < kend) pages(k0 + 2 * kStride, p0);
      if (more1) load(k0 + kStride, p1, s1);
      compute(k0, s0);
      if (!more1) break;
      k0 += kStride;
      const bool more0 = k0 + kStride < kend;
      if (k0 + 2 * kStride < kend) pages(k0 + 2 * kStride, p1);
      if (more0) load(k0 + kStride, p0, s0);
      compute(k0, s1);
      if (!more0) break;
      k0 += kStride;
    }
  }
  pr_finish<TF32, D, NW>(a, it, sh, o, m_run, l_run, bad, rows, r0, kbeg, kend);
}

// Many rows per KV head: 128 rows a block, a wave owns 32, 64 keys a step through LDS. The pipeline of fa_fwd2
// (attention.hip: S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16, K and V by LDS DMA two stages deep, V
// read transposed by ds_read_b64_tr_b16, each MFMA burst beside the other product's softmax work, the
// lazily raised exp2 base). What is different:
//   * A row is a (token, head of the group) pair, so the query heads of a KV head share its K and V tiles.
//   * A wave brings 16 consecutive keys of a tile, which with pages of a multiple of 16 slots lie in one page,
//     through a buffer resource of that page's address and as many bytes as the slice has keys left there (the
//     rest arrives as zeros). The resources of 64 tiles are made at once, one per lane.
//   * No pass over what a row does not see: V of masked keys only has to be finite. Where a row's result is
//     NaN, or a page lies outside the cache, the item's rows are computed again by pa_row.
// Bound by the MFMA and the softmax VALU work, as fa_fwd2 is. 512 tokens after 16001 (32 heads of 128, 8 KV heads,
// bf16): 156 us, 875 TFLOP/s, MFMA busy 40 % of the time, half of it waiting; four prompts of 2048: 167 to 186 us, 740
// to 820. A prompt of 8192 runs at 992 TFLOP/s, fa_fwd2 on dense keys at 1074.
constexpr int kPtRows = 32 * kPaWaves;

// fa2_dma16 for a resource made right before it: its words come from v_readlane / v_readfirstlane, and a vector
// memory instruction may read a scalar register that the VALU wrote only five wait states later. The compiler
// keeps that distance for its own instructions but does not see the load in here.
__device__ __forceinline__ void pa_dma16(const u32x4& rsrc, uint32_t voff, uint32_t lds) {
  asm volatile(
      "s_nop 4\n\t"
      "buffer_load_dwordx4 %0, %1, 0 offen lds"
      :
      : "v"(voff), "s"(rsrc), "{m0}"(lds)
      : "memory");
}
template <int D>
struct PtShared {
  uint16_t k[2 * kFaBKV * D], v[2 * kFaBKV * D];
  int again;
};
template <typename T, int D>
__device__ __forceinline__ void pa_tiles_item(const PaArgs& a, uint32_t item, PtShared<D>& sh) {
  constexpr int DC = D / 8;                            // 16-byte chunks per key
  constexpr int RPI = 64 / DC;                         // keys per 1 KB transfer
  constexpr int NIW = kFaBKV / RPI / kPaWaves;         // transfers per wave and tile, per matrix
  constexpr int NS = D / 16, NDB = D / 32;             // 16-deep steps of S^T, 32-row blocks of O^T
  constexpr int TILE = kFaBKV * D;
  PaItem it;
  if (!pa_find<kPtRows, 1>(a, item, it)) return;
  if (threadIdx.x == 0) sh.again = 0;
  const int lane = lane_id(), l32 = lane & 31, hh = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(wave_id());
  const int rows = it.seq.n * a.G, r0 = it.tile * kPtRows, rw0 = r0 + 32 * w;  // this wave's first row
  const int my_r = rw0 + l32;
  const int kbeg = pa_begin(it), kend = pa_end(it, pa_seen(it, min(rows, r0 + kPtRows) - 1, a.f_g));
  const int tk = (int)fdiv((uint32_t)min(my_r, rows - 1), a.f_g);
  const int64_t head = it.hk * a.G + min(my_r, rows - 1) - tk * a.G, tok = it.seq.t0 + tk;
  const int nt = pa_uniform((max(kend - kbeg, 0) + kFaBKV - 1) / kFaBKV);
  float m_run = -INFINITY, l_run = 0.f;
  f32x16 o[NDB];
#pragma unroll
  for (int i = 0; i < NDB; ++i)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[i][v] = 0.f;
  bool bad = false;

  if (nt > 0) {
    // keys seen by this lane's row, by the wave's first row and by its last
    const int lim = min(pa_seen(it, min(my_r, rows - 1), a.f_g), kend);
    const int lim0 = pa_uniform(min(pa_seen(it, min(rw0, rows - 1), a.f_g), kend));
    const int lim1 = pa_uniform(min(pa_seen(it, min(rw0 + 31, rows - 1), a.f_g), kend));
    const int jw = pa_uniform(rw0 < rows && lim1 > kbeg ? (lim1 - 1 - kbeg) / kFaBKV : -1);  // the wave's last tile

    const uint16_t* Qr = (const uint16_t*)a.q + tok * a.qst + head * a.qsh;
    u32x4 qf[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] = my_r < rows ? ld16(Qr + s * 16 + hh * 8) : u32x4{0u, 0u, 0u, 0u};

    // Byte offsets of a lane inside its wave's 16 keys: transfer i writes rows 16 w + i RPI .. of the tile, lane L
    // physical chunk L % DC of row L / DC of them, and so fetches the logical chunk that the swizzle maps there.
    uint32_t offk[NIW], offv[NIW];
#pragma unroll
    for (int i = 0; i < NIW; ++i) {
      const int in16 = i * RPI + lane / DC;
      offk[i] = (uint32_t)(in16 * (int)a.kct * 2 + (((lane % DC) ^ fa2_kswz<D>(in16)) * 16));
      offv[i] = (uint32_t)(in16 * (int)a.vct * 2 + (((lane % DC) ^ fa2_vswz<D>(in16)) * 16));
    }
    const uint32_t sK_lds = (uint32_t)(uintptr_t)(lds_void*)sh.k, sV_lds = (uint32_t)(uintptr_t)(lds_void*)sh.v;
    // Where the wave's keys of tile (j & ~63) + lane lie: address and bytes, all 64 tiles side by side. (Made for
    // each tile and transfer by the scalar unit, 35 instructions each, this cost a third of the kernel's time.)
    struct Where {
      uint32_t lo, hi, n;
    };
    const int32_t* tab = a.s.table + it.b * a.s.table_stride;
    auto find = [&](int j, const uint16_t* base, uint32_t page_bytes, uint32_t slot_bytes) {
      const int key = kbeg + ((j & ~63) + lane) * kFaBKV + 16 * w, left = min(kend - key, 16);
      const bool any = left > 0;
      const uint32_t e = fdiv((uint32_t)min(key, kend - 1), a.s.page_div);
      const uint32_t slot = (uint32_t)min(key, kend - 1) - e * (uint32_t)a.s.page_size;
      const uint32_t page = (uint32_t)tab[e];
      const bool in = page < (uint32_t)a.s.num_pages;
      bad |= any && !in;
      const uint64_t at = (uint64_t)(uintptr_t)base + (uint64_t)page * page_bytes + (uint64_t)slot * slot_bytes;
      return Where{(uint32_t)at, (uint32_t)(at >> 32) & 0xffffu,
                   any && in ? (uint32_t)(left - 1) * slot_bytes + D * 2 : 0u};
    };
    auto issue = [&](const Where& x, int j, const uint32_t (&off)[NIW], uint32_t lds) {
      const u32x4 rs = {(uint32_t)__builtin_amdgcn_readlane((int)x.lo, j & 63),
                        (uint32_t)__builtin_amdgcn_readlane((int)x.hi, j & 63),
                        (uint32_t)__builtin_amdgcn_readlane((int)x.n, j & 63), 0x00020000u};
#pragma unroll
      for (int i = 0; i < NIW; ++i) pa_dma16(rs, off[i], lds + (w * NIW + i) * 1024);
    };
    const uint16_t* Kb = (const uint16_t*)a.kc + it.hk * a.kch;
    const uint16_t* Vb = (const uint16_t*)a.vc + it.hk * a.vch;
    Where wk, wv;
    auto issue_k = [&](int j, int stage) {
      if ((j & 63) == 0) wk = find(j, Kb, (uint32_t)a.kcp * 2, (uint32_t)a.kct * 2);
      issue(wk, j, offk, sK_lds + stage * TILE * 2);
    };
    auto issue_v = [&](int j, int stage) {
      if ((j & 63) == 0) wv = find(j, Vb, (uint32_t)a.vcp * 2, (uint32_t)a.vct * 2);
      issue(wv, j, offv, sV_lds + stage * TILE * 2);
    };

    auto qk = [&](const uint16_t* ks, f32x16 (&s)[2]) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int v = 0; v < 16; ++v) s[kb][v] = 0.f;
#pragma unroll
      for (int st = 0; st < NS; ++st)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const int r = kb * 32 + l32, c = st * 2 + hh;
          const u32x4 kf = *reinterpret_cast<const u32x4*>(&ks[r * D + (c ^ fa2_kswz<D>(r)) * 8]);
          s[kb] = mfma32x32x16<T>(kf, qf[st], s[kb]);
        }
    };
    const int g16 = lane >> 4, i16 = lane & 15;
    const int vrow = 4 * (g16 >> 1) + (i16 >> 2), vcol = 16 * (g16 & 1) + 4 * (i16 & 3), vsw = fa2_vswz<D>(vrow);
    u32x4 pf[4];
    auto pv = [&](const uint16_t* vs) {
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int col = db * 32 + vcol;
          const uint16_t* p = vs + (16 * t + vrow) * D + (((col >> 3) ^ vsw) * 8) + (col & 7);
          const u32x2 lo = fa2_tr16(p), hi = fa2_tr16(p + 8 * D);
          o[db] = mfma32x32x16<T>(u32x4{lo[0], lo[1], hi[0], hi[1]}, pf[t], o[db]);
        }
    };
    // Row statistics of S_j: mask, tile max, lazy base update (alpha = 1 unless it moved).
    auto stats = [&](f32x16 (&s)[2], int k0, bool masked, float& alpha, float& base) {
      if (masked) {
        const int t = lim - (k0 + hh * 4);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int off = kb * 32 + (v >> 2) * 8 + (v & 3);
            if (off >= t) s[kb][v] = -INFINITY;
          }
      }
      float m4[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int kb = c >> 1, v0 = (c & 1) * 8;
        float m = fa2_max(fa2_max(s[kb][v0], s[kb][v0 + 1]), s[kb][v0 + 2]);
        m = fa2_max(fa2_max(m, s[kb][v0 + 3]), s[kb][v0 + 4]);
        m4[c] = fa2_max(fa2_max(m, s[kb][v0 + 5]), s[kb][v0 + 6]);
      }
      float mt = fa2_max(fa2_max(m4[0], s[0][7]), m4[1]);
      mt = fa2_max(fa2_max(mt, s[0][15]), m4[2]);
      mt = fa2_max(fa2_max(mt, s[1][7]), m4[3]);
      mt = fa2_max(mt, s[1][15]);
      const float mts = fa2_halves_max(mt) * a.c_log2;
      const float m_new = (mts > m_run + kFa2Slack || m_run == -INFINITY) ? fmaxf(m_run, mts) : m_run;
      base = (m_new == -INFINITY) ? 0.f : m_new;
      alpha = (m_new == m_run) ? 1.0f : __builtin_amdgcn_exp2f(m_run - base);
      m_run = m_new;
    };
    auto exp_args = [&](f32x16 (&s)[2], float base) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int v = 0; v < 16; ++v) s[kb][v] = __builtin_fmaf(s[kb][v], a.c_log2, -base);
    };
    auto exp_pack = [&](const f32x16 (&s)[2]) -> float {
      float ps = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int v = 8 * (t & 1) + 2 * e;
          pf[t][e] = fa2_pack<T>(__builtin_amdgcn_exp2f(s[t >> 1][v]), __builtin_amdgcn_exp2f(s[t >> 1][v + 1]));
          ps = fa2_sum2<T>(pf[t][e], ps);
        }
      return ps;
    };
    auto rescale = [&](float alpha) {
      if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[db][v] *= alpha;
      }
    };
    // The DMA schedule and its waits are fa_fwd2's: tile t lives in stage t & 1; V_{j+1} is issued after
    // phase 1 of iteration j, K_{j+3} after phase 2, and a wait leaves the transfers issued later in flight.
    // (The compiler's own waits cover find's global load.)
    auto barrier_after = [&](int later) {
      if (later >= 2) dma_barrier<2 * NIW>();
      else if (later == 1) dma_barrier<NIW>();
      else dma_barrier<0>();
    };
    auto sync_mid = [&](int j, int par) {
      barrier_after(j == 0 ? (nt > 2) : 1 + (j + 2 < nt));
      if (j + 1 < nt) issue_v(j + 1, par ^ 1);
    };
    auto sync_end = [&](int j, int par) {
      barrier_after((j + 2 < nt) + (j + 1 < nt));
      if (j + 3 < nt) issue_k(j + 3, par ^ 1);
    };
    f32x16 sa[2], sb[2];
    auto iter = [&](int j, int par, f32x16 (&S)[2], f32x16 (&Sn)[2]) {
      const int k0 = kbeg + j * kFaBKV;
      if (j > 0 && j - 1 <= jw) pv(sh.v + (par ^ 1) * TILE);  // V_{j-1}
      float alpha = 1.0f, base = 0.f;
      const bool act = j <= jw;
      if (act) stats(S, k0, k0 + kFaBKV > lim0, alpha, base);
      sync_mid(j, par);
      if (j + 1 <= jw) qk(sh.k + (par ^ 1) * TILE, Sn);  // K_{j+1}
      if (act) {
        exp_args(S, base);
        const float ps = exp_pack(S);
        l_run = l_run * alpha + ps;
        rescale(alpha);
      }
      sync_end(j, par);
    };
    constexpr int kPhaseMfma = D / 8, kP1Valu = D == 128 ? 4 : 8, kP2Valu = D == 128 ? 5 : 9;
    auto iter_fast = [&](int j, int par, f32x16 (&S)[2], f32x16 (&Sn)[2]) {
      pv(sh.v + (par ^ 1) * TILE);
      float alpha, base;
      stats(S, kbeg + j * kFaBKV, false, alpha, base);
      exp_args(S, base);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) asm volatile("" ::"v"(S[kb]));
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for (int i = 0; i < kPhaseMfma - 2; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, kP1Valu, 0);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, kP1Valu, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      sync_mid(j, par);
      qk(sh.k + (par ^ 1) * TILE, Sn);
      const float ps = exp_pack(S);
#pragma unroll
      for (int t = 0; t < 4; ++t) asm volatile("" ::"v"(pf[t]));
      asm volatile("" ::"v"(ps));
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
#pragma unroll
      for (int i = 0; i < kPhaseMfma - 2; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
        __builtin_amdgcn_sched_group_barrier(0x402, kP2Valu, 1);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
        __builtin_amdgcn_sched_group_barrier(0x402, kP2Valu, 1);
      }
      __builtin_amdgcn_sched_barrier(0);
      rescale(alpha);
      l_run = l_run * alpha + ps;
      sync_end(j, par);
    };

    issue_k(0, 0);
    if (nt > 1) issue_k(1, 1);
    issue_v(0, 0);
    dma_barrier<0>();
    qk(sh.k, sa);
    dma_barrier<0>();
    if (nt > 2) issue_k(2, 0);
    const int jm = max(lim0 - kbeg, 0) / kFaBKV;  // the wave's first masked tile
    const int jf = max(1, min(jm, jw));
    iter(0, 0, sa, sb);
    int j = 1;
    for (; j + 1 < jf; j += 2) {
      iter_fast(j, 1, sb, sa);
      iter_fast(j + 1, 0, sa, sb);
    }
    if (j < jf) {
      iter_fast(j, 1, sb, sa);
      ++j;
    } else {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) sa[kb] = sb[kb];
    }
    for (; j < nt; ++j) {
      iter(j, j & 1, sa, sb);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) sa[kb] = sb[kb];
    }
    if (nt - 1 <= jw) pv(sh.v + ((nt - 1) & 1) * TILE);
    wait_vmcnt<0>();  // no transfer outlives the block
    l_run = fa2_halves_sum(l_run);
    if (my_r < rows) {
      bad |= l_run != l_run;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) bad |= o[db][v] != o[db][v];
    }
  }
  __syncthreads();  // (the flag is cleared by now)
  if (__builtin_amdgcn_ballot_w64(bad) && lane == 0) atomicOr(&sh.again, 1);
  __syncthreads();
  if (sh.again) {
    pa_one_by_one<T, kPtRows, 1>(a, it, r0, min(rows, r0 + kPtRows), kbeg, kend);
    return;
  }
  if (my_r >= rows) return;
  if (it.nsplit > 1) {
    const int64_t slot = (int64_t)it.slot * kPtRows + 32 * w + l32;
    float* p = a.c[1].part + slot * a.Dp;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(p + db * 32 + g * 8 + hh * 4) =
            f32x4{o[db][g * 4], o[db][g * 4 + 1], o[db][g * 4 + 2], o[db][g * 4 + 3]};
    if (hh == 0) {
      a.c[1].stat[slot * 2] = m_run;
      a.c[1].stat[slot * 2 + 1] = l_run;
    }
    return;
  }
  const float inv = pa_inv(it.seq, pa_seen(it, my_r, a.f_g) > 0, l_run);
  uint16_t* orow = (uint16_t*)a.o + tok * a.ost + head * a.osh;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      u32x2 pk2;
      pk2[0] = fa2_pack<T>(o[db][g * 4] * inv, o[db][g * 4 + 1] * inv);
      pk2[1] = fa2_pack<T>(o[db][g * 4 + 2] * inv, o[db][g * 4 + 3] * inv);
      *reinterpret_cast<u32x2*>(orow + db * 32 + g * 8 + hh * 4) = pk2;
    }
}

template <typename T, int D, int PG, int NW, bool STREAM>
__global__ __launch_bounds__(NW* kWave, 2) void pa_rows(const PaArgs a) {
  __shared__ __attribute__((aligned(16))) PrShared<D, NW> sh;
  if constexpr (T::kCode == AK_F32) pa_rows_f32_item<D, PG == 8 ? 4 : 1, NW>(a, blockIdx.x, sh);
  else pa_rows_item<T, D, PG, NW, STREAM>(a, blockIdx.x, sh);
}
// Both classes in one launch: the blocks of the large tiles first.
template <typename T, int D>
__global__ __launch_bounds__(kPaThreads, 2) void pa_mixed(const PaArgs a) {
  __shared__ __attribute__((aligned(1024))) union {
    PtShared<D> t;
    PrShared<D, kPaWaves> r;
  } sh;
  if (blockIdx.x < a.c[1].items) pa_tiles_item<T, D>(a, blockIdx.x, sh.t);
  else pa_rows_item<T, D, 8, kPaWaves, true>(a, blockIdx.x - a.c[1].items, sh.r);
}

// What a call launches: the most items of each class and their partials. Keys are sliced only where some
// sequence can be longer than kPaMinSliced, below which the merge costs what the shorter walk saves (one
// sequence of 1000 keys: 5 us each).
// Items aimed at: 1536 tiles of 16 rows (64 ragged sequences 120.4 us; 1024: 123.2, 2048: 120.9; two thirds for
// sequences of about one length, see pa_chunk), 512 of 128
// rows (512 tokens after 16001 157 us; 1024: 172).
// A sequence of more rows than one tile of 16 takes tiles of 128, which read its keys once (64 sequences over 2000
// tokens, 32 / 64 rows each: 103 / 109 us, in tiles of 16: 179 / 204), in calls where that pays:
//   * With sliced keys, where some sequence has several new tokens (two of 8 over 8000: 24.4 us, 28.6 without), or with
//     more than kPaTiledRows rows. The rows of up to 16 single tokens stay with blocks of eight waves (8 / 16
//     sequences of 1000, 4 rows each: 15.7 / 17.4 us, 19.4 / 21.1 beside empty large tiles).
//   * With whole keys, where the tiles of 16 would be more than two per CU, about what runs at a time: a wave of the
//     large tiles walks all the keys, a wave of the small ones a fourth (30 tokens each of 4 sequences of 1000: 17.7 us,
//     31.8 with the large tiles; 100 tokens each: 32.3, 44.0 without).
constexpr int64_t kPaSplitRows = 16, kPaTiledRows = 64, kPaMinSliced = 1536, kPaOneEach = 256;
struct PaPlan {
  int bm0;
  int64_t items[2], target[2], ws[2];  // ws: floats of a class's partials
  int64_t bytes() const { return (ws[0] + ws[1]) * (int64_t)sizeof(float); }
};
// fast: the MFMA kernels; pa_tiles needs pages of a multiple of 16 slots
static PaPlan pa_plan(int dtype, int64_t T, int64_t B, int64_t Hq, int64_t Hk, int64_t D, int64_t page_size,
                      int64_t width, bool fast) {
  PaPlan p{};
  const int64_t keys = page_size * width, G = Hq / Hk, rows = T * G, seqs = std::min(B, T);
  const bool sliced = keys > kPaMinSliced;
  p.bm0 = fast ? kPrRows : kPaRowTile;
  p.items[0] = (rows / p.bm0 + seqs) * Hk;
  const bool tiles = fast && dtype != AK_F32 && page_size % 16 == 0 && rows > kPaSplitRows &&
                     (sliced ? T > B || rows > kPaTiledRows : (rows / kPrRows + seqs / 2) * Hk > 2 * kPaOneEach);
  if (tiles) {
    p.items[0] = std::min(p.items[0], seqs * ((kPaSplitRows + p.bm0 - 1) / p.bm0) * Hk);
    p.items[1] = (rows / kPtRows + std::min(seqs, rows / (kPaSplitRows + 1))) * Hk;
  }
  if (sliced) {
    p.target[0] = 1536;
    // two tiles per CU at a time; four times that many are work enough unsliced
    if (tiles && rows / kPtRows * Hk < 4 * 512) p.target[1] = 512;
  }
  const int64_t row = (D + 3) / 4 * 4 + 2;
  for (int c = 0; c < 2; ++c)
    if (p.target[c] > 0) {
      p.items[c] += p.target[c];
      p.ws[c] = p.items[c] * (c ? kPtRows : p.bm0) * row;
    }
  return p;
}

static void pa_set(PaArgs& a, const PaPlan& p, void* ws) {
  float* f = (float*)ws;
  for (int c = 0; c < 2; ++c) {
    a.c[c].items = (uint32_t)p.items[c];
    a.c[c].target = (float)p.target[c];
    a.c[c].part = f;
    a.c[c].stat = f ? f + p.items[c] * (c ? kPtRows : p.bm0) * a.Dp : nullptr;
    if (f) f += p.ws[c];
  }
  a.split_rows = p.items[1] > 0 ? (int)kPaSplitRows : INT_MAX;
}
template <typename T, int BM0, int BM1, int JN>
static void pa_launch_merge(PaArgs& a, hipStream_t st) {
  if (a.c[0].target <= 0.f && a.c[1].target <= 0.f) return;
  const int64_t rows = (int64_t)a.s.T * a.Hq;
  // 64 tokens of 32 heads, up to 7 slices: a block per row costs the call 2.4 us more than a group
  const bool wide = rows < 1024;
  a.f_units = make_fastdiv((uint32_t)(wide ? a.Hq : (a.Hq + 3) / 4));
  // where only sequences with few rows may be sliced, blocks for as many rows as these can have
  const int64_t most = a.c[1].target > 0.f || a.c[1].items == 0 ? rows : (int64_t)a.s.B * a.split_rows * a.Hk;
  const int64_t blocks = std::min<int64_t>(cdiv(std::min(rows, most), 4 * kPaWaves), 2048);
  if (wide) pa_merge<T, BM0, BM1, JN, true><<<dim3((unsigned)rows), kPaThreads, 0, st>>>(a);
  else pa_merge<T, BM0, BM1, JN, false><<<dim3((unsigned)blocks), kPaThreads, 0, st>>>(a);
}
template <typename T>
static int launch_general(PaArgs a, const PaPlan& p, void* ws, hipStream_t st) {
  pa_set(a, p, ws);
  pa_general<T><<<dim3((unsigned)p.items[0]), kPaThreads, 0, st>>>(a);
  pa_launch_merge<T, kPaRowTile, kPaRowTile, 4>(a, st);
  return record_launch();
}
// Blocks of eight waves where a batch has at most one per CU: each wave walks half as many keys (one sequence of
// 1000: 14.4 us, 15.8 with four). With more blocks than that four waves leave room for a second one on the CU.
// Single tokens over long caches stream their keys (16 over 8000: 105 -> 97 us); fp32 keys, which take several loads per
// 128 bytes, do not (210 -> 375).
template <typename T, int D, int PG>
static void launch_rows(const PaArgs& a, const PaPlan& p, hipStream_t st) {
  const dim3 grid((unsigned)p.items[0]);
  if (p.items[0] <= kPaOneEach) {
    pa_rows<T, D, PG, 8, false><<<grid, 8 * kWave, 0, st>>>(a);
    return;
  }
  if constexpr (T::kCode != AK_F32) {
    if (p.target[0] > 0 && a.s.T <= a.s.B) {
      pa_rows<T, D, PG, kPaWaves, true><<<grid, kPaThreads, 0, st>>>(a);
      return;
    }
  }
  pa_rows<T, D, PG, kPaWaves, false><<<grid, kPaThreads, 0, st>>>(a);
}
template <typename T, int D>
static int launch_fast(PaArgs a, const PaPlan& p, void* ws, hipStream_t st) {
  pa_set(a, p, ws);
  if constexpr (T::kCode != AK_F32) {
    if (p.items[1] > 0) {
      pa_mixed<T, D><<<dim3((unsigned)(p.items[0] + p.items[1])), kPaThreads, 0, st>>>(a);
      pa_launch_merge<T, kPrRows, kPtRows, D / 64>(a, st);
      return record_launch();
    }
  }
  if (a.s.page_size % 8 == 0) launch_rows<T, D, 8>(a, p, st);
  else launch_rows<T, D, 1>(a, p, st);
  pa_launch_merge<T, kPrRows, kPrRows, D / 64>(a, st);
  return record_launch();
}
template <typename T>
static int launch_fast(const PaArgs& a, const PaPlan& p, void* ws, hipStream_t st) {
  return a.D == 64 ? launch_fast<T, 64>(a, p, ws, st) : launch_fast<T, 128>(a, p, ws, st);
}

static bool pa_sizes_ok(int64_t T, int64_t B, int64_t Hq, int64_t Hk, int64_t D) {
  if (T < 0 || B < 0 || Hq < 0 || Hk <= 0 || D <= 0 || Hq % Hk != 0 || Hq > 65536) return false;
  return T <= INT_MAX && B < INT_MAX && T * Hq < (int64_t)1 << 31 && std::min(B, T) * Hk < (int64_t)1 << 31;
}
static bool pa_plan_fits(const PaPlan& p) { return grid_fits(p.items[0] + p.items[1], 8 * kWave); }

}  // namespace ak

using namespace ak;

// The workspace is sized for the MFMA kernels wherever dtype and head_dim allow them; a call that turns out
// unaligned needs less.
extern "C" int64_t ak_paged_attn_workspace_bytes(int dtype, int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                                                 int64_t page_size, int64_t max_pages) {
  if (dtype != AK_F32 && dtype != AK_F16 && dtype != AK_BF16) return 0;
  if (!pa_sizes_ok(T, B, Hq, Hkv, D) || T == 0 || B == 0 || Hq == 0 || page_size <= 0 || max_pages < 0) return 0;
  if (page_size > INT_MAX || max_pages > INT_MAX) return 0;
  const PaPlan f = pa_plan(dtype, T, B, Hq, Hkv, D, page_size, max_pages, D == 64 || D == 128);
  const PaPlan g = pa_plan(dtype, T, B, Hq, Hkv, D, page_size, max_pages, false);
  return std::max(pa_plan_fits(f) ? f.bytes() : 0, pa_plan_fits(g) ? g.bytes() : 0);
}

extern "C" int ak_paged_attn(int dtype, const void* q, const void* k_cache, const void* v_cache, void* o,
                             const int32_t* page_table, const int32_t* q_starts, const int32_t* kv_lens, int64_t T,
                             int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t num_pages, int64_t page_size,
                             int64_t max_pages, int64_t table_stride, const int64_t* q_strides,
                             const int64_t* k_cache_strides, const int64_t* v_cache_strides, const int64_t* o_strides,
                             float sm_scale, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  if (dtype != AK_F32 && dtype != AK_F16 && dtype != AK_BF16) return AK_EINVAL;
  if (!pa_sizes_ok(T, B, Hq, Hkv, D)) return AK_EINVAL;
  if (D > 256) return AK_EUNSUPPORTED;
  if (!paged_args_ok(page_table, q_starts, kv_lens, T, B, num_pages, page_size, max_pages, table_stride))
    return AK_EINVAL;
  if (T == 0 || B == 0 || Hq == 0) return AK_OK;
  if (!q || !o || !q_strides || !o_strides || !k_cache_strides || !v_cache_strides) return AK_EINVAL;
  if (num_pages > 0 && (!k_cache || !v_cache)) return AK_EINVAL;
  if (!(sm_scale > 0.f) || sm_scale > 2e38f) return AK_EINVAL;  // (log2(e) times it is finite)
  for (int i = 0; i < 3; ++i)
    if (k_cache_strides[i] < 0 || v_cache_strides[i] < 0) return AK_EINVAL;
  const int64_t need = ak_paged_attn_workspace_bytes(dtype, T, B, Hq, Hkv, D, page_size, max_pages);
  if (need > 0 && (!host_aligned16(workspace) || !workspace || workspace_bytes < need)) return AK_EINVAL;
  PaArgs a{};
  a.q = q, a.kc = k_cache, a.vc = v_cache, a.o = o;
  a.qst = q_strides[0], a.qsh = q_strides[1], a.ost = o_strides[0], a.osh = o_strides[1];
  a.kcp = k_cache_strides[0], a.kch = k_cache_strides[1], a.kct = k_cache_strides[2];
  a.vcp = v_cache_strides[0], a.vch = v_cache_strides[1], a.vct = v_cache_strides[2];
  a.Hq = (int)Hq, a.Hk = (int)Hkv, a.G = (int)(Hq / Hkv), a.D = (int)D, a.Dp = (int)((D + 3) / 4 * 4);
  a.c_log2 = sm_scale * kFaLog2e;
  a.f_g = make_fastdiv((uint32_t)a.G);
  a.f_hk = make_fastdiv((uint32_t)a.Hk);
  a.s = make_paged(page_table, q_starts, kv_lens, T, B, num_pages, page_size, max_pages, table_stride);
  // K rows in 16-byte vectors
  const int vw = dtype == AK_F32 ? 4 : 8;
  a.vec = D % vw == 0 && host_aligned16(k_cache) && a.kcp % vw == 0 && a.kch % vw == 0 && a.kct % vw == 0;
  bool fast = a.vec && (D == 64 || D == 128) && host_aligned16(v_cache) && host_aligned16(q) && host_aligned16(o);
  for (const int64_t x : {a.vcp, a.vch, a.vct, a.qst, a.qsh, a.ost, a.osh})
    if (x % vw != 0) fast = false;
  // the fast kernels look a few steps past the last key with 32-bit positions; pa_tiles addresses inside a page
  // with 32 bits
  if (page_size * max_pages > INT_MAX - (1 << 16)) fast = false;
  for (const int64_t x : {a.kct, a.vct})
    if (x < D || x > (1 << 24) || x * page_size >= (int64_t)1 << 31) fast = false;
  for (const int64_t x : {a.kcp, a.vcp})
    if (x >= (int64_t)1 << 31) fast = false;
  const PaPlan p = pa_plan(dtype, T, B, Hq, Hkv, D, page_size, max_pages, fast);
  if (!pa_plan_fits(p)) return AK_EINVAL;
  AK_DISPATCH(dtype, T_, {
    return fast ? launch_fast<T_>(a, p, workspace, stream) : launch_general<T_>(a, p, workspace, stream);
  });
}
