// paged_attention.hip -- attention of new tokens over a paged cache.
//
//   o_i = softmax_j(q_i . K_j sm_scale) V_j over the cached keys j <= pos(i) of the token's sequence
// (paged_common.h: rows, positions, pages), grouped-query heads, one softmax pass with fp32 statistics.
// A row that sees no key (a position below zero) is zero; rows outside every sequence are not written; a
// row that sees a key in a page outside the cache is NaN, and so is every row of a sequence longer than
// its page table.
//
// Work split. The rows of a (sequence, KV head) are its group's query heads of each new token, token by
// token (row r: token r / group, head r % group), cut into tiles. A tile's keys are cut into slices of C
// keys, and a block takes one (tile, slice). The lengths are device data, so every block finds its item
// itself: it adds up the batch's work, derives C (about `target` items in all) and walks the sequences'
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

struct PaArgs {
  const void *q, *kc, *vc;
  void* o;
  float *part, *stat;  // [items][tile rows][Dp], [items][tile rows][2] (exp2 base, sum)
  int64_t qst, qsh, ost, osh;            // row and head strides (elements)
  int64_t kcp, kch, kct, vcp, vch, vct;  // cache: page, head, slot strides
  int Hq, Hk, G, D, Dp, vec;  // Dp: floats of a partial row, D rounded up to 4
  float c_log2;
  float target;    // items aimed at; 0: keys are not sliced
  uint32_t items;  // grid of the attention kernel: the most items there can be
  FastDiv f_g, f_hk;
  PagedSeqs s;
};

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
  int b, hk, tile, split, nsplit, chunk, tiles;
  uint32_t first;  // index of the sequence's first item
  PaSeq seq;
};

__device__ __forceinline__ int pa_wave_scan(int v) {  // inclusive
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int x = __shfl_up(v, o, kWave);
    if (lane_id() >= o) v += x;
  }
  return v;
}

// Keys per slice: all of them when the batch's work fills the chip without slicing, else the work over
// `target`, in multiples of kPaSlice.
constexpr int kPaSlice = 256;
template <int BM>
__device__ __forceinline__ int pa_chunk(const PaArgs& a) {
  if (a.target <= 0.f) return INT_MAX;
  float w = 0.f;
  for (int i = 0; i < a.s.B; i += kWave) {
    const int b = i + lane_id();
    if (b >= a.s.B) break;
    const PaSeq q = pa_seq(a.s, b);
    w += (float)((q.n * a.G + BM - 1) / BM) * (float)q.len;
  }
  w = wave_sum(w) * (float)a.Hk * 1.001f;
  const float c = ceilf(w / a.target / (float)kPaSlice) * (float)kPaSlice;
  return c >= 1e9f ? INT_MAX : max((int)c, kPaSlice);
}
__device__ __forceinline__ int pa_splits(int len, int chunk) {
  return chunk == INT_MAX ? 1 : max(1, (len + chunk - 1) / chunk);
}

// Item `it` of the batch; false when there are fewer. Within a sequence the KV heads run fastest (one
// per XCD, whose L2 then serves the tiles that share a head's keys), then tiles, last rows first (they see
// the most keys), then slices.
template <int BM>
__device__ __forceinline__ bool pa_find(const PaArgs& a, uint32_t it, PaItem& o) {
  o.chunk = pa_chunk<BM>(a);
  uint32_t base = 0;
  for (int i = 0; i < a.s.B; i += kWave) {
    const int b = i + lane_id();
    int cnt = 0, tiles = 0;
    if (b < a.s.B) {
      const PaSeq q = pa_seq(a.s, b);
      tiles = (q.n * a.G + BM - 1) / BM;
      cnt = tiles * a.Hk * pa_splits(q.len, o.chunk);
    }
    const int inc = pa_wave_scan(cnt);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(it - base < (uint32_t)inc && cnt > 0);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      o.b = i + l;
      o.tiles = __builtin_amdgcn_readlane(tiles, l);
      o.first = base + (uint32_t)__builtin_amdgcn_readlane(inc - cnt, l);
      o.seq = pa_seq(a.s, o.b);
      o.nsplit = pa_splits(o.seq.len, o.chunk);
      const uint32_t rel = it - o.first;
      const uint32_t x = fdiv(rel, a.f_hk);
      o.hk = (int)(rel - x * a.Hk);
      o.split = (int)(x / (uint32_t)o.tiles);
      o.tile = o.tiles - 1 - (int)(x - (uint32_t)o.split * o.tiles);
      return o.split < o.nsplit;
    }
    base += (uint32_t)__builtin_amdgcn_readlane(inc, kWave - 1);
  }
  return false;
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

// Row r of a tile: its output row, and the end of the keys that it sees in [.., hi).
__device__ __forceinline__ int pa_seen(const PaItem& it, int r, FastDiv f_g) {
  return max(0, it.seq.len - it.seq.n + (int)fdiv((uint32_t)r, f_g) + 1);
}

// What a row's weighted values are multiplied with: 1 / sum, 0 for a row that sees no key.
__device__ __forceinline__ float pa_inv(const PaSeq& q, bool sees, float l) {
  return q.overlong ? __builtin_nanf("") : sees ? 1.0f / l : 0.f;
}

// Rows r_begin .. r_end - 1 of an item's tile (of `bm` rows) over keys [lo, hi), one wave per row: results, or
// partials when the keys are sliced.
template <typename T>
__device__ void pa_rows_again(const PaArgs& a, const PaItem& it, int r_begin, int r_end, int lo, int hi, int bm) {
  using S = typename T::S;
  const int lane = lane_id();
  for (int r = r_begin + wave_id(); r < r_end; r += kPaWaves) {
    const int tk = (int)fdiv((uint32_t)r, a.f_g);
    const int tok = it.seq.t0 + tk, h = it.hk * a.G + r - tk * a.G;
    const int seen = pa_seen(it, r, a.f_g);
    float m, l, acc[4];
    pa_row<T>(a, it.b, it.hk, (const S*)a.q + tok * a.qst + h * a.qsh, lo, min(seen, hi), m, l, acc);
    if (it.nsplit > 1) {
      const int64_t slot = (int64_t)blockIdx.x * bm + (r - r_begin);
      float* p = a.part + slot * a.Dp;
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (lane + 64 * x < a.D) p[lane + 64 * x] = acc[x];
      if (lane == 0) {
        a.stat[slot * 2] = m;
        a.stat[slot * 2 + 1] = l;
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

// Any type, head_dim and alignment: one wave per row, four rows per block.
constexpr int kPaRowTile = kPaWaves;
template <typename T>
__global__ __launch_bounds__(kPaThreads) void pa_general(const PaArgs a) {
  PaItem it;
  if (!pa_find<kPaRowTile>(a, blockIdx.x, it)) return;
  const int r0 = it.tile * kPaRowTile, lo = it.nsplit == 1 ? 0 : it.split * it.chunk;
  pa_rows_again<T>(a, it, r0, min(it.seq.n * a.G, r0 + kPaRowTile), lo, it.nsplit == 1 ? INT_MAX : lo + it.chunk,
                   kPaRowTile);
}

// Sliced rows: W waves per (row, query head). A group of 16 lanes adds the partials of slices g, g + 4 W, ..
// (lane c: dims 4 c .. 4 c + 3 of each 64), then the groups' sums combine in group order. Four groups of one
// wave for many rows; with few rows sixteen, so that 64 slices' partials are in flight at once.
template <typename T, int BM, int W>
__global__ __launch_bounds__(kPaThreads) void pa_merge(const PaArgs a) {
  using S = typename T::S;
  constexpr int NG = 4 * W, NR = kPaWaves / W;  // groups of a row, rows of a block
  __shared__ float so[kPaWaves * 4][260], sm[kPaWaves * 4], sl[kPaWaves * 4];
  const int lane = lane_id(), c = lane & 15;
  const int slot_in = wave_id() / W, g = (wave_id() % W) * 4 + lane / 16;
  const int64_t row = (int64_t)blockIdx.x * NR + slot_in;
  const int64_t tok = row / a.Hq;
  const int h = (int)(row - tok * a.Hq);
  PaSeq q{0, 0, 0, false};
  int b = a.s.B, nsplit = 1, chunk = 0;
  if (tok < a.s.T) b = paged_seq_of(a.s, (int)tok);
  if (b < a.s.B) {
    q = pa_seq(a.s, b);
    if (tok >= q.t0 && tok < q.t0 + q.n) {
      chunk = pa_chunk<BM>(a);
      nsplit = pa_splits(q.len, chunk);
    }
  }
  float m = -INFINITY, l = 0.f, acc[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
  if (nsplit > 1) {
    // items of the sequences before this one
    int first = 0;
    for (int i = lane; i < b; i += kWave) {
      const PaSeq x = pa_seq(a.s, i);
      first += (x.n * a.G + BM - 1) / BM * a.Hk * pa_splits(x.len, chunk);
    }
    first = __builtin_amdgcn_readlane(pa_wave_scan(first), kWave - 1);
    const int tiles = (q.n * a.G + BM - 1) / BM;
    const int hk = h / a.G, r = ((int)tok - q.t0) * a.G + h % a.G;
    const uint32_t it0 = (uint32_t)first + (uint32_t)(tiles - 1 - r / BM) * a.Hk + hk;
    for (int sp = g; sp < nsplit; sp += 4 * NG) {
      float ms[4], ls[4];
      f32x4 v[4][4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t it = it0 + (uint32_t)(sp + u * NG) * tiles * a.Hk;
        ms[u] = -INFINITY;
        ls[u] = 0.f;
        if (sp + u * NG >= nsplit || it >= a.items) continue;
        const int64_t slot = (int64_t)it * BM + r % BM;
        ms[u] = a.stat[slot * 2];
        ls[u] = a.stat[slot * 2 + 1];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (64 * j + 4 * c < a.D) v[u][j] = *reinterpret_cast<const f32x4*>(a.part + slot * a.Dp + 64 * j + 4 * c);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (ms[u] == -INFINITY && ls[u] == 0.f) continue;  // a slice without a key that the row sees
        const float m_new = nan_max(m, ms[u]);
        const float f0 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
        const float f1 = ms[u] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms[u] - m_new);
        m = m_new;
        l = l * f0 + ls[u] * f1;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (64 * j + 4 * c < a.D)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][e] = acc[j][e] * f0 + v[u][j][e] * f1;
      }
    }
  }
  const int me = slot_in * NG + g;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (64 * j + 4 * c < a.D) *reinterpret_cast<f32x4*>(&so[me][64 * j + 4 * c]) = f32x4{acc[j][0], acc[j][1], acc[j][2], acc[j][3]};
  if (c == 0) {
    sm[me] = m;
    sl[me] = l;
  }
  __syncthreads();
  if (nsplit == 1) return;
  float mb = -INFINITY, lb = 0.f;
  for (int x = 0; x < NG; ++x) mb = nan_max(mb, sm[slot_in * NG + x]);
  float f[NG];
#pragma unroll
  for (int x = 0; x < NG; ++x) {
    const float mx = sm[slot_in * NG + x];
    f[x] = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - mb);
    lb += sl[slot_in * NG + x] * f[x];
  }
  const float inv = pa_inv(q, q.len - (q.t0 + q.n - (int)tok) >= 0, lb);  // its position
  S* o = (S*)a.o + tok * a.ost + h * a.osh;
  for (int d = (wave_id() % W) * kWave + lane; d < a.D; d += W * kWave) {
    float v = 0.f;
#pragma unroll
    for (int x = 0; x < NG; ++x) v += so[slot_in * NG + x][d] * f[x];
    o[d] = T::from_f(v * inv);
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

template <typename T, int D, int PG>
__global__ __launch_bounds__(kPaThreads, 2) void pa_rows(const PaArgs a) {
  constexpr int NS = D / 32, VW = D / 16;
  constexpr int NK = PG == 8 ? 1 : 2, NV = PG == 8 ? 1 : 8;  // page numbers of a lane and step
  using VV = typename PrVec<D>::type;
  __shared__ __attribute__((aligned(16))) float so[kPaWaves][kPrRows][D + 4];
  __shared__ float sst[kPaWaves][kPrRows][2];
  __shared__ int again;

  PaItem it;
  if (!pa_find<kPrRows>(a, blockIdx.x, it)) return;
  if (threadIdx.x == 0) again = 0;
  const int lane = lane_id(), w = wave_id();
  const int i16 = lane & 15, g = lane >> 4;
  const uint16_t* Kb = (const uint16_t*)a.kc + it.hk * a.kch + g * 8;
  const uint16_t* Vb = (const uint16_t*)a.vc + it.hk * a.vch + i16 * VW;
  const int rows = it.seq.n * a.G, r0 = it.tile * kPrRows, r = r0 + i16;
  const int lim = r < rows ? (int)pa_seen(it, r, a.f_g) : 0;  // keys that this lane's row sees
  u32x4 qf[NS];
  {
    const int tk = (int)fdiv((uint32_t)min(r, rows - 1), a.f_g);
    const uint16_t* q = (const uint16_t*)a.q + (int64_t)(it.seq.t0 + tk) * a.qst +
                        (int64_t)(it.hk * a.G + min(r, rows - 1) - tk * a.G) * a.qsh;
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] = r < rows ? ld16(q + s * 32 + g * 8) : u32x4{0u, 0u, 0u, 0u};
  }
  const int rl = min(rows, r0 + kPrRows) - 1;  // the tile's last row sees the most
  const int kbeg = it.nsplit == 1 ? 0 : it.split * it.chunk;
  const int kend = min((int)pa_seen(it, rl, a.f_g), it.nsplit == 1 ? INT_MAX : kbeg + it.chunk);
  const int full = (int)pa_seen(it, r0, a.f_g);  // every row sees the keys below

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
      for (int s = 0; s < NS; ++s) st.k[t][s] = in ? ld16(src + s * 32) : u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int key = k0 + 8 * g + e;
      const int pg = p.v[PG == 8 ? 0 : e];
      const bool in = (uint32_t)pg < a.s.num_pages && (!tail || key < kend);
      const uint32_t slot = (uint32_t)key - fdiv((uint32_t)key, a.s.page_div) * a.s.page_size;
      if (in) {
        st.v[e] = *reinterpret_cast<const VV*>(Vb + pg * a.vcp + slot * a.vct);
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

  constexpr int kStride = kPaWaves * kPrKeys;
  int k0 = kbeg + w * kPrKeys;
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
  l_run = pr_groups(l_run, OpAdd());
  bad |= l_run != l_run;
#pragma unroll
  for (int e = 0; e < VW; ++e)
#pragma unroll
    for (int v = 0; v < 4; ++v) bad |= o[e][v] != o[e][v];

  // Merge the waves: lane (i16, g) holds of row i16, in o[e][v], dim VW (4 g + v) + e.
#pragma unroll
  for (int v = 0; v < 4; ++v)
#pragma unroll
    for (int e = 0; e < VW; ++e) so[w][i16][VW * (4 * g + v) + e] = o[e][v];
  if (g == 0) {
    sst[w][i16][0] = m_run;
    sst[w][i16][1] = l_run;
  }
  __syncthreads();  // (the flag is cleared by now)
  if (__builtin_amdgcn_ballot_w64(bad) && lane == 0) atomicOr(&again, 1);
  __syncthreads();
  if (again) {
    pa_rows_again<T>(a, it, r0, min(rows, r0 + kPrRows), kbeg, kend, kPrRows);
    return;
  }
  const int q = threadIdx.x >> 4, c = threadIdx.x & 15;  // row of the tile, VW dims at c * VW
  if (r0 + q >= rows) return;
  float mb = -INFINITY, l = 0.f, acc[VW];
#pragma unroll
  for (int x = 0; x < kPaWaves; ++x) mb = fmaxf(mb, sst[x][q][0]);
#pragma unroll
  for (int e = 0; e < VW; ++e) acc[e] = 0.f;
#pragma unroll
  for (int x = 0; x < kPaWaves; ++x) {
    const float f = sst[x][q][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sst[x][q][0] - mb);
    l += sst[x][q][1] * f;
#pragma unroll
    for (int e = 0; e < VW; ++e) acc[e] += so[x][q][c * VW + e] * f;
  }
  if (it.nsplit > 1) {
    const int64_t slot = (int64_t)blockIdx.x * kPrRows + q;
    float* p = a.part + slot * a.Dp + c * VW;
#pragma unroll
    for (int e = 0; e < VW; e += 4) *reinterpret_cast<f32x4*>(p + e) = f32x4{acc[e], acc[e + 1], acc[e + 2], acc[e + 3]};
    if (c == 0) {
      a.stat[slot * 2] = mb;
      a.stat[slot * 2 + 1] = l;
    }
    return;
  }
  const float inv = pa_inv(it.seq, pa_seen(it, r0 + q, a.f_g) > 0, l);
  const int tk = (int)fdiv((uint32_t)(r0 + q), a.f_g);
  typename PrVec<D>::type pk;
#pragma unroll
  for (int e = 0; e < VW / 2; ++e) pk[e] = fa2_pack<T>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  *reinterpret_cast<VV*>((uint16_t*)a.o + (int64_t)(it.seq.t0 + tk) * a.ost +
                         (int64_t)(it.hk * a.G + r0 + q - tk * a.G) * a.osh + c * VW) = pk;
}

// Most items a call can have, and its workspace. Keys are sliced only where some sequence can be longer
// than one slice.
struct PaPlan {
  int64_t items, ws_bytes;
  float target;
};
static PaPlan pa_plan(int64_t T, int64_t B, int64_t Hq, int64_t Hk, int64_t D, int64_t keys, int bm, int64_t target) {
  PaPlan p;
  const int64_t tiles = (T * (Hq / Hk)) / bm + std::min(B, T);
  p.items = tiles * Hk;
  p.target = 0.f;
  p.ws_bytes = 0;
  if (keys > kPaSlice) {
    p.items += target;
    p.target = (float)target;
    p.ws_bytes = p.items * bm * ((D + 3) / 4 * 4 + 2) * (int64_t)sizeof(float);
  }
  return p;
}

template <typename T, int BM, typename K>
static int pa_launch(K kernel, PaArgs a, const PaPlan& p, void* ws, hipStream_t st) {
  a.items = (uint32_t)p.items;
  a.target = p.target;
  a.part = (float*)ws;
  a.stat = a.part ? a.part + p.items * BM * a.Dp : nullptr;
  kernel<<<dim3((unsigned)p.items), kPaThreads, 0, st>>>(a);
  if (a.target > 0.f) {
    const int64_t rows = (int64_t)a.s.T * a.Hq;
    if (rows <= 4096) pa_merge<T, BM, 4><<<dim3((unsigned)rows), kPaThreads, 0, st>>>(a);
    else pa_merge<T, BM, 1><<<dim3((unsigned)cdiv(rows, kPaWaves)), kPaThreads, 0, st>>>(a);
  }
  return record_launch();
}
template <typename T, int D>
static int launch_rows(const PaArgs& a, const PaPlan& p, void* ws, hipStream_t st) {
  return a.s.page_size % 8 == 0 ? pa_launch<T, kPrRows>(pa_rows<T, D, 8>, a, p, ws, st)
                                : pa_launch<T, kPrRows>(pa_rows<T, D, 1>, a, p, ws, st);
}

static bool pa_sizes_ok(int64_t T, int64_t B, int64_t Hq, int64_t Hk, int64_t D) {
  if (T < 0 || B < 0 || Hq < 0 || Hk <= 0 || D <= 0 || Hq % Hk != 0 || Hq > 65536) return false;
  return T <= INT_MAX && B < INT_MAX && T * Hq < (int64_t)1 << 31 && (std::min(B, T) + T * (Hq / Hk)) * Hk < (int64_t)1 << 24;
}
constexpr int64_t kPaTarget = 1024;
// Rows of a tile. The workspace is sized for the MFMA kernels' tiles wherever dtype and head_dim allow them; a
// call that turns out unaligned has smaller tiles.
static int pa_tile(int dtype, int64_t D) { return dtype != AK_F32 && (D == 64 || D == 128) ? kPrRows : kPaRowTile; }

}  // namespace ak

using namespace ak;

extern "C" int64_t ak_paged_attn_workspace_bytes(int dtype, int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                                                 int64_t page_size, int64_t max_pages) {
  if (dtype != AK_F32 && dtype != AK_F16 && dtype != AK_BF16) return 0;
  if (!pa_sizes_ok(T, B, Hq, Hkv, D) || T == 0 || B == 0 || Hq == 0 || page_size <= 0 || max_pages < 0) return 0;
  if (page_size > INT_MAX || max_pages > INT_MAX) return 0;
  return pa_plan(T, B, Hq, Hkv, D, page_size * max_pages, pa_tile(dtype, D), kPaTarget).ws_bytes;
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
  if (!(sm_scale > 0.f) || sm_scale > 3e38f) return AK_EINVAL;
  const int64_t keys = page_size * max_pages;
  const int64_t need = pa_plan(T, B, Hq, Hkv, D, keys, pa_tile(dtype, D), kPaTarget).ws_bytes;
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
  bool mfma = a.vec && dtype != AK_F32 && (D == 64 || D == 128) && host_aligned16(v_cache) && host_aligned16(q) &&
              host_aligned16(o);
  for (const int64_t x : {a.vcp, a.vch, a.vct, a.qst, a.qsh, a.ost, a.osh})
    if (x % 8 != 0) mfma = false;
  if (mfma) {
    const PaPlan p = pa_plan(T, B, Hq, Hkv, D, keys, kPrRows, kPaTarget);
    if (dtype == AK_F16)
      return D == 64 ? launch_rows<TF16, 64>(a, p, workspace, stream) : launch_rows<TF16, 128>(a, p, workspace, stream);
    return D == 64 ? launch_rows<TBF16, 64>(a, p, workspace, stream) : launch_rows<TBF16, 128>(a, p, workspace, stream);
  }
  const PaPlan p = pa_plan(T, B, Hq, Hkv, D, keys, kPaRowTile, kPaTarget);
  AK_DISPATCH(dtype, T_, return (pa_launch<T_, kPaRowTile>(pa_general<T_>, a, p, workspace, stream)));
}
