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
#include "paged_common.h"

namespace ak {

constexpr int kPaWaves = 4;
constexpr int kPaThreads = kPaWaves * kWave;

struct PaArgs {
  const void *q, *kc, *vc;
  void* o;
  float *part, *stat;  // [items][tile rows][D], [items][tile rows][2] (exp2 base, sum)
  int64_t qst, qsh, ost, osh;            // row and head strides (elements)
  int64_t kcp, kch, kct, vcp, vch, vct;  // cache: page, head, slot strides
  int Hq, Hk, G, D, vec;
  float c_log2;
  float target;  // items aimed at; 0: keys are not sliced
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
__device__ __forceinline__ int64_t pa_seen(const PaItem& it, int r, int G) {
  return max((int64_t)0, min((int64_t)it.seq.len, (int64_t)it.seq.len - it.seq.n + r / G + 1));
}

// What a row's weighted values are multiplied with: 1 / sum, 0 for a row that sees no key.
__device__ __forceinline__ float pa_inv(const PaSeq& q, bool sees, float l) {
  return q.overlong ? __builtin_nanf("") : sees ? 1.0f / l : 0.f;
}

// Any type, head_dim and alignment: one wave per row, four rows per block.
constexpr int kPaRowTile = kPaWaves;
template <typename T>
__global__ __launch_bounds__(kPaThreads) void pa_general(const PaArgs a) {
  using S = typename T::S;
  PaItem it;
  if (!pa_find<kPaRowTile>(a, blockIdx.x, it)) return;
  const int lane = lane_id(), w = wave_id();
  const int r = it.tile * kPaRowTile + w;
  if (r >= it.seq.n * a.G) return;
  const int tok = it.seq.t0 + r / a.G, h = it.hk * a.G + r % a.G;
  const int64_t lo = it.nsplit == 1 ? 0 : (int64_t)it.split * it.chunk;
  const int64_t hi = min(pa_seen(it, r, a.G), it.nsplit == 1 ? (int64_t)INT_MAX : lo + it.chunk);
  float m, l, acc[4];
  pa_row<T>(a, it.b, it.hk, (const S*)a.q + tok * a.qst + h * a.qsh, lo, hi, m, l, acc);
  if (it.nsplit > 1) {
    float* p = a.part + ((int64_t)blockIdx.x * kPaRowTile + w) * a.D;
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (lane + 64 * x < a.D) p[lane + 64 * x] = acc[x];
    if (lane == 0) {
      float* st = a.stat + ((int64_t)blockIdx.x * kPaRowTile + w) * 2;
      st[0] = m;
      st[1] = l;
    }
    return;
  }
  S* o = (S*)a.o + tok * a.ost + h * a.osh;
  const float inv = pa_inv(it.seq, hi > lo, l);
#pragma unroll
  for (int x = 0; x < 4; ++x)
    if (lane + 64 * x < a.D) o[lane + 64 * x] = T::from_f(it.seq.overlong ? inv : acc[x] * inv);
}

// Sliced rows: one wave per (row, query head) adds its partials in slice order.
template <typename T, int BM>
__global__ __launch_bounds__(kPaThreads) void pa_merge(const PaArgs a) {
  using S = typename T::S;
  const int lane = lane_id();
  const int64_t row = (int64_t)blockIdx.x * kPaWaves + wave_id();
  const int64_t tok = row / a.Hq;
  const int h = (int)(row - tok * a.Hq);
  if (tok >= a.s.T) return;
  const int b = paged_seq_of(a.s, (int)tok);
  if (b >= a.s.B) return;
  const PaSeq q = pa_seq(a.s, b);
  if (tok < q.t0 || tok >= q.t0 + q.n) return;
  const int chunk = pa_chunk<BM>(a);
  const int nsplit = pa_splits(q.len, chunk);
  if (nsplit == 1) return;
  // items of the sequences before this one
  int first = 0;
  for (int i = lane; i < b; i += kWave) {
    const PaSeq x = pa_seq(a.s, i);
    first += (x.n * a.G + BM - 1) / BM * a.Hk * pa_splits(x.len, chunk);
  }
  first = __builtin_amdgcn_readlane(pa_wave_scan(first), kWave - 1);
  const int tiles = (q.n * a.G + BM - 1) / BM;
  const int hk = h / a.G, r = ((int)tok - q.t0) * a.G + h % a.G;
  const int tile = r / BM;
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int sp = 0; sp < nsplit; ++sp) {
    const uint32_t it = (uint32_t)first + ((uint32_t)sp * tiles + (tiles - 1 - tile)) * a.Hk + hk;
    if (it >= a.items) break;
    const int64_t slot = (int64_t)it * BM + r % BM;
    const float ms = a.stat[slot * 2], ls = a.stat[slot * 2 + 1];
    if (ms == -INFINITY && ls == 0.f) continue;  // a slice without a key that the row sees
    const float m_new = nan_max(m, ms);
    const float f0 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
    const float f1 = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - m_new);
    m = m_new;
    l = l * f0 + ls * f1;
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (lane + 64 * x < a.D) acc[x] = acc[x] * f0 + a.part[slot * a.D + lane + 64 * x] * f1;
  }
  const float inv = pa_inv(q, q.len - (q.t0 + q.n - tok) >= 0, l);  // its position
  S* o = (S*)a.o + tok * a.ost + h * a.osh;
#pragma unroll
  for (int x = 0; x < 4; ++x)
    if (lane + 64 * x < a.D) o[lane + 64 * x] = T::from_f(acc[x] * inv);
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
    p.ws_bytes = p.items * bm * (D + 2) * (int64_t)sizeof(float);
  }
  return p;
}

template <typename T>
static int launch_general(PaArgs a, const PaPlan& p, void* ws, hipStream_t st) {
  constexpr int BM = kPaRowTile;
  a.items = (uint32_t)p.items;
  a.target = p.target;
  a.part = (float*)ws;
  a.stat = a.part ? a.part + p.items * BM * a.D : nullptr;
  pa_general<T><<<dim3((unsigned)p.items), kPaThreads, 0, st>>>(a);
  if (a.target > 0.f)
    pa_merge<T, BM><<<dim3((unsigned)cdiv((int64_t)a.s.T * a.Hq, kPaWaves)), kPaThreads, 0, st>>>(a);
  return record_launch();
}

static bool pa_sizes_ok(int64_t T, int64_t B, int64_t Hq, int64_t Hk, int64_t D) {
  if (T < 0 || B < 0 || Hq < 0 || Hk <= 0 || D <= 0 || Hq % Hk != 0 || Hq > 65536) return false;
  return T <= INT_MAX && B < INT_MAX && T * Hq < (int64_t)1 << 31 && (std::min(B, T) + T * (Hq / Hk)) * Hk < (int64_t)1 << 24;
}
constexpr int64_t kPaTarget = 2048;

}  // namespace ak

using namespace ak;

extern "C" int64_t ak_paged_attn_workspace_bytes(int dtype, int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                                                 int64_t page_size, int64_t max_pages) {
  if (dtype != AK_F32 && dtype != AK_F16 && dtype != AK_BF16) return 0;
  if (!pa_sizes_ok(T, B, Hq, Hkv, D) || T == 0 || B == 0 || Hq == 0 || page_size <= 0 || max_pages < 0) return 0;
  if (page_size > INT_MAX || max_pages > INT_MAX) return 0;
  return pa_plan(T, B, Hq, Hkv, D, page_size * max_pages, kPaRowTile, kPaTarget).ws_bytes;
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
  const PaPlan p = pa_plan(T, B, Hq, Hkv, D, page_size * max_pages, kPaRowTile, kPaTarget);
  if (p.ws_bytes > 0 && (!host_aligned16(workspace) || !workspace || workspace_bytes < p.ws_bytes)) return AK_EINVAL;
  PaArgs a{};
  a.q = q, a.kc = k_cache, a.vc = v_cache, a.o = o;
  a.qst = q_strides[0], a.qsh = q_strides[1], a.ost = o_strides[0], a.osh = o_strides[1];
  a.kcp = k_cache_strides[0], a.kch = k_cache_strides[1], a.kct = k_cache_strides[2];
  a.vcp = v_cache_strides[0], a.vch = v_cache_strides[1], a.vct = v_cache_strides[2];
  a.Hq = (int)Hq, a.Hk = (int)Hkv, a.G = (int)(Hq / Hkv), a.D = (int)D;
  a.c_log2 = sm_scale * kFaLog2e;
  a.f_g = make_fastdiv((uint32_t)a.G);
  a.f_hk = make_fastdiv((uint32_t)a.Hk);
  a.s = make_paged(page_table, q_starts, kv_lens, T, B, num_pages, page_size, max_pages, table_stride);
  // K rows in 16-byte vectors
  const int vw = dtype == AK_F32 ? 4 : 8;
  a.vec = D % vw == 0 && host_aligned16(k_cache) && a.kcp % vw == 0 && a.kch % vw == 0 && a.kct % vw == 0;
  AK_DISPATCH(dtype, T_, return launch_general<T_>(a, p, workspace, stream));
}
