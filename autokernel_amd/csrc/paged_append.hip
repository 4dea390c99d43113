// paged_append.hip -- new tokens' keys and values written to a paged cache, q and k rotated on the way.
//
// Row t of sequence b has position pos (paged_common.h). Its q and k heads turn by the fp32 table rows
// cos[pos], sin[pos], in pairs (2i, 2i + 1) or (i, i + rot / 2):
//   y0 = x0 c - x1 s,  y1 = x0 s + x1 c    (products and sums rounded in fp32, one rounding to the type)
// and k, v go to slot pos % page_size of the position's page. Bound by HBM: q, k, v read once, written
// once; a decode step's few tokens by the launch. A wave takes 16-byte vectors of one token's heads (q,
// then k, then v). Its lanes keep one column each, so a lane reads its table entries once for all heads;
// the page comes from one table read per wave. Few tokens are spread over more waves per token.
// 8000 tokens of prompts (32 + 2 x 8 heads of 128, bf16): 196 MB in 35 us, 5.6 TB/s (a large copy 5.1); 48 tokens: 4 us,
// the launch and the chain of lengths, page number and row.
#include <limits.h>

#include <algorithm>

#include "paged_common.h"

namespace ak {

constexpr int kApWaves = 4;
constexpr int kApUnroll = 4;  // vectors a lane has in flight

struct AppendArgs {
  const void *q, *k, *v;
  void *qo, *kc, *vc;
  const float *ct, *st;  // [table_rows][rot / 2] or null
  int64_t qst, qsh, kst, ksh, vst, vsh, ost, osh;    // row and head strides (elements)
  int64_t kcp, kch, kct, vcp, vch, vct;              // cache: page, head, slot strides
  int64_t table_rows;
  int Hq, Hk, D, rot;
  int units, per_step, steps, wpt;  // lanes of a head, heads and steps of a wave, waves per token
  FastDiv f_wpt;
  PagedSeqs s;
};

#pragma clang fp contract(off)
template <typename T>
__device__ __forceinline__ void ap_turn(float& x0, float& x1, float c, float s) {
  const float y0 = x0 * c - x1 * s, y1 = x0 * s + x1 * c;
  x0 = y0;
  x1 = y1;
}

// What a wave knows of its token.
struct ApToken {
  int64_t pos, page;
  bool turn;  // its position has table rows (or no table is used)
};
__device__ __forceinline__ bool ap_token(const AppendArgs& a, int t, ApToken& k) {
  const int b = paged_seq_of(a.s, t);
  if (b >= a.s.B || t < a.s.starts[b]) return false;  // a row outside every sequence
  k.pos = (int64_t)a.s.lens[b] - ((int64_t)a.s.starts[b + 1] - t);
  k.turn = k.pos >= 0 && (!a.ct || k.pos < a.table_rows);
  k.page = k.turn ? paged_page_of(a.s, b, k.pos) : -1;
  return true;
}

// Source and destination of head slot h (q heads, k heads, v heads) of token t at column 0; dst is null
// when nothing is to be written.
template <typename S>
__device__ __forceinline__ void ap_head(const AppendArgs& a, const ApToken& k, int t, int slot, int h, const S*& src,
                                        S*& dst) {
  if (h < a.Hq) {
    src = (const S*)a.q + t * a.qst + h * a.qsh;
    dst = (S*)a.qo + t * a.ost + h * a.osh;
  } else if (h < a.Hq + a.Hk) {
    src = (const S*)a.k + t * a.kst + (h - a.Hq) * a.ksh;
    dst = k.page < 0 ? nullptr : (S*)a.kc + k.page * a.kcp + (h - a.Hq) * a.kch + slot * a.kct;
  } else {
    src = (const S*)a.v + t * a.vst + (h - a.Hq - a.Hk) * a.vsh;
    dst = k.page < 0 ? nullptr : (S*)a.vc + k.page * a.vcp + (h - a.Hq - a.Hk) * a.vch + slot * a.vct;
  }
}

// 16-byte vectors: head_dim, rot (rot / 2 for HALVES) and every stride multiples of the vector, bases aligned.
template <typename T, bool HALVES>
__global__ __launch_bounds__(kApWaves* kWave) void append_vec(const AppendArgs a) {
  using S = typename T::S;
  constexpr int V = T::kVec, NT = HALVES ? V : V / 2;  // table entries of a lane
  const uint32_t gw = blockIdx.x * kApWaves + wave_id();
  const int t = (int)fdiv(gw, a.f_wpt), part = (int)(gw - (uint32_t)t * a.wpt);
  if (t >= a.s.T) return;
  ApToken k;
  if (!ap_token(a, t, k)) return;
  const int lane = lane_id();
  const int sub = lane / a.units, c = lane - sub * a.units;
  if (sub >= a.per_step) return;
  const int slot = k.page < 0 ? 0 : (int)((uint32_t)k.pos - fdiv((uint32_t)k.pos, a.s.page_div) * a.s.page_size);
  const int half = a.rot / 2;
  // columns of this lane: e0 .. e0 + V - 1 and, when it turns halves, e0 + half ..
  const bool turns = HALVES ? c < half / V : c * V < a.rot;
  const int e0 = !HALVES || turns ? c * V : a.rot + (c - half / V) * V;
  float cs[NT], sn[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) cs[i] = sn[i] = 0.f;
  if (turns && a.ct) {
    const float* cp = a.ct + (k.turn ? k.pos : 0) * half + (HALVES ? e0 : e0 / 2);
    const float* sp = a.st + (k.turn ? k.pos : 0) * half + (HALVES ? e0 : e0 / 2);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      cs[i] = k.turn ? cp[i] : __builtin_nanf("");  // q of a token without a position: NaN
      sn[i] = k.turn ? sp[i] : __builtin_nanf("");
    }
  }
  const int heads = a.Hq + 2 * a.Hk;
  const int spw = (a.steps + a.wpt - 1) / a.wpt;  // steps of this wave
  const int s_end = min(a.steps, (part + 1) * spw);
  for (int s0 = part * spw; s0 < s_end; s0 += kApUnroll) {
    u32x4 x0[kApUnroll], x1[kApUnroll];
    S* dst[kApUnroll];
#pragma unroll
    for (int u = 0; u < kApUnroll; ++u) {
      const int h = (s0 + u) * a.per_step + sub;
      dst[u] = nullptr;
      if (s0 + u >= s_end || h >= heads) continue;
      const S* src;
      ap_head<S>(a, k, t, slot, h, src, dst[u]);
      x0[u] = ld16(src + e0);
      if (HALVES && turns) x1[u] = ld16(src + e0 + half);
    }
#pragma unroll
    for (int u = 0; u < kApUnroll; ++u) {
      if (!dst[u]) continue;
      const int h = (s0 + u) * a.per_step + sub;
      if (turns && a.ct && h < a.Hq + a.Hk) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          float y0, y1;
          if constexpr (HALVES) {
            y0 = T::lane_elem(x0[u], i), y1 = T::lane_elem(x1[u], i);
            ap_turn<T>(y0, y1, cs[i], sn[i]);
            T::set_elem(x0[u], i, y0);
            T::set_elem(x1[u], i, y1);
          } else {
            y0 = T::lane_elem(x0[u], 2 * i), y1 = T::lane_elem(x0[u], 2 * i + 1);
            ap_turn<T>(y0, y1, cs[i], sn[i]);
            T::set_elem(x0[u], 2 * i, y0);
            T::set_elem(x0[u], 2 * i + 1, y1);
          }
        }
      }
      st16(dst[u] + e0, x0[u]);
      if (HALVES && turns) st16(dst[u] + e0 + half, x1[u]);
    }
  }
}

// Any alignment, element by element: a wave walks its token's heads one pair or one unturned element per lane.
template <typename T, bool HALVES>
__global__ __launch_bounds__(kApWaves* kWave) void append_scalar(const AppendArgs a) {
  using S = typename T::S;
  const uint32_t gw = blockIdx.x * kApWaves + wave_id();
  const int t = (int)fdiv(gw, a.f_wpt), part = (int)(gw - (uint32_t)t * a.wpt);
  if (t >= a.s.T) return;
  ApToken k;
  if (!ap_token(a, t, k)) return;
  const int slot = k.page < 0 ? 0 : (int)((uint32_t)k.pos - fdiv((uint32_t)k.pos, a.s.page_div) * a.s.page_size);
  const int half = a.rot / 2;
  const int total = (a.Hq + 2 * a.Hk) * a.units;
  for (int i = part * kWave + lane_id(); i < total; i += a.wpt * kWave) {
    const int h = i / a.units, c = i - h * a.units;
    const S* src;
    S* dst;
    ap_head<S>(a, k, t, slot, h, src, dst);
    if (!dst) continue;
    if (c >= half) {
      dst[half + c] = src[half + c];
      continue;
    }
    const int e0 = HALVES ? c : 2 * c, e1 = HALVES ? c + half : 2 * c + 1;
    if (a.ct && h < a.Hq + a.Hk) {
      float y0 = T::to_f(src[e0]), y1 = T::to_f(src[e1]);
      ap_turn<T>(y0, y1, k.turn ? a.ct[k.pos * half + c] : __builtin_nanf(""),
                 k.turn ? a.st[k.pos * half + c] : __builtin_nanf(""));
      dst[e0] = T::from_f(y0);
      dst[e1] = T::from_f(y1);
    } else {
      const S y0 = src[e0], y1 = src[e1];
      dst[e0] = y0;
      dst[e1] = y1;
    }
  }
}

template <typename T>
static int launch_append(AppendArgs a, bool vec, bool halves, hipStream_t st) {
  const int heads = a.Hq + 2 * a.Hk;
  if (vec) {
    a.units = halves ? (a.D - a.rot / 2) / T::kVec : a.D / T::kVec;
    a.per_step = kWave / a.units;
    a.steps = (int)cdiv(heads, a.per_step);
  } else {
    a.units = a.D - a.rot / 2;
    a.per_step = 0;
    a.steps = (int)cdiv((int64_t)heads * a.units, kWave);
  }
  // Enough waves to fill the chip from few tokens, one per token from 4096 tokens on.
  a.wpt = (int)std::min<int64_t>(a.steps, std::max<int64_t>(1, cdiv(4096, a.s.T)));
  const int64_t waves = (int64_t)a.s.T * a.wpt, blocks = cdiv(waves, kApWaves);
  if (waves > INT_MAX || !grid_fits(blocks, kApWaves * kWave)) return AK_EINVAL;
  a.f_wpt = make_fastdiv((uint32_t)a.wpt);
  const dim3 grid((unsigned)blocks), block(kApWaves * kWave);
  if (vec && halves) append_vec<T, true><<<grid, block, 0, st>>>(a);
  else if (vec) append_vec<T, false><<<grid, block, 0, st>>>(a);
  else if (halves) append_scalar<T, true><<<grid, block, 0, st>>>(a);
  else append_scalar<T, false><<<grid, block, 0, st>>>(a);
  return record_launch();
}

}  // namespace ak

using namespace ak;

extern "C" int ak_kv_append(int dtype, const void* q, const void* k, const void* v, void* q_out, void* k_cache,
                            void* v_cache, const float* cos_t, const float* sin_t, const int32_t* page_table,
                            const int32_t* q_starts, const int32_t* kv_lens, int64_t T, int64_t B, int64_t Hq,
                            int64_t Hkv, int64_t D, int64_t rot_dim, int64_t table_rows, int64_t num_pages,
                            int64_t page_size, int64_t max_pages, int64_t table_stride, const int64_t* q_strides,
                            const int64_t* k_strides, const int64_t* v_strides, const int64_t* q_out_strides,
                            const int64_t* k_cache_strides, const int64_t* v_cache_strides, int interleaved,
                            hipStream_t stream) {
  if (dtype != AK_F32 && dtype != AK_F16 && dtype != AK_BF16) return AK_EINVAL;
  if (Hq < 0 || Hkv < 0 || D <= 0 || Hq > 65536 || Hkv > 65536) return AK_EINVAL;
  if (D > 256) return AK_EUNSUPPORTED;
  if (!paged_args_ok(page_table, q_starts, kv_lens, T, B, num_pages, page_size, max_pages, table_stride))
    return AK_EINVAL;
  if (rot_dim < 0 || rot_dim > D || rot_dim % 2 != 0 || table_rows < 0) return AK_EINVAL;
  const bool turn = rot_dim > 0;
  if (turn && (!cos_t || !sin_t)) return AK_EINVAL;
  if (Hq > 0 && !turn) return AK_EINVAL;  // q is here to be rotated
  if (T == 0 || B == 0 || Hq + Hkv == 0) return AK_OK;
  if ((Hq > 0 && (!q || !q_out || !q_strides || !q_out_strides)) ||
      (Hkv > 0 && (!k || !v || !k_strides || !v_strides || !k_cache_strides || !v_cache_strides)) ||
      (Hkv > 0 && num_pages > 0 && (!k_cache || !v_cache)))
    return AK_EINVAL;
  for (int i = 0; i < 3; ++i)
    if (Hkv > 0 && (k_cache_strides[i] < 0 || v_cache_strides[i] < 0)) return AK_EINVAL;
  AppendArgs a{};
  a.q = q, a.k = k, a.v = v, a.qo = q_out, a.kc = k_cache, a.vc = v_cache;
  a.ct = turn ? cos_t : nullptr, a.st = turn ? sin_t : nullptr;
  a.table_rows = table_rows;
  a.Hq = (int)Hq, a.Hk = (int)Hkv, a.D = (int)D, a.rot = (int)rot_dim;
  a.s = make_paged(page_table, q_starts, kv_lens, T, B, num_pages, page_size, max_pages, table_stride);
  const int vw = dtype == AK_F32 ? 4 : 8;
  const bool halves = turn && !interleaved;
  bool vec = D % vw == 0 && (halves ? rot_dim / 2 : rot_dim) % vw == 0;
  auto take = [&](const void* p, const int64_t* s, int n, int64_t* o0, int64_t* o1, int64_t* o2) {
    if (!host_aligned16(p)) vec = false;
    for (int i = 0; i < n; ++i)
      if (s[i] % vw != 0) vec = false;
    *o0 = s[0], *o1 = s[1];
    if (o2) *o2 = s[2];
  };
  if (Hq > 0) {
    take(q, q_strides, 2, &a.qst, &a.qsh, nullptr);
    take(q_out, q_out_strides, 2, &a.ost, &a.osh, nullptr);
  }
  if (Hkv > 0) {
    take(k, k_strides, 2, &a.kst, &a.ksh, nullptr);
    take(v, v_strides, 2, &a.vst, &a.vsh, nullptr);
    take(k_cache, k_cache_strides, 3, &a.kcp, &a.kch, &a.kct);
    take(v_cache, v_cache_strides, 3, &a.vcp, &a.vch, &a.vct);
  }
  AK_DISPATCH(dtype, T_, return launch_append<T_>(a, vec, halves, stream));
}
