// sample.hip -- a token from each row of logits and one given random number: temperature, min-p, top-k, top-p.
//
// Of a row x with maximum M, temperature t and w_i = exp((x_i - M) / t), in falling order of x (ties: lowest
// index first):
//   min-p keeps w_i >= min_p, top-k the first k of these, top-p the shortest prefix of these whose mass
//   reaches top_p of theirs; the token is the first whose running mass passes u times the kept mass.
// Each step keeps a prefix of the falling order, so all of it is a search along one sequence of running sums,
// and the row is never sorted as a whole.
//
// The token is a whole number that a rounding error could change, so weights and sums are exact where it
// counts: w is computed in 64-bit floating point (2^x by a polynomial, error below 1e-12) and added as
// an integer multiple of 2^-42. Integer sums do not depend on their order, so LDS atomics add them and the
// token is the same on every run. A row of 2^20 weights stays below 2^62.
//
// One block of 16 waves per row:
//   1. maximum (as an order-preserving integer key, its lowest index, NaN check)
//   2. histogram of the row over kBins equal steps of log w, from the maximum down to 2^-44 (below, a weight
//      adds nothing): counts, and masses unless top-k makes them needless
//   3. the bins' running sums name the bin where a border lies. Where the bins down to it hold few enough
//      elements they are gathered as (key, index) pairs and sorted in LDS, and every border falls out of one
//      scan. Otherwise each border's own bin is gathered, cut into finer bins first while it holds too many.
#include <limits.h>

#include "ak_common.h"

namespace ak {

constexpr int kSmThreads = 1024;
constexpr int kSmWaves = kSmThreads / kWave;
constexpr int kBins = 4096, kBinsPer = kBins / kSmThreads;
constexpr int kList = 4096, kListPer = kList / kSmThreads;
constexpr float kSpan = 44.0f;                // octaves of weight that the bins cover
constexpr uint64_t kFixOne = 1ull << 42;      // weight 1

struct SampleArgs {
  const void* x;
  int64_t stride;
  const float* u;
  const float *tp, *pp, *mp;  // per-row settings, or null: the values below
  const int32_t* kp;
  float t, p, m;
  int k, V;
  int64_t* out;
};

struct SampleShared {
  uint64_t mass[kBins];
  uint32_t cnt[kBins];
  uint64_t list[kList];
  uint64_t red[kSmWaves];
  uint64_t red2[kSmWaves];
  uint64_t found[4];   // a border's element or bin, count and mass before it
  uint32_t n;
};

// Order-preserving key of a float (the two zeros are equal); larger key, larger value.
__device__ __forceinline__ uint32_t sm_key(float x) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  return b ^ ((int32_t)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float sm_val(uint32_t k) {
  return __uint_as_float(k ^ ((int32_t)k < 0 ? 0x80000000u : 0xffffffffu));
}
// (key, index) as one number whose falling order is the sorting order
__device__ __forceinline__ uint64_t sm_pair(uint32_t key, int i) { return (uint64_t)key << 32 | (uint32_t)~i; }

struct SampleRow {
  double top, c;   // maximum; log2(e) / t
  float topf, step;  // maximum; bins per unit of x
  uint32_t low;    // smallest key that min-p keeps
};

// 2^y for y <= 0: rounded to an integer n plus |f| <= 1/2, the Taylor polynomial of 2^f (its first term left
// out is below 2.3e-13) and a shift of the exponent.
__device__ __forceinline__ double sm_exp2(double y) {
  const double n = __builtin_rint(y), f = y - n;
  double r = 7.0549116208011232e-09;
  r = __builtin_fma(r, f, 1.0178086009239699e-07);
  r = __builtin_fma(r, f, 1.3215486790144309e-06);
  r = __builtin_fma(r, f, 1.5252733804059841e-05);
  r = __builtin_fma(r, f, 1.5403530393381608e-04);
  r = __builtin_fma(r, f, 1.3333558146428443e-03);
  r = __builtin_fma(r, f, 9.6181291076284772e-03);
  r = __builtin_fma(r, f, 5.5504108664821576e-02);
  r = __builtin_fma(r, f, 2.4022650695910069e-01);
  r = __builtin_fma(r, f, 6.9314718055994529e-01);
  r = __builtin_fma(r, f, 1.0);
  return __builtin_ldexp(r, (int)n);
}
__device__ __forceinline__ double sm_weight(const SampleRow& r, float x) {
  if (x == r.topf) return 1.0;
  const double y = ((double)x - r.top) * r.c;
  return y < -1000.0 ? 0.0 : sm_exp2(y);
}
// weight in units of 2^-42, rounded to nearest: 2^10 has this unit as its last place
__device__ __forceinline__ uint64_t sm_fixed(const SampleRow& r, float x) {
  return __builtin_bit_cast(uint64_t, sm_weight(r, x) + 1024.0) - 0x4090000000000000ull;
}
// Bin of x (falls with x), or -1: too light to count, or below min-p.
__device__ __forceinline__ int sm_bin(const SampleRow& r, float x) {
  if (x == r.topf) return 0;
  const float f = (r.topf - x) * r.step;
  return f < (float)kBins && sm_key(x) >= r.low ? (int)f : -1;
}

// f(value, index) for every element of the row, 16-byte vectors between an unaligned head and tail. HEAVY: a
// long f stands in the code once per 32-bit word of a vector, not once per element of it.
template <typename T, bool HEAVY, typename F>
__device__ __forceinline__ void sm_each(const typename T::S* x, int V, F f) {
  constexpr int W = T::kVec;
  const int head = min(V, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(typename T::S));
  const int nv = (V - head) / W, tail = head + nv * W;
  if ((int)threadIdx.x < head) f(T::to_f(x[threadIdx.x]), (int)threadIdx.x);
  if ((int)threadIdx.x < V - tail) f(T::to_f(x[tail + threadIdx.x]), tail + (int)threadIdx.x);
  // the next vector is in flight while one is worked on
  u32x4 next = (int)threadIdx.x < nv ? ld16(x + head + (int64_t)threadIdx.x * W) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll 1
  for (int i = threadIdx.x; i < nv; i += kSmThreads) {
    const u32x4 v = next;
    if (i + kSmThreads < nv) next = ld16(x + head + (int64_t)(i + kSmThreads) * W);
    if constexpr (HEAVY) {
      u32x4 w = v;
#pragma unroll 1
      for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int e = 0; e < W / 4; ++e) f(T::lane_elem(w, e), head + i * W + q * (W / 4) + e);
        w = u32x4{w[1], w[2], w[3], w[0]};
      }
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) f(T::lane_elem(v, e), head + i * W + e);
    }
  }
}

__device__ __forceinline__ uint64_t sm_wave_max(uint64_t v) {
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor((unsigned long long)v, o, kWave);
    v = w > v ? w : v;
  }
  return v;
}
// Sum over the lower threads of the block (exclusive); total gets everyone's.
__device__ __forceinline__ uint64_t sm_scan(uint64_t v, uint64_t* red, uint64_t& total) {
  uint64_t s = v;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint64_t w = __shfl_up((unsigned long long)s, o, kWave);
    if (lane_id() >= o) s += w;
  }
  __syncthreads();
  if (lane_id() == kWave - 1) red[wave_id()] = s;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kSmWaves; ++i) {
    if (i < wave_id()) before += red[i];
    total += red[i];
  }
  return before + s - v;
}

// Falling order of list[0 .. n), padded with zeros to a power of two.
__device__ __forceinline__ void sm_sort(SampleShared& sh, int n) {
  int n2 = 1;
  while (n2 < n) n2 <<= 1;
  for (int i = n + threadIdx.x; i < n2; i += kSmThreads) sh.list[i] = 0;
  for (int k = 2; k <= n2; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n2 / 2; i += kSmThreads) {
        const int a = 2 * i - (i & (j - 1)), b = a + j;
        const uint64_t p = sh.list[a], q = sh.list[b];
        if ((p < q) == ((a & k) == 0)) {
          sh.list[a] = q;
          sh.list[b] = p;
        }
      }
    }
  __syncthreads();
}

enum SampleRule { kByCount, kReaches, kPasses };
// Whether a running (count, mass) has arrived at the border.
__device__ __forceinline__ bool sm_there(SampleRule rule, double target, uint64_t cnt, uint64_t mass) {
  return rule == kByCount ? (double)cnt >= target : rule == kReaches ? (double)mass >= target : (double)mass > target;
}

// The bins' running sums, this thread's part: bins kBinsPer * tid ...
struct SampleBins {
  uint32_t cnt[kBinsPer + 1];
  uint64_t mass[kBinsPer + 1];
  uint64_t all_cnt, all_mass;
};
__device__ __forceinline__ void sm_sum_bins(SampleShared& sh, SampleBins& b) {
  uint64_t c = 0, m = 0;
#pragma unroll
  for (int i = 0; i < kBinsPer; ++i) {
    c += sh.cnt[threadIdx.x * kBinsPer + i];
    m += sh.mass[threadIdx.x * kBinsPer + i];
  }
  b.cnt[0] = (uint32_t)sm_scan(c, sh.red, b.all_cnt);
  b.mass[0] = sm_scan(m, sh.red2, b.all_mass);
#pragma unroll
  for (int i = 0; i < kBinsPer; ++i) {
    b.cnt[i + 1] = b.cnt[i] + sh.cnt[threadIdx.x * kBinsPer + i];
    b.mass[i + 1] = b.mass[i] + sh.mass[threadIdx.x * kBinsPer + i];
  }
}
// Bin of the border and the count and mass before it (the last bin if rounding puts the border past it).
struct SampleBin {
  int bin;
  uint32_t n;  // its elements
  uint64_t cnt, mass;
};
__device__ __forceinline__ SampleBin sm_find_bin(SampleShared& sh, const SampleBins& b, SampleRule rule, double target) {
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kBinsPer; ++i)
    if (!sm_there(rule, target, b.cnt[i], b.mass[i]) && sm_there(rule, target, b.cnt[i + 1], b.mass[i + 1])) {
      sh.found[0] = threadIdx.x * kBinsPer + i;
      sh.found[1] = b.cnt[i];
      sh.found[2] = b.mass[i];
      sh.found[3] = b.cnt[i + 1] - b.cnt[i];
    }
  __syncthreads();
  return SampleBin{(int)sh.found[0], (uint32_t)sh.found[3], sh.found[1], sh.found[2]};
}

__device__ __forceinline__ void sm_clear_bins(SampleShared& sh) {
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kSmThreads) {
    sh.cnt[i] = 0;
    sh.mass[i] = 0;
  }
  __syncthreads();
}

// Running sums over the sorted list (this thread's entries kListPer * tid ..), starting from (cnt, mass).
struct SampleList {
  uint64_t mass[kListPer + 1];
  uint32_t cnt0;
  int n;
};
__device__ __forceinline__ void sm_sum_list(SampleShared& sh, const SampleRow& r, int n, uint64_t cnt, uint64_t mass,
                                            SampleList& l) {
  uint64_t w[kListPer], s = 0, total;
#pragma unroll
  for (int i = 0; i < kListPer; ++i) {
    const int e = threadIdx.x * kListPer + i;
    w[i] = e < n ? sm_fixed(r, sm_val((uint32_t)(sh.list[e] >> 32))) : 0;
    s += w[i];
  }
  l.mass[0] = mass + sm_scan(s, sh.red, total);
#pragma unroll
  for (int i = 0; i < kListPer; ++i) l.mass[i + 1] = l.mass[i] + w[i];
  l.cnt0 = (uint32_t)cnt;
  l.n = n;
}
// The element at the border: index, and the mass up to and with it.
struct SampleHit {
  int index;
  uint64_t mass;
};
__device__ __forceinline__ SampleHit sm_find_list(SampleShared& sh, const SampleList& l, SampleRule rule, double target) {
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kListPer; ++i) {
    const int e = threadIdx.x * kListPer + i;
    if (e < l.n && !sm_there(rule, target, l.cnt0 + e, l.mass[i]) &&
        sm_there(rule, target, l.cnt0 + e + 1, l.mass[i + 1])) {
      sh.found[0] = (uint32_t)~(uint32_t)sh.list[e];
      sh.found[1] = l.mass[i + 1];
    }
  }
  __syncthreads();
  return SampleHit{(int)sh.found[0], sh.found[1]};
}

template <typename T>
__device__ __forceinline__ void sm_gather(SampleShared& sh, const SampleRow& r, const typename T::S* x, int V, int b0,
                                          int b1, uint64_t lo, uint64_t hi) {
  __syncthreads();
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  sm_each<T, true>(x, V, [&](float v, int i) {
    const int b = sm_bin(r, v);
    if (b < b0 || b > b1) return;
    const uint64_t e = sm_pair(sm_key(v), i);
    if (e < lo || e > hi) return;
    const uint32_t at = atomicAdd(&sh.n, 1u);
    if (at < kList) sh.list[at] = e;
  });
  __syncthreads();
}

// A bin of more than kList elements is cut into kBins equal ranges of (key, index) until the border's range
// [lo, hi] is small enough; `at` becomes that range.
template <typename T>
__device__ __forceinline__ void sm_narrow(SampleShared& sh, const SampleRow& r, const typename T::S* x, int V,
                                          SampleBin& at, SampleRule rule, double target, uint64_t& lo, uint64_t& hi) {
#pragma unroll 1
  while (at.n > kList) {
    // the range that the elements really take
    uint64_t a = 0, z = 0;  // largest, and largest complement
    sm_each<T, true>(x, V, [&](float v, int i) {
      if (sm_bin(r, v) != at.bin) return;
      const uint64_t e = sm_pair(sm_key(v), i);
      if (e < lo || e > hi) return;
      a = e > a ? e : a;
      z = ~e > z ? ~e : z;
    });
    a = sm_wave_max(a);
    z = sm_wave_max(z);
    __syncthreads();
    if (lane_id() == 0) {
      sh.red[wave_id()] = a;
      sh.red2[wave_id()] = z;
    }
    __syncthreads();
    for (int i = 0; i < kSmWaves; ++i) {
      a = sh.red[i] > a ? sh.red[i] : a;
      z = sh.red2[i] > z ? sh.red2[i] : z;
    }
    hi = a;
    lo = ~z;
    int shift = 0;
    while (((hi - lo) >> shift) >= kBins) ++shift;
    sm_clear_bins(sh);
    sm_each<T, true>(x, V, [&](float v, int i) {
      if (sm_bin(r, v) != at.bin) return;
      const uint64_t e = sm_pair(sm_key(v), i);
      if (e < lo || e > hi) return;
      const int q = (int)((hi - e) >> shift);
      atomicAdd(&sh.cnt[q], 1u);
      atomicAdd((unsigned long long*)&sh.mass[q], (unsigned long long)sm_fixed(r, v));
    });
    __syncthreads();
    SampleBins b;
    sm_sum_bins(sh, b);
    // the border counts from the row's start
#pragma unroll
    for (int i = 0; i <= kBinsPer; ++i) {
      b.cnt[i] += (uint32_t)at.cnt;
      b.mass[i] += at.mass;
    }
    const SampleBin in = sm_find_bin(sh, b, rule, target);
    const uint64_t width = (1ull << shift) - 1;
    hi -= (uint64_t)in.bin << shift;
    if (hi >= width && hi - width > lo) lo = hi - width;
    at.n = in.n;
    at.cnt = in.cnt;
    at.mass = in.mass;
  }
}

template <typename T>
__device__ __forceinline__ void sm_histogram(SampleShared& sh, const SampleRow& r, const typename T::S* x, int V,
                                             bool masses) {
  sm_clear_bins(sh);
  if (masses) {
    sm_each<T, true>(x, V, [&](float v, int) {
      const int b = sm_bin(r, v);
      if (b < 0) return;
      atomicAdd(&sh.cnt[b], 1u);
      atomicAdd((unsigned long long*)&sh.mass[b], (unsigned long long)sm_fixed(r, v));
    });
  } else {
    sm_each<T, false>(x, V, [&](float v, int) {
      const int b = sm_bin(r, v);
      if (b >= 0) atomicAdd(&sh.cnt[b], 1u);
    });
  }
  __syncthreads();
}

template <typename T>
__global__ __launch_bounds__(kSmThreads) void sample_rows(const SampleArgs a) {
  using S = typename T::S;
  __shared__ SampleShared sh;
  const int64_t row = blockIdx.x;
  const S* x = (const S*)a.x + row * a.stride;
  const int V = a.V;
  const float t = a.tp ? a.tp[row] : a.t, top_p = a.pp ? a.pp[row] : a.p;
  float min_p = a.mp ? a.mp[row] : a.m;
  const int top_k = a.kp ? a.kp[row] : a.k;
  float uf = a.u[row];
  uf = uf >= 0.f ? fminf(uf, 1.0f - 0x1p-24f) : 0.f;
  const double u = uf;

  // 1. maximum
  uint64_t best = 0;
  bool nan = false;
  sm_each<T, false>(x, V, [&](float v, int i) {
    nan |= v != v;
    const uint64_t e = sm_pair(sm_key(v), i);
    best = e > best ? e : best;
  });
  best = sm_wave_max(best);
  const bool wnan = __builtin_amdgcn_ballot_w64(nan) != 0;
  if (lane_id() == 0) {
    sh.red[wave_id()] = best;
    sh.red2[wave_id()] = wnan;
  }
  __syncthreads();
  for (int i = 0; i < kSmWaves; ++i) {
    best = sh.red[i] > best ? sh.red[i] : best;
    nan |= sh.red2[i] != 0;
  }
  __syncthreads();
  SampleRow r;
  r.topf = sm_val((uint32_t)(best >> 32));
  // a NaN, nothing to draw, or settings that are no numbers
  const bool none = nan || r.topf == -INFINITY || !(t >= 0.f && t < INFINITY) || top_p != top_p || min_p != min_p;
  if (none || t == 0.f) {
    if (threadIdx.x == 0) a.out[row] = none ? -1 : (int64_t)(uint32_t)~(uint32_t)best;
    return;
  }
  r.top = r.topf;
  r.c = 1.4426950408889634 / (double)t;
  r.step = (float)(r.c * (kBins / (double)kSpan));
  r.low = 0;
  if (min_p > 0.f) {
    // smallest key of weight >= min_p, 64 candidates a step (weights rise with the key)
    min_p = fminf(min_p, 1.0f);
    uint32_t lo = 0, hi = (uint32_t)(best >> 32);  // the border is in (lo, hi], hi is kept
    while (hi - lo > 1) {
      const uint32_t step = max(1u, (hi - lo) / kWave);
      const uint32_t at = lo + step * (lane_id() + 1);
      const bool in = step * (uint64_t)(lane_id() + 1) < hi - lo;
      const float v = sm_val(at);
      const bool keep = !in || (v == v && sm_weight(r, v) >= (double)min_p);
      const uint64_t m = __builtin_amdgcn_ballot_w64(keep);
      const int first = m ? __builtin_ctzll(m) : kWave;  // candidates rise: the first that is kept
      const uint32_t nlo = lo + step * first;
      if (first < kWave) hi = min(hi, lo + step * (first + 1));
      lo = nlo;
    }
    r.low = hi;
  }

  // 2. histogram: with top-k the counts alone, unless the first top_k elements are more than a list holds
  SampleBins b;
  const bool has_k = top_k > 0 && top_k < V, has_p = top_p < 1.0f;
  bool cuts = false;  // top-k cuts something off
#pragma unroll 1
  for (bool masses = !has_k;; masses = true) {
    sm_histogram<T>(sh, r, x, V, masses);
    sm_sum_bins(sh, b);
    cuts = has_k && (uint64_t)top_k < b.all_cnt;
    if (masses) break;
    uint64_t upto = b.all_cnt;
    if (cuts) {
      const SampleBin kb = sm_find_bin(sh, b, kByCount, top_k);
      upto = kb.cnt + kb.n;
    }
    if (upto <= kList) break;
  }

  // 3. the borders, one after another: top-k, top-p, the token. A list that starts at the row's maximum holds
  // the later borders too.
  double z = (double)b.all_mass;  // mass up to the last border
  bool listed = false;
  SampleList l;
  SampleHit hit;
#pragma unroll 1
  for (int step = 0; step < 3; ++step) {
    if (step == 0 ? !has_k : step == 1 ? !has_p : false) continue;
    const SampleRule rule = step == 0 ? kByCount : step == 1 ? kReaches : kPasses;
    // (a row with fewer elements than top_k ends at its last one)
    const double target = step == 0 ? fmin((double)top_k, (double)b.all_cnt)
                                    : step == 1 ? fmax((double)top_p * z, 1.0) : u * z;
    if (!listed) {
      SampleBin at = sm_find_bin(sh, b, rule, target);
      uint64_t lo = 0, hi = ~0ull;
      const int last = at.bin;
      listed = at.cnt + at.n <= kList;
      if (listed) at = SampleBin{0, (uint32_t)(at.cnt + at.n), 0, 0};
      else sm_narrow<T>(sh, r, x, V, at, rule, target, lo, hi);
      sm_gather<T>(sh, r, x, V, at.bin, last, lo, hi);
      const int n = min((int)sh.n, kList);
      sm_sort(sh, n);
      sm_sum_list(sh, r, n, at.cnt, at.mass, l);
    }
    hit = sm_find_list(sh, l, rule, target);
    z = (double)hit.mass;
  }
  if (threadIdx.x == 0) a.out[row] = hit.index;
}

}  // namespace ak

using namespace ak;

extern "C" int ak_sample(int dtype, const void* logits, const float* u, int64_t* tokens, int64_t rows, int64_t vocab,
                         int64_t row_stride, const float* temperature_rows, float temperature,
                         const int32_t* top_k_rows, int32_t top_k, const float* top_p_rows, float top_p,
                         const float* min_p_rows, float min_p, hipStream_t stream) {
  if (dtype != AK_F32 && dtype != AK_F16 && dtype != AK_BF16) return AK_EINVAL;
  if (rows < 0 || vocab <= 0 || row_stride < 0 || rows > INT_MAX || (rows > 1 && row_stride < vocab)) return AK_EINVAL;
  if (!temperature_rows && !(temperature >= 0.f && temperature < INFINITY)) return AK_EINVAL;
  if (!top_p_rows && top_p != top_p) return AK_EINVAL;
  if (!min_p_rows && min_p != min_p) return AK_EINVAL;
  if (vocab > (1 << 20)) return AK_EUNSUPPORTED;
  if (!grid_fits(rows, kSmThreads)) return AK_EINVAL;
  if (rows == 0) return AK_OK;
  if (!logits || !u || !tokens) return AK_EINVAL;
  const SampleArgs a{logits, row_stride, u, temperature_rows, top_p_rows, min_p_rows, top_k_rows,
                     temperature, top_p, min_p, top_k, (int)vocab, tokens};
  AK_DISPATCH(dtype, T, {
    sample_rows<T><<<dim3((unsigned)rows), kSmThreads, 0, stream>>>(a);
    return record_launch();
  });
}
