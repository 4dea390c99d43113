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
// counts: w is computed in 64-bit floating point (2^x by a polynomial, error below 1e-13) and added as
// an integer multiple of 2^-42. Integer sums do not depend on their order, so LDS atomics add them and the
// token is the same on every run. A row of 2^20 weights stays below 2^62.
//
// One block of 16 waves per row. Rows of 16-bit values are counted by value (sm_counted, below); the others, by sm_any:
//   1. the maximum
//      With top-k up to kQuickK, or min-p, a bound on what they keep usually leads straight to the list of 3.
//   2. a histogram of the row over kBins equal steps of log w, from the maximum down to 2^-44 (below, a weight
//      adds nothing): of masses, or of counts while top-k is to be found
//   3. the bins' running sums name the bin where a border lies. Where the bins down to it hold few enough
//      elements, these are gathered as (key, index) pairs and sorted in LDS, and the borders fall out of one
//      scan. Otherwise the border's own bin is gathered, cut into finer ranges first while it holds too many.
//      (A top-k border found that way becomes a bound on the row, and step 2 is done again with masses.)
// What bounds sm_any: the 64-bit weights of a whole row where no top-k spares them, about 25 instructions an
// element. So everything else an element meets is one or two comparisons: a bin, or min-p, is a range of
// floats, whose end is found once per row by trying 64 candidates at a time.
// 64 rows of 50257 fp32 with settings of all kinds: 33 to 42 us, of which 4 read the row; the slowest rows are those with
// top-p alone (28 us for 131072 weights, 16 with a constant in place of the weight, and 28 without the atomics).
#include <float.h>
#include <limits.h>

#include "ak_common.h"

namespace ak {

constexpr int kSmThreads = 1024;
constexpr int kSmWaves = kSmThreads / kWave;
constexpr int kBinsPer = 8, kListPer = 4;       // of a thread
constexpr int kBins = kBinsPer * kSmThreads, kList = kListPer * kSmThreads;
constexpr int kFine = kList;
constexpr int kRanked = 512;                    // lists up to this are ordered by counting, not by a sort network
constexpr int kQuickK = 512;                    // top-k up to this starts from the threads' maxima
constexpr float kMinTemperature = 1e-20f, kMaxTemperature = 1e30f;  // (bins per unit of x stay a float)
constexpr float kSpan = 44.0f;                  // octaves of weight that the bins cover

static_assert(2 * kRanked == kSmThreads, "two threads an entry");

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

struct SampleBins {
  uint64_t hist[kBins];
  alignas(16) uint64_t list[kList];
  uint64_t fine[kFine];  // finer bins, while a bin is cut up
};
constexpr int kGroups = 1024, kGroup = 64;        // of 16-bit values, in falling order
struct SamplePlace {
  uint32_t d, m, n;  // place among the values, number among its equals (from 1), how many these are
  uint64_t upto;     // the running mass up to it
};
struct SampleKeys {
  alignas(16) uint32_t count[1 << 15];            // two 16-bit counts a word; later a bit per element of the row
  uint64_t mass[kGroups];
  uint32_t size[kGroups], before[kGroups];        // elements of a group, and of those before it
  uint16_t list[kGroups];
  uint32_t times, nan, top;
  SamplePlace at[2];
};
struct SampleShared {
  union {
    SampleBins b;
    SampleKeys k;
  };
  uint64_t red[kSmWaves], red2[kSmWaves];
  uint64_t found[3];     // a border: its entry, the sum up to it, the sum before it
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
__device__ __forceinline__ uint64_t sm_pair(float x, int i) { return (uint64_t)sm_key(x) << 32 | (uint32_t)~i; }

struct SampleRow {
  double top, c;     // maximum; log2(e) / t
  float topf, step;  // maximum; bins per unit of x
  float low;         // smallest value that counts (min-p, the bins' span, top-k); of its equals those up to
  int low_last;      // index low_last
  float min_p;
};

// (2^f - 1) / f for |f| <= 1/2: interpolated at the nine Chebyshev nodes in long double. 1 + f q(f) is 2^f to
// 3.7e-14, and 1 at 0.
// (The instruction itself, its constant in scalar registers: the compiler takes the two-operand form and copies a
// constant into place before each of them.)
__device__ __forceinline__ double sm_fma(double a, double b, double c) {
  double d;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "s"(c));
  return d;
}
__device__ __forceinline__ double sm_q(double f) {
  double q = sm_fma(f, 1.0203121156603192e-07, 1.325522487537687e-06);
  q = sm_fma(q, f, 1.5252686845879443e-05);
  q = sm_fma(q, f, 0.0001540345585246757);
  q = sm_fma(q, f, 0.001333355817904356);
  q = sm_fma(q, f, 0.009618129159402543);
  q = sm_fma(q, f, 0.055504108664760424);
  q = sm_fma(q, f, 0.2402265069581299);
  return sm_fma(q, f, 0.6931471805599453);
}
// w of x <= topf
__device__ __forceinline__ double sm_weight(const SampleRow& r, float x) {
  const double y = fmax(((double)x - r.top) * r.c, -999.0), n = __builtin_rint(y), f = y - n;
  return __builtin_ldexp(__builtin_fma(sm_q(f), f, 1.0), (int)n);
}
// w in units of 2^-42, rounded to nearest, for x within the bins: log2 of it is between -2.1 and 42. Adding 1.5 2^52
// leaves the nearest integer in the low word (and, taken off again, as a double), adding 2^52 the rounded result
// in the mantissa.
__device__ __forceinline__ uint64_t sm_fixed(const SampleRow& r, float x) {
  const double y = __builtin_fma((double)x - r.top, r.c, 42.0), t = y + 6755399441055744.0;
  const double f = y - (t - 6755399441055744.0);
  uint64_t b = __builtin_bit_cast(uint64_t, __builtin_fma(sm_q(f), f, 1.0));
  b += (uint64_t)(uint32_t)__builtin_bit_cast(uint64_t, t) << 52;
  return __builtin_bit_cast(uint64_t, __builtin_bit_cast(double, b) + 4503599627370496.0) & 0xfffffffffffffull;
}
// Bin of x <= topf: rises as x falls (each operation rounds monotonically). kBins and more: too light.
__device__ __forceinline__ float sm_bin(const SampleRow& r, float x) { return (r.topf - x) * r.step; }

// Smallest float of bin `last` or an earlier one with w >= min_p, on every wave: 64 candidates a round, the first
// round next to where it should be. (topf is one.)
__device__ __forceinline__ float sm_first(const SampleRow& r, float last) {
  uint32_t lo = 0, hi = sm_key(r.topf);  // in (lo, hi]; hi is one
  const auto is = [&](uint32_t key) {
    const float v = sm_val(key);
    return sm_bin(r, v) < last + 1.0f && (r.min_p <= 0.f || sm_weight(r, v) >= (double)r.min_p);
  };
  float guess = r.topf - (last + 1.0f) / r.step;
  if (r.min_p > 0.f) guess = fmaxf(guess, r.topf + __builtin_amdgcn_logf(r.min_p) / (float)r.c);
  const uint32_t near = sm_key(guess);
  if (near > kWave && near + kWave < hi) {
    const uint64_t m = __builtin_amdgcn_ballot_w64(is(near - kWave / 2 + lane_id()));
    const int first = m ? __builtin_ctzll(m) : kWave;
    if (first > 0) lo = near - kWave / 2 + first - 1;
    if (first < kWave) hi = near - kWave / 2 + first;
  }
#pragma unroll 1
  while (hi - lo > 1) {
    const uint32_t step = max(1u, (hi - lo) / kWave);
    const bool past = step * (uint64_t)(lane_id() + 1) >= hi - lo;
    const uint64_t m = __builtin_amdgcn_ballot_w64(past || is(lo + step * (lane_id() + 1)));  // all after the first
    const int first = m ? __builtin_ctzll(m) : kWave;
    if (first < kWave) hi = min(hi, lo + step * (first + 1));
    lo += step * first;
  }
  return sm_val(hi);
}

// (v_minimum: fminf takes a second instruction for signalling NaNs)
__device__ __forceinline__ float sm_finite(float x) { return __builtin_elementwise_minimum(x, FLT_MAX); }

// f(value, index) for every element of the row, 16-byte vectors between an unaligned head and tail, the next two
// vectors in flight. +infinity counts as the largest finite float. HEAVY: a long f stands in the code once per
// 32-bit word of a vector, not once per element of it.
template <typename T, bool HEAVY, typename F>
__device__ __forceinline__ void sm_each(const typename T::S* x, int V, F f) {
  constexpr int W = T::kVec;
  const int tid = threadIdx.x;
  const int head = min(V, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(typename T::S));
  const int nv = (V - head) / W, tail = head + nv * W;
  const typename T::S* p = x + head;
  auto load = [&](int i) { return ld16(p + (int64_t)min(i, nv - 1) * W); };
  // head and tail: at most W - 1 elements each, on the first lanes of two waves
  const int edge = tid < kWave ? (tid < head ? tid : -1) : (tid - kWave < V - tail ? tail + tid - kWave : -1);
  if (tid < 2 * kWave && edge >= 0) f(sm_finite(T::to_f(x[edge])), edge);
  if (nv == 0) return;
  u32x4 next = load(tid), after = load(tid + kSmThreads);
#pragma unroll 1
  for (int i = tid; i < nv; i += kSmThreads) {
    const u32x4 v = next;
    next = after;
    after = load(i + 2 * kSmThreads);
    if constexpr (HEAVY) {
      u32x4 w = v;
#pragma unroll 1
      for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int e = 0; e < W / 4; ++e) f(sm_finite(T::lane_elem(w, e)), head + i * W + q * (W / 4) + e);
        w = u32x4{w[1], w[2], w[3], w[0]};
      }
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) f(sm_finite(T::lane_elem(v, e)), head + i * W + e);
    }
  }
}

__device__ __forceinline__ uint64_t sm_wave_max(uint64_t v) {
#pragma unroll 1
  for (int o = kWave / 2; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor((unsigned long long)v, o, kWave);
    v = w > v ? w : v;
  }
  return v;
}
__device__ __forceinline__ uint64_t sm_block_max(uint64_t v, uint64_t* red) {
  v = sm_wave_max(v);
  __syncthreads();
  if (lane_id() == 0) red[wave_id()] = v;
  __syncthreads();
  return sm_wave_max(red[lane_id() % kSmWaves]);
}

// v plus the lower lanes' values: within rows of 16 lanes by row_shr, then each row's last lane to the rows after
// it by row_bcast (a shuffle goes through LDS, twice for 64 bits).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t sm_scan_step(uint64_t v) {
  const int lo = __builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xf, false);
  return v + ((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
}
__device__ __forceinline__ uint64_t sm_wave_scan(uint64_t v) {
  v = sm_scan_step<0x111, 0xf>(v);
  v = sm_scan_step<0x112, 0xf>(v);
  v = sm_scan_step<0x114, 0xf>(v);
  v = sm_scan_step<0x118, 0xf>(v);
  v = sm_scan_step<0x142, 0xa>(v);
  return sm_scan_step<0x143, 0xc>(v);
}
__device__ __forceinline__ uint32_t sm_wave_scan(uint32_t v) {
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);
  return v + __builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
}
__device__ __forceinline__ uint32_t sm_lane(uint32_t v, int l) { return __builtin_amdgcn_readlane((int)v, l); }
__device__ __forceinline__ uint64_t sm_lane(uint64_t v, int l) {
  return (uint64_t)sm_lane((uint32_t)(v >> 32), l) << 32 | sm_lane((uint32_t)v, l);
}

// Running sums over the threads' values: of all of them, of those before this thread's, and up to each of its own.
template <int PER, typename N = uint64_t>
struct SampleSums {
  N total, before, upto[PER];
};
template <int PER, typename N>
__device__ __forceinline__ void sm_sums(SampleShared& sh, const N (&v)[PER], SampleSums<PER, N>& s) {
  N sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) s.upto[i] = sum += v[i];
  const N run = sm_wave_scan(sum);
  __syncthreads();
  if (lane_id() == kWave - 1) sh.red[wave_id()] = run;
  __syncthreads();
  // the waves' totals, one a lane
  const int wave = __builtin_amdgcn_readfirstlane(wave_id());
  const N waves = sm_wave_scan((N)sh.red[lane_id() % kSmWaves]);  // (of the first 16 lanes)
  s.total = sm_lane(waves, kSmWaves - 1);
  s.before = run - sum + (wave > 0 ? sm_lane(waves, wave - 1) : 0);
#pragma unroll
  for (int i = 0; i < PER; ++i) s.upto[i] += s.before;
}
template <int PER>
__device__ __forceinline__ void sm_sum_bins(SampleShared& sh, const uint64_t* bins, SampleSums<PER>& s) {
  uint64_t v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i] = bins[threadIdx.x * PER + i];
  sm_sums(sh, v, s);
}
template <int PER>
__device__ __forceinline__ void sm_clear(uint64_t* bins) {
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) bins[threadIdx.x + i * kSmThreads] = 0;
  __syncthreads();
}
// The first of the values whose running sum, with `base` before them all, reaches the target; at is -1 if none does.
struct SampleBorder {
  int at;
  uint64_t upto, before;
};
template <int PER>
__device__ __forceinline__ SampleBorder sm_find(SampleShared& sh, const SampleSums<PER>& s, uint64_t base,
                                                uint64_t target) {
  __syncthreads();
  if (base + s.before < target && base + s.upto[PER - 1] >= target) {
    int i = 0;
    uint64_t upto = s.upto[0], before = s.before;
#pragma unroll
    for (int j = 1; j < PER; ++j)
      if (base + upto < target) i = j, before = upto, upto = s.upto[j];
    sh.found[0] = threadIdx.x * PER + i;
    sh.found[1] = base + upto;
    sh.found[2] = base + before;
  } else if (threadIdx.x == kSmThreads - 1 && base + s.upto[PER - 1] < target) {
    sh.found[0] = ~0ull;
  }
  __syncthreads();
  return SampleBorder{(int)sh.found[0], sh.found[1], sh.found[2]};
}
// The running sum up to value `at`.
template <int PER>
__device__ __forceinline__ uint64_t sm_last(SampleShared& sh, const SampleSums<PER>& s, int at) {
  __syncthreads();
  if ((int)threadIdx.x == at / PER) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (at % PER == i) sh.found[1] = s.upto[i];
  }
  __syncthreads();
  return sh.found[1];
}
// About how many elements the bins up to `at` hold: their masses over the weight in a bin's middle.
__device__ __forceinline__ uint32_t sm_upto(SampleShared& sh, const SampleSums<kBinsPer>& s, int at) {
  __syncthreads();
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  float n = 0.f;
  uint64_t before = s.before;
#pragma unroll
  for (int i = 0; i < kBinsPer; ++i) {
    const int b = threadIdx.x * kBinsPer + i;
    const float in = (float)(s.upto[i] - before);
    if (b <= at) n += in * __builtin_amdgcn_exp2f(((float)b + 0.5f) * (kSpan / kBins) - 42.0f);
    before = s.upto[i];
  }
  n = wave_sum(n);
  if (lane_id() == 0 && n >= 0.5f) atomicAdd(&sh.n, (uint32_t)fminf(n + 0.5f, 1e8f));
  __syncthreads();
  return sh.n;
}

// What an element adds: 1, or its weight.
template <typename T>
__device__ __forceinline__ void sm_histogram(SampleShared& sh, const SampleRow& r, const typename T::S* x, int V,
                                             bool counts, SampleSums<kBinsPer>& s) {
  sm_clear<kBinsPer>(sh.b.hist);
  auto add = [&](float v, uint64_t w) {
    atomicAdd((unsigned long long*)&sh.b.hist[(int)sm_bin(r, v)], (unsigned long long)w);
  };
  if (counts) {
    sm_each<T, true>(x, V, [&](float v, int) {
      if (v >= r.low) add(v, 1);
    });
  } else if (r.low_last == INT_MAX) {
    sm_each<T, false>(x, V, [&](float v, int) {
      if (v >= r.low) add(v, sm_fixed(r, v));
    });
  } else {
    sm_each<T, true>(x, V, [&](float v, int i) {
      if (v > r.low || (v == r.low && i <= r.low_last)) add(v, sm_fixed(r, v));
    });
  }
  __syncthreads();
  sm_sum_bins(sh, sh.b.hist, s);
}

// Pairs in [lo, hi] of the row, into the list. sh.n: how many there are, which may be more than it holds.
template <typename T>
__device__ __forceinline__ void sm_gather(SampleShared& sh, const SampleRow& r, const typename T::S* x, int V, uint64_t lo,
                                          uint64_t hi) {
  __syncthreads();
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  const float vlo = sm_val((uint32_t)(lo >> 32)), vhi = sm_val((uint32_t)(hi >> 32));
  sm_each<T, false>(x, V, [&](float v, int i) {
    if (v >= vlo && v <= vhi) {
      const uint64_t e = sm_pair(v, i);
      if (e >= lo && e <= hi) {
        const uint32_t at = atomicAdd(&sh.n, 1u);
        if (at < kList) sh.b.list[at] = e;
      }
    }
  });
  __syncthreads();
}

// The list in falling order, and its running sums (of ones, or of weights).
__device__ __forceinline__ void sm_order(SampleShared& sh, const SampleRow& r, int n, bool counts,
                                         SampleSums<kListPer>& s) {
  if (n <= kRanked) {
    // an entry's place is the number of larger ones: two threads an entry, one half of the list each
    const int me_at = threadIdx.x % kRanked, part = threadIdx.x / kRanked;
    const uint64_t me = me_at < n ? sh.b.list[me_at] : 0;
    if (threadIdx.x < 4) sh.b.list[n + threadIdx.x] = 0;  // (kList is larger)
    __syncthreads();
    const int half = (n + 3) / 4 * 2;
    uint32_t place = 0;
    if (me_at < (n + kWave - 1) / kWave * kWave)
#pragma unroll 2
      for (int i = part * half; i < (part + 1) * half; i += 2) {
        const u32x4 p = ld16(&sh.b.list[i]);
        place += ((uint64_t)p[1] << 32 | p[0]) > me;
        place += ((uint64_t)p[3] << 32 | p[2]) > me;
      }
    if (part) sh.b.fine[me_at] = place;
    __syncthreads();
    if (!part && me_at < n) sh.b.list[place + (uint32_t)sh.b.fine[me_at]] = me;
  } else {
    int n2 = kRanked;
    while (n2 < n) n2 <<= 1;
    for (int i = n + threadIdx.x; i < n2; i += kSmThreads) sh.b.list[i] = 0;
#pragma unroll 1
    for (int k = 2; k <= n2; k <<= 1)
#pragma unroll 1
      for (int j = k >> 1; j > 0; j >>= 1) {
        __syncthreads();
#pragma unroll 1
        for (int i = threadIdx.x; i < n2 / 2; i += kSmThreads) {
          const int a = 2 * i - (i & (j - 1)), b = a + j;
          const uint64_t p = sh.b.list[a], q = sh.b.list[b];
          if ((p < q) == ((a & k) == 0)) {
            sh.b.list[a] = q;
            sh.b.list[b] = p;
          }
        }
      }
  }
  __syncthreads();
  uint64_t v[kListPer];
#pragma unroll 1
  for (int i = 0; i < kListPer; ++i) {
    const int e = threadIdx.x * kListPer + i;
    const uint64_t w = e >= n ? 0 : counts ? 1 : sm_fixed(r, sm_val((uint32_t)(sh.b.list[e] >> 32)));
    v[0] = i == 0 ? w : v[0], v[1] = i == 1 ? w : v[1], v[2] = i == 2 ? w : v[2], v[3] = i == 3 ? w : v[3];
  }
  sm_sums(sh, v, s);
}

// The finer bins of a border's surroundings: equal ranges of the pairs that its elements take. each(f) calls f on
// this thread's pairs; `before` is the sum of the pairs above them. lo, hi and before become the border's range.
template <typename E>
__device__ __forceinline__ void sm_cut(SampleShared& sh, const SampleRow& r, bool counts, uint64_t target, uint64_t& lo,
                                       uint64_t& hi, uint64_t& before, E each) {
  uint64_t a = 0, z = 0;  // largest, and largest complement
  each([&](uint64_t e) {
    a = e > a ? e : a;
    z = ~e > z ? ~e : z;
  });
  hi = sm_block_max(a, sh.red);
  lo = ~sm_block_max(z, sh.red2);
  int shift = 0;
  while (((hi - lo) >> shift) >= kFine) ++shift;
  sm_clear<kListPer>(sh.b.fine);
  const uint64_t top = hi;
  each([&](uint64_t e) {
    atomicAdd((unsigned long long*)&sh.b.fine[(top - e) >> shift],
              (unsigned long long)(counts ? 1 : sm_fixed(r, sm_val((uint32_t)(e >> 32)))));
  });
  __syncthreads();
  SampleSums<kListPer> s;
  sm_sum_bins(sh, sh.b.fine, s);
  const SampleBorder in = sm_find(sh, s, before, target);
  const uint64_t width = (1ull << shift) - 1;
  hi -= (uint64_t)in.at << shift;
  if (hi >= width && hi - width > lo) lo = hi - width;
  before = in.before;
}
// ... of the row's pairs in [lo, hi], too many for the list
template <typename T>
__device__ __forceinline__ void sm_narrow(SampleShared& sh, const SampleRow& r, const typename T::S* x, int V, bool counts,
                                          uint64_t target, uint64_t& lo, uint64_t& hi, uint64_t& before) {
  const uint64_t lo0 = lo, hi0 = hi;
  const float vlo = sm_val((uint32_t)(lo >> 32)), vhi = sm_val((uint32_t)(hi >> 32));
  sm_cut(sh, r, counts, target, lo, hi, before, [&](auto f) {
    sm_each<T, true>(x, V, [&](float v, int i) {
      if (!(v >= vlo && v <= vhi)) return;
      const uint64_t e = sm_pair(v, i);
      if (e >= lo0 && e <= hi0) f(e);
    });
  });
}
// ... of the list, too many to be ordered by counting: the pairs outside the border's range leave it
__device__ __forceinline__ void sm_thin(SampleShared& sh, const SampleRow& r, bool counts, uint64_t target,
                                        uint64_t& before) {
  uint64_t mine[kListPer], lo, hi;
  const int n = (int)sh.n;
#pragma unroll
  for (int i = 0; i < kListPer; ++i) {
    const int at = threadIdx.x + i * kSmThreads;
    mine[i] = at < n ? sh.b.list[at] : 0;  // (no pair is 0)
  }
  sm_cut(sh, r, counts, target, lo, hi, before, [&](auto f) {
#pragma unroll
    for (int i = 0; i < kListPer; ++i)
      if (mine[i]) f(mine[i]);
  });
  __syncthreads();
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kListPer; ++i)
    if (mine[i] >= lo && mine[i] <= hi && mine[i]) sh.b.list[atomicAdd(&sh.n, 1u)] = mine[i];
  __syncthreads();
}

// A row's settings.
struct SampleSet {
  float t, p, m, u;
  int k;
};
__device__ __forceinline__ SampleSet sm_settings(const SampleArgs& a, int64_t row) {
  const float u = a.u[row];
  return SampleSet{a.tp ? a.tp[row] : a.t, a.pp ? a.pp[row] : a.p, a.mp ? a.mp[row] : a.m,
                   u >= 0.f ? fminf(u, 1.0f - 0x1p-24f) : 0.f, a.kp ? a.kp[row] : a.k};
}
__device__ __forceinline__ bool sm_numbers(const SampleSet& g) {
  return g.t >= 0.f && g.t <= kMaxTemperature && g.p == g.p && g.m == g.m;
}
__device__ __forceinline__ void sm_row(SampleRow& r, const SampleSet& g) {
  r.top = r.topf;
  r.c = 1.4426950408889634 / (double)fmaxf(g.t, kMinTemperature);
  r.step = (float)(r.c * (kBins / (double)kSpan));
  r.min_p = fminf(g.m, 1.0f);
}
// The running masses that end what top-p keeps, of z, and that reach the token.
__device__ __forceinline__ uint64_t sm_target_p(float p, uint64_t z) {
  return max((uint64_t)__builtin_ceil((double)fmaxf(p, 0.f) * (double)z), (uint64_t)1);
}
__device__ __forceinline__ uint64_t sm_target_u(float u, uint64_t z) { return (uint64_t)((double)u * (double)z) + 1; }

// The token of a row of any type.
template <typename T>
__device__ void sm_any(SampleShared& sh, const SampleSet& g, const typename T::S* x, int V, int64_t* out) {
  using S = typename T::S;
  SampleRow r;
  // 1. maximum (v_maximum hands a NaN on, fminf above would lose it: the raw values)
  float top, mine = -INFINITY;  // of the row, of this thread's elements
  {
    const int head = min(V, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(S));
    const int nv = (V - head) / T::kVec, tail = head + nv * T::kVec;
    for (int i = threadIdx.x; i < head; i += kSmThreads) mine = __builtin_elementwise_maximum(mine, T::to_f(x[i]));
    for (int i = tail + threadIdx.x; i < V; i += kSmThreads) mine = __builtin_elementwise_maximum(mine, T::to_f(x[i]));
#pragma unroll 4
    for (int i = threadIdx.x; i < nv; i += kSmThreads) {
      const u32x4 v = ld16(x + head + (int64_t)i * T::kVec);
#pragma unroll
      for (int e = 0; e < T::kVec; ++e) mine = __builtin_elementwise_maximum(mine, T::lane_elem(v, e));
    }
    const uint64_t nan = __builtin_amdgcn_ballot_w64(mine != mine) ? 1 : 0;
    const uint64_t best = (uint64_t)sm_key(mine) << 1 | nan;
    const uint64_t all = sm_block_max((nan << 40) | best, sh.red);
    top = all >> 40 ? __builtin_nanf("") : sm_val((uint32_t)(all >> 1));
  }
  // a NaN, nothing to draw, or settings that are no numbers
  if (!(top > -INFINITY) || !sm_numbers(g)) {
    if (threadIdx.x == 0) *out = -1;
    return;
  }
  r.topf = fminf(top, FLT_MAX);
  if (g.t == 0.f) {  // the maximum's lowest index
    uint64_t first = 0;
    sm_each<T, true>(x, V, [&](float v, int i) {
      if (v == r.topf) first = (uint32_t)~i > first ? (uint32_t)~i : first;
    });
    first = sm_block_max(first, sh.red);
    if (threadIdx.x == 0) *out = (int64_t)(uint32_t)~(uint32_t)first;
    return;
  }
  sm_row(r, g);
  const int top_k = g.k;
  r.low = sm_first(r, kBins - 1);
  r.low_last = INT_MAX;

  // 2, 3. the borders, one after another: top-k (while it is looked for, elements count 1 each), top-p, the
  // token. A list that starts at the row's maximum holds the later borders too.
  bool counts = top_k > 0 && top_k < V, listed = false;
  SampleSums<kBinsPer> s;
  SampleSums<kListPer> l;
  uint64_t z = 0;
  int token = -1;
  const uint64_t least = sm_pair(r.low, r.low_last), most = sm_pair(r.topf, 0);
  // Short cuts to the list, without a histogram of the row: the top_k-th largest of the threads' maxima is a
  // bound that at least top_k elements pass, and few more; min-p mostly leaves few elements.
  const bool quick = counts && top_k <= kQuickK;
  if (quick || r.min_p > 0.f) {
    uint64_t lo = least;
    if (quick) {
      // coarse bins, one a thread: bin b is kBinsPer of the row's
      sh.b.hist[threadIdx.x] = 0;
      __syncthreads();
      mine = fminf(mine, FLT_MAX);
      if (mine >= r.low) atomicAdd((unsigned long long*)&sh.b.hist[(int)sm_bin(r, mine) / kBinsPer], 1ull);
      __syncthreads();
      const uint64_t v[1] = {sh.b.hist[threadIdx.x]};
      SampleSums<1> c;
      sm_sums(sh, v, c);
      const int bin = sm_find(sh, c, 0, top_k).at;
      if (bin >= 0) {
        const uint64_t bound = sm_pair(sm_first(r, (float)(bin * kBinsPer + kBinsPer - 1)), INT_MAX);
        if (bound > lo) lo = bound;
      }
    }
    sm_gather<T>(sh, r, x, V, lo, most);
    listed = sh.n <= (quick ? kList : kRanked);
    if (listed) {
      sm_order(sh, r, (int)sh.n, false, l);
      z = sm_last(sh, l, (counts ? min((uint32_t)top_k, sh.n) : sh.n) - 1);
      counts = false;
    }
  }
#pragma unroll 1
  for (int step = counts ? 0 : 1; step < 3; ++step) {
    if (!listed && step < 2) {
      sm_histogram<T>(sh, r, x, V, counts, s);
      z = s.total;  // everything that is left
    }
    if (step == 1 && !(g.p < 1.0f)) continue;
    const uint64_t target = step == 0   ? min((uint64_t)top_k, z)  // a row with fewer elements ends at its last one
                            : step == 1 ? sm_target_p(g.p, z)
                                        : sm_target_u(g.u, z);
    uint64_t before = 0;
    if (!listed) {
      const SampleBorder bin = sm_find(sh, s, 0, target);
      uint64_t lo = sm_pair(sm_first(r, (float)bin.at), INT_MAX), hi = most;
      const uint64_t end = sm_pair(r.low, r.low_last);
      if (lo < end) lo = end;
      if (step > 0 && sm_upto(sh, s, bin.at) <= kRanked) {
        sm_gather<T>(sh, r, x, V, lo, hi);
        listed = sh.n <= kList;
      }
      if (!listed) {
        if (bin.at > 0) hi = ((uint64_t)sm_key(sm_first(r, (float)(bin.at - 1))) << 32) - 1;
        before = bin.before;
#pragma unroll 1
        while (true) {
          sm_gather<T>(sh, r, x, V, lo, hi);
          if (sh.n <= kList) break;
          sm_narrow<T>(sh, r, x, V, counts, target, lo, hi, before);
        }
#pragma unroll 1
        while (sh.n > kRanked) sm_thin(sh, r, counts, target, before);
      }
      sm_order(sh, r, (int)sh.n, counts, l);
    }
    const SampleBorder at = sm_find(sh, l, before, target);
    const uint64_t e = sh.b.list[at.at];
    z = at.upto;
    if (step == 0) {  // the row ends there
      r.low = sm_val((uint32_t)(e >> 32));
      r.low_last = (int)~(uint32_t)e;
      counts = false;
    }
    token = (int)~(uint32_t)e;
  }
  if (threadIdx.x == 0) *out = token;
}

// Rows of 16-bit values: at most 65536 different ones, so a row is counted by value first, in one pass, and everything
// but the order of equal values follows from the counts. A weight is computed once for a value that occurs, not
// for each element, and nothing needs the maximum beforehand.
//   1. counts: 16 bits each, for all values (128 KB). 64 samples of the row tell whether one value fills much of it (a
//      mask, mostly); that one is counted in registers, as atomics of one address wait for each other. A count that
//      overflows leaves fewer counted than there are elements: such a row (another value more than 65535
//      times) is left to sm_any.
//   2. by groups of 64 values in falling order: the elements of each and before each, then the mass of each that
//      the cuts leave anything of
//   3. the border's group, in it the border's value, and how many of the equal elements are before the border
//   4. the token: the m-th element of its value, found in a bit map of the row's elements with that value
// What bounds it: reading the row, and one LDS atomic per element; for short rows the latency of the steps. The
// two ways on the same rows, sm_any after sm_counted, no cut / top-p 0.9 / top-k 50 (us):
//   bf16  1 x 1000: 9 10 8 / 12 16 11   64 x 32000: 13 14 11 / 29 36 14   256 x 131072: 27 28 24 / 66 79 29
//   f16   1 x 1000: 13 14 8 / 13 15 11  64 x 32000: 22 23 11 / 28 35 14   256 x 131072: 36 36 24 / 67 78 29
// (f16 has eight times as many values in a range, so eight times the weights.) 256 x 131072 bf16, top-p 0.95: 15 us
// for the counts (HBM's 67 MB take 13), 6 for the second look at the row, 8 for what is between.
template <typename T>
constexpr uint32_t kInfBits = T::kCode == AK_F16 ? 0x7c00 : 0x7f80;

// A value's place in falling order: x ^ 0x7fff without its sign bit, x with it. The zeros are 0x7fff and 0x8000.
__device__ __forceinline__ uint32_t sm_place(uint32_t x) { return x & 0x8000 ? x : x ^ 0x7fff; }
template <typename T>
__device__ __forceinline__ float sm_placed(uint32_t d) {  // (sm_place is its own inverse)
  return sm_finite(T::to_f(__builtin_bit_cast(typename T::S, (uint16_t)sm_place(d))));
}

// vec(16 bytes of the row, index of their first element) and one(bits, index) over the row, from its end if BACK.
template <bool BACK, typename S, typename FV, typename F1>
__device__ __forceinline__ void sm_each16(const S* x, int V, FV vec, F1 one) {
  const int tid = threadIdx.x;
  const int head = min(V, (int)((16 - ((uintptr_t)x & 15)) & 15) / 2);
  const int nv = (V - head) / 8, tail = head + nv * 8;
  const S* p = x + head;
  auto load = [&](int i) { return ld16(p + (int64_t)(BACK ? max(nv - 1 - i, 0) : min(i, nv - 1)) * 8); };
  const int edge = tid < kWave ? (tid < head ? tid : -1) : (tid - kWave < V - tail ? tail + tid - kWave : -1);
  if (tid < 2 * kWave && edge >= 0) one((uint32_t)__builtin_bit_cast(uint16_t, x[edge]), edge);
  if (nv == 0) return;
  u32x4 next = load(tid), after = load(tid + kSmThreads);
#pragma unroll 1
  for (int i = tid; i < nv; i += kSmThreads) {
    const u32x4 v = next;
    next = after;
    after = load(i + 2 * kSmThreads);
    vec(v, head + (BACK ? nv - 1 - i : i) * 8);
  }
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));

// The counts, and the value that is counted apart from them (negative zeros count as zeros).
struct SampleCounts {
  const SampleKeys& k;
  uint32_t common, times;  // its place (none: 0x8000, which no element has), how often it occurs
  __device__ __forceinline__ uint32_t operator[](uint32_t d) const {
    const uint32_t c = k.count[d & 0x7fff], n = d & 0x8000 ? c >> 16 : c & 0xffff;
    return d == 0x8000 ? 0 : n + (d == common ? times : 0) + (d == 0x7fff ? k.count[0] >> 16 : 0);
  }
};
template <typename T>
__device__ __forceinline__ uint64_t sm_place_weight(const SampleRow& r, uint32_t d) {
  const float v = sm_placed<T>(d);
  const bool counts = sm_bin(r, v) < (float)kBins && (r.min_p <= 0.f || sm_weight(r, v) >= (double)r.min_p);
  return counts ? sm_fixed(r, v) : 0;
}
// A lane's value of group g: its weight, how many elements have it, and how many of these top-k leaves.
struct SampleLane {
  uint64_t w;
  uint32_t all, n;
};
template <typename T>
__device__ __forceinline__ SampleLane sm_group_lane(const SampleCounts& c, const SampleRow& r, int g, uint32_t top_k) {
  const uint32_t d = g * kGroup + lane_id(), all = c[d], before = c.k.before[g];
  uint32_t n = all;
  if (before + c.k.size[g] > top_k) {
    const uint32_t upto = sm_wave_scan(n) + before;
    n = upto <= top_k ? n : upto - n < top_k ? n - (upto - top_k) : 0;
  }
  return SampleLane{n > 0 ? sm_place_weight<T>(r, d) : 0, all, n};
}
// The first element whose running mass reaches target, which is not above s.total: one wave has the border's group
// and finds the value.
template <typename T>
__device__ __forceinline__ void sm_find_value(const SampleCounts& c, const SampleRow& r, const SampleSums<1>& s,
                                              uint64_t target, uint32_t top_k, SamplePlace& at) {
  const uint64_t hit = __builtin_amdgcn_ballot_w64(s.before < target && s.upto[0] >= target);
  if (!hit) return;
  const int gl = __builtin_ctzll(hit), g = __builtin_amdgcn_readfirstlane(wave_id()) * kWave + gl;
  const SampleLane e = sm_group_lane<T>(c, r, g, top_k);
  const uint64_t mass = e.w * e.n, upto = sm_lane(s.before, gl) + sm_wave_scan(mass);
  if (upto < target || upto - mass >= target) return;
  // its number among its equals: the quotient is below 2^20, so in floats it is off by one at most
  const uint64_t need = target - (upto - mass) - 1;
  uint32_t m = (uint32_t)((float)need / (float)e.w);
  if (m * e.w > need) --m;
  else if ((m + 1) * e.w <= need) ++m;
  at = SamplePlace{g * kGroup + (uint32_t)lane_id(), m + 1, e.all, upto - mass + (m + 1) * e.w};
}

// The m-th element (from 1) of the value at place d, of which there are n.
template <typename S>
__device__ __forceinline__ void sm_nth(SampleShared& sh, const S* x, int V, uint32_t d, uint32_t m, uint32_t n,
                                       int64_t* out) {
  const uint32_t bits = sm_place(d), mask = bits == 0 ? 0x7fff : 0xffff;  // (either zero)
  const uint32_t words = (V + 31) / 32;
  __syncthreads();  // the counts have been read
  if (n > 1) {
    for (uint32_t i = threadIdx.x; i < words; i += kSmThreads) sh.k.count[i] = 0;
    __syncthreads();
  }
  auto one = [&](uint32_t b, int i) {
    if ((b & mask) != bits) return;
    if (n == 1) *out = i;
    else atomicOr(&sh.k.count[i >> 5], 1u << (i & 31));
  };
  const uint32_t mask2 = mask << 16 | mask, bits2 = bits << 16 | bits;
  sm_each16<true>(  // (what was read last is the nearest)
      x, V,
      [&](const u32x4& v, int i0) {
        u16x2 z[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) z[q] = __builtin_bit_cast(u16x2, (v[q] & mask2) ^ bits2);
        const u16x2 least = __builtin_elementwise_min(__builtin_elementwise_min(z[0], z[1]),
                                                      __builtin_elementwise_min(z[2], z[3]));
        if (least[0] != 0 && least[1] != 0) return;
        if (n == 1) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            one(v[q] & 0xffff, i0 + 2 * q);
            one(v[q] >> 16, i0 + 2 * q + 1);
          }
          return;
        }
        // eight bits, which the row's alignment may spread over two words
        uint32_t set = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) set |= (z[q][0] == 0) << 2 * q | (z[q][1] == 0) << (2 * q + 1);
        const int at = i0 & 31;
        atomicOr(&sh.k.count[i0 >> 5], set << at);
        if (at > 24 && set >> (32 - at)) atomicOr(&sh.k.count[(i0 >> 5) + 1], set >> (32 - at));
      },
      one);
  if (n == 1) return;
  __syncthreads();
  const uint32_t per = (words + kSmThreads - 1) / kSmThreads, w0 = threadIdx.x * per, w1 = min(w0 + per, words);
  uint32_t have = 0;
  for (uint32_t i = w0; i < w1; ++i) have += __builtin_popcount(sh.k.count[i]);
  const uint32_t v[1] = {have};
  SampleSums<1, uint32_t> s;
  sm_sums(sh, v, s);
  if (s.before >= m || s.upto[0] < m) return;
  uint32_t left = m - s.before, i = w0, word = sh.k.count[i];
  while (left > (uint32_t)__builtin_popcount(word)) {
    left -= __builtin_popcount(word);
    word = sh.k.count[++i];
  }
  for (; left > 1; --left) word &= word - 1;
  *out = (int64_t)i * 32 + __builtin_ctz(word);
}

// The row's counts and its common value.
template <typename T>
__device__ __forceinline__ SampleCounts sm_count(SampleShared& sh, const typename T::S* x, int V) {
  SampleKeys& k = sh.k;
  const uint32_t pick = __builtin_bit_cast(uint16_t, x[((int64_t)lane_id() * V) >> 6]);
  for (int i = threadIdx.x; i < (1 << 15) / 4; i += kSmThreads) st16(&k.count[4 * i], u32x4{0u, 0u, 0u, 0u});
  k.mass[threadIdx.x] = 0;
  if (threadIdx.x == 0) k.times = k.nan = 0;
  // the most frequent of three samples
  uint32_t common = 0, often = 0;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const uint32_t c = __builtin_amdgcn_readlane(pick, 21 * i);
    const uint32_t n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(pick == c));
    if (n > often) common = c, often = n;
  }
  const bool apart = often >= 4;  // four lanes of an atomic at one address take hardly longer than four addresses
  __syncthreads();
  uint32_t times = 0;
  auto one = [&](uint32_t b, int) {
    if (apart && b == common) ++times;
    else atomicAdd(&k.count[sm_place(b) & 0x7fff], b & 0x8000 ? 0x10000u : 1u);
  };
  sm_each16<false>(
      x, V,
      [&](const u32x4& v, int) {
        if (apart) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            one(v[q] & 0xffff, 0);
            one(v[q] >> 16, 0);
          }
          return;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t p = v[q];  // (a bit cast of v[q] itself takes element 0)
          const uint32_t neg = __builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2, p) >> 15);
          const uint32_t d = p ^ (~neg & 0x7fff7fffu);
          atomicAdd(&k.count[d & 0x7fff], (neg & 0xffff) + 1);
          atomicAdd(&k.count[d >> 16 & 0x7fff], (neg >> 16) + 1);
        }
      },
      one);
  if (apart && times) atomicAdd(&k.times, times);
  __syncthreads();
  const uint32_t d = sm_place(common);
  return SampleCounts{k, !apart ? 0x8000 : d == 0x8000 ? 0x7fff : d, k.times};
}

// The token of a row of 16-bit values; false if a count has overflowed.
template <typename T>
__device__ bool sm_counted(SampleShared& sh, const SampleSet& set, const typename T::S* x, int V, int64_t* out) {
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), tid = threadIdx.x;
  SampleKeys& k = sh.k;
  // 1. counts
  const SampleCounts c = sm_count<T>(sh, x, V);
  // 2. the groups' elements
  {
    // two threads to the words of a group and of the one in their upper halves; 16 lanes start at 16 different
    // vectors of them, which lie in different banks
    const int g = tid >> 1, w0 = g * kGroup + (tid & 1) * (kGroup / 2);
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int i = 0; i < kGroup / 2 / 4; ++i) {
      const u32x4 v = ld16(&k.count[w0 + 4 * ((i + g) % (kGroup / 2 / 4))]);
#pragma unroll
      for (int q = 0; q < 4; ++q) lo += v[q] & 0xffff, hi += v[q] >> 16;
    }
    lo += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)lo, 0xb1, 0xf, 0xf, false);  // its neighbour's
    hi += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)hi, 0xb1, 0xf, 0xf, false);
    const uint32_t zeros = k.count[0] >> 16;
    if (g == kGroups / 2 - 1) lo += zeros;
    if (g == 0) hi -= zeros;
    const int mine = g + (tid & 1) * (kGroups / 2);
    k.size[mine] = (tid & 1 ? hi : lo) + ((int)c.common / kGroup == mine ? c.times : 0);
  }
  __syncthreads();
  const uint32_t size[1] = {k.size[tid]};
  SampleSums<1, uint32_t> e;
  sm_sums(sh, size, e);
  k.before[tid] = e.before;
  if (e.before == 0 && size[0] > 0) k.top = tid;
  constexpr uint32_t kMinusInf = 0x8000 | kInfBits<T>;  // the last place but for NaN
  static_assert(kMinusInf % kGroup == 0, "first of its group");
  if (tid >= (int)(kMinusInf / kGroup) && size[0] != (tid == kMinusInf / kGroup ? c[kMinusInf] : 0)) k.nan = 1;
  __syncthreads();
  if (e.total != (uint32_t)V) return false;
  const int top_g = (int)k.top;
  const uint32_t top_n = c[top_g * kGroup + lane];
  const int top_l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(top_n != 0));
  const uint32_t top_d = top_g * kGroup + top_l;
  if (k.nan || top_d < (kInfBits<T> ^ 0x7fff) || top_d >= kMinusInf || !sm_numbers(set)) {
    if (tid == 0) *out = -1;
    return true;
  }
  SampleRow r;
  r.topf = sm_placed<T>(top_d);
  SamplePlace at{top_d, 1, (uint32_t)__builtin_amdgcn_readlane(top_n, top_l), 0};
  if (set.t > 0.f) {
    sm_row(r, set);
    const uint32_t top_k = set.k > 0 ? set.k : UINT_MAX;
    // The groups' masses. Those that count are listed, and as many threads share a group as there are for it. The
    // group in which top-k ends is one wave's.
    const auto counts = [&](float v) {  // the group's largest value
      return sm_bin(r, v) < (float)kBins && (r.min_p <= 0.f || sm_weight(r, v) >= (double)r.min_p);
    };
    const bool any = size[0] > 0 && e.before < top_k && (tid == top_g || counts(sm_placed<T>(tid * kGroup)));
    const bool cut = any && e.before + size[0] > top_k;
    const uint64_t cuts = __builtin_amdgcn_ballot_w64(cut), whole = __builtin_amdgcn_ballot_w64(any && !cut);
    if (lane == 0) sh.red[wave] = __builtin_popcountll(whole);
    __syncthreads();
    const uint32_t waves = sm_wave_scan((uint32_t)sh.red[lane % kSmWaves]);
    const uint32_t listed = sm_lane(waves, kSmWaves - 1);
    if (any && !cut)
      k.list[(wave > 0 ? sm_lane(waves, wave - 1) : 0) + __builtin_popcountll(whole & ((1ull << lane) - 1))] = (uint16_t)tid;
    if (cuts) {
      const int g = wave * kWave + __builtin_ctzll(cuts);
      const SampleLane b = sm_group_lane<T>(c, r, g, top_k);
      const uint64_t sum = sm_wave_scan(b.w * b.n);
      if (lane == kWave - 1) k.mass[g] = sum;
    }
    __syncthreads();
    int share = 6;  // log2 of a group's threads
    while (listed << share > kSmThreads) --share;
    const int slot = tid >> share, each = kGroup >> share;
    if (slot < (int)listed) {
      const int g = k.list[slot];
      uint64_t sum = 0;
#pragma unroll 1
      for (int i = 0; i < each; ++i) {  // (groups start at different values, which lie in different banks)
        const uint32_t d = g * kGroup + ((i + slot & each - 1) << share) + (tid & (1 << share) - 1), n = c[d];
        if (n) sum += sm_place_weight<T>(r, d) * n;
      }
      if (sum) atomicAdd((unsigned long long*)&k.mass[g], (unsigned long long)sum);
    }
    __syncthreads();
    // 3. the borders
    const uint64_t mass[1] = {k.mass[tid]};
    SampleSums<1> s;
    sm_sums(sh, mass, s);
    uint64_t z = s.total;
#pragma unroll 1
    for (int step = set.p < 1.0f ? 0 : 1; step < 2; ++step) {
      sm_find_value<T>(c, r, s, step == 0 ? sm_target_p(set.p, z) : sm_target_u(set.u, z), top_k, k.at[step]);
      __syncthreads();
      at = k.at[step];
      z = at.upto;
    }
  }
  // 4. the token
  sm_nth(sh, x, V, at.d, at.m, at.n, out);
  return true;
}

template <typename T>
__global__ __launch_bounds__(kSmThreads) void sample_rows(const SampleArgs a) {
  __shared__ SampleShared sh;
  const int64_t row = blockIdx.x;
  const typename T::S* x = (const typename T::S*)a.x + row * a.stride;
  const SampleSet g = sm_settings(a, row);
  if constexpr (T::kCode != AK_F32) {
    if (sm_counted<T>(sh, g, x, a.V, a.out + row)) return;
    __syncthreads();
  }
  sm_any<T>(sh, g, x, a.V, a.out + row);
}

}  // namespace ak

using namespace ak;

extern "C" int ak_sample(int dtype, const void* logits, const float* u, int64_t* tokens, int64_t rows, int64_t vocab,
                         int64_t row_stride, const float* temperature_rows, float temperature,
                         const int32_t* top_k_rows, int32_t top_k, const float* top_p_rows, float top_p,
                         const float* min_p_rows, float min_p, hipStream_t stream) {
  if (dtype != AK_F32 && dtype != AK_F16 && dtype != AK_BF16) return AK_EINVAL;
  if (rows < 0 || vocab <= 0 || row_stride < 0 || rows > INT_MAX || (rows > 1 && row_stride < vocab)) return AK_EINVAL;
  if (!temperature_rows && !(temperature >= 0.f && temperature <= kMaxTemperature)) return AK_EINVAL;
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
