// attention_common.h -- what the attention sources share: softmax helpers, LDS DMA and transpose reads of the
// tiled kernels, and the few-row kernel's launcher (attention_rows.hip) for the dispatch in attention.hip.
#pragma once
#include "ak_common.h"

namespace ak {

constexpr float kFaLog2e = 1.4426950408889634f;

template <typename T>
__device__ __forceinline__ uint32_t fa2_pack(float a, float b);
template <>
__device__ __forceinline__ uint32_t fa2_pack<TF16>(float a, float b) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, f16x2));
}
template <>
__device__ __forceinline__ uint32_t fa2_pack<TBF16>(float a, float b) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, b2));
}
// acc + p.lo + p.hi (p: two packed values)
template <typename T>
__device__ __forceinline__ float fa2_sum2(uint32_t p, float acc);
template <>
__device__ __forceinline__ float fa2_sum2<TF16>(uint32_t p, float acc) {
  const f16x2 one = {(_Float16)1.0f, (_Float16)1.0f};
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, p), one, acc, false);
}
template <>
__device__ __forceinline__ float fa2_sum2<TBF16>(uint32_t p, float acc) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  const b2 one = {(__bf16)1.0f, (__bf16)1.0f};
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, p), one, acc, false);
}
// NaN-propagating max (v_maximum3_f32 / v_maximum_f32). fmaxf would ignore a NaN score, and on
// MFMA results the compiler then quiets each operand first (one v_max_f32 per operand: 11 more
// instructions per 64-key tile). A row whose scores hold a NaN comes out NaN either way: its true
// max fails the overflow test below.
__device__ __forceinline__ float fa2_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

constexpr int kFaBKV = 64;   // keys per tile
// fa_fwd2's lazy exp2 base: a row's base is raised only when a tile's max passes it by more than
// this (log2 units), so P <= 2^8 (exact range in f16 / bf16) and, after a row's first tile, the
// O rescale is almost never needed.
constexpr float kFa2Slack = 8.0f;

template <typename T>
__device__ __forceinline__ f32x16 mfma32x32x16(const u32x4& a, const u32x4& b, const f32x16& c);
template <>
__device__ __forceinline__ f32x16 mfma32x32x16<TF16>(const u32x4& a, const u32x4& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x16 mfma32x32x16<TBF16>(const u32x4& a, const u32x4& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// LDS swizzles of fa_fwd2's K and V tiles (attention.hip).
template <int D>
__device__ __forceinline__ int fa2_kswz(int r) {
  if constexpr (D == 128) return r & 15;
  else return (r >> 1) & 7;
}
template <int D>
__device__ __forceinline__ int fa2_vswz(int r) {
  if constexpr (D == 128) return 4 * (r & 3) + 2 * ((r >> 2) & 1);
  else return 4 * ((r >> 1) & 1) + 2 * ((r >> 2) & 1);
}

// Raw buffer resource: loads at byte offsets >= nbytes return zeros.
__device__ __forceinline__ u32x4 fa2_rsrc(const void* base, uint32_t nbytes) {
  const uint64_t a = (uint64_t)(uintptr_t)base;
  u32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((uint32_t)a);
  r[1] = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xffffu);  // stride 0
  r[2] = __builtin_amdgcn_readfirstlane(nbytes);
  r[3] = 0x00020000u;  // 32-bit data format, untyped access
  return r;
}

// One 1 KB LDS-DMA transfer: lane L's 16 bytes from rsrc + voff land at LDS byte lds + 16 L.
// Inline assembly, so the compiler inserts no waits for it: every wait is an explicit vmcnt. The
// LDS destination is an input operand bound to M0 ("{m0}"): the compiler writes M0 itself, so no
// register changes behind its back. One wait state separates the M0 write from the load.
__device__ __forceinline__ void fa2_dma16(const u32x4& rsrc, uint32_t voff, uint32_t lds) {
  asm volatile(
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %0, %1, 0 offen lds"
      :
      : "v"(voff), "s"(rsrc), "{m0}"(lds)
      : "memory");
}

typedef short fa2_s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x2 fa2_tr16(const uint16_t* p) {
  return __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) fa2_s16x4*)(p)));
}

// Keeps the computation of x ahead of this point (an empty use the compiler cannot move).
__device__ __forceinline__ void fa2_pin(const f32x16& x) { asm volatile("" ::"v"(x)); }
// max over the two 32-lane halves (every lane gets the same value, combined in the same order)
__device__ __forceinline__ float fa2_halves_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fa2_max(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float fa2_halves_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Few query rows per KV head (decode): see attention_rows.hip.
struct FaRowsPlan {
  bool ok;          // the kernel serves this shape
  int64_t splits;   // key slices; > 1 needs a workspace of ws_bytes
  int64_t ws_bytes;
};
FaRowsPlan fa_rows_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Sk, int64_t D, bool causal);
template <typename T>
int launch_fa_rows(const void* Q, const void* K, const void* V, void* O, int64_t B, int64_t Hq, int64_t Hkv,
                   int64_t Sq, int64_t Sk, int64_t D, const int64_t* qs, const int64_t* ks, const int64_t* vs,
                   const int64_t* os, float sm_scale, float* ws, int64_t ws_bytes, hipStream_t st);

}  // namespace ak
