// paged_common.h -- what the paged-cache sources share: the batch of sequences of a call.
//
// A call's tokens are one row each, the sequences' new tokens one after another: sequence b has rows
// starts[b] .. starts[b + 1] - 1, and its cache holds lens[b] tokens, these new ones last. So the
// position of row t is lens[b] - (starts[b + 1] - t). Token p of sequence b lives in slot p % page_size
// of page table[b][p / page_size]. All of it is device data that the host never sees, so every index made
// from it is checked here before it becomes an address.
#pragma once
#include "ak_common.h"

namespace ak {

struct PagedSeqs {
  const int32_t* table;   // [B][width], rows table_stride elements apart
  const int32_t* starts;  // [B + 1]
  const int32_t* lens;    // [B]
  int64_t table_stride, num_pages;
  int B, T, width, page_size;
  FastDiv page_div;
};

// The sequence of row t: how many of starts[1 .. B] are at most t (B for a row behind the last
// sequence). One 64-wide load and ballot per 64 sequences instead of a search's chain of loads. t is
// wave-uniform; every lane gets the result.
__device__ __forceinline__ int paged_seq_of(const PagedSeqs& s, int t) {
  int b = 0;
  for (int i = 0; i < s.B; i += kWave) {
    const int j = i + lane_id();
    b += __builtin_popcountll(__builtin_amdgcn_ballot_w64(j < s.B && s.starts[min(j, s.B - 1) + 1] <= t));
  }
  return b;
}

// Page of position pos (>= 0) of sequence b, or -1 if the table has none inside the cache.
__host__ __device__ __forceinline__ int64_t paged_page_of(const PagedSeqs& s, int b, int64_t pos) {
  if (pos >= (int64_t)s.width * s.page_size) return -1;
  const int pg = s.table[b * s.table_stride + fdiv((uint32_t)pos, s.page_div)];
  return (uint32_t)pg < s.num_pages ? pg : -1;
}

// Host checks shared by the entry points. Positions stay below 2^31 (FastDiv).
inline bool paged_args_ok(const void* table, const void* starts, const void* lens, int64_t T, int64_t B,
                          int64_t num_pages, int64_t page_size, int64_t width, int64_t table_stride) {
  constexpr int64_t kMax = INT32_MAX;
  if (T < 0 || B < 0 || num_pages < 0 || page_size <= 0 || width < 0 || table_stride < 0) return false;
  if (T > kMax || B > kMax - 1 || num_pages > kMax || page_size > kMax || width > kMax || width * page_size > kMax)
    return false;
  if (B > 0 && (!starts || !lens || (width > 0 && !table))) return false;
  return B <= 1 || table_stride >= width;
}
inline PagedSeqs make_paged(const int32_t* table, const int32_t* starts, const int32_t* lens, int64_t T, int64_t B,
                            int64_t num_pages, int64_t page_size, int64_t width, int64_t table_stride) {
  return PagedSeqs{table,  starts,     lens,           table_stride, num_pages, (int)B, (int)T,
                   (int)width, (int)page_size, make_fastdiv((uint32_t)page_size)};
}

}  // namespace ak
