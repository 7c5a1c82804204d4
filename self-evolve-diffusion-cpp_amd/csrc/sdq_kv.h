// The paged cache's addressing on the device, shared by its kernels.
#pragma once

#include "sdq_internal.h"

namespace sdq {
namespace kv {

constexpr int kHd = 128;

// The cache and the batch as the kernels see them (include/sdq.h).
struct View {
  int8_t* k;
  float* ks;
  int8_t* v;
  float* vs;
  int64_t pages;
  int page_log2;
  int kv_heads;
  const int32_t* q_start;
  const int32_t* lens;
  const int32_t* table;
  int nseq;
  int64_t max_pages;
  int64_t T;
};

// Token runs that several sequences of a batch share (include/sdq.h): part g is the
// beginning of sequences s_start[g] .. s_start[g + 1] - 1.
struct Shared {
  const int32_t* s_start;
  const int32_t* lens;
  const int32_t* table;
  int n;
  int64_t max_pages;
  int nseq;  // of the batch
  __device__ __forceinline__ int seq_of(int g) const {
    const int s = s_start[g];
    return s < 0 ? 0 : s > nseq ? nseq : s;
  }
};

// Where an eviction's kept tokens go (include/sdq.h).
struct Kept {
  int64_t first, last, keep;
  const int32_t* table;
  int64_t max_pages;
  int32_t* lens;
  int32_t* kept;
};

// Row range of sequence s inside the call's T rows, and its length inside the
// table, whatever the arrays hold.
__device__ __forceinline__ int64_t row_of(const View& c, int s) {
  const int64_t r = c.q_start[s];
  return r < 0 ? 0 : r > c.T ? c.T : r;
}
__device__ __forceinline__ int64_t length_of(const View& c, int s) {
  const int64_t n = c.lens[s], most = c.max_pages << c.page_log2;
  return n < 0 ? 0 : n > most ? most : n;
}

// The sequence that row t belongs to (the last one that starts at or before
// it), or -1: rows before the first and behind the last sequence.
__device__ __forceinline__ int seq_of(const View& c, int64_t t) {
  if (t < row_of(c, 0) || t >= row_of(c, c.nseq)) return -1;
  int lo = 0, hi = c.nseq;  // row_of(lo) <= t < row_of(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (row_of(c, mid) <= t)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// The (page, head, row) index of position p of sequence s, or -1 where the
// table names no page of the pool.
__device__ __forceinline__ int64_t place_of(const View& c, int s, int64_t p, int head) {
  const int64_t page = c.table[s * c.max_pages + (p >> c.page_log2)];
  if (page < 0 || page >= c.pages) return -1;
  return ((page * c.kv_heads + head) << c.page_log2) + (p & ((1 << c.page_log2) - 1));
}

}  // namespace kv
}  // namespace sdq
