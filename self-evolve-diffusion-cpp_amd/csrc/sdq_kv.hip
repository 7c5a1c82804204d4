// The paged int8 cache's writes and reads (gfx950).
//
// A row of 128 values of one token and head becomes 128 codes and one scale,
// as sdq_quant.hip's quantizer makes them (maximum / 127, products with the
// scale's reciprocal rounded to fp32, to the nearest even integer). 32 lanes
// hold a row, four values each, and the maximum is five lane exchanges.
//
// Bound by HBM: per row 512 bytes read and 132 written, the other way round for
// the reads. A workgroup takes 64 consecutive tokens of one head and tensor: their
// places are looked up once, a lane has up to eight rows in flight, and the
// scales of a page's rows, which lie side by side, are written together
// (a workgroup of eight heads of one token wrote them one by one: 27280 tokens x 24
// heads 369 us the write and 255 the read; now 207-222 and 134-139, 3.9 and 6.2 TB/s).
#include <algorithm>

#include "sdq_device.h"
#include "sdq_kv.h"

#pragma clang fp contract(off)

namespace sdq {
namespace {

using kv::kHd;
using kv::View;

constexpr int kTokens = 64;              // of a workgroup
constexpr int kRows = kTokens / 8;       // of a half-wave
constexpr int64_t kMaxBlocks = 1 << 22;  // a grid's threads are a 32-bit number

// Where token t of the call goes: the (page, row) index without the head, page
// * page_size + row; -1: nowhere, -2: the row is no sequence's.
__device__ __forceinline__ int64_t token_place(const View& c, int64_t t) {
  if (t >= c.T) return -2;
  const int s = kv::seq_of(c, t);
  if (s < 0) return -2;
  const int64_t p = kv::length_of(c, s) - kv::row_of(c, s + 1) + t;
  if (p < 0) return -1;
  const int64_t page = c.table[s * c.max_pages + (p >> c.page_log2)];
  if (page < 0 || page >= c.pages) return -1;
  return (page << c.page_log2) + (p & ((1 << c.page_log2) - 1));
}
// The same with the head: an index of rows.
__device__ __forceinline__ int64_t with_head(const View& c, int64_t place, int head) {
  const int64_t page = place >> c.page_log2;
  return ((page * c.kv_heads + head) << c.page_log2) + (place - (page << c.page_log2));
}

// Work item i: (64 tokens, tensor, head), the head fastest.
struct Item {
  int64_t t0;
  bool value;  // v, else k
  int head;
};
__device__ __forceinline__ Item item_at(const View& c, int64_t i) {
  const int64_t per = 2 * (int64_t)c.kv_heads;
  const int64_t b = i / per;
  const int r = (int)(i - b * per);
  return {b * kTokens, r >= c.kv_heads, r >= c.kv_heads ? r - c.kv_heads : r};
}

__global__ void __launch_bounds__(256)
kv_write_kernel(View c, const float* __restrict__ k, int64_t ldk, const float* __restrict__ v,
                int64_t ldv, int64_t items) {
  __shared__ int64_t places[kTokens];
  const int j = threadIdx.x & 31, hw = threadIdx.x >> 5;
  for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const Item it = item_at(c, i);
    const float* src = (it.value ? v : k) + (int64_t)it.head * kHd;
    const int64_t ld = it.value ? ldv : ldk;
    float4 f[kRows];
#pragma unroll
    for (int r = 0; r < kRows; r++) {
      const int64_t t = it.t0 + hw + 8 * r;
      f[r] = t < c.T ? reinterpret_cast<const float4*>(src + t * ld)[j]
                     : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncthreads();  // the last item's places are read
    if (threadIdx.x < kTokens) places[threadIdx.x] = token_place(c, it.t0 + threadIdx.x);
    __syncthreads();
    int8_t* codes = it.value ? c.v : c.k;
    float* scales = it.value ? c.vs : c.ks;
#pragma unroll
    for (int r = 0; r < kRows; r++) {
      const int64_t place = places[hw + 8 * r];
      if (place < 0) continue;
      float mx = 0.f;
      for (float a : {f[r].x, f[r].y, f[r].z, f[r].w}) mx = mx < fabsf(a) ? fabsf(a) : mx;
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        const float u = __shfl_xor(mx, o);
        mx = mx < u ? u : mx;
      }
      float sc = mx / 127.f;
      if (sc == 0.f) sc = 1.f;
      const int64_t at = with_head(c, place, it.head);
      reinterpret_cast<uint32_t*>(codes + at * kHd)[j] =
          dev::quant_pack4(f[r].x, f[r].y, f[r].z, f[r].w, 1.f / sc);
      if (j == 0) scales[at] = sc;
    }
  }
}

__global__ void __launch_bounds__(256)
kv_read_kernel(View c, float* __restrict__ k, int64_t ldk, float* __restrict__ v, int64_t ldv,
               int64_t items) {
  __shared__ int64_t places[kTokens];
  const int j = threadIdx.x & 31, hw = threadIdx.x >> 5;
  for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const Item it = item_at(c, i);
    __syncthreads();
    if (threadIdx.x < kTokens) places[threadIdx.x] = token_place(c, it.t0 + threadIdx.x);
    __syncthreads();
    const int8_t* codes = it.value ? c.v : c.k;
    const float* scales = it.value ? c.vs : c.ks;
    uint32_t q[kRows];
    float sc[kRows];
#pragma unroll
    for (int r = 0; r < kRows; r++) {
      const int64_t place = places[hw + 8 * r];
      q[r] = 0;
      sc[r] = 0.f;
      if (place >= 0) {
        const int64_t at = with_head(c, place, it.head);
        q[r] = reinterpret_cast<const uint32_t*>(codes + at * kHd)[j];
        sc[r] = scales[at];
      }
    }
    float* dst = (it.value ? v : k) + (int64_t)it.head * kHd;
    const int64_t ld = it.value ? ldv : ldk;
#pragma unroll
    for (int r = 0; r < kRows; r++)
      if (places[hw + 8 * r] != -2)
        reinterpret_cast<float4*>(dst + (it.t0 + hw + 8 * r) * ld)[j] =
            make_float4((float)(int8_t)q[r] * sc[r], (float)(int8_t)(q[r] >> 8) * sc[r],
                        (float)(int8_t)(q[r] >> 16) * sc[r], (float)(int8_t)(q[r] >> 24) * sc[r]);
  }
}

}  // namespace

hipError_t launch_kv_write(const View& c, const float* k, int64_t ldk, const float* v,
                           int64_t ldv, hipStream_t s) {
  const int64_t items = ceil_div(c.T, kTokens) * 2 * c.kv_heads;
  const int64_t blocks = std::min(items, kMaxBlocks);
  hipLaunchKernelGGL(kv_write_kernel, dim3((unsigned)blocks), dim3(256), 0, s, c, k, ldk, v, ldv,
                     items);
  return hipGetLastError();
}

hipError_t launch_kv_read(const View& c, float* k, int64_t ldk, float* v, int64_t ldv,
                          hipStream_t s) {
  const int64_t items = ceil_div(c.T, kTokens) * 2 * c.kv_heads;
  const int64_t blocks = std::min(items, kMaxBlocks);
  hipLaunchKernelGGL(kv_read_kernel, dim3((unsigned)blocks), dim3(256), 0, s, c, k, ldk, v, ldv,
                     items);
  return hipGetLastError();
}

}  // namespace sdq
