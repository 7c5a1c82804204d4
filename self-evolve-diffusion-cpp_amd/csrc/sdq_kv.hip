// The paged int8 cache's writes and reads (gfx950).
//
// A row of 128 values of one token and head becomes 128 codes and one scale,
// as sdq_quant.hip's quantizer makes them (maximum / 127, products with the
// scale's reciprocal rounded to fp32, to the nearest even integer). 32 lanes
// hold a row, four values each, so a wave moves two rows' 1 KiB at a time and
// the maximum is five lane exchanges. Bound by HBM: per row 512 bytes read and 132
// written, and the other way round for the reads; small calls by the launch.
#include <algorithm>

#include "sdq_device.h"
#include "sdq_kv.h"

#pragma clang fp contract(off)

namespace sdq {
namespace {

using kv::kHd;
using kv::View;

constexpr int64_t kMaxBlocks = 1 << 22;  // a grid's threads are a 32-bit number

// Half-wave i of the grid: (token, tensor, head), the head fastest.
struct Row {
  int64_t t;
  int which, head;
};
__device__ __forceinline__ Row row_at(const View& c, int64_t i) {
  const int64_t per = 2 * (int64_t)c.kv_heads;
  const int64_t t = i / per;
  const int r = (int)(i - t * per);
  return {t, r >= c.kv_heads, r >= c.kv_heads ? r - c.kv_heads : r};
}

// Place of the row's token in the cache, -1 none, -2: the row is no sequence's.
__device__ __forceinline__ int64_t place(const View& c, const Row& r) {
  const int s = kv::seq_of(c, r.t);
  if (s < 0) return -2;
  const int64_t p = kv::length_of(c, s) - kv::row_of(c, s + 1) + r.t;
  return p < 0 ? -1 : kv::place_of(c, s, p, r.head);
}

__global__ void __launch_bounds__(256)
kv_write_kernel(View c, const float* __restrict__ k, int64_t ldk, const float* __restrict__ v,
                int64_t ldv) {
  const int j = threadIdx.x & 31;
  const int64_t rows = c.T * 2 * c.kv_heads;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < rows;
       i += (int64_t)gridDim.x * 8) {
    const Row r = row_at(c, i);
    const int64_t at = place(c, r);
    if (at < 0) continue;
    const float* x = (r.which ? v + r.t * ldv : k + r.t * ldk) + (int64_t)r.head * kHd;
    const float4 f = reinterpret_cast<const float4*>(x)[j];
    float mx = 0.f;
    for (float a : {f.x, f.y, f.z, f.w}) mx = mx < fabsf(a) ? fabsf(a) : mx;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float u = __shfl_xor(mx, o);
      mx = mx < u ? u : mx;
    }
    float sc = mx / 127.f;
    if (sc == 0.f) sc = 1.f;
    reinterpret_cast<uint32_t*>((r.which ? c.v : c.k) + at * kHd)[j] =
        dev::quant_pack4(f.x, f.y, f.z, f.w, 1.f / sc);
    if (j == 0) (r.which ? c.vs : c.ks)[at] = sc;
  }
}

__global__ void __launch_bounds__(256)
kv_read_kernel(View c, float* __restrict__ k, int64_t ldk, float* __restrict__ v, int64_t ldv) {
  const int j = threadIdx.x & 31;
  const int64_t rows = c.T * 2 * c.kv_heads;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < rows;
       i += (int64_t)gridDim.x * 8) {
    const Row r = row_at(c, i);
    const int64_t at = place(c, r);
    if (at == -2) continue;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    if (at >= 0) {
      const uint32_t q = reinterpret_cast<const uint32_t*>((r.which ? c.v : c.k) + at * kHd)[j];
      const float sc = (r.which ? c.vs : c.ks)[at];
      y = make_float4((float)(int8_t)q * sc, (float)(int8_t)(q >> 8) * sc,
                      (float)(int8_t)(q >> 16) * sc, (float)(int8_t)(q >> 24) * sc);
    }
    float* o = (r.which ? v + r.t * ldv : k + r.t * ldk) + (int64_t)r.head * kHd;
    reinterpret_cast<float4*>(o)[j] = y;
  }
}

}  // namespace

hipError_t launch_kv_write(const View& c, const float* k, int64_t ldk, const float* v,
                           int64_t ldv, hipStream_t s) {
  const int64_t blocks = std::min<int64_t>(ceil_div(c.T * 2 * c.kv_heads, 8), kMaxBlocks);
  hipLaunchKernelGGL(kv_write_kernel, dim3((unsigned)blocks), dim3(256), 0, s, c, k, ldk, v, ldv);
  return hipGetLastError();
}

hipError_t launch_kv_read(const View& c, float* k, int64_t ldk, float* v, int64_t ldv,
                          hipStream_t s) {
  const int64_t blocks = std::min<int64_t>(ceil_div(c.T * 2 * c.kv_heads, 8), kMaxBlocks);
  hipLaunchKernelGGL(kv_read_kernel, dim3((unsigned)blocks), dim3(256), 0, s, c, k, ldk, v, ldv);
  return hipGetLastError();
}

}  // namespace sdq
