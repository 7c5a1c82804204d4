// Linears with 4-bit weights and group scales (gfx950): the weight's layout and
// the few-row product.
//
//   Y[m, n] = epilogue( sum_g scale[n, g] sum_{k in g} (u[n, k] - zero[n, g]) x[m, k] )
//
// Layout: blocks of 16 outputs, cut along K into units of 128 values: 1024
// bytes, lane l's 16 bytes at l * 16 belong to output l % 16 and lane group
// g = l / 16. A byte holds two codes u - 8 in two's complement, so that
// masking a half leaves 16 times the signed code in a byte. Group sizes 64 and
// 128: byte b's low half is k = 16 g + b, its high half k = 64 + 16 g + b.
// Group size 32: the low halves of bytes 0-7 and 8-15 are k = 8 g + b % 8 of the
// unit's first and second 32, the high halves those of its third and fourth.
// scale [block][group][16] f32, zero - 8 [block][group][16] int8. Rows and
// values past N and K are zero codes with scale 0.
#include <algorithm>

#include "sdq_device.h"
#include "sdq_internal.h"

#pragma clang fp contract(off)

namespace sdq {
namespace {

// k inside its unit of the nibble (byte b, half h) of lane group g.
__host__ __device__ __forceinline__ int unit_k(int group, int b, int h, int g) {
  return group == 32 ? 32 * ((b >> 3) + 2 * h) + 8 * g + (b & 7) : 64 * h + 16 * g + b;
}

// One wave a unit: gathers the lane's 32 codes from the row-major nibbles.
__global__ void __launch_bounds__(256)
w4_repack_kernel(const uint8_t* __restrict__ u, int64_t N, int64_t K, int group, int64_t units,
                 int64_t total, uint8_t* __restrict__ out) {
  const int l = threadIdx.x & 63;
  const int64_t rb = (K + 1) / 2;
  for (int64_t f = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); f < total;
       f += (int64_t)gridDim.x * 4) {
    const int64_t n = f / units * 16 + (l & 15), k0 = f % units * 128;
    uint32_t w[4] = {0, 0, 0, 0};
    for (int b = 0; b < 16; b++)
      for (int h = 0; h < 2; h++) {
        const int64_t k = k0 + unit_k(group, b, h, l >> 4);
        if (n < N && k < K) {
          const uint32_t c = ((uint32_t)u[n * rb + k / 2] >> (4 * (k & 1))) & 15;
          w[b >> 2] |= (c ^ 8) << (8 * (b & 3) + 4 * h);
        }
      }
    *reinterpret_cast<uint4*>(out + f * 1024 + l * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

__global__ void __launch_bounds__(256)
w4_scales_kernel(const float* __restrict__ scale, const uint8_t* __restrict__ zero, int64_t N,
                 int64_t G, int64_t Gp, int64_t total, float* __restrict__ scale_out,
                 int8_t* __restrict__ zero_out) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t n = i / (16 * Gp) * 16 + (i & 15), g = i / 16 % Gp;
    const bool ok = n < N && g < G;
    scale_out[i] = ok ? scale[n * G + g] : 0.f;
    if (zero_out) zero_out[i] = ok ? (int8_t)((int)zero[n * G + g] - 8) : (int8_t)0;
  }
}

// Output (m, n) from its sum.
__device__ __forceinline__ void store_one(const EpiArgs& e, float* y, int64_t m, int64_t n,
                                          int64_t N, float v) {
  if (e.bias) v = v + e.bias[n];
  const int64_t i = m * N + n;
  if (e.kind == SDQ_EPI_GELU)
    v = dev::gelu_tanh(v);
  else if (e.kind == SDQ_EPI_GATED)
    v = e.gate_fma ? __builtin_fmaf(v, e.gate[n], e.resid[i]) : e.resid[i] + v * e.gate[n];
  else if (e.kind == SDQ_EPI_RESID)
    v = e.resid[i] + v;
  y[i] = v;
}

// One wave a block of 16 outputs, rows one after the other.
template <int GROUP, bool ZERO>
__global__ void __launch_bounds__(64)
w4_simple_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scale,
                 const int8_t* __restrict__ zero, const float* __restrict__ x, int64_t M,
                 int64_t K, int64_t N, int64_t units, EpiArgs epi, float* __restrict__ y) {
  const int l = threadIdx.x, r = l & 15, g = l >> 4;
  const int64_t nb = blockIdx.x, m = blockIdx.y;
  constexpr int per = 128 / GROUP;
  float sum = 0.f;
  for (int64_t u = 0; u < units; u++) {
    const uint4 q = *reinterpret_cast<const uint4*>(codes + (nb * units + u) * 1024 + l * 16);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    float part[per] = {}, xs[per] = {};
#pragma unroll
    for (int b = 0; b < 16; b++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int64_t k = u * 128 + unit_k(GROUP, b, h, g);
        const int at = (GROUP == 32 ? (b >> 3) + 2 * h : GROUP == 64 ? h : 0);
        const int c = (int)(w[b >> 2] << (28 - 8 * (b & 3) - 4 * h)) >> 28;
        float v = k < K ? x[m * K + k] : 0.f;
        if (!(fabsf(v) <= 3.402823466e38f)) v = __builtin_nanf("");  // the row's result: NaN
        part[at] += (float)c * v;
        xs[at] += v;
      }
#pragma unroll
    for (int i = 0; i < per; i++) {
      const int64_t at = ((nb * units + u) * per + i) * 16 + r;
      const float z = ZERO ? (float)zero[at] : 0.f;
      sum += scale[at] * (part[i] - z * xs[i]);
    }
  }
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  const int64_t n = nb * 16 + r;
  if (g == 0 && n < N) store_one(epi, y, m, n, N, sum);
}

}  // namespace

hipError_t launch_w4_repack(const uint8_t* u, const float* scale, const uint8_t* zero, int64_t N,
                            int64_t K, int group, uint8_t* codes, float* scale_out,
                            int8_t* zero_out, hipStream_t s) {
  const int64_t nb = ceil_div(N, 16), units = ceil_div(K, 128), total = nb * units;
  constexpr int64_t kMaxBlocks = 1 << 22;  // a grid's threads are a 32-bit number
  hipLaunchKernelGGL(w4_repack_kernel,
                     dim3((unsigned)std::min(ceil_div(total, 4), kMaxBlocks)), dim3(256), 0, s, u, N, K,
                     group, units, total, codes);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t Gp = units * (128 / group), n = nb * Gp * 16;
  hipLaunchKernelGGL(w4_scales_kernel, dim3((unsigned)std::min(ceil_div(n, 256), kMaxBlocks)), dim3(256), 0, s, scale,
                     zero, N, ceil_div(K, group), Gp, n, scale_out, zero_out);
  return hipGetLastError();
}

hipError_t launch_w4(const W4View& w, const float* x, int64_t M, const EpiArgs& epi, float* y,
                     hipStream_t s) {
  const dim3 grid((unsigned)ceil_div(w.N, 16), (unsigned)M);
  const int64_t units = ceil_div(w.K, 128);
#define SDQ_W4(G, Z)                                                                             \
  hipLaunchKernelGGL((w4_simple_kernel<G, Z>), grid, dim3(64), 0, s, w.codes, w.scale, w.zero, x, \
                     M, w.K, w.N, units, epi, y)
  if (w.group == 32) {
    if (w.zero) SDQ_W4(32, true); else SDQ_W4(32, false);
  } else if (w.group == 64) {
    if (w.zero) SDQ_W4(64, true); else SDQ_W4(64, false);
  } else {
    if (w.zero) SDQ_W4(128, true); else SDQ_W4(128, false);
  }
#undef SDQ_W4
  return hipGetLastError();
}

}  // namespace sdq
