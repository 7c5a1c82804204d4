// Attention of new tokens over the paged int8 cache (gfx950).
//
// Per row (token i at position p, head h): logits t_j = scale q . k_j over the
// sequence's keys (j <= p where causal), out = sum_j 2^(t_j - m) v_j / sum_j
// 2^(t_j - m) with t in units of log2 and m the running maximum.
#include <algorithm>

#include "sdq_device.h"
#include "sdq_kv.h"

#pragma clang fp contract(off)

namespace sdq {
namespace {

using kv::kHd;
using kv::View;

// One wave a row and head; lane l holds dims 2l and 2l + 1.
__global__ void __launch_bounds__(64)
kv_attn_simple_kernel(View c, const float* __restrict__ q, int64_t ldq, float* __restrict__ out,
                      int64_t ldo, int heads, float scale2, int causal) {
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, l = threadIdx.x;
  const int s = kv::seq_of(c, t);
  if (s < 0) return;
  const int64_t len = kv::length_of(c, s);
  const int64_t p = len - kv::row_of(c, s + 1) + t;
  const int64_t end = causal ? (p + 1 < len ? p + 1 : len) : len;
  const int kvh = h / (heads / c.kv_heads);
  const float2 a = reinterpret_cast<const float2*>(q + t * ldq + (int64_t)h * kHd)[l];
  float m = -INFINITY, z = 0.f, o0 = 0.f, o1 = 0.f;
  for (int64_t j = 0; p >= 0 && j < end; j++) {
    const int64_t at = kv::place_of(c, s, j, kvh);
    if (at < 0) continue;
    const uint16_t kk = reinterpret_cast<const uint16_t*>(c.k + at * kHd)[l];
    const uint16_t vv = reinterpret_cast<const uint16_t*>(c.v + at * kHd)[l];
    float dot = a.x * (float)(int8_t)kk + a.y * (float)(int8_t)(kk >> 8);
#pragma unroll
    for (int o = 32; o; o >>= 1) dot += __shfl_xor(dot, o);
    const float x = dot * c.ks[at] * scale2;
    const float top = m < x ? x : m;
    const float f = m == top ? 1.f : __builtin_exp2f(m - top);
    const float e = __builtin_exp2f(x - top);
    const float w = e * c.vs[at];
    z = z * f + e;
    o0 = o0 * f + w * (float)(int8_t)vv;
    o1 = o1 * f + w * (float)(int8_t)(vv >> 8);
    m = top;
  }
  const float inv = z == 0.f ? 0.f : 1.f / z;
  reinterpret_cast<float2*>(out + t * ldo + (int64_t)h * kHd)[l] = float2{o0 * inv, o1 * inv};
}

}  // namespace

hipError_t launch_kv_attn(const View& c, const float* q, int64_t ldq, float* out, int64_t ldo,
                          int heads, float scale, int causal, hipStream_t s) {
  hipLaunchKernelGGL(kv_attn_simple_kernel, dim3((unsigned)c.T, (unsigned)heads), dim3(64), 0, s, c,
                     q, ldq, out, ldo, heads, scale * 1.44269504088896341f, causal);
  return hipGetLastError();
}

}  // namespace sdq
