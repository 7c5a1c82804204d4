// Residual addition + root-mean-square norm + int8 row codes in one pass
// (gfx950), the codes' way back to fp32, and their way into the GEMM's
// fragment layout.
//
//   h = fl(x + d);  y = fl(h / sqrt(mean(h^2) + eps) * w);  codes of y
//
// A code is decided by y * 127 / max|y| next to a half, where one fp32
// rounding of the norm moves it by a whole step; so the sum of squares and the
// product are 64-bit (the card runs them at the fp32 rate, and the kernel waits
// for memory either way) and rounded once. From y on the steps are those of
// the plain quantizer (sdq_quant.hip), in fp32.
//
// Bound by HBM: with a residual and its sum 8 bytes read and 5 written per value. A
// row is read once and stays in the registers of its threads (T of them, NV groups of
// four values each) over the two reductions; rows past the register form are read
// again. 27280 x 5120: 358 us, 5.07 TB/s, the rate of a large copy (the codes' way
// back 116 us, 6.0 TB/s); 509 x 4096 10.2 us, 2.6 TB/s (a load a thread and array, and the
// weight's behind the first reduction), and one row 4.1 us, which is latency. Rows past
// the register form: 1000 x 20000 104 us, 2.5 TB/s of what it has to move.
#include <algorithm>

#include "sdq_device.h"
#include "sdq_internal.h"

#pragma clang fp contract(off)

namespace sdq {
namespace {

struct RmsqArgs {
  const float* x;
  int64_t ldx;
  const float* d;  // nullable
  int64_t ldd;
  int64_t M, K;
  const float* w;  // nullable
  double eps;
  float* sum;  // nullable; may be x or d
  int64_t ldsum;
  int8_t* aq;
  float* as;
};

// Sum (64-bit) or maximum over the T threads of a row; every thread gets it.
// T == 64: a wave owns its row and needs no barrier.
template <int T>
__device__ __forceinline__ double row_sum(double v, double* red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  if constexpr (T > 64) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[w] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int i = 0; i < T / 64; i++) v += red[i];
  }
  return v;
}
template <int T>
__device__ __forceinline__ float row_max(float v, float* red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const float u = __shfl_xor(v, o);
    v = v < u ? u : v;
  }
  if constexpr (T > 64) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[w] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < T / 64; i++) v = v < red[i] ? red[i] : v;
  }
  return v;
}

// The scale of a row whose largest magnitude is mx, and its reciprocal.
__device__ __forceinline__ float2 scale_of(float mx) {
  float sc = mx / 127.f;
  if (sc == 0.f) sc = 1.f;
  return float2{sc, 1.f / sc};
}

// R rows a workgroup, T threads a row, up to 4 * NV * T values. VEC: four
// consecutive values a thread and group (K and the row strides multiples of 4,
// 16-byte aligned arrays); else single values, T apart.
template <int T, int R, int NV, bool VEC>
__global__ void __launch_bounds__(T * R) rmsnorm_quant_kernel(RmsqArgs a) {
  static_assert(T == 64 || R == 1, "rows of several waves have the workgroup to themselves");
  __shared__ double red_sum[T / 64];
  __shared__ float red_max[T / 64];
  const int t = threadIdx.x % T;
  const int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / T;
  if (R > 1 && row >= a.M) return;
  const float* xr = a.x + row * a.ldx;
  const float* dr = a.d ? a.d + row * a.ldd : nullptr;
  float* sr = a.sum ? a.sum + row * a.ldsum : nullptr;
  const int K = (int)a.K;  // fits the register form
  float h[NV][4];
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < NV; i++) {
    if constexpr (VEC) {
      const int k = (t + i * T) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k < K) {
        v = *reinterpret_cast<const float4*>(xr + k);
        if (dr) {
          const float4 u = *reinterpret_cast<const float4*>(dr + k);
          v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
        }
        if (sr) *reinterpret_cast<float4*>(sr + k) = v;
      }
      h[i][0] = v.x; h[i][1] = v.y; h[i][2] = v.z; h[i][3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int k = t + (4 * i + e) * T;
        float v = 0.f;
        if (k < K) {
          v = xr[k];
          if (dr) v += dr[k];
          if (sr) sr[k] = v;
        }
        h[i][e] = v;
      }
    }
#pragma unroll
    for (int e = 0; e < 4; e++) ss = __builtin_fma((double)h[i][e], (double)h[i][e], ss);
  }
  ss = row_sum<T>(ss, red_sum);
  const double inv = 1.0 / __builtin_sqrt(ss / (double)a.K + a.eps);
  float mx = 0.f;
#pragma unroll
  for (int i = 0; i < NV; i++) {
    float wv[4] = {1.f, 1.f, 1.f, 1.f};
    if (a.w) {
      if constexpr (VEC) {
        const int k = (t + i * T) * 4;
        if (k < K) {
          const float4 u = *reinterpret_cast<const float4*>(a.w + k);
          wv[0] = u.x; wv[1] = u.y; wv[2] = u.z; wv[3] = u.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int k = t + (4 * i + e) * T;
          wv[e] = k < K ? a.w[k] : 0.f;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float y = (float)((double)h[i][e] * inv * (double)wv[e]);
      h[i][e] = y;
      const float m = fabsf(y);
      // the padding's zeros times an infinite inv are NaN: they never win
      mx = mx < m ? m : mx;
    }
  }
  mx = row_max<T>(mx, red_max);
  const float2 sc = scale_of(mx);
  if (t == 0) a.as[row] = sc.x;
  int8_t* q = a.aq + row * a.K;
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const uint32_t p = dev::quant_pack4(h[i][0], h[i][1], h[i][2], h[i][3], sc.y);
    if constexpr (VEC) {
      const int k = (t + i * T) * 4;
      if (k < K) *reinterpret_cast<uint32_t*>(q + k) = p;
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int k = t + (4 * i + e) * T;
        if (k < K) q[k] = (int8_t)(p >> (8 * e));
      }
    }
  }
}

// Rows past the register form: one workgroup a row, three passes over it. With
// a sum the later passes read it (each thread the values that it wrote), so
// that x or d may be the sum.
__global__ void __launch_bounds__(1024) rmsnorm_quant_long_kernel(RmsqArgs a) {
  __shared__ double red_sum[16];
  __shared__ float red_max[16];
  const int64_t row = blockIdx.x;
  const float* xr = a.x + row * a.ldx;
  const float* dr = a.d ? a.d + row * a.ldd : nullptr;
  float* sr = a.sum ? a.sum + row * a.ldsum : nullptr;
  double ss = 0.0;
  for (int64_t k = threadIdx.x; k < a.K; k += 1024) {
    float v = xr[k];
    if (dr) v += dr[k];
    if (sr) sr[k] = v;
    ss = __builtin_fma((double)v, (double)v, ss);
  }
  ss = row_sum<1024>(ss, red_sum);
  const double inv = 1.0 / __builtin_sqrt(ss / (double)a.K + a.eps);
  auto value = [&](int64_t k) {
    float v = sr ? sr[k] : xr[k];
    if (!sr && dr) v += dr[k];
    return (float)((double)v * inv * (a.w ? (double)a.w[k] : 1.0));
  };
  float mx = 0.f;
  for (int64_t k = threadIdx.x; k < a.K; k += 1024) {
    const float m = fabsf(value(k));
    mx = mx < m ? m : mx;
  }
  mx = row_max<1024>(mx, red_max);
  const float2 sc = scale_of(mx);
  if (threadIdx.x == 0) a.as[row] = sc.x;
  for (int64_t k = threadIdx.x; k < a.K; k += 1024)
    a.aq[row * a.K + k] = (int8_t)dev::quant_one(value(k), sc.y);
}

// A grid's threads are a 32-bit number: many rows run in ranges of 2^21.
template <class F>
hipError_t in_ranges(RmsqArgs a, F launch) {
  constexpr int64_t kRange = 1 << 21;
  const int64_t M = a.M;
  for (int64_t r = 0; r < M; r += kRange) {
    a.M = std::min(kRange, M - r);
    launch(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    a.x += kRange * a.ldx;
    if (a.d) a.d += kRange * a.ldd;
    if (a.sum) a.sum += kRange * a.ldsum;
    a.aq += kRange * a.K;
    a.as += kRange;
  }
  return hipSuccess;
}

template <int T, int R, int NV>
hipError_t launch_rows(const RmsqArgs& args, bool vec, hipStream_t s) {
  return in_ranges(args, [&](const RmsqArgs& a) {
    const dim3 grid((unsigned)ceil_div(a.M, R)), block(T * R);
    if (vec)
      hipLaunchKernelGGL((rmsnorm_quant_kernel<T, R, NV, true>), grid, block, 0, s, a);
    else
      hipLaunchKernelGGL((rmsnorm_quant_kernel<T, R, NV, false>), grid, block, 0, s, a);
  });
}

__global__ void __launch_bounds__(256)
dequant_kernel(const int8_t* __restrict__ aq, const float* __restrict__ as, int64_t M, int64_t K,
               int vec, float* __restrict__ y) {
  const int64_t n = M * K;
  if (vec) {  // K % 4 == 0: a group of four stays inside its row
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n;
         i += (int64_t)gridDim.x * 1024) {
      const uint32_t q = *reinterpret_cast<const uint32_t*>(aq + i);
      const float s = as[i / K];
      *reinterpret_cast<float4*>(y + i) =
          make_float4((float)(int8_t)q * s, (float)(int8_t)(q >> 8) * s,
                      (float)(int8_t)(q >> 16) * s, (float)(int8_t)(q >> 24) * s);
    }
  } else {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
      y[i] = (float)aq[i] * as[i / K];
  }
}

// Row-major codes -> fragments of Mp rows and KFp fragments (zeros past M and
// K), and the padded column copies, as the quantizers leave them. One wave a
// fragment; the first workgroups copy the columns.
__global__ void __launch_bounds__(256)
codes_frags_kernel(const int8_t* __restrict__ aq, const float* __restrict__ as, int64_t M,
                   int64_t K, int64_t KFp, int64_t nfrags, int64_t Mp, int vec,
                   int8_t* __restrict__ frags, float* __restrict__ as_out, ColCopy cc) {
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < std::max(cc.CP, Mp); i += step) {
    if (i < cc.CP && cc.bias_pad) cc.bias_pad[i] = i < cc.N ? cc.bias[i] : 0.f;
    if (i < cc.CP && cc.gate_pad) cc.gate_pad[i] = i < cc.N ? cc.gate[i] : 0.f;
    if (i < Mp) as_out[i] = i < M ? as[i] : 0.f;
  }
  const int l = threadIdx.x & 63;
  for (int64_t f = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); f < nfrags;
       f += (int64_t)gridDim.x * 4) {
    const int64_t rb = f / KFp, kb = f - rb * KFp;
    const int64_t row = rb * 32 + (l & 31);
    const int64_t k0 = kb * 32 + (l >> 5) * 16;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < M) {
      const int8_t* src = aq + row * K;
      if (vec && k0 + 16 <= K) {
        v = *reinterpret_cast<const uint4*>(src + k0);
      } else {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 16; e++)
          if (k0 + e < K) w[e >> 2] |= (uint32_t)(uint8_t)src[k0 + e] << (8 * (e & 3));
        v = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    *reinterpret_cast<uint4*>(frags + f * 1024 + l * 16) = v;
  }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

hipError_t launch_rmsnorm_quant(const float* x, int64_t ldx, const float* d, int64_t ldd,
                                int64_t M, int64_t K, const float* w, float eps, float* sum,
                                int64_t ldsum, int8_t* aq, float* as, int cu_count,
                                hipStream_t s) {
  RmsqArgs a{x, ldx, d, ldd, M, K, w, (double)eps, sum, ldsum, aq, as};
  const bool vec = K % 4 == 0 && al16(x) && ldx % 4 == 0 && (!d || (al16(d) && ldd % 4 == 0)) &&
                   (!w || al16(w)) && (!sum || (al16(sum) && ldsum % 4 == 0)) && al16(aq);
  if (K <= 256) return launch_rows<64, 4, 1>(a, vec, s);
  if (K <= 512) return launch_rows<64, 4, 2>(a, vec, s);
  if (K <= 1024) return launch_rows<256, 1, 1>(a, vec, s);
  // Few rows leave the machine idle: more threads a row, fewer values each.
  if (M <= 2 * cu_count) {
    if (K <= 4096) return launch_rows<1024, 1, 1>(a, vec, s);
    if (K <= 8192) return launch_rows<1024, 1, 2>(a, vec, s);
  }
  if (K <= 2048) return launch_rows<256, 1, 2>(a, vec, s);
  if (K <= 4096) return launch_rows<256, 1, 4>(a, vec, s);
  if (K <= 6144) return launch_rows<256, 1, 6>(a, vec, s);
  if (K <= 8192) return launch_rows<256, 1, 8>(a, vec, s);
  if (K <= 16384) return launch_rows<1024, 1, 4>(a, vec, s);
  return in_ranges(a, [&](const RmsqArgs& r) {
    hipLaunchKernelGGL(rmsnorm_quant_long_kernel, dim3((unsigned)r.M), dim3(1024), 0, s, r);
  });
}

hipError_t launch_dequant(const int8_t* aq, const float* as, int64_t M, int64_t K, float* y,
                          hipStream_t s) {
  const int vec = K % 4 == 0 && al16(aq) && al16(y);
  const int64_t blocks = ceil_div(M * K, vec ? 1024 : 256);
  hipLaunchKernelGGL(dequant_kernel, dim3((unsigned)std::min<int64_t>(blocks, 1 << 16)), dim3(256),
                     0, s, aq, as, M, K, vec, y);
  return hipGetLastError();
}

hipError_t launch_codes_frags(const int8_t* aq, const float* as, int64_t M, int64_t K, int64_t Mp,
                              int64_t KFp, int8_t* at, float* as_out, const ColCopy& cc,
                              hipStream_t s) {
  const int64_t nfrags = (Mp / kFragRows) * KFp;
  const int vec = K % 16 == 0 && al16(aq);
  hipLaunchKernelGGL(codes_frags_kernel,
                     dim3((unsigned)std::min<int64_t>(ceil_div(nfrags, 4), 1 << 22)), dim3(256), 0, s, aq,
                     as, M, K, KFp, nfrags, Mp, vec, at, as_out, cc);
  return hipGetLastError();
}

}  // namespace sdq
