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

typedef int v2i __attribute__((ext_vector_type(2)));
using dev::v4i;

// ---- activations as three signed bytes a value ----
//
// A group's values become X = rint(x 2^p), p the largest power with |X| <=
// 8355711 = 127 (2^16 + 2^8 + 1), and X = d0 2^16 + d1 2^8 + d2 with signed
// bytes d: the bytes of X + 0x808080 with their top bits flipped. Their
// products with the codes are int8 MFMAs, exact over a group, and need no
// unpacking of the weight beyond a mask: the codes stand in the bytes' upper
// halves, 16 times their value.

// Power of a group whose largest magnitude is mx (finite).
__device__ __forceinline__ int group_power(float mx) {
  if (!(mx > 0.f)) return 0;
  const int p = 23 - __builtin_amdgcn_frexp_expf(mx);
  return __builtin_ldexpf(mx, p) > 8355711.f ? p - 1 : p;
}
__device__ __forceinline__ uint32_t biased(float x, int p) {
  return (uint32_t)((int)__builtin_rintf(__builtin_ldexpf(x, p)) + 0x808080);
}
// Digit D (0 the highest) of eight biased values as two dwords.
template <int D>
__device__ __forceinline__ v2i digits8(const uint32_t y[8]) {
  constexpr uint32_t b = 2 - D;
  constexpr uint32_t lo = 0x0c0c0000u | b | ((b + 4) << 8), hi = (lo << 16) | 0x0c0cu;
  auto four = [&](int i) {
    const uint32_t v = __builtin_amdgcn_perm(y[i + 1], y[i], lo) |
                       __builtin_amdgcn_perm(y[i + 3], y[i + 2], hi);
    return (int)(v ^ 0x80808080u);
  };
  return v2i{four(0), four(4)};
}
__device__ __forceinline__ int sum8(v2i d) {
  return __builtin_amdgcn_sdot4(d[0], 0x01010101,
                                __builtin_amdgcn_sdot4(d[1], 0x01010101, 0, false), false);
}

// Eight consecutive values of a row (zeros past K), and their largest finite
// magnitude; bad: one was not finite (it enters as 0, its row ends as NaN).
__device__ __forceinline__ float load8(const float* row, int64_t k, int64_t K, bool vec,
                                       float v[8], bool& bad) {
  if (vec && k + 8 <= K) {
    const float4 a = *reinterpret_cast<const float4*>(row + k);
    const float4 b = *reinterpret_cast<const float4*>(row + k + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = k + i < K ? row[k + i] : 0.f;
  }
  float mx = 0.f;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const bool fine = fabsf(v[i]) <= 3.402823466e38f;
    bad |= !fine;
    v[i] = fine ? v[i] : 0.f;
    mx = fmaxf(mx, fabsf(v[i]));
  }
  return mx;
}

// The group's power and digits of eight values; the threads of a group are
// GROUP / 8 consecutive lanes. Returns the power; ds[d]: the digits; with SUM,
// sums[d]: the group's digit sums.
template <int GROUP, bool SUM>
__device__ __forceinline__ int digitize(const float v[8], float mx, v2i ds[3], int sums[3]) {
#pragma unroll
  for (int o = 1; o < GROUP / 8; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
  const int p = group_power(mx);
  uint32_t y[8];
#pragma unroll
  for (int i = 0; i < 8; i++) y[i] = biased(v[i], p);
  ds[0] = digits8<0>(y);
  ds[1] = digits8<1>(y);
  ds[2] = digits8<2>(y);
  if constexpr (SUM) {
#pragma unroll
    for (int d = 0; d < 3; d++) {
      sums[d] = sum8(ds[d]);
#pragma unroll
      for (int o = 1; o < GROUP / 8; o <<= 1) sums[d] += __shfl_xor(sums[d], o);
    }
  }
  return p;
}

// One 64-value step of a weight's unit as an MFMA operand: the low halves of
// the lane's bytes (H = 0) or the high ones.
template <int H>
__device__ __forceinline__ v4i half_of(const uint4& q) {
  if constexpr (H == 0)
    return v4i{(int)((q.x << 4) & 0xf0f0f0f0u), (int)((q.y << 4) & 0xf0f0f0f0u),
               (int)((q.z << 4) & 0xf0f0f0f0u), (int)((q.w << 4) & 0xf0f0f0f0u)};
  else
    return v4i{(int)(q.x & 0xf0f0f0f0u), (int)(q.y & 0xf0f0f0f0u), (int)(q.z & 0xf0f0f0f0u),
               (int)(q.w & 0xf0f0f0f0u)};
}
__device__ __forceinline__ long as_long(int a, int b) {
  return (long)(((uint64_t)(uint32_t)b << 32) | (uint32_t)a);
}

// A unit's codes with their scales and zero points (lane group g: outputs
// 4 g .. 4 g + 3 of the block).
template <int GROUP, bool ZERO>
struct Unit {
  static constexpr int kPer = 128 / GROUP;
  uint4 q;
  float4 s[kPer];
  uint32_t z[kPer];
};
template <int GROUP, bool ZERO>
__device__ __forceinline__ void load_unit(const W4View& w, int64_t unit, int l,
                                          Unit<GROUP, ZERO>& u) {
  u.q = *reinterpret_cast<const uint4*>(w.codes + unit * 1024 + l * 16);
#pragma unroll
  for (int i = 0; i < Unit<GROUP, ZERO>::kPer; i++) {
    const int64_t at = (unit * Unit<GROUP, ZERO>::kPer + i) * 16 + 4 * (l >> 4);
    u.s[i] = *reinterpret_cast<const float4*>(w.scale + at);
    if constexpr (ZERO) u.z[i] = *reinterpret_cast<const uint32_t*>(w.zero + at);
  }
}
// Start of a group's sum: -16 (zero - 8) times the digit sum, so that the sum
// ends as 16 sum (u - zero) d.
template <bool ZERO>
__device__ __forceinline__ v4i start_of(uint32_t z, int digit_sum) {
  if constexpr (!ZERO) return v4i{0, 0, 0, 0};
  const int s = -16 * digit_sum;
  return v4i{__mul24((int8_t)z, s), __mul24((int8_t)(z >> 8), s), __mul24((int8_t)(z >> 16), s),
             __mul24((int8_t)(z >> 24), s)};
}

// ---- fewest rows (3 M <= 15 columns of one MFMA tile): one launch ----
//
// A workgroup of eight waves makes the digits of all of A in LDS (its first
// weight units already on their way), then its waves take every eighth unit of
// NB blocks of 16 outputs. Bound by the weight read; the tile's spare columns
// cost nothing.

constexpr int kWaves = 8;
constexpr int64_t kFewMaxLds = 60 * 1024;

struct FewLds {  // offsets of the dynamic LDS, for the host too
  int64_t digits, power, sums, bytes;
  __host__ __device__ FewLds(int64_t units, int per, int M, bool zero) {
    digits = 0;
    power = units * 128 * 3 * M;
    sums = power + units * per * M * 4;
    bytes = sums + (zero ? units * per * 3 * M * 4 : 0);
  }
};

template <int GROUP, bool ZERO, int NB>
__global__ void __launch_bounds__(64 * kWaves)
w4_few_kernel(W4View wt, const float* __restrict__ x, int M, int vec, EpiArgs epi,
              float* __restrict__ y) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ int bad_row[5];
  using U = Unit<GROUP, ZERO>;
  constexpr int per = U::kPer;
  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 4;
  const int64_t units = (wt.K + 127) / 128, nblk = (wt.N + 15) / 16;
  const int64_t nb0 = (int64_t)blockIdx.x * NB;
  const FewLds at(units, per, M, ZERO);
  const int C = 3 * M;
  int* power = reinterpret_cast<int*>(lds + at.power);
  int* sums = reinterpret_cast<int*>(lds + at.sums);

  U cur[NB];
  auto load = [&](int64_t u, U (&o)[NB]) {
#pragma unroll
    for (int j = 0; j < NB; j++)  // past the last block: any block, not stored
      load_unit(wt, (nb0 + j < nblk ? nb0 + j : nblk - 1) * units + u, l, o[j]);
  };
  if (w < units) load(w, cur);

  if (tid < 5) bad_row[tid] = 0;
  __syncthreads();
  for (int m = 0; m < M; m++) {
    const float* row = x + m * wt.K;
    for (int64_t k = tid * 8; k < units * 128; k += 64 * kWaves * 8) {
      float v[8];
      bool bad = false;
      const float mx = load8(row, k, wt.K, vec != 0, v, bad);
      if (bad) bad_row[m] = 1;
      v2i ds[3];
      int sm[3];
      const int p = digitize<GROUP, ZERO>(v, mx, ds, sm);
#pragma unroll
      for (int d = 0; d < 3; d++)
        *reinterpret_cast<v2i*>(lds + ((k >> 6) * C + d * M + m) * 64 + (k & 63)) = ds[d];
      if ((k & (GROUP - 1)) == 0) {
        const int64_t grp = k / GROUP;
        power[grp * M + m] = p;
        if constexpr (ZERO) {
#pragma unroll
          for (int d = 0; d < 3; d++) sums[grp * C + d * M + m] = sm[d];
        }
      }
    }
  }
  __syncthreads();

  const int col = (l & 15) < C ? l & 15 : C - 1, m = col % M;
  const int place = 12 - 8 * (col / M);  // the digit's 2^16, 2^8, 1 and the codes' 1/16
  float f[NB][4] = {};
  for (int64_t u = w; u < units; u += kWaves) {
    U nxt[NB];
    if (u + kWaves < units) load(u + kWaves, nxt);
    const char* b = lds + (2 * u * C + col) * 64;
    int pw[per], sm[per] = {};
#pragma unroll
    for (int i = 0; i < per; i++) {
      pw[i] = place - power[(u * per + i) * M + m];
      if constexpr (ZERO) sm[i] = sums[(u * per + i) * C + col];
    }
    v4i acc[NB][per];
    if constexpr (GROUP == 32) {
#pragma unroll
      for (int st = 0; st < 4; st++) {  // 32 values each
        const v2i d = *reinterpret_cast<const v2i*>(b + (st >> 1) * C * 64 + (st & 1) * 32 + 8 * g);
#pragma unroll
        for (int j = 0; j < NB; j++) {
          const v4i a = st < 2 ? half_of<0>(cur[j].q) : half_of<1>(cur[j].q);
          acc[j][st] = __builtin_amdgcn_mfma_i32_16x16x32_i8(
              st & 1 ? as_long(a[2], a[3]) : as_long(a[0], a[1]), as_long(d[0], d[1]),
              start_of<ZERO>(cur[j].z[st], sm[st]), 0, 0, 0);
        }
      }
    } else {
      const v4i d0 = *reinterpret_cast<const v4i*>(b + 16 * g);
      const v4i d1 = *reinterpret_cast<const v4i*>(b + C * 64 + 16 * g);
#pragma unroll
      for (int j = 0; j < NB; j++) {
        acc[j][0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
            half_of<0>(cur[j].q), d0, start_of<ZERO>(cur[j].z[0], sm[0]), 0, 0, 0);
        acc[j][per - 1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
            half_of<1>(cur[j].q), d1,
            per == 1 ? acc[j][0] : start_of<ZERO>(cur[j].z[per - 1], sm[per - 1]), 0, 0, 0);
      }
    }
#pragma unroll
    for (int j = 0; j < NB; j++)
#pragma unroll
      for (int i = 0; i < per; i++) {
        const float s[4] = {cur[j].s[i].x, cur[j].s[i].y, cur[j].s[i].z, cur[j].s[i].w};
#pragma unroll
        for (int e = 0; e < 4; e++)
          f[j][e] = __builtin_fmaf(__builtin_ldexpf((float)acc[j][i][e], pw[i]), s[e], f[j][e]);
      }
#pragma unroll
    for (int j = 0; j < NB; j++) cur[j] = nxt[j];
  }

  // Join the waves and the digits, the lowest first.
  __syncthreads();
  float* red = reinterpret_cast<float*>(lds);  // [wave][block][16 outputs][16 columns]
#pragma unroll
  for (int j = 0; j < NB; j++)
#pragma unroll
    for (int e = 0; e < 4; e++) red[((w * NB + j) * 16 + 4 * g + e) * 16 + (l & 15)] = f[j][e];
  __syncthreads();
  for (int i = tid; i < NB * 16 * M; i += 64 * kWaves) {
    const int n = i % (NB * 16), mm = i / (NB * 16);
    float v = 0.f;
#pragma unroll
    for (int d = 2; d >= 0; d--) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < kWaves; k++) t += red[(k * NB * 16 + n) * 16 + d * M + mm];
      v += t;
    }
    if (bad_row[mm]) v = __builtin_nanf("");
    if (nb0 * 16 + n < wt.N) store_one(epi, y, mm, nb0 * 16 + n, wt.N, v);
  }
}

// ---- more rows: digits made once by a kernel of their own ----
//
// digits [16-row block][64-value step][digit][row][64 bytes], power [block][group][row],
// digit sums [block][group][digit][row], bad [row]. One workgroup a row (rows past M: zeros).

struct Digits {
  int8_t* d;
  int* power;
  int* sums;
  int* bad;
};

template <int GROUP, bool ZERO>
__global__ void __launch_bounds__(256)
w4_digits_kernel(const float* __restrict__ x, int64_t M, int64_t K, int vec, Digits o) {
  const int64_t r = blockIdx.x, units = (K + 127) / 128;
  const int64_t rb = r >> 4, groups = units * (128 / GROUP);
  const int r16 = (int)(r & 15);
  __shared__ int any;
  if (threadIdx.x == 0) any = 0;
  __syncthreads();
  const float* row = x + (r < M ? r : 0) * K;
  for (int64_t k = threadIdx.x * 8; k < units * 128; k += 2048) {
    float v[8];
    bool bad = false;
    const float mx = load8(row, r < M ? k : K, K, vec != 0, v, bad);
    if (bad) any = 1;
    v2i ds[3];
    int sm[3];
    const int p = digitize<GROUP, ZERO>(v, mx, ds, sm);
#pragma unroll
    for (int d = 0; d < 3; d++)
      *reinterpret_cast<v2i*>(o.d + (((rb * 2 * units + (k >> 6)) * 3 + d) * 16 + r16) * 64 +
                              (k & 63)) = ds[d];
    if ((k & (GROUP - 1)) == 0) {
      const int64_t at = rb * groups + k / GROUP;
      o.power[at * 16 + r16] = p;
      if constexpr (ZERO) {
#pragma unroll
        for (int d = 0; d < 3; d++) o.sums[(at * 3 + d) * 16 + r16] = sm[d];
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) o.bad[r] = any;
}

// RT blocks of 16 rows against NB blocks of 16 outputs, units [units z / S,
// units (z+1) / S) shared out over eight waves. Columns of an MFMA are the 16
// rows of one digit, so that a lane holds the three digits' sums of its
// output and row and joins them at once: d1 2^8 + d2 in int32 (below 2^30), then
// one fma, the power, the scale.
template <int GROUP, bool ZERO, int RT, int NB>
__global__ void __launch_bounds__(64 * kWaves)
w4_batch_kernel(W4View wt, Digits dg, int64_t M, int splits, EpiArgs epi, float* __restrict__ y,
                float* __restrict__ part) {
  using U = Unit<GROUP, ZERO>;
  constexpr int per = U::kPer;
  constexpr int kRowsP = 16 * RT + 1;  // LDS row of the joined sums
  __shared__ float red[kWaves][NB * 16][kRowsP];
  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 4, r16 = l & 15;
  const int64_t units = (wt.K + 127) / 128, nblk = (wt.N + 15) / 16;
  const int64_t ntiles = (nblk + NB - 1) / NB;
  const int z = (int)(blockIdx.x % splits);
  const int64_t nb0 = blockIdx.x / splits % ntiles * NB;
  const int64_t rb0 = blockIdx.x / splits / ntiles * RT;
  const int64_t u0 = units * z / splits, u1 = units * (z + 1) / splits;

  float f[NB][RT][4] = {};
  U cur[NB];
  auto load = [&](int64_t u, U (&o)[NB]) {
#pragma unroll
    for (int j = 0; j < NB; j++)
      load_unit(wt, (nb0 + j < nblk ? nb0 + j : nblk - 1) * units + u, l, o[j]);
  };
  if (u0 + w < u1) load(u0 + w, cur);
  for (int64_t u = u0 + w; u < u1; u += kWaves) {
    U nxt[NB];
    if (u + kWaves < u1) load(u + kWaves, nxt);
    int pw[RT][per], sm[RT][per][3] = {};
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
      for (int i = 0; i < per; i++) {
        const int64_t at = (rb0 + rt) * units * per + u * per + i;
        pw[rt][i] = -4 - dg.power[at * 16 + r16];
        if constexpr (ZERO) {
#pragma unroll
          for (int d = 0; d < 3; d++) sm[rt][i][d] = dg.sums[(at * 3 + d) * 16 + r16];
        }
      }
    auto join = [&](const v4i a[3], int j, int rt, int i) {
      const float s[4] = {cur[j].s[i].x, cur[j].s[i].y, cur[j].s[i].z, cur[j].s[i].w};
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float c = __builtin_fmaf((float)a[0][e], 65536.f, (float)((a[1][e] << 8) + a[2][e]));
        f[j][rt][e] = __builtin_fmaf(__builtin_ldexpf(c, pw[rt][i]), s[e], f[j][rt][e]);
      }
    };
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
      const int8_t* b = dg.d + ((rb0 + rt) * 2 * units + 2 * u) * 3072 + r16 * 64;
      if constexpr (GROUP == 32) {
#pragma unroll
        for (int st = 0; st < 4; st++) {
          v2i d[3];
#pragma unroll
          for (int i = 0; i < 3; i++)
            d[i] = *reinterpret_cast<const v2i*>(b + (st >> 1) * 3072 + i * 1024 + (st & 1) * 32 +
                                                 8 * g);
#pragma unroll
          for (int j = 0; j < NB; j++) {
            const v4i q = st < 2 ? half_of<0>(cur[j].q) : half_of<1>(cur[j].q);
            v4i acc[3];
#pragma unroll
            for (int i = 0; i < 3; i++)
              acc[i] = __builtin_amdgcn_mfma_i32_16x16x32_i8(
                  st & 1 ? as_long(q[2], q[3]) : as_long(q[0], q[1]), as_long(d[i][0], d[i][1]),
                  start_of<ZERO>(cur[j].z[st], sm[rt][st][i]), 0, 0, 0);
            join(acc, j, rt, st);
          }
        }
      } else {
        v4i d[2][3];
#pragma unroll
        for (int st = 0; st < 2; st++)
#pragma unroll
          for (int i = 0; i < 3; i++)
            d[st][i] = *reinterpret_cast<const v4i*>(b + st * 3072 + i * 1024 + 16 * g);
#pragma unroll
        for (int j = 0; j < NB; j++) {
          v4i acc[3];
#pragma unroll
          for (int i = 0; i < 3; i++)
            acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                half_of<0>(cur[j].q), d[0][i], start_of<ZERO>(cur[j].z[0], sm[rt][0][i]), 0, 0, 0);
          if constexpr (per == 2) join(acc, j, rt, 0);
#pragma unroll
          for (int i = 0; i < 3; i++)
            acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                half_of<1>(cur[j].q), d[1][i],
                per == 1 ? acc[i] : start_of<ZERO>(cur[j].z[per - 1], sm[rt][per - 1][i]), 0, 0, 0);
          join(acc, j, rt, per - 1);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NB; j++) cur[j] = nxt[j];
  }

#pragma unroll
  for (int j = 0; j < NB; j++)
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
      for (int e = 0; e < 4; e++) red[w][j * 16 + 4 * g + e][rt * 16 + r16] = f[j][rt][e];
  __syncthreads();
  for (int i = tid; i < NB * 16 * RT * 16; i += 64 * kWaves) {
    const int n = i % (NB * 16), r = i / (NB * 16);
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kWaves; k++) v += red[k][n][r];
    const int64_t row = rb0 * 16 + r, at = nb0 * 16 + n;
    if (row >= M || at >= wt.N) continue;
    if (splits > 1) {
      part[((int64_t)z * M + row) * wt.N + at] = v;
    } else {
      if (dg.bad[row]) v = __builtin_nanf("");
      store_one(epi, y, row, at, wt.N, v);
    }
  }
}

__global__ void __launch_bounds__(256)
w4_join_kernel(const float* __restrict__ part, const int* __restrict__ bad, int64_t M, int64_t N,
               int splits, EpiArgs epi, float* __restrict__ y) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < M * N;
       i += (int64_t)gridDim.x * 256) {
    float v = 0.f;
    for (int z = 0; z < splits; z++) v += part[z * M * N + i];
    const int64_t m = i / N;
    if (bad[m]) v = __builtin_nanf("");
    store_one(epi, y, m, i - m * N, N, v);
  }
}

template <int GROUP, bool ZERO>
hipError_t launch_form(const W4View& w, const float* x, int64_t M, EpiArgs epi, float* y,
                       const W4Plan& p, char* scratch, hipStream_t s) {
  const int vec = w.K % 4 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const int64_t units = ceil_div(w.K, 128), nblk = ceil_div(w.N, 16);
  if (p.few) {
    const FewLds lds(units, 128 / GROUP, (int)M, ZERO);
    const int64_t bytes = std::max<int64_t>(lds.bytes, kWaves * p.nb * 256 * 4);
    const dim3 grid((unsigned)ceil_div(nblk, p.nb)), block(64 * kWaves);
    if (p.nb == 1)
      hipLaunchKernelGGL((w4_few_kernel<GROUP, ZERO, 1>), grid, block, (unsigned)bytes, s, w, x,
                         (int)M, vec, epi, y);
    else
      hipLaunchKernelGGL((w4_few_kernel<GROUP, ZERO, 2>), grid, block, (unsigned)bytes, s, w, x,
                         (int)M, vec, epi, y);
    return hipGetLastError();
  }
  const Digits dg{reinterpret_cast<int8_t*>(scratch), reinterpret_cast<int*>(scratch + p.power_at),
                  reinterpret_cast<int*>(scratch + p.sums_at),
                  reinterpret_cast<int*>(scratch + p.bad_at)};
  float* part = reinterpret_cast<float*>(scratch + p.part_at);
  for (int64_t r = 0; r < M; r += p.rows) {  // p.rows rows at a time
    const int64_t n = std::min(p.rows, M - r);
    const int64_t blocks = ceil_div(n, 16 * p.rt);
    hipLaunchKernelGGL((w4_digits_kernel<GROUP, ZERO>), dim3((unsigned)(blocks * 16 * p.rt)),
                       dim3(256), 0, s, x + r * w.K, n, w.K, vec, dg);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    EpiArgs ep = epi;
    if (ep.resid) ep.resid += r * w.N;
    const dim3 grid((unsigned)(blocks * ceil_div(nblk, p.nb) * p.splits)), block(64 * kWaves);
#define SDQ_W4B(RT, NB)                                                                         \
  hipLaunchKernelGGL((w4_batch_kernel<GROUP, ZERO, RT, NB>), grid, block, 0, s, w, dg, n,       \
                     p.splits, ep, y + r * w.N, part)
    if (p.rt == 1) {
      if (p.nb == 2) SDQ_W4B(1, 2); else SDQ_W4B(1, 4);
    } else {
      if (p.nb == 2) SDQ_W4B(2, 2); else SDQ_W4B(2, 4);
    }
#undef SDQ_W4B
    e = hipGetLastError();
    if (e == hipSuccess && p.splits > 1) {
      hipLaunchKernelGGL(w4_join_kernel,
                         dim3((unsigned)std::min<int64_t>(ceil_div(n * w.N, 256), 1 << 16)),
                         dim3(256), 0, s, part, dg.bad, n, w.N, p.splits, ep, y + r * w.N);
      e = hipGetLastError();
    }
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
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

W4Plan plan_w4(const W4View& w, int64_t M, int cu_count) {
  W4Plan p{};
  const int64_t units = ceil_div(w.K, 128), nblk = ceil_div(w.N, 16);
  const int per = 128 / w.group;
  p.splits = 1;
  p.few = M <= 5 && FewLds(units, per, (int)M, w.zero != nullptr).bytes <= kFewMaxLds;
  if (p.few) {
    p.nb = nblk >= 4 * cu_count ? 2 : 1;
    return p;
  }
  p.rt = M > 16 ? 2 : 1;
  const int64_t high = 16 * p.rt;
  // digits of at most about 256 MiB at a time
  p.rows = std::max<int64_t>(1, std::min<int64_t>(ceil_div(M, high),
                                                  (int64_t(1) << 28) / (units * 384 * high))) * high;
  const int64_t blocks = ceil_div(std::min(M, p.rows), high);
  p.nb = nblk * blocks >= 2 * cu_count ? 4 : 2;
  const int64_t groups = ceil_div(nblk, p.nb) * blocks;
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({cu_count / std::max<int64_t>(groups, 1) + 1,
                                                          units / (2 * kWaves), 8}));
  // a grid's threads are a 32-bit number
  while (p.rows > high && ceil_div(p.rows, high) * ceil_div(nblk, p.nb) * p.splits > (1 << 22))
    p.rows -= high;
  auto put = [&](int64_t bytes) {
    const int64_t at = p.bytes;
    p.bytes += round_up(bytes, 256);
    return at;
  };
  put(p.rows * units * 384);
  p.power_at = put(p.rows * units * per * 4);
  p.sums_at = put(w.zero ? p.rows * units * per * 12 : 0);
  p.bad_at = put(p.rows * 4);
  p.part_at = put(p.splits > 1 ? p.splits * std::min(M, p.rows) * w.N * 4 : 0);
  return p;
}

hipError_t launch_w4(const W4View& w, const float* x, int64_t M, const EpiArgs& epi, float* y,
                     const W4Plan& p, void* scratch, hipStream_t s) {
  char* sc = static_cast<char*>(scratch);
  if (w.group == 32)
    return w.zero ? launch_form<32, true>(w, x, M, epi, y, p, sc, s)
                  : launch_form<32, false>(w, x, M, epi, y, p, sc, s);
  if (w.group == 64)
    return w.zero ? launch_form<64, true>(w, x, M, epi, y, p, sc, s)
                  : launch_form<64, false>(w, x, M, epi, y, p, sc, s);
  return w.zero ? launch_form<128, true>(w, x, M, epi, y, p, sc, s)
                : launch_form<128, false>(w, x, M, epi, y, p, sc, s);
}

}  // namespace sdq
