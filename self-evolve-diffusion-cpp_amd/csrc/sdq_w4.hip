// Linears with 4-bit weights and group scales (gfx950): the weight's layout and
// the few-row product.
//
//   Y[m, n] = epilogue( sum_g scale[n, g] sum_{k in g} (u[n, k] - zero[n, g]) x[m, k] )
//
// What bounds it: the weight read, half a byte a value; the matrix cores multiply
// the codes as they are, so that unpacking them and joining the groups' sums (fp32,
// one scale each) is what the vector units do. Two forms, by the row count:
//
// Up to five rows: x as three signed bytes a value, exact int8 MFMAs of the codes,
// all bytes of all rows in one tile of 16 columns. Three operations unpack eight
// codes (fp16 ones take nine: 1 x 4096 -> 18432 14.0 us with those, 11.5 so).
//
// More rows: x as two fp16 parts, u - zero as exact fp16. Rows fill the tile's
// columns, both parts add into one sum and a group costs one fma an output (as
// bytes: eight to join three sums, the powers and the zero points).
//
// Layout: blocks of 16 outputs, cut along K into units of 128 values: 1024
// bytes, lane l's 16 bytes at l * 16 belong to output l % 16. Dword st holds values
// k = 32 st + 8 (l / 16) + 0..7 of the unit, value 2 t in nibble t and 2 t + 1 in
// nibble t + 4: a mask leaves two codes in the low mantissa bits of a pair of fp16
// (1024 + u, or 1024 + 16 u four bits higher), or four codes as bytes.
// scale [block][unit][group][16] f32; zero [block][unit][16][group] bytes. Rows
// and values past N and K are codes 0 with zero 0 or scale 0.
#include <algorithm>

#include "sdq_device.h"
#include "sdq_internal.h"

#pragma clang fp contract(off)

namespace sdq {
namespace {

using dev::v4f;
using dev::v4i;
typedef int v2i __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kWaves = 8;
constexpr int64_t kFewMaxLds = 60 * 1024;
constexpr int kNbTall = 4;  // blocks of outputs of a workgroup of 32 rows
constexpr int kTop = 15;  // a row's largest value below 2^kTop

// One wave a unit: gathers the lane's 32 codes from the row-major nibbles.
__global__ void __launch_bounds__(256)
w4_repack_kernel(const uint8_t* __restrict__ u, int64_t N, int64_t K, int64_t units, int64_t total,
                 uint8_t* __restrict__ out) {
  const int l = threadIdx.x & 63;
  const int64_t rb = (K + 1) / 2;
  for (int64_t f = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); f < total;
       f += (int64_t)gridDim.x * 4) {
    const int64_t n = f / units * 16 + (l & 15), k0 = f % units * 128 + 8 * (l >> 4);
    uint32_t w[4] = {0, 0, 0, 0};
    for (int st = 0; st < 4; st++)
      for (int i = 0; i < 8; i++) {
        const int64_t k = k0 + 32 * st + i;
        if (n < N && k < K)
          w[st] |= (((uint32_t)u[n * rb + k / 2] >> (4 * (k & 1))) & 15)
                   << (4 * ((i >> 1) + 4 * (i & 1)));
      }
    *reinterpret_cast<uint4*>(out + f * 1024 + l * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

__global__ void __launch_bounds__(256)
w4_scales_kernel(const float* __restrict__ scale, const uint8_t* __restrict__ zero, int64_t N,
                 int64_t G, int64_t Gp, int per, int64_t total, float* __restrict__ scale_out,
                 uint8_t* __restrict__ zero_out) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t n = i / (16 * Gp) * 16 + (i & 15), g = i / 16 % Gp;
    const bool ok = n < N && g < G;
    scale_out[i] = ok ? scale[n * G + g] : 0.f;
    if (zero_out) zero_out[((i / 16 - g % per) * 16) + (i & 15) * per + g % per] =
        ok ? zero[n * G + g] & 15 : 0;
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

// ---- activations ----

// Eight consecutive values of a row, zeros past K.
__device__ __forceinline__ void load8(const float* row, int64_t k, int64_t K, bool vec,
                                      float v[8]) {
  if (vec && k + 8 <= K) {
    const float4 a = *reinterpret_cast<const float4*>(row + k);
    const float4 b = *reinterpret_cast<const float4*>(row + k + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = k + i < K ? row[k + i] : 0.f;
  }
}

// ---- weights ----

// What a group's zero point takes off: 1024 + z and 64 + z as pairs of fp16.
struct ZeroPair {
  v2h a, b;
};
__device__ __forceinline__ ZeroPair zero_pair(uint32_t zz) {  // z in both halves
  return {__builtin_bit_cast(v2h, 0x64006400u + zz),
          __builtin_bit_cast(v2h, 0x54005400u + (zz << 4))};
}
// A dword's eight codes as an MFMA operand.
__device__ __forceinline__ v8h operand(uint32_t w, const ZeroPair& z) {
  const v2h sixteenth{(_Float16)0.0625f, (_Float16)0.0625f};
  auto low = [&](uint32_t x) {
    return __builtin_bit_cast(v2h, (x & 0x000f000fu) | 0x64006400u) - z.a;
  };
  auto high = [&](uint32_t x) {
    return __builtin_elementwise_fma(__builtin_bit_cast(v2h, (x & 0x00f000f0u) | 0x64006400u),
                                     sixteenth, -z.b);
  };
  const v2h a = low(w), b = high(w), c = low(w >> 8), d = high(w >> 8);
  return v8h{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A unit of a block as it is loaded: the codes, the zero points of the lane's
// output, and the unit's scales spread over the lanes (one each at most): 16
// lanes share every scale, and they get it through LDS.
struct Unit {
  uint4 q;
  uint32_t z;
  float s;
};
template <int GROUP, bool ZERO>
__device__ __forceinline__ void load_unit(const W4View& w, int64_t unit, int l, Unit& u) {
  constexpr int per = 128 / GROUP;
  u.q = *reinterpret_cast<const uint4*>(w.codes + unit * 1024 + l * 16);
  if (per == 4 || l < per * 16) u.s = w.scale[unit * per * 16 + l];
  if constexpr (ZERO) {
    const uint8_t* z = w.zero + unit * per * 16 + (l & 15) * per;
    if constexpr (per == 4)
      u.z = *reinterpret_cast<const uint32_t*>(z);
    else if constexpr (per == 2)
      u.z = *reinterpret_cast<const uint16_t*>(z);
    else
      u.z = *z;
  }
}
template <int GROUP, bool ZERO>
__device__ __forceinline__ ZeroPair zeros_of(const Unit& u, int group) {
  // byte `group` of the word, to the low byte of either half
  return zero_pair(ZERO ? __builtin_amdgcn_perm(0u, u.z, 0x0c000c00u + 0x00010001u * group)
                        : 0x00080008u);
}

// A wave's LDS words for the scales of NB units.
template <int GROUP, int NB>
struct ScaleLds {
  __attribute__((aligned(16))) float s[NB][128 / GROUP * 16];
};
template <int GROUP, int NB>
__device__ __forceinline__ void put_scales(ScaleLds<GROUP, NB>& o, const Unit (&u)[NB], int l) {
  __builtin_amdgcn_wave_barrier();  // the wave's own words: its LDS accesses stay in order
#pragma unroll
  for (int j = 0; j < NB; j++)
    if (GROUP == 32 || l < 128 / GROUP * 16) o.s[j][l] = u[j].s;
  __builtin_amdgcn_wave_barrier();
}

// ---- fewest rows (3 M <= 15 columns of one MFMA tile): one launch ----
//
// A group's values become X = rint(x 2^p), p the largest power with |X| <=
// 8355711 = 127 (2^16 + 2^8 + 1), and X = d0 2^16 + d1 2^8 + d2 with signed
// bytes d: the bytes of X + 0x808080 with their top bits flipped. Their sums
// with the codes are exact over a group. A sum in its row's own units, before the
// weight's scale, passes fp32's range for values from 2^117 on: a row that holds one
// of 2^64 or more is summed in units 2^32 larger, and the result shifted back.
//
// A workgroup of eight waves makes the bytes of all of A in LDS (its first weight
// units already on their way), then its waves take every eighth unit of NB blocks
// of 16 outputs. The tile's spare columns cost nothing. (1 x 4096 -> 18432 11.3 us, 3.6
// TB/s: 576 workgroups on 256 CUs, so that some have three and most two.)

// Power of a group whose largest magnitude is mx (finite).
__device__ __forceinline__ int group_power(float mx) {
  if (!(mx > 0.f)) return 0;
  const int p = 23 - __builtin_amdgcn_frexp_expf(mx);
  return __builtin_ldexpf(mx, p) > 8355711.f ? p - 1 : p;
}
// Digit D (0 the highest) of eight biased values as two dwords, in the order in
// which a weight dword's low and high halves hold them.
template <int D>
__device__ __forceinline__ v2i digits8(const uint32_t y[8]) {
  constexpr uint32_t b = 2 - D;
  constexpr uint32_t lo = 0x0c0c0000u | b | ((b + 4) << 8), hi = (lo << 16) | 0x0c0cu;
  auto four = [&](int i) {  // values i, i + 4, i + 1, i + 5
    const uint32_t v = __builtin_amdgcn_perm(y[i + 4], y[i], lo) |
                       __builtin_amdgcn_perm(y[i + 5], y[i + 1], hi);
    return (int)(v ^ 0x80808080u);
  };
  return v2i{four(0), four(2)};
}
__device__ __forceinline__ int sum8(v2i d) {
  return __builtin_amdgcn_sdot4(d[0], 0x01010101,
                                __builtin_amdgcn_sdot4(d[1], 0x01010101, 0, false), false);
}
__device__ __forceinline__ int low_half(uint32_t w) { return (int)(w & 0x0f0f0f0fu); }
__device__ __forceinline__ int high_half(uint32_t w) { return (int)((w >> 4) & 0x0f0f0f0fu); }
__device__ __forceinline__ long as_long(int a, int b) {
  return (long)(((uint64_t)(uint32_t)b << 32) | (uint32_t)a);
}

constexpr int kFewMaxRows = 5;
constexpr float kHuge = 0x1p64f;
constexpr int kHugeShift = 32;  // values under 2^128, their sums with 128 codes under 2^139

struct FewLds {  // offsets of the dynamic LDS, for the host too
  int64_t power, sums, scales, bytes;
  __host__ __device__ FewLds(int64_t units, int per, int M, int nb) {
    power = units * 128 * 3 * M;  // [64-value step][column][lane group][16 bytes] before it
    sums = power + units * per * M * 4;
    scales = (sums + units * per * 3 * M * 4 + 15) & ~(int64_t)15;
    bytes = scales + (int64_t)kWaves * nb * per * 16 * 4;
    const int64_t red = (int64_t)kWaves * nb * 256 * 4;  // the waves' sums, at the end
    bytes = bytes > red ? bytes : red;
  }
};

template <int GROUP, bool ZERO, int NB>
__global__ void __launch_bounds__(64 * kWaves)
w4_few_kernel(W4View wt, const float* __restrict__ x, int M, int vec, EpiArgs epi,
              float* __restrict__ y) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ int bad_row[kFewMaxRows], shift_row[kFewMaxRows];
  constexpr int per = 128 / GROUP;
  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 4;
  const int64_t units = (wt.K + 127) / 128, nblk = (wt.N + 15) / 16;
  const int64_t nb0 = (int64_t)blockIdx.x * NB;
  const FewLds at(units, per, M, NB);
  const int C = 3 * M;
  int* power = reinterpret_cast<int*>(lds + at.power);
  int* sums = reinterpret_cast<int*>(lds + at.sums);

  // The zero points here are those of the lane's four outputs of the sum.
  Unit cur[NB];
  uint32_t zcur[NB][per] = {};
  auto load = [&](int64_t u, Unit (&o)[NB], uint32_t (&z)[NB][per]) {
#pragma unroll
    for (int j = 0; j < NB; j++) {  // past the last block: any block, not stored
      const int64_t unit = (nb0 + j < nblk ? nb0 + j : nblk - 1) * units + u;
      load_unit<GROUP, false>(wt, unit, l, o[j]);
      if constexpr (ZERO) {
#pragma unroll
        for (int i = 0; i < per; i++)
          z[j][i] = reinterpret_cast<const uint32_t*>(wt.zero + (unit * 16 + 4 * g) * per)[i];
      }
    }
  };
  if (w < units) load(w, cur, zcur);

  if (tid < kFewMaxRows) bad_row[tid] = shift_row[tid] = 0;
  __syncthreads();
  for (int m = 0; m < M; m++) {
    for (int64_t k = tid * 8; k < units * 128; k += 64 * kWaves * 8) {
      float v[8];
      load8(x + m * wt.K, k, wt.K, vec != 0, v);
      float mx = 0.f;
      bool bad = false;  // not finite: enters as 0, its row ends as NaN
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const bool fine = fabsf(v[i]) <= 3.402823466e38f;
        bad |= !fine;
        v[i] = fine ? v[i] : 0.f;
        mx = fmaxf(mx, fabsf(v[i]));
      }
      if (bad) bad_row[m] = 1;
      if (mx >= kHuge) shift_row[m] = kHugeShift;
#pragma unroll
      for (int o = 1; o < GROUP / 8; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
      const int p = group_power(mx);
      uint32_t b[8];
#pragma unroll
      for (int i = 0; i < 8; i++)
        b[i] = (uint32_t)((int)__builtin_rintf(__builtin_ldexpf(v[i], p)) + 0x808080);
      const v2i ds[3] = {digits8<0>(b), digits8<1>(b), digits8<2>(b)};
      int sm[3];
#pragma unroll
      for (int d = 0; d < 3; d++) {
        // lane group (k / 8) % 4 of its step: the dwords of 32 values side by side
        int* o = reinterpret_cast<int*>(
            lds + (((k >> 6) * C + d * M + m) * 4 + ((k >> 3) & 3)) * 16 + ((k >> 5) & 1) * 4);
        o[0] = ds[d][0];
        o[2] = ds[d][1];
        sm[d] = sum8(ds[d]);
#pragma unroll
        for (int i = 1; i < GROUP / 8; i <<= 1) sm[d] += __shfl_xor(sm[d], i);
      }
      if ((k & (GROUP - 1)) == 0) {
        const int64_t grp = k / GROUP;
        power[grp * M + m] = p;
#pragma unroll
        for (int d = 0; d < 3; d++) sums[grp * C + d * M + m] = sm[d];
      }
    }
  }
  __syncthreads();

  auto& sl = *reinterpret_cast<ScaleLds<GROUP, NB>*>(lds + at.scales +
                                                     w * (int64_t)sizeof(ScaleLds<GROUP, NB>));
  const int col = (l & 15) < C ? l & 15 : C - 1, m = col % M;
  const int place = 16 - 8 * (col / M) - shift_row[m];  // the digit's 2^16, 2^8, 1
  float f[NB][4] = {};
  for (int64_t u = w; u < units; u += kWaves) {
    Unit nxt[NB];
    uint32_t znxt[NB][per] = {};
    if (u + kWaves < units) load(u + kWaves, nxt, znxt);
    put_scales<GROUP, NB>(sl, cur, l);
    const char* b = lds + ((2 * u * C + col) * 4 + g) * 16;
    const v4i d0 = *reinterpret_cast<const v4i*>(b);
    const v4i d1 = *reinterpret_cast<const v4i*>(b + C * 64);
#pragma unroll
    for (int j = 0; j < NB; j++) {
      const uint32_t q[4] = {cur[j].q.x, cur[j].q.y, cur[j].q.z, cur[j].q.w};
      // a group's sum starts at -z times its digit sum
      auto start = [&](int i) {
        const int s = -sums[(u * per + i) * C + col];
        if constexpr (!ZERO) return v4i{8 * s, 8 * s, 8 * s, 8 * s};
        auto z = [&](int e) {
          const int b = e * per + i;
          return __mul24((int)((zcur[j][b / 4] >> (8 * (b & 3))) & 255u), s);
        };
        return v4i{z(0), z(1), z(2), z(3)};
      };
      auto join = [&](const v4i& a, int i) {
        const int p = place - power[(u * per + i) * M + m];
        const v4f s = *reinterpret_cast<const v4f*>(&sl.s[j][i * 16 + 4 * g]);
#pragma unroll
        for (int e = 0; e < 4; e++)
          f[j][e] = __builtin_fmaf(__builtin_ldexpf((float)a[e], p), s[e], f[j][e]);
      };
      if constexpr (GROUP == 32) {
#pragma unroll
        for (int st = 0; st < 4; st++) {  // 32 values each
          const v4i d = st < 2 ? d0 : d1;
          join(__builtin_amdgcn_mfma_i32_16x16x32_i8(
                   as_long(low_half(q[st]), high_half(q[st])),
                   as_long(d[st & 1], d[2 + (st & 1)]), start(st), 0, 0, 0),
               st);
        }
      } else {
        const v4i a0{low_half(q[0]), low_half(q[1]), high_half(q[0]), high_half(q[1])};
        const v4i a1{low_half(q[2]), low_half(q[3]), high_half(q[2]), high_half(q[3])};
        v4i acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a0, d0, start(0), 0, 0, 0);
        if constexpr (per == 2) {
          join(acc, 0);
          acc = start(1);
        }
        join(__builtin_amdgcn_mfma_i32_16x16x64_i8(a1, d1, acc, 0, 0, 0), per - 1);
      }
    }
#pragma unroll
    for (int j = 0; j < NB; j++) {
      cur[j] = nxt[j];
#pragma unroll
      for (int i = 0; i < per; i++) zcur[j][i] = znxt[j][i];
    }
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
    const int n = i % (NB * 16), r = i / (NB * 16);
    float v = 0.f;
#pragma unroll
    for (int d = 2; d >= 0; d--) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < kWaves; k++) t += red[(k * NB * 16 + n) * 16 + d * M + r];
      v += t;
    }
    v = __builtin_ldexpf(v, shift_row[r]);
    if (bad_row[r]) v = __builtin_nanf("");
    if (nb0 * 16 + n < wt.N) store_one(epi, y, r, nb0 * 16 + n, wt.N, v);
  }
}

// ---- more rows ----
//
// A first kernel scales each row's units (128 values) by a power of two that puts the
// largest value into [2^14, 2^15) and splits them into fp16 parts, x = hi + lo to 22 bits
// of every value down to 2^-18 of the largest and an absolute 2^-40 of it below. A
// wave takes a unit of 16 rows in the layout that it writes, so that a unit's maximum
// needs no other wave and its stores are whole kilobytes (a workgroup a row with one
// power for all of it, 16 bytes at a time: 4.3 us for 13 x 5120 and 7.2 for 32 x
// 14336; now 4.3 and 5.1, and the product takes the powers out, 1 us of its 20).
//
// A workgroup takes NB blocks of 16 outputs and RT blocks of 16 rows, its eight waves
// every eighth unit of K, their codes and the parts one unit ahead. With few outputs a
// workgroup the parts' traffic (128 bytes a value and 32 rows) is the bound, with
// many the parallelism: a wave has about five units, and each waits for memory. (32 x
// 14336 -> 5120, the product alone: 32 outputs a workgroup 31 us, 64 and K in three
// ranges 20, the parts a unit instead of a step ahead 19; codes two units ahead, or two
// or four waves over the outputs of one unit: 20-22. The
// waves over outputs instead, 256 of them, and the parts of a range of K in LDS:
// 28-45 us, filling the LDS and the join of many ranges took what the traffic had;
// the rows split in that kernel too: no faster.)
//
// parts [rows / 16 RT][unit][32-value step][row block][part][lane group][row][16 bytes],
// power [rows / 16 RT][unit][row block][row].

struct Rows {
  char* parts;
  int* power;
};

// Wave i: unit and row block of i (rows past M are zeros).
template <int RT>
__global__ void __launch_bounds__(256)
w4_parts_kernel(const float* __restrict__ x, int64_t M, int64_t K, int vec, int64_t total,
                Rows o) {
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), units = (K + 127) / 128;
  if (i >= total) return;
  const int l = threadIdx.x & 63, g = l >> 4, rb = (int)(i % RT);
  const int64_t tu = i / RT, tile = tu / units, u = tu - tile * units;
  const int64_t r = (tile * RT + rb) * 16 + (l & 15);
  const int64_t k1 = r < M ? K : 0;
  const float* row = x + (r < M ? r : 0) * K;
  float v[4][8];
  // the largest finite one: what is not makes its own row NaN by itself
  float mx = 0.f;
#pragma unroll
  for (int st = 0; st < 4; st++) load8(row, u * 128 + 32 * st + 8 * g, k1, vec != 0, v[st]);
#pragma unroll
  for (int st = 0; st < 4; st++)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float a = fabsf(v[st][e]);
      mx = a <= 3.402823466e38f ? fmaxf(mx, a) : mx;
    }
  mx = fmaxf(mx, __shfl_xor(mx, 16));
  mx = fmaxf(mx, __shfl_xor(mx, 32));
  const int fit = mx > 0.f ? kTop - __builtin_amdgcn_frexp_expf(mx) : 0;
  const int p = fit > 126 ? 126 : fit;  // 2^-p is a normal float
  if (g == 0) o.power[i * 16 + l] = p;
  char* to = o.parts + (tu * 4 * RT + rb) * 2048 + l * 16;
#pragma unroll
  for (int st = 0; st < 4; st++) {
    v8h hi, lo;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float f = __builtin_ldexpf(v[st][e], p);
      hi[e] = (_Float16)f;
      lo[e] = (_Float16)(f - (float)hi[e]);
    }
    *reinterpret_cast<v8h*>(to + st * 2048 * RT) = hi;
    *reinterpret_cast<v8h*>(to + st * 2048 * RT + 1024) = lo;
  }
}

template <int GROUP, bool ZERO, int RT, int NB>
__global__ void __launch_bounds__(64 * kWaves, 2)
w4_batch_kernel(W4View wt, Rows rows, int64_t M, int splits, EpiArgs epi, float* __restrict__ y,
                float* __restrict__ part) {
  constexpr int kOut = NB * 16, kRowsT = 16 * RT;
  __shared__ union {
    float red[kWaves][kRowsT][kOut + 4];
    ScaleLds<GROUP, NB> s[kWaves];
  } lds;
  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 4, r16 = l & 15;
  const int64_t units = (wt.K + 127) / 128, nblk = (wt.N + 15) / 16;
  const int64_t ntiles = (nblk + NB - 1) / NB;
  const int z = (int)(blockIdx.x % splits);
  const int64_t nb0 = blockIdx.x / splits % ntiles * NB;
  const int64_t row0 = blockIdx.x / splits / ntiles * kRowsT;
  const int u0 = (int)(units * z / splits), u1 = (int)(units * (z + 1) / splits);

  float f[NB][RT][4] = {};
  Unit cur[NB];
  auto load = [&](int u, Unit (&o)[NB]) {
#pragma unroll
    for (int j = 0; j < NB; j++)  // past the last block: any block, not stored
      load_unit<GROUP, ZERO>(wt, (nb0 + j < nblk ? nb0 + j : nblk - 1) * units + u, l, o[j]);
  };
  struct Step {
    v8h hi[RT], lo[RT];
  };
  const char* parts = rows.parts + row0 / 16 * units * 8192 + l * 16;
  const int* powers = rows.power + row0 * units + r16;
  int power[RT];
  auto load_power = [&](int u, int (&p)[RT]) {
#pragma unroll
    for (int rt = 0; rt < RT; rt++) p[rt] = powers[(u * RT + rt) * 16];
  };
  auto load_step = [&](int u, int st, Step& x) {
    const char* b = parts + (u * 4 + st) * (int64_t)(2048 * RT);
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
      x.hi[rt] = *reinterpret_cast<const v8h*>(b + rt * 2048);
      x.lo[rt] = *reinterpret_cast<const v8h*>(b + rt * 2048 + 1024);
    }
  };
  Step x[4];
  if (u0 + w < u1) {
    load(u0 + w, cur);
    load_power(u0 + w, power);
#pragma unroll
    for (int st = 0; st < 4; st++) load_step(u0 + w, st, x[st]);
  }
  for (int u = u0 + w; u < u1; u += kWaves) {
    // The last unit loads itself again: a branch here, between the matrix
    // instructions and what reads their results, could make the compiler miss the
    // wait between the two (tests/test_mfma_hazards.py).
    const int un = u + kWaves < u1 ? u + kWaves : u;
    Unit nxt[NB];
    load(un, nxt);
    int power_next[RT];
    load_power(un, power_next);
    put_scales<GROUP, NB>(lds.s[w], cur, l);
    v4f acc[NB][RT];
    float sum[NB][RT][4];  // of the unit
#pragma unroll
    for (int st = 0; st < 4; st++) {
      constexpr int steps = GROUP / 32;  // of a group
      const int i = st / steps;
      const Step& now = x[st];
#pragma unroll
      for (int j = 0; j < NB; j++) {
        const uint32_t q[4] = {cur[j].q.x, cur[j].q.y, cur[j].q.z, cur[j].q.w};
        const v8h a = operand(q[st], zeros_of<GROUP, ZERO>(cur[j], i));
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
          if (st % steps == 0) acc[j][rt] = v4f{0.f, 0.f, 0.f, 0.f};
          acc[j][rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, now.lo[rt], acc[j][rt], 0, 0, 0);
          acc[j][rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, now.hi[rt], acc[j][rt], 0, 0, 0);
        }
      }
      load_step(un, st, x[st]);
      if (st % steps == steps - 1) {
#pragma unroll
        for (int j = 0; j < NB; j++) {
          const v4f s = *reinterpret_cast<const v4f*>(&lds.s[w].s[j][i * 16 + 4 * g]);
#pragma unroll
          for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int e = 0; e < 4; e++)
              sum[j][rt][e] = st == steps - 1 ? acc[j][rt][e] * s[e]
                                              : __builtin_fmaf(acc[j][rt][e], s[e], sum[j][rt][e]);
        }
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
      const float back = __builtin_ldexpf(1.f, -power[rt]);
      power[rt] = power_next[rt];
#pragma unroll
      for (int j = 0; j < NB; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) f[j][rt][e] = __builtin_fmaf(sum[j][rt][e], back, f[j][rt][e]);
    }
#pragma unroll
    for (int j = 0; j < NB; j++) cur[j] = nxt[j];
  }

  __syncthreads();
#pragma unroll
  for (int rt = 0; rt < RT; rt++)
#pragma unroll
    for (int j = 0; j < NB; j++)
      *reinterpret_cast<v4f*>(&lds.red[w][rt * 16 + r16][j * 16 + 4 * g]) =
          v4f{f[j][rt][0], f[j][rt][1], f[j][rt][2], f[j][rt][3]};
  __syncthreads();
  // kOut divides the step: a thread keeps its output column
  const int c = tid % kOut;
  const int64_t n = nb0 * 16 + c;
  if (n >= wt.N) return;
#pragma unroll 1
  for (int r = tid / kOut; r < kRowsT && row0 + r < M; r += 64 * kWaves / kOut) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kWaves; k++) v += lds.red[k][r][c];
    if (splits > 1)
      part[((int64_t)z * M + row0 + r) * wt.N + n] = v;
    else
      store_one(epi, y, row0 + r, n, wt.N, v);
  }
}

__global__ void __launch_bounds__(256)
w4_join_kernel(const float* __restrict__ part, int64_t M, int64_t N, int splits, EpiArgs epi,
               float* __restrict__ y) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < M * N;
       i += (int64_t)gridDim.x * 256) {
    float v = 0.f;
#pragma unroll 8
    for (int z = 0; z < splits; z++) v += part[z * M * N + i];
    const int64_t m = i / N;
    store_one(epi, y, m, i - m * N, N, v);
  }
}

template <int GROUP, bool ZERO>
hipError_t launch_form(const W4View& w, const float* x, int64_t M, EpiArgs epi, float* y,
                       const W4Plan& p, char* scratch, hipStream_t s) {
  const int vec = w.K % 4 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const int64_t units = ceil_div(w.K, 128), nblk = ceil_div(w.N, 16);
  if (p.few) {
    const unsigned bytes = (unsigned)FewLds(units, 128 / GROUP, (int)M, p.nb).bytes;
    const dim3 grid((unsigned)ceil_div(nblk, p.nb)), block(64 * kWaves);
    if (p.nb == 1)
      hipLaunchKernelGGL((w4_few_kernel<GROUP, ZERO, 1>), grid, block, bytes, s, w, x, (int)M, vec,
                         epi, y);
    else
      hipLaunchKernelGGL((w4_few_kernel<GROUP, ZERO, 2>), grid, block, bytes, s, w, x, (int)M, vec,
                         epi, y);
    return hipGetLastError();
  }
  const Rows rows{scratch, reinterpret_cast<int*>(scratch + p.power_at)};
  float* part = reinterpret_cast<float*>(scratch + p.part_at);
  for (int64_t r = 0; r < M; r += p.rows) {  // p.rows rows at a time
    const int64_t n = std::min(p.rows, M - r);
    const int64_t waves = ceil_div(n, 16 * p.rt) * p.rt * units;
    const dim3 all((unsigned)ceil_div(waves, 4));
    if (p.rt == 1)
      hipLaunchKernelGGL((w4_parts_kernel<1>), all, dim3(256), 0, s, x + r * w.K, n, w.K, vec,
                         waves, rows);
    else
      hipLaunchKernelGGL((w4_parts_kernel<2>), all, dim3(256), 0, s, x + r * w.K, n, w.K, vec,
                         waves, rows);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    EpiArgs ep = epi;
    if (ep.resid) ep.resid += r * w.N;
    const dim3 grid((unsigned)(ceil_div(n, 16 * p.rt) * ceil_div(nblk, p.nb) * p.splits));
#define SDQ_W4B(RT, NB)                                                                         \
  hipLaunchKernelGGL((w4_batch_kernel<GROUP, ZERO, RT, NB>), grid, dim3(64 * kWaves), 0, s, w,  \
                     rows, n, p.splits, ep, y + r * w.N, part)
    if (p.rt == 1) SDQ_W4B(1, 2); else SDQ_W4B(2, kNbTall);
#undef SDQ_W4B
    e = hipGetLastError();
    if (e == hipSuccess && p.splits > 1) {
      hipLaunchKernelGGL(w4_join_kernel,
                         dim3((unsigned)std::min<int64_t>(ceil_div(n * w.N, 256), 1 << 16)),
                         dim3(256), 0, s, part, n, w.N, p.splits, ep, y + r * w.N);
      e = hipGetLastError();
    }
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_w4_repack(const uint8_t* u, const float* scale, const uint8_t* zero, int64_t N,
                            int64_t K, int group, uint8_t* codes, float* scale_out,
                            uint8_t* zero_out, hipStream_t s) {
  const int64_t nb = ceil_div(N, 16), units = ceil_div(K, 128), total = nb * units;
  constexpr int64_t kMaxBlocks = 1 << 22;  // a grid's threads are a 32-bit number
  hipLaunchKernelGGL(w4_repack_kernel,
                     dim3((unsigned)std::min(ceil_div(total, 4), kMaxBlocks)), dim3(256), 0, s, u, N,
                     K, units, total, codes);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int per = 128 / group;
  const int64_t Gp = units * per, n = nb * Gp * 16;
  hipLaunchKernelGGL(w4_scales_kernel, dim3((unsigned)std::min(ceil_div(n, 256), kMaxBlocks)),
                     dim3(256), 0, s, scale, zero, N, ceil_div(K, group), Gp, per, n, scale_out,
                     zero_out);
  return hipGetLastError();
}

W4Plan plan_w4(const W4View& w, int64_t M, int cu_count) {
  W4Plan p{};
  const int64_t units = ceil_div(w.K, 128), nblk = ceil_div(w.N, 16);
  p.splits = 1;
  p.nb = nblk >= 4 * cu_count ? 2 : 1;
  p.few = M <= kFewMaxRows && FewLds(units, 128 / w.group, (int)M, p.nb).bytes <= kFewMaxLds;
  if (p.few) return p;
  p.rt = M > 16 ? 2 : 1;
  p.nb = p.rt == 2 ? kNbTall : 2;
  // Ranges of K while all workgroups run at once (two fit a CU of the short form, one
  // of the tall one) and every wave keeps two units.
  const int64_t rows = ceil_div(M, 16 * p.rt);
  p.splits = (int)std::max<int64_t>(
      1, std::min<int64_t>({(p.rt == 2 ? 1 : 2) * cu_count / (ceil_div(nblk, p.nb) * rows),
                            units / (2 * kWaves), 16}));
  // rows at a time: at most 2^22 workgroups (a grid's threads are a 32-bit number)
  // and 256 MiB of parts, or of partial sums
  const int64_t high = 16 * p.rt, tiles = ceil_div(nblk, p.nb) * p.splits;
  int64_t most = std::min((int64_t(1) << 22) / std::max(tiles, high),
                          (int64_t(1) << 28) / (units * 512 * high));
  if (p.splits > 1) most = std::min(most, (int64_t(1) << 28) / (p.splits * high * w.N * 4));
  p.rows = std::min(rows, std::max<int64_t>(1, most)) * high;
  auto put = [&](int64_t bytes) {
    const int64_t at = p.bytes;
    p.bytes += round_up(bytes, 256);
    return at;
  };
  put(p.rows * units * 512);
  p.power_at = put(p.rows * units * 4);
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
