// The softmax weights that each cached key was given, summed over a call's rows (gfx950).
//
// Per key j and cached head, over the call's rows r of the head's group that see it, with
// t_rj = scale log2(e) q_r . k_j + e_j, row r's maximum m_r of t and denominator d_r as the
// attention left them (e_j: the exponent of the key's value scale, see sdq_kv_attn.hip):
//   sum_r 2^(t_rj - m_r - e_j) / d_r.
//
// The logits are formed again, bit for bit as the attention forms them (a row's weights then
// sum to 1 however large they are), two MFMA products each: half of the attention's. A wave keeps 64 keys in registers, the workgroup 256, and the rows pass by in
// LDS, 32 at a time in two buffers; a lane sums the weights of 16 of its keys for one row of
// 16, the lanes' sums are joined once a block of keys. One workgroup sums a key over all
// rows, in their order: no atomics, the same bits every time.
#include <algorithm>

#include "sdq_kv_attn.h"

#pragma clang fp contract(off)

namespace sdq {
namespace {

using namespace kvattn;

constexpr int kWaves = 4;
constexpr int kTiles = 4;                        // of 16 keys, a wave
constexpr int kBlock = 16 * kTiles * kWaves;     // keys of a workgroup
constexpr int kRows = 32;                        // in LDS

struct RowInfo {
  float qk, m, inv;
  int see;  // keys; 0: the row adds nothing
};
struct Stage {
  __attribute__((aligned(16))) char q[2][kRows / 16][4][1024];  // [hi, lo][tile][kb][lane 16 B]
  RowInfo row[kRows];
};

__global__ void __launch_bounds__(64 * kWaves, 2)
kv_weights_kernel(Args a, float* __restrict__ sums, int across) {
  __shared__ Stage buf[2];
  const View& c = a.c;
  const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, r16 = l & 15, g = l >> 4;
  const int x = (int)(blockIdx.x % across);
  const int64_t sh = blockIdx.x / across;
  const int h = (int)(sh % c.kv_heads), s = (int)(sh / c.kv_heads);
  Tile t{s, 0, 0, kv::row_of(c, s), 0, 0};
  const int64_t tokens = kv::row_of(c, s + 1) - t.row0;
  if (tokens <= 0) return;
  t.rows = tokens * a.group;
  t.len = (int)kv::length_of(c, s);
  t.first = t.len - (int)tokens;
  const int32_t* table = c.table + s * c.max_pages;
  const int e0 = first_exp(c, t, h);

  for (int64_t b = x; b * kBlock < t.len; b += across) {
    // the wave's keys as MFMA operands and their scales
    const int k0 = (int)(b * kBlock) + 16 * kTiles * w;
    v8h key[kTiles][4];
    v4f kc[kTiles], ke[kTiles];
    bool there[kTiles];
    int64_t at[kTiles];
#pragma unroll
    for (int kt = 0; kt < kTiles; kt++) {
      const int p = k0 + 16 * kt;
      const int page = p < t.len ? table[p >> c.page_log2] : -1;
      there[kt] = page >= 0 && page < c.pages;
      at[kt] = (((there[kt] ? page : 0) * (int64_t)c.kv_heads + h) << c.page_log2) +
               (p & ((1 << c.page_log2) - 1));
      const int8_t* kp = c.k + (at[kt] + r16) * kHd + 16 * g;
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const uint4 r = *reinterpret_cast<const uint4*>(kp + 64 * j);
        key[kt][2 * j] = codes8(r.x, r.y);
        key[kt][2 * j + 1] = codes8(r.z, r.w);
      }
      const v4f ks = *reinterpret_cast<const v4f_any*>(c.ks + at[kt] + 4 * g);
      const v4f vs = *reinterpret_cast<const v4f_any*>(c.vs + at[kt] + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const KeyTerms k =
            key_terms(ks[i], vs[i], there[kt] && p + 4 * g + i < t.len, 1.f, e0);
        kc[kt][i] = k.c, ke[kt][i] = k.e;
      }
    }
    v4f sum[kTiles];
#pragma unroll
    for (int kt = 0; kt < kTiles; kt++) sum[kt] = v4f{0.f, 0.f, 0.f, 0.f};

    // rows that see a key of the block: from the first one's place on
    const int64_t i0 = a.causal ? std::max<int64_t>(0, b * kBlock - t.first) : 0;
    const int64_t first = i0 * a.group / kRows * kRows;
    auto stage = [&](int64_t r0, Stage& d) {
      const int row = tid >> 3, j = tid & 7;
      const int64_t r = r0 + row;
      float v[16];
      float mx = 0.f;
      const bool ok = r < t.rows;
      const int64_t tok = (ok ? r : 0) / a.group;
      const int head = h * a.group + (int)((ok ? r : 0) - tok * a.group);
      const float* q = a.q + (t.row0 + tok) * a.ldq + (int64_t)head * kHd + 16 * j;
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const v4f f = *reinterpret_cast<const v4f*>(q + i);
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const bool fine = fabsf(f[k]) <= 3.402823466e38f;
          v[i + k] = ok && fine ? f[k] : 0.f;
          mx = fmaxf(mx, fabsf(v[i + k]));
        }
      }
#pragma unroll
      for (int o = 4; o; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
      const int e = q_exp(mx);
#pragma unroll
      for (int i = 0; i < 16; i++) v[i] = __builtin_ldexpf(v[i], e);
#pragma unroll
      for (int p = 0; p < 2; p++) {  // dims 16 j + 8 p ..: k slot 8 (j % 4) + i of step 2 (j / 4) + p
        v8h hi, lo;
        parts8(v + 8 * p, hi, lo);
        const int off = (16 * (j & 3) + (row & 15)) * 16;
        *reinterpret_cast<v8h*>(d.q[0][row >> 4][2 * (j >> 2) + p] + off) = hi;
        *reinterpret_cast<v8h*>(d.q[1][row >> 4][2 * (j >> 2) + p] + off) = lo;
      }
      if (j == 0) {
        const float2 st = ok ? a.stats[(t.row0 + tok) * a.heads + head] : float2{0.f, 0.f};
        d.row[row] = RowInfo{__builtin_ldexpf(a.scale2, -e), st.x, st.y,
                             st.y > 0.f ? keys_of(t, r, a.group, a.causal) : 0};
      }
    };
    __syncthreads();  // the last block's rows are read
    if (first < t.rows) stage(first, buf[0]);
    __syncthreads();
    int n = 0;
    for (int64_t r0 = first; r0 < t.rows; r0 += kRows, n ^= 1) {
      if (r0 + kRows < t.rows) stage(r0 + kRows, buf[n ^ 1]);
      const Stage& d = buf[n];
#pragma unroll
      for (int rt = 0; rt < kRows / 16; rt++) {
        const RowInfo ri = d.row[16 * rt + r16];
        if (!__any(ri.see > k0)) continue;
        v4f sc[kTiles];
#pragma unroll
        for (int kt = 0; kt < kTiles; kt++) sc[kt] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < 4; kb++) {
          const v8h lo = *reinterpret_cast<const v8h*>(d.q[1][rt][kb] + l * 16);
          const v8h hi = *reinterpret_cast<const v8h*>(d.q[0][rt][kb] + l * 16);
#pragma unroll
          for (int kt = 0; kt < kTiles; kt++) sc[kt] = mma(key[kt][kb], lo, sc[kt]);
#pragma unroll
          for (int kt = 0; kt < kTiles; kt++) sc[kt] = mma(key[kt][kb], hi, sc[kt]);
        }
        const bool all = __all(ri.see >= k0 + 16 * kTiles);
#pragma unroll
        for (int kt = 0; kt < kTiles; kt++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float x = __builtin_fmaf(sc[kt][i], kc[kt][i] * ri.qk, ke[kt][i]);
            const float e = __builtin_amdgcn_exp2f(x - ri.m - ke[kt][i]);
            if (all || k0 + 16 * kt + 4 * g + i < ri.see)
              sum[kt][i] = __builtin_fmaf(e, ri.inv, sum[kt][i]);
          }
      }
      __syncthreads();
    }
    // the 16 rows' sums of a key lie in 16 lanes; lane r16 then keeps key 4 g + r16 % 4 of tile r16 / 4
    float mine = 0.f;
    int64_t place = 0;
    bool ok = false;
#pragma unroll
    for (int kt = 0; kt < kTiles; kt++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float v = sum[kt][i];
#pragma unroll
        for (int o = 8; o; o >>= 1) v += __shfl_xor(v, o);
        if (r16 == 4 * kt + i) {
          mine = v;
          place = at[kt] + 4 * g + i;
          ok = there[kt];
        }
      }
    const int p = k0 + 16 * (r16 >> 2) + 4 * g + (r16 & 3);
    if (ok && p < t.len) sums[place] = p < t.first ? sums[place] + mine : mine;
  }
}

}  // namespace

hipError_t launch_kv_weights(const View& c, const KvRows& r, const float2* stats, float* w,
                             int cu_count, hipStream_t s) {
  Args a{};
  a.c = c;
  a.q = r.q, a.ldq = r.ldq;
  a.heads = r.heads, a.group = r.heads / c.kv_heads;
  a.scale2 = r.scale * 1.44269504088896341f;
  a.causal = r.causal;
  a.stats = const_cast<float2*>(stats);
  // Blocks of a sequence and head go round `across` workgroups.
  const int64_t pairs = (int64_t)c.nseq * c.kv_heads;
  const int64_t blocks = ceil_div(std::max<int64_t>(c.max_pages << c.page_log2, 1), kBlock);
  const int64_t across = std::min(blocks, ceil_div(8 * (int64_t)cu_count, pairs));
  // sequences at a time that a grid's 32-bit thread count takes
  const int per = (int)std::max<int64_t>(1, (int64_t(1) << 22) / (across * c.kv_heads));
  for (int s0 = 0; s0 < c.nseq; s0 += per) {
    View v = c;
    v.q_start += s0, v.lens += s0, v.table += s0 * c.max_pages;
    v.nseq = std::min(per, c.nseq - s0);
    a.c = v;
    hipLaunchKernelGGL(kv_weights_kernel, dim3((unsigned)(across * v.nseq * c.kv_heads)),
                       dim3(64 * kWaves), 0, s, a, w, (int)across);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace sdq
