// Eviction from the paged int8 cache by a weight for each token and head (gfx950).
//
// select: one workgroup a sequence and head. Every token gets a number whose order is the
// order of keeping (tokens that stay whatever their weight, then weights from the largest, NaN
// last, then places without a token); the keep-th largest number is found digit by digit (11,
// 11 and 10 bits, counted in LDS), and the tokens from it on are listed in order of their
// position, of those that equal it the first ones. A thread takes 16 tokens that lie side by
// side, a tile of one page, so that one scan over the workgroup numbers 16384 of them.
// move: 64 kept tokens a workgroup: codes of 128 bytes by 8 lanes, scales and weights.
#include <algorithm>

#include "sdq_device.h"
#include "sdq_kv.h"

#pragma clang fp contract(off)

namespace sdq {
namespace {

using kv::Kept;
using kv::kHd;
using kv::View;
using dev::v4f;
typedef v4f v4f_any __attribute__((aligned(4)));

constexpr int kThreads = 1024;
constexpr int kRun = 16;  // tokens of a thread: page_size is at least that

constexpr uint32_t kAlways = 0xffffffffu, kAbsent = 0u;
// Weights in order as numbers 2 .. 0xfffffffe - 1, zeros of either sign the same; NaN 1.
__device__ __forceinline__ uint32_t rank_of(float w) {
  if (!(w == w)) return 1u;
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;  // -inf is 0x007fffff, inf 0xff800000
}

// Tokens [p, p + 16) of a sequence as ranks, and how many of them hold a token.
__device__ __forceinline__ int load_ranks(const View& c, const float* w, const int32_t* table, int h,
                                          int64_t len, int64_t first, int64_t last, int64_t p,
                                          uint32_t r[kRun]) {
#pragma unroll
  for (int i = 0; i < kRun; i++) r[i] = kAbsent;
  if (p >= len) return 0;
  const int64_t page = table[p >> c.page_log2];
  if (page < 0 || page >= c.pages) return 0;
  const float* at =
      w + ((page * c.kv_heads + h) << c.page_log2) + (p & ((1 << c.page_log2) - 1));
#pragma unroll
  for (int i = 0; i < kRun; i += 4) {
    const v4f v = *reinterpret_cast<const v4f_any*>(at + i);
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int64_t q = p + i + k;
      if (q < len) r[i + k] = q < first || q >= last ? kAlways : rank_of(v[k]);
    }
  }
  return (int)(len - p < kRun ? len - p : kRun);
}

// Sum over the workgroup, the same in every thread.
__device__ __forceinline__ int64_t all_sum(int64_t v, int64_t* lds) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < kThreads / 64; i++) v += lds[i];
  return v;
}

__global__ void __launch_bounds__(kThreads) kv_select_kernel(View c, const float* __restrict__ w, Kept k) {
  __shared__ uint32_t hist[2048];
  __shared__ int64_t lds[kThreads / 64];
  __shared__ uint32_t found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = (int)(blockIdx.x % c.kv_heads), s = (int)(blockIdx.x / c.kv_heads);
  const int32_t* table = c.table + s * c.max_pages;
  const int64_t len = kv::length_of(c, s), last = len - k.last;
  int32_t* kept = k.kept + ((int64_t)s * c.kv_heads + h) * k.keep;
  uint32_t r[kRun];

  int64_t n = 0;
  for (int64_t p = (int64_t)tid * kRun; p < len; p += kThreads * kRun)
    n += load_ranks(c, w, table, h, len, k.first, last, p, r);
  const int64_t present = all_sum(n, lds);
  const int64_t keep = present < k.keep ? present : k.keep;
  if (h == 0 && tid == 0) k.lens[s] = (int32_t)keep;

  // the keep-th largest rank, and how many of its equals are kept
  uint32_t border = 1;      // all that hold a token
  int64_t equals = present;
  if (present > keep) {
    uint32_t prefix = 0, need = (uint32_t)keep;
    int shift = 32;
    for (int bits : {11, 11, 10}) {
      shift -= bits;
      for (int i = tid; i < 2048; i += kThreads) hist[i] = 0;
      __syncthreads();
      for (int64_t p = (int64_t)tid * kRun; p < len; p += kThreads * kRun) {
        load_ranks(c, w, table, h, len, k.first, last, p, r);
#pragma unroll
        for (int i = 0; i < kRun; i++)
          if (r[i] != kAbsent && (shift + bits == 32 || r[i] >> (shift + bits) == prefix))
            atomicAdd(&hist[(r[i] >> shift) & ((1u << bits) - 1)], 1u);
      }
      __syncthreads();
      if (wave == 0) {  // from the largest digit down: 32 of them a lane
        uint32_t sum = 0;
        for (int i = 0; i < 32; i++) sum += hist[2047 - (lane * 32 + i)];
        uint32_t upto = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const uint32_t v = __shfl_up(upto, o);
          if (lane >= o) upto += v;
        }
        uint32_t before = upto - sum;
        if (before < need && need <= upto) {
          int i = 0;
          while (before + hist[2047 - (lane * 32 + i)] < need) before += hist[2047 - (lane * 32 + i++)];
          found[0] = 2047 - (lane * 32 + i);
          found[1] = need - before;
        }
      }
      __syncthreads();
      prefix = prefix << bits | found[0];
      need = found[1];
      __syncthreads();
    }
    border = prefix;
    equals = need;
  }

  int64_t above0 = 0, equal0 = 0;  // before this round's tokens
  for (int64_t base = 0; base < len; base += kThreads * kRun) {
    load_ranks(c, w, table, h, len, k.first, last, base + (int64_t)tid * kRun, r);
    uint32_t above = 0, equal = 0;
#pragma unroll
    for (int i = 0; i < kRun; i++) {
      above += present > keep ? r[i] > border : 0;
      equal += present > keep ? r[i] == border : r[i] != kAbsent;
    }
    // both counts at once: a round has at most 2^14 of either
    uint32_t v = above | equal << 16, upto = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t u = __shfl_up(upto, o);
      if (lane >= o) upto += u;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = upto;
    __syncthreads();
    uint32_t ahead = 0, total = 0;
    for (int i = 0; i < kThreads / 64; i++) {
      const uint32_t u = (uint32_t)lds[i];
      ahead += i < wave ? u : 0;
      total += u;
    }
    ahead += upto - v;
    int64_t a = above0 + (ahead & 0xffff), e = equal0 + (ahead >> 16);
#pragma unroll
    for (int i = 0; i < kRun; i++) {
      const bool is_above = present > keep && r[i] > border;
      const bool is_equal = present > keep ? r[i] == border : r[i] != kAbsent;
      if (is_above || (is_equal && e < equals))
        kept[a + (e < equals ? e : equals)] = (int32_t)(base + (int64_t)tid * kRun + i);
      a += is_above;
      e += is_equal;
    }
    above0 += total & 0xffff;
    equal0 += total >> 16;
  }
  for (int64_t i = keep + tid; i < k.keep; i += kThreads) kept[i] = -1;
}

__global__ void __launch_bounds__(256) kv_move_kernel(View c, float* __restrict__ w, Kept k, int64_t items) {
  const int j = threadIdx.x & 7, row = threadIdx.x >> 3;
  const int64_t chunks = (k.keep + 63) / 64;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int h = (int)(item % c.kv_heads);
    const int64_t rest = item / c.kv_heads;
    const int64_t to0 = rest % chunks * 64;
    const int64_t s = rest / chunks;
    const int32_t* kept = k.kept + (s * c.kv_heads + h) * k.keep;
    uint4 kc[2], vc[2];
    float sc[2];
    int64_t at[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int64_t to = to0 + 32 * u + row;
      const int64_t from = to < k.keep ? kept[to] : -1;
      at[u] = -1;
      if (from < 0) continue;
      const int64_t page = k.table[s * k.max_pages + (to >> c.page_log2)];
      if (page < 0 || page >= c.pages) continue;
      const int64_t slot = (1 << c.page_log2) - 1;
      at[u] = ((page * c.kv_heads + h) << c.page_log2) + (to & slot);
      // kept tokens have a page
      const int64_t src = ((c.table[s * c.max_pages + (from >> c.page_log2)] * (int64_t)c.kv_heads + h)
                           << c.page_log2) + (from & slot);
      kc[u] = reinterpret_cast<const uint4*>(c.k + src * kHd)[j];
      vc[u] = reinterpret_cast<const uint4*>(c.v + src * kHd)[j];
      if (j < 3) sc[u] = (j == 0 ? c.ks : j == 1 ? c.vs : w)[src];
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
      if (at[u] < 0) continue;
      reinterpret_cast<uint4*>(c.k + at[u] * kHd)[j] = kc[u];
      reinterpret_cast<uint4*>(c.v + at[u] * kHd)[j] = vc[u];
      if (j < 3) (j == 0 ? c.ks : j == 1 ? c.vs : w)[at[u]] = sc[u];
    }
  }
}

}  // namespace

hipError_t launch_kv_evict(const View& c, float* w, const Kept& k, hipStream_t s) {
  // sequences at a time that a grid's 32-bit thread count takes
  const int per = (int)std::max<int64_t>(1, (int64_t(1) << 21) / c.kv_heads);
  for (int s0 = 0; s0 < c.nseq; s0 += per) {
    View v = c;
    v.lens += s0, v.table += s0 * c.max_pages;
    v.nseq = std::min(per, c.nseq - s0);
    Kept q = k;
    q.lens += s0, q.table += s0 * k.max_pages, q.kept += (int64_t)s0 * c.kv_heads * k.keep;
    hipLaunchKernelGGL(kv_select_kernel, dim3((unsigned)(v.nseq * c.kv_heads)), dim3(kThreads), 0, s,
                       v, w, q);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t items = ceil_div(k.keep, 64) * v.nseq * c.kv_heads;
    hipLaunchKernelGGL(kv_move_kernel, dim3((unsigned)std::min<int64_t>(items, 1 << 22)), dim3(256), 0,
                       s, v, w, q, items);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace sdq
