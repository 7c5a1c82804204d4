// Eviction from the paged int8 cache by a weight for each token and head (gfx950).
//
// select: one workgroup a sequence and head, for tables of up to 16384 tokens. Every token gets a number whose order is the
// order of keeping (tokens that stay whatever their weight, then weights from the largest, NaN
// last, then places without a token); the keep-th largest number is found digit by digit (11,
// 11 and 10 bits, counted in LDS), and the tokens from it on are listed in order of their
// position, of those that equal it the first ones. The tokens stay in registers, four that lie
// side by side to a load. Wider tables: chunks of whole times 16384 tokens, a workgroup each, and four
// launches (three that count a digit, one that lists), each of which reads the weights again.
// move: 32 kept rows of codes a workgroup, 8 lanes a row.
#include <algorithm>

#include "sdq_device.h"
#include "sdq_kv.h"
#include "sdq_kv_plan.h"

#pragma clang fp contract(off)

namespace sdq {
namespace {

using kv::Kept;
using kv::kHd;
using kv::View;
using dev::v4f;
typedef v4f v4f_any __attribute__((aligned(4)));

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kRun = 4;  // tokens of a thread that lie side by side
constexpr int kRound = kThreads * kRun;
static_assert(4 * kRound == kvplan::kEvictRegisters);

constexpr uint32_t kAlways = 0xffffffffu, kAbsent = 0u;
// Weights in order as numbers 2 .. 0xfffffffe - 1, zeros of either sign the same; NaN 1.
__device__ __forceinline__ uint32_t rank_of(float w) {
  if (!(w == w)) return 1u;
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;  // -inf is 0x007fffff, inf 0xff800000
}

// A sequence's and head's tokens.
struct Tokens {
  const float* w;  // of the head, from page 0 on
  const int32_t* table;
  int64_t pages;
  int page_log2, kv_heads;
  int len, first, last;

  // Tokens p .. p + 3 of N rounds (absent from `end` on) as ranks. No branch stands between the
  // loads: all pages first, then all weights, of the pool's first page where there is none.
  template <int N>
  __device__ __forceinline__ void load(int64_t p, int64_t end, uint32_t (&r)[N][kRun]) const {
    int page[N];
    v4f v[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int64_t q = p + j * kRound;
      page[j] = table[(q < end ? q : end - 1) >> page_log2];
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int64_t q = p + j * kRound;
      const bool there = q < end && page[j] >= 0 && page[j] < pages;
      if (!there) page[j] = -1;
      v[j] = *reinterpret_cast<const v4f_any*>(
          w + (((there ? page[j] : 0) * (int64_t)kv_heads) << page_log2) + (q & ((1 << page_log2) - 1)));
    }
#pragma unroll
    for (int j = 0; j < N; j++)
#pragma unroll
      for (int i = 0; i < kRun; i++) {
        const int64_t q = p + j * kRound + i;
        r[j][i] = page[j] < 0 || q >= len ? kAbsent : q < first || q >= last ? kAlways : rank_of(v[j][i]);
      }
  }
};

// Many weights have the same high digit, and lanes that count the same one wait for each other
// (131073 tokens' first launch: one copy of the counts 9.2 us, two 7.2, four 6.4).
constexpr int kCopies = 4;
struct Lds {
  __attribute__((aligned(16))) uint32_t hist[2048 * kCopies];  // [digit][lane % kCopies]
  uint32_t wave[kWaves];
  uint32_t rounds[4][kWaves];
  uint32_t found[3];
};

// The counts of 2 digits from `first` on, of all copies.
__device__ __forceinline__ uint2 counts_of(const Lds& s, int first) {
  uint32_t n[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int c = 0; c < kCopies; c++) n[i] += s.hist[(first + i) * kCopies + c];
  return uint2{n[0], n[1]};
}
__device__ __forceinline__ void clear_counts(Lds& s) {
#pragma unroll
  for (int c = 0; c < 2 * kCopies; c += 4)
    *reinterpret_cast<uint4*>(&s.hist[c * kThreads + 4 * threadIdx.x]) = uint4{0, 0, 0, 0};
}

// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ uint32_t scan(uint32_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t u = __shfl_up(v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// The digit that holds the need-th token from the largest down: the thread has the counts of
// digits 2047 - 2 * tid and one less. need: how many of its `count` tokens are meant; total: of
// all digits (no more than need: nothing is found).
struct Digit {
  uint32_t digit, need, count, total;
};
__device__ __forceinline__ Digit find_digit(uint32_t hi, uint32_t lo, uint32_t need, Lds& s) {
  const int tid = threadIdx.x, wave = tid >> 6;
  const uint32_t sum = scan(hi + lo);
  if ((tid & 63) == 63) s.wave[wave] = sum;
  __syncthreads();
  uint32_t before = sum - hi - lo, total = 0;
#pragma unroll
  for (int i = 0; i < kWaves; i++) {
    const uint32_t u = s.wave[i];
    before += i < wave ? u : 0;
    total += u;
  }
  if (before < need && need <= before + hi + lo) {
    const bool second = need > before + hi;
    s.found[0] = 2047 - 2 * tid - second;
    s.found[1] = need - before - (second ? hi : 0);
    s.found[2] = second ? lo : hi;
  }
  __syncthreads();
  return Digit{s.found[0], s.found[1], s.found[2], total};
}
// The thread's share of the round's counts (v: of the lane's tokens) before its own, and the
// round's.
__device__ __forceinline__ uint32_t before_me(uint32_t v, uint32_t& total, Lds& s) {
  const int wave = threadIdx.x >> 6;
  const uint32_t sum = scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s.wave[wave] = sum;
  __syncthreads();
  uint32_t before = sum - v;
  total = 0;
#pragma unroll
  for (int i = 0; i < kWaves; i++) {
    const uint32_t u = s.wave[i];
    before += i < wave ? u : 0;
    total += u;
  }
  return before;
}

// What is kept: ranks above the border, and the first `equals` of those on it.
struct Border {
  uint32_t border, equals;
  // Both counts of four tokens in one word.
  __device__ __forceinline__ uint32_t count(const uint32_t (&x)[kRun]) const {
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < kRun; i++) v += (x[i] > border) | (x[i] == border && border) << 16;
    return v;
  }
  // Four tokens from p on, behind a above the border and e on it.
  __device__ __forceinline__ void put(int32_t* kept, int p, const uint32_t (&x)[kRun], uint32_t a,
                                      uint32_t e) const {
#pragma unroll
    for (int i = 0; i < kRun; i++) {
      const bool above = x[i] > border, on = x[i] == border && border;
      if (above || (on && e < equals)) kept[a + (e < equals ? e : equals)] = p + i;
      a += above;
      e += on;
    }
  }
};

// Lists tokens p .. p + 3 of N rounds, behind a above the border and e on it, and counts on.
template <int N>
__device__ __forceinline__ void list(Border b, const uint32_t (&r)[N][kRun], int p, uint32_t& a,
                                     uint32_t& e, int32_t* kept, Lds& s) {
  const int wave = threadIdx.x >> 6;
  uint32_t upto[N];
#pragma unroll
  for (int j = 0; j < N; j++) {
    upto[j] = scan(b.count(r[j]));
    if ((threadIdx.x & 63) == 63) s.rounds[j][wave] = upto[j];
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < N; j++) {
    // Compared again: the masks of all rounds kept from above are more than the scalar registers.
    asm volatile("" : "+v"(b.border));
    // the counts of a round are at most 4096 each: no carry
    uint32_t v = upto[j] - b.count(r[j]), total = 0;
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
      const uint32_t u = s.rounds[j][i];
      v += i < wave ? u : 0;
      total += u;
    }
    b.put(kept, p + j * kRound, r[j], a + (v & 0xffff), e + (v >> 16));
    a += total & 0xffff;
    e += total >> 16;
  }
}

template <int N>
__device__ __forceinline__ void count_digits(const uint32_t (&r)[N][kRun], int shift, int bits,
                                             uint32_t prefix, Lds& s) {
  const int copy = threadIdx.x % kCopies;
#pragma unroll
  for (int j = 0; j < N; j++)
#pragma unroll
    for (int i = 0; i < kRun; i++)
      if (r[j][i] != kAbsent && (shift == 21 || r[j][i] >> (shift + bits) == prefix))
        atomicAdd(&s.hist[((r[j][i] >> shift) & ((1u << bits) - 1)) * kCopies + copy], 1u);
}

// A sequence of up to N rounds, in registers.
template <int N>
__device__ __forceinline__ void select(const Tokens& t, int64_t most, int32_t* kept, int32_t* len,
                                       Lds& s) {
  const int tid = threadIdx.x;
  uint32_t r[N][kRun];
  t.load<N>(tid * kRun, t.len, r);
  // The border's digits from the highest; as soon as a digit's tokens are all kept the rest
  // does not matter.
  Border b{0, 0};
  uint32_t keep = (uint32_t)most, need = keep, prefix = 0;
  int shift = 32;
#pragma unroll 1
  for (int level = 0; level < 3; level++) {
    const int bits = level < 2 ? 11 : 10;
    shift -= bits;
    clear_counts(s);
    __syncthreads();
    count_digits<N>(r, shift, bits, prefix, s);
    __syncthreads();
    const uint2 n = counts_of(s, 2046 - 2 * tid);
    const Digit d = find_digit(n.y, n.x, need, s);
    if (shift == 21 && d.total <= keep) {  // all that hold a token
      keep = d.total;
      break;
    }
    prefix = prefix << bits | d.digit;
    need = d.need;
    b = Border{prefix << shift, need};
    if (d.count == need) {
      b = Border{(prefix << shift) - 1, 0};
      break;
    }
  }
  if (len && tid == 0) *len = (int32_t)keep;

  uint32_t a = 0, e = 0;
  list<N>(b, r, tid * kRun, a, e, kept, s);
  for (int64_t i = keep + tid; i < most; i += kThreads) kept[i] = -1;
}

__device__ __forceinline__ Tokens tokens_of(const View& c, const float* w, const Kept& k, int s, int h) {
  const int len = (int)kv::length_of(c, s);
  const int64_t last = len - k.last;
  return Tokens{w + ((int64_t)h << c.page_log2), c.table + s * c.max_pages, c.pages, c.page_log2,
                c.kv_heads, len, (int)k.first, (int)(last < 0 ? 0 : last)};
}

__global__ void __launch_bounds__(kThreads) kv_select_kernel(View c, const float* __restrict__ w, Kept k) {
  __shared__ Lds lds;
  const int h = (int)(blockIdx.x % c.kv_heads), s = (int)(blockIdx.x / c.kv_heads);
  const Tokens t = tokens_of(c, w, k, s, h);
  int32_t* kept = k.kept + ((int64_t)s * c.kv_heads + h) * k.keep;
  int32_t* to = h == 0 ? k.lens + s : nullptr;
  if (t.len == 0) {
    if (to && threadIdx.x == 0) *to = 0;
    for (int64_t i = threadIdx.x; i < k.keep; i += kThreads) kept[i] = -1;
  } else if (t.len <= kRound)
    select<1>(t, k.keep, kept, to, lds);
  else
    select<4>(t, k.keep, kept, to, lds);
}

// ---- sequences that may be longer: their tokens in chunks, a workgroup each ----
//
// Launch `level` counts the chunks' tokens by digit `level` below the digits that are known by
// then, which every workgroup of a sequence and head finds from all chunks' counts of the
// launch before; the fourth launch lists. What a chunk has to list before its own is in the
// counts of those ahead of it.
struct Found {
  uint32_t prefix, need, keep;
  uint32_t digit[3];
  int levels;  // digits that matter
  int done;    // 1: all of the last digit's tokens are kept, 2: all tokens are
};
static_assert(3 * sizeof(Found) == kvplan::kEvictFound);
struct Long {
  uint32_t* hist;  // [pair][chunk][level][2048]
  Found* found;    // [pair][level]
  int chunks;      // a pair has at most
  int64_t chunk;   // tokens, whole times 4 rounds
};

template <int level>
__global__ void __launch_bounds__(kThreads)
kv_select_long_kernel(View c, const float* __restrict__ w, Kept k, Long g) {
  __shared__ Lds lds;
  const int tid = threadIdx.x;
  const int chunk = (int)(blockIdx.x % g.chunks);
  const int64_t pair = blockIdx.x / g.chunks;
  const int h = (int)(pair % c.kv_heads), s = (int)(pair / c.kv_heads);
  const Tokens t = tokens_of(c, w, k, s, h);
  const int64_t begin = chunk * g.chunk;
  const int chunks = (int)((t.len + g.chunk - 1) / g.chunk);
  if (chunk > 0 && begin >= t.len) return;
  auto hist = [&](int64_t ch, int lv) { return g.hist + ((pair * g.chunks + ch) * 3 + lv) * 2048; };
  auto bits = [](int lv) { return lv < 2 ? 11 : 10; };
  auto shift = [](int lv) { return lv == 0 ? 21 : lv == 1 ? 10 : 0; };

  Found f{0, (uint32_t)k.keep, (uint32_t)k.keep, {0, 0, 0}, 0, 0};
  if (level > 0) {
    if constexpr (level > 1) f = g.found[pair * 3 + level - 2];
    if (!f.done) {
      const int lv = level - 1;
      uint32_t hi = 0, lo = 0;
#pragma unroll 8
      for (int ch = 0; ch < chunks; ch++) {
        const uint2 u = *reinterpret_cast<const uint2*>(hist(ch, lv) + 2046 - 2 * tid);
        lo += u.x;
        hi += u.y;
      }
      const Digit d = find_digit(hi, lo, f.need, lds);
      f.levels = level;
      if (lv == 0 && d.total <= f.keep) {
        f.keep = d.total;
        f.done = 2;
      } else {
        f.digit[lv] = d.digit;
        f.prefix = f.prefix << bits(lv) | d.digit;
        f.need = d.need;
        f.done = d.count == d.need;
      }
    }
    if constexpr (level < 3)
      if (chunk == 0 && tid == 0) g.found[pair * 3 + level - 1] = f;
  }
  const int64_t end = begin + g.chunk < t.len ? begin + g.chunk : t.len;
  if constexpr (level < 3) {
    if (f.done) return;
    clear_counts(lds);
    __syncthreads();
    for (int64_t p = begin + tid * kRun; p < end; p += 4 * kRound) {
      uint32_t r[4][kRun];
      t.load<4>(p, end, r);
      count_digits<4>(r, shift(level), bits(level), f.prefix, lds);
    }
    __syncthreads();
    *reinterpret_cast<uint2*>(hist(chunk, level) + 2 * tid) = counts_of(lds, 2 * tid);
    return;
  }

  const int last = f.levels - 1;
  const uint32_t edge = f.prefix << shift(last);
  const Border b = f.done == 2 ? Border{0, 0} : f.done ? Border{edge - 1, 0} : Border{edge, f.need};
  // what the chunks ahead list: tokens of higher digits, and of the last one where all are kept
  uint32_t a = 0, e = 0;
#pragma unroll 1
  for (int lv = 0; lv < f.levels; lv++) {
    const uint32_t at = lv == 0 ? f.digit[0] : lv == 1 ? f.digit[1] : f.digit[2];
#pragma unroll 4
    for (int ch = 0; ch < chunk; ch++) {
      const uint2 u = *reinterpret_cast<const uint2*>(hist(ch, lv) + 2 * tid);
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const uint32_t digit = 2 * tid + i, n = i ? u.y : u.x;
        a += f.done == 2 || digit > at || (f.done && lv == last && digit == at) ? n : 0;
        e += !f.done && lv == last && digit == at ? n : 0;
      }
    }
  }
  uint32_t all_a, all_e;
  before_me(a, all_a, lds);
  before_me(e, all_e, lds);
  int32_t* kept = k.kept + pair * k.keep;
  a = all_a, e = all_e;
  for (int64_t base = begin; base < end; base += 4 * kRound) {
    uint32_t r[4][kRun];
    const int64_t p = base + tid * kRun;
    t.load<4>(p, end, r);
    __syncthreads();  // the last rounds' counts are read
    list<4>(b, r, (int)p, a, e, kept, lds);
  }
  if (chunk == 0) {
    if (h == 0 && tid == 0) k.lens[s] = (int32_t)f.keep;
    for (int64_t i = f.keep + tid; i < k.keep; i += kThreads) kept[i] = -1;
  }
}

// Rows of codes: workgroups of (32 kept rows, keys or values, head, sequence); the scales and
// weights go with them.
__global__ void __launch_bounds__(256) kv_move_kernel(View c, float* __restrict__ w, Kept k, int64_t items) {
  const int j = threadIdx.x & 7, row = threadIdx.x >> 3;
  const int64_t chunks = (k.keep + 31) / 32;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const bool value = item & 1;
    const int h = (int)((item >> 1) % c.kv_heads);
    const int64_t rest = (item >> 1) / c.kv_heads, s = rest / chunks;
    const int64_t to = (rest - s * chunks) * 32 + row;
    if (to >= k.keep) continue;
    const int64_t from = k.kept[(s * c.kv_heads + h) * k.keep + to];
    const int64_t page = k.table[s * k.max_pages + (to >> c.page_log2)];
    if (from < 0 || page < 0 || page >= c.pages) continue;
    const int64_t slot = (1 << c.page_log2) - 1;
    const int64_t at = ((page * c.kv_heads + h) << c.page_log2) + (to & slot);
    // kept tokens have a page
    const int64_t src = ((c.table[s * c.max_pages + (from >> c.page_log2)] * (int64_t)c.kv_heads + h)
                         << c.page_log2) + (from & slot);
    int8_t* codes = value ? c.v : c.k;
    float* scales = value ? c.vs : c.ks;
    const uint4 x = reinterpret_cast<const uint4*>(codes + src * kHd)[j];
    const float sc = j == 0 ? scales[src] : j == 1 && !value ? w[src] : 0.f;
    reinterpret_cast<uint4*>(codes + at * kHd)[j] = x;
    if (j == 0) scales[at] = sc;
    if (j == 1 && !value) w[at] = sc;
  }
}

}  // namespace

hipError_t launch_kv_evict(const View& c, float* w, const Kept& k, const kvplan::EvictPlan& p, void* scratch,
                           hipStream_t s) {
  for (int s0 = 0; s0 < c.nseq; s0 += p.seqs) {
    View v = c;
    v.lens += s0, v.table += s0 * c.max_pages;
    v.nseq = std::min(p.seqs, c.nseq - s0);
    Kept q = k;
    q.lens += s0, q.table += s0 * k.max_pages, q.kept += (int64_t)s0 * c.kv_heads * k.keep;
    const unsigned pairs = (unsigned)(v.nseq * c.kv_heads);
    hipError_t e;
    if (p.chunks) {
      uint32_t* hist = static_cast<uint32_t*>(scratch);
      const Long g{hist, reinterpret_cast<Found*>(hist + (int64_t)pairs * p.chunks * 3 * 2048), p.chunks,
                   p.chunk};
      for (auto kernel : {kv_select_long_kernel<0>, kv_select_long_kernel<1>, kv_select_long_kernel<2>,
                          kv_select_long_kernel<3>}) {
        hipLaunchKernelGGL(kernel, dim3(pairs * p.chunks), dim3(kThreads), 0, s, v, w, q, g);
        if ((e = hipGetLastError()) != hipSuccess) return e;
      }
    } else {
      hipLaunchKernelGGL(kv_select_kernel, dim3(pairs), dim3(kThreads), 0, s, v, w, q);
      if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    const int64_t items = 2 * ceil_div(k.keep, 32) * pairs;
    hipLaunchKernelGGL(kv_move_kernel, dim3((unsigned)std::min<int64_t>(items, 1 << 22)), dim3(256), 0,
                       s, v, w, q, items);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace sdq
