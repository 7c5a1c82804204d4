// Attention of new tokens over the paged int8 cache (gfx950).
//
// Per row (token i at position p, head h), over the keys j that it sees, with
// s_j = scale log2(e) q . k_j:   out = sum_j 2^s_j v_j / sum_j 2^s_j.
//
// Numbers. A cached value is code * scale; the codes are exact in fp16, so each
// fp32 product costs two fp16 MFMA products: q = (hi + lo) 2^-r, r a power of two
// for each row that puts its largest element into [2^14, 2^15), and the softmax
// weight = hi + lo below. Both parts are rounded: hi + lo is off by at most 2^-22
// of the value, or half of fp16's smallest step, an absolute 2^-39 of the row's largest
// element and 2^-34 of its largest weight. (Truncated parts lost up to 1.4e-4 where 2^17 equal
// light keys stand beside a heavy one, of values of 2.5; now 1.7e-5. A reference that
// rises by 2^2 instead of 2^6, the weights 2^4 further from the smallest step: 0.9e-5, and
// 2% slower for 768 tokens.) The key's scale multiplies the finished sum. The value's scale is v_j = f_j 2^(e_j + E0), f_j in
// [1/2, 1), E0 the exponent of the sequence's first value, at least -16: its exponent
// goes into the softmax,
//   t_j = s_j + e_j,  X_j = 2^(t_j - m), m near the running maximum of t,
//   out = 2^E0 sum_j X_j f_j code_j / sum_j X_j 2^-e_j,
// one exponential a key as before, and the weights that are split into parts
// are those that count: no value is lost beside another, however far apart the
// scales of heavy and light keys are. e_j is held to -60 .. 60 (2^-e_j and the sums have to
// be floats); a value under that counts with fewer bits, one over it makes its rows NaN.
// X_j can lie under the smallest float where X_j 2^-e_j, at most 2^(60 + 60) larger, is
// still most of the denominator: such terms are formed apart (add_faint, times_exp2).
//
// Scores are computed transposed, S^T = K Q^T (16x16x32): a lane then holds one
// query's scores for keys 4 g + 0..3 (g = lane / 16) of two 16-key tiles, which
// is the B operand of out^T = V^T P^T with no exchange between lanes, where the
// eight k slots of lane group g stand for keys 4 g .. 4 g + 3 of either tile.
// Dims: k slot 8 g + i of step kb is dim 64 (kb / 2) + 16 g + 8 (kb % 2) + i (16
// bytes of a cached row a lane), and row c of V's tile e is dim 8 c + e (8
// bytes), so that lane group g ends with dims 32 g .. 32 g + 31 of its query.
#include <algorithm>

#include "sdq_device.h"
#include "sdq_kv.h"
#include "sdq_kv_plan.h"

#pragma clang fp contract(off)

namespace sdq {
namespace {

using kv::kHd;
using kv::View;
using dev::v4f;
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// Four scales as they lie in the cache, whose scales need no more than a float's alignment.
typedef v4f v4f_any __attribute__((aligned(4)));

constexpr int kTop = 15;      // largest q of a row below 2^kTop
constexpr int kSlack = 6;     // X stays below 2^kSlack
constexpr int kWeight = 9;    // weights X f enter as X f 2^kWeight, below 2^15
constexpr int kFar = 60;      // e_j is held to -kFar .. kFar
constexpr int kLeast = -16;   // of E0
// A key with e >= kNear whose X is under 2^-126 is less than 2^(-126 - kNear) of a
// denominator that holds at least 2^-kFar: 2^30 of them less than 2^-26 of it.
constexpr float kNear = -10.f;

struct Args {
  View c;
  const float* q;
  int64_t ldq;
  float* out;
  int64_t ldo;
  int heads, group;  // query heads, query heads per cached head
  float scale2;      // scale * log2(e)
  int causal;
  int splits;
  int64_t tile0;     // first tile of this launch
  float* part;       // [tile][kv head][split][row][128], unscaled sums
  float2* part_ml;   // the same without dims: maximum, denominator
};

// A tile of rows: rows [r0, r0 + RT) of sequence s, row r = token r / group,
// query head r % group of the tile's cached head.
struct Tile {
  int s;          // -1: none
  int64_t r0;
  int64_t rows;   // of the sequence
  int64_t row0;   // the sequence's first row in q
  int len;        // keys, at most 2^30
  int first;      // position of the sequence's first row
};

// A lane's value that is the same in the whole wave, as a scalar.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Tile number `tile`. Sequence s, whose rows start at row a and end before row b of all
// (row: a token's head of the group), has the numbers from a / RT + s to b / RT + s, at
// least as many as it has tiles of RT rows: a number without a tile is none. So the
// sequence is found by search, 64 ways at a time, with no sum over those before it
// (a scan over them took a fifth of a microsecond for each 64). The same in every wave.
template <int RT>
__device__ __forceinline__ Tile find_tile(const View& c, int group, int64_t tile) {
  const int l = threadIdx.x & 63;
  Tile t{-1, 0, 0, 0, 0, 0};
  auto first = [&](int s) { return kv::row_of(c, s) * group / RT + s; };
  int lo = 0, n = c.nseq, step;
  do {
    step = (n + 63) / 64;
    const uint64_t upto = __ballot((int64_t)l * step < n && first(min(lo + l * step, c.nseq)) <= tile);
    if (!upto) return t;
    const int k = 63 - __builtin_clzll(upto);
    lo += k * step;
    n = min(step, n - k * step);
  } while (step > 1);
  lo = uniform(lo);
  t.row0 = kv::row_of(c, lo);
  const int64_t tokens = kv::row_of(c, lo + 1) - t.row0;
  t.r0 = (tile - first(lo)) * RT;
  t.rows = tokens > 0 ? tokens * group : 0;
  t.len = (int)kv::length_of(c, lo);
  t.first = t.len - (int)(tokens > 0 ? tokens : 0);
  if (t.r0 < t.rows) t.s = lo;
  return t;
}

// Keys that row r sees (0: it has no position, or is none).
__device__ __forceinline__ int keys_of(const Tile& t, int64_t r, int group, int causal) {
  if (r >= t.rows) return 0;
  const int p = t.first + (int)(r / group);
  return p < 0 ? 0 : causal ? (p + 1 < t.len ? p + 1 : t.len) : t.len;
}
// And the rows [r, r + n) at most: the last one.
__device__ __forceinline__ int keys_of_rows(const Tile& t, int64_t r, int n, int group,
                                            int causal) {
  return keys_of(t, (r + n < t.rows ? r + n : t.rows) - 1, group, causal);
}

__device__ __forceinline__ v4f mma(v8h a, v8h b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Eight codes (two dwords) as fp16: 0x6400 | u is 1024 + u, with u = code + 128.
__device__ __forceinline__ v2h less1152(uint32_t x) {
  return __builtin_bit_cast(v2h, x) + v2h{(_Float16)-1152.f, (_Float16)-1152.f};
}
__device__ __forceinline__ v8h codes8(uint32_t a, uint32_t b) {
  a ^= 0x80808080u;
  b ^= 0x80808080u;
  const v2h x = less1152(__builtin_amdgcn_perm(0x64646464u, a, 0x04010400u));
  const v2h y = less1152(__builtin_amdgcn_perm(0x64646464u, a, 0x04030402u));
  const v2h z = less1152(__builtin_amdgcn_perm(0x64646464u, b, 0x04010400u));
  const v2h w = less1152(__builtin_amdgcn_perm(0x64646464u, b, 0x04030402u));
  return v8h{x[0], x[1], y[0], y[1], z[0], z[1], w[0], w[1]};
}
// Byte I of two dwords (codes xor 0x80) as a pair of fp16.
template <int I>
__device__ __forceinline__ v2h pair_of(uint32_t a, uint32_t b) {
  constexpr uint32_t sel = 0x0c000c00u | (uint32_t)I | ((uint32_t)(I + 4) << 16);
  return less1152(__builtin_amdgcn_perm(b, a, sel) | 0x64006400u);
}

// Over the four lanes l, l ^ 16, l ^ 32, l ^ 48 of a query, by swaps of lane rows.
template <class F>
__device__ __forceinline__ float quad(float v, F f) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float quad_max(float v) {
  return quad(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float quad_sum(float v) {
  return quad(v, [](float a, float b) { return a + b; });
}

// x - hi of either half of a pair of fp16, exact, in one operation.
__device__ __forceinline__ float less_low(v2h hi, float x) {
  float r;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(hi), "v"(x));
  return r;
}
__device__ __forceinline__ float less_high(v2h hi, float x) {
  float r;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
      : "=v"(r)
      : "v"(hi), "v"(x));
  return r;
}
// fp32 to two fp16 parts, both rounded (two conversions at a time): the high
// part's remainder is exact, so the pair is off by at most 2^-22.
__device__ __forceinline__ v2h rounded(float a, float b) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  return __builtin_convertvector((v2f{a, b}), v2h);
}
__device__ __forceinline__ void parts8(const float x[8], v8h& hi, v8h& lo) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const v2h h = rounded(x[i], x[i + 1]);
    const v2h r = rounded(less_low(h, x[i]), less_high(h, x[i + 1]));
    hi[i] = h[0];
    hi[i + 1] = h[1];
    lo[i] = r[0];
    lo[i + 1] = r[1];
  }
}

// The lane's slice of a query row (head of a token), zeros where it is none.
__device__ __forceinline__ void load_q(const Args& a, const Tile& t, int h, int64_t r, int g,
                                       float x[4][8]) {
  const bool ok = r < t.rows;
  const int64_t rr = ok ? r : 0;
  const int64_t tok = rr / a.group;
  const float* p =
      a.q + (t.row0 + tok) * a.ldq + (int64_t)(h * a.group + (int)(rr - tok * a.group)) * kHd;
#pragma unroll
  for (int kb = 0; kb < 4; kb++)
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const float4 v =
          ok ? *reinterpret_cast<const float4*>(p + 64 * (kb >> 1) + 16 * g + 8 * (kb & 1) + 4 * j)
             : make_float4(0.f, 0.f, 0.f, 0.f);
      x[kb][4 * j] = v.x;
      x[kb][4 * j + 1] = v.y;
      x[kb][4 * j + 2] = v.z;
      x[kb][4 * j + 3] = v.w;
    }
}
// The largest magnitude of a row's slice. NaN and infinities become zeros, and the row (of
// four lanes) is `bad`: its denominator is NaN once it has seen a key, and 0 before.
__device__ __forceinline__ float clean(float x[4][8], bool& bad) {
  float m = 0.f, b = 0.f;
#pragma unroll
  for (int kb = 0; kb < 4; kb++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const bool fine = fabsf(x[kb][i]) <= 3.402823466e38f;
      x[kb][i] = fine ? x[kb][i] : 0.f;
      b = fine ? b : 1.f;
      m = fmaxf(m, fabsf(x[kb][i]));
    }
  bad = quad_max(b) != 0.f;
  return quad_max(m);
}
__device__ __forceinline__ float den_of(float l, bool bad) {
  const float den = quad_sum(l);
  return bad && den != 0.f ? __builtin_nanf("") : den;
}
// Exponent that scales a row's largest |q| below 2^kTop; within what a float's power
// of two can hold. Each row has its own: one of the same tile that holds something
// huge takes no bits from it.
__device__ __forceinline__ int q_exp(float m) {
  const int e = m > 0.f ? kTop - __builtin_amdgcn_frexp_expf(m) : 0;
  return e > 100 ? 100 : e;
}

// What a key contributes: c (score to log2 units), e, 2^-e and f 2^kWeight. One
// that is not there (masked, no page) gives zeros, so that whatever its memory
// holds stays out.
struct KeyTerms {
  float c, e, w, f;
};
__device__ __forceinline__ KeyTerms key_terms(float ks, float vs, bool ok, float qk, int e0) {
  const float top = __builtin_ldexpf(1.f, kFar + e0);  // inf: every finite scale fits
  KeyTerms k;
  int e = vs != 0.f ? __builtin_amdgcn_frexp_expf(vs) - e0 : 0;
  e = e < -kFar ? -kFar : e > kFar ? kFar : e;
  k.c = ok ? ks * qk : 0.f;
  k.e = ok ? (float)e : 0.f;
  k.w = ok ? __builtin_ldexpf(1.f, -e) : 0.f;
  // past kFar the weights would not fit fp16, and the conversion would cut them off
  k.f = !ok ? 0.f : fabsf(vs) >= top ? __builtin_nanf("") : __builtin_ldexpf(vs, kWeight - e - e0);
  return k;
}
// E0: the exponent of the sequence's first value scale; from kLeast on, so that a
// first value of next to nothing leaves those after it their range.
__device__ __forceinline__ int first_exp(const View& c, const Tile& t, int h) {
  if (t.len <= 0) return 0;
  const int64_t at = kv::place_of(c, t.s, 0, h);
  const float v = at >= 0 ? c.vs[at] : 0.f;
  const int e = v != 0.f ? __builtin_amdgcn_frexp_expf(v) : 0;
  return e < kLeast ? kLeast : e;
}

// One query's softmax state in a lane: the reference m (the maximum of t, or up
// to kSlack below it; -inf: no key yet) is the same in the query's four lanes,
// the denominator is the lane's own share.
struct State {
  float m, l;
};

// A 32-key block's logits of one query tile, in place of its scores (tiles kt,
// elements i: key 16 kt + 4 g + i), and their largest. seen(kt, i): the row sees
// that key.
template <bool MASK, class Seen>
__device__ __forceinline__ float logits(v4f s[2], const v4f c[2], const v4f e[2], Seen seen) {
  float mx = -INFINITY;
#pragma unroll
  for (int kt = 0; kt < 2; kt++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float v = __builtin_fmaf(s[kt][i], c[kt][i], e[kt][i]);
      if (MASK && !seen(kt, i)) v = -INFINITY;
      s[kt][i] = v;
      mx = fmaxf(mx, v);
    }
  return quad_max(mx);
}
// Logits to the two parts of the weights.
template <bool MASK, class Seen>
__device__ __forceinline__ void weights(const v4f t[2], const v4f w[2], const v4f f[2], State& st,
                                        Seen seen, v8h& hi, v8h& lo) {
  const float ref = st.m == -INFINITY ? 0.f : st.m;
  float p[8], l = 0.f;  // the block's share first: an eighth of the roundings of a long sum
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float x = __builtin_amdgcn_exp2f(t[j >> 2][j & 3] - ref);
    l = __builtin_fmaf(x, w[j >> 2][j & 3], l);
    p[j] = x * f[j >> 2][j & 3];
    if (MASK && !seen(j >> 2, j & 3)) p[j] = 0.f;  // its scale may be NaN
  }
  st.l += l;
  parts8(p, hi, lo);
}
// a 2^d, also where 2^d alone is under the smallest float (exp2 gives 0 there).
__device__ __forceinline__ float times_exp2(float a, float d) {
  const float h = __builtin_amdgcn_exp2f(0.5f * d);
  return a * h * h;
}
// The denominator's terms 2^(t - m - e) of keys whose X is under the smallest float (what
// is 2^-1000 is nothing, masked keys among it); their X is 0 from here on. Called
// where a block has a key with e < kNear.
__device__ __forceinline__ void add_faint(v4f t[2], const v4f e[2], State& st) {
  const float ref = st.m == -INFINITY ? 0.f : st.m;
  float l = 0.f;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float x = t[j >> 2][j & 3] - ref;
    const bool faint = x < -126.f && x > -1000.f;
    l += __builtin_amdgcn_exp2f(faint ? x - e[j >> 2][j & 3] : -INFINITY);
    t[j >> 2][j & 3] = faint ? -INFINITY : t[j >> 2][j & 3];
  }
  st.l += l;
}
// The reference rises only when a block's largest logit passes it by more than
// kSlack (the weights then stay below 2^kSlack, inside fp16 with kWeight):
// rarely. The branch is the wave's, the rise each row's own, so that no row's bits
// depend on its neighbours.
__device__ __forceinline__ bool rises(const State& st, float mx) { return mx > st.m + kSlack; }
__device__ __forceinline__ void raise(State& st, float mx, v4f acc[8]) {
  const float m = rises(st, mx) ? mx : st.m;
  const float d = m == -INFINITY ? 0.f : st.m - m;
  const float shrink = __builtin_amdgcn_exp2f(d);
  st.m = m;
  st.l = times_exp2(st.l, d);
#pragma unroll
  for (int e = 0; e < 8; e++) acc[e] = acc[e] * shrink;
}

// ---- few rows: a tile of 16, the workgroup's waves share out the keys ----
//
// Bound by the cache's bytes, 264 a key and cached head, each read once by the wave
// that uses it, straight into the MFMA operands' lanes, a block of 32 keys ahead: 1
// token x 262145 keys, 8 cached heads, 111 us, 5.0 TB/s, the rate of a large copy.
// 8 tokens of ragged sequences up to 4099 keys, 24 heads: 34 us, 3.4 TB/s; there a wave
// has eight blocks at most, and every sequence has the same number of shares: the longest
// has shares of 1025 keys, where the mean is 652. Two tiles read their keys twice (8
// sequences of up to 24 rows 45 us).

constexpr int kFewRows = kvplan::kFewRows;
constexpr int kFewWaves = kvplan::kFewWaves;
constexpr int kFewStride = kHd + 4;  // LDS row of a merged sum (bank spread)

__global__ void __launch_bounds__(64 * kFewWaves, 2) kv_attn_few_kernel(Args a) {
  const View& c = a.c;
  const int w = uniform((int)threadIdx.x >> 6), l = threadIdx.x & 63, r16 = l & 15, g = l >> 4;
  const int z = (int)(blockIdx.x % a.splits);
  const int64_t th = blockIdx.x / a.splits;
  const int h = (int)(th % c.kv_heads);
  const int64_t tile = a.tile0 + th / c.kv_heads;
  const Tile t = find_tile<kFewRows>(c, a.group, tile);
  if (t.s < 0) return;

  float x[4][8];
  load_q(a, t, h, t.r0 + r16, g, x);
  bool bad;
  const int qe = q_exp(clean(x, bad));
  v8h qh[4], ql[4];
#pragma unroll
  for (int kb = 0; kb < 4; kb++) {
#pragma unroll
    for (int i = 0; i < 8; i++) x[kb][i] = __builtin_ldexpf(x[kb][i], qe);
    parts8(x[kb], qh[kb], ql[kb]);
  }
  const float qk = __builtin_ldexpf(a.scale2, -qe);
  const int e0 = first_exp(c, t, h);

  const int keys = keys_of_rows(t, t.r0, kFewRows, a.group, a.causal);
  const int blocks = (keys + 31) / 32;
  const int b0 = (int)((int64_t)blocks * z / a.splits);
  const int b1 = (int)((int64_t)blocks * (z + 1) / a.splits);
  // what this lane's row sees, and what every row of the tile does
  const int mine = keys_of(t, t.r0 + r16, a.group, a.causal);
  const int all = keys_of(t, t.r0, a.group, a.causal);  // the first row

  State st{-INFINITY, 0.f};
  v4f acc[8];
#pragma unroll
  for (int e = 0; e < 8; e++) acc[e] = v4f{0.f, 0.f, 0.f, 0.f};

  // A block's codes and scales, loaded one block ahead, its pages another one.
  struct Raw {
    uint4 k[2][2];
    uint2 v[2][4];
    v4f ks[2], vs[2];
    bool there[2];
  };
  const int32_t* table = c.table + t.s * c.max_pages;
  auto page_at = [&](int b, int kt) {
    const int p = b * 32 + 16 * kt;
    return b < b1 && p < keys ? table[p >> c.page_log2] : -1;
  };
  auto load = [&](int b, const int pages[2], Raw& r) {
#pragma unroll
    for (int kt = 0; kt < 2; kt++) {
      const int p = b * 32 + 16 * kt;
      r.there[kt] = pages[kt] >= 0 && pages[kt] < c.pages;
      const int64_t at = (((r.there[kt] ? pages[kt] : 0) * (int64_t)c.kv_heads + h)
                          << c.page_log2) + (p & ((1 << c.page_log2) - 1));
      const int8_t* kp = c.k + (at + r16) * kHd + 16 * g;
      r.k[kt][0] = *reinterpret_cast<const uint4*>(kp);
      r.k[kt][1] = *reinterpret_cast<const uint4*>(kp + 64);
#pragma unroll
      for (int i = 0; i < 4; i++)
        r.v[kt][i] = *reinterpret_cast<const uint2*>(c.v + (at + 4 * g + i) * kHd + 8 * r16);
      r.ks[kt] = *reinterpret_cast<const v4f_any*>(c.ks + at + 4 * g);
      r.vs[kt] = *reinterpret_cast<const v4f_any*>(c.vs + at + 4 * g);
    }
  };
  Raw cur;
  int pages[2];
  if (b0 + w < b1) {
    pages[0] = page_at(b0 + w, 0), pages[1] = page_at(b0 + w, 1);
    load(b0 + w, pages, cur);
    pages[0] = page_at(b0 + w + kFewWaves, 0), pages[1] = page_at(b0 + w + kFewWaves, 1);
  }
  for (int b = b0 + w; b < b1; b += kFewWaves) {
    Raw nxt;
    if (b + kFewWaves < b1) {
      load(b + kFewWaves, pages, nxt);
      pages[0] = page_at(b + 2 * kFewWaves, 0), pages[1] = page_at(b + 2 * kFewWaves, 1);
    }
    v4f s[2], kc[2], ke[2], kw[2], kf[2];
#pragma unroll
    for (int kt = 0; kt < 2; kt++) {
      s[kt] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kb = 0; kb < 4; kb++) {
        const uint4 r = cur.k[kt][kb >> 1];
        const v8h ka = kb & 1 ? codes8(r.z, r.w) : codes8(r.x, r.y);
        s[kt] = mma(ka, ql[kb], s[kt]);
        s[kt] = mma(ka, qh[kb], s[kt]);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const KeyTerms k = key_terms(cur.ks[kt][i], cur.vs[kt][i],
                                     cur.there[kt] && b * 32 + 16 * kt + 4 * g + i < t.len, qk, e0);
        kc[kt][i] = k.c, ke[kt][i] = k.e, kw[kt][i] = k.w, kf[kt][i] = k.f;
      }
    }
    v8h ph, pl;
    float least = ke[0][0];
#pragma unroll
    for (int j = 1; j < 8; j++) least = fminf(least, ke[j >> 2][j & 3]);
    auto softmax = [&](auto mask, auto seen) {
      constexpr bool kMask = decltype(mask)::value;
      const float mx = logits<kMask>(s, kc, ke, seen);
      if (__any(rises(st, mx))) raise(st, mx, acc);
      if (__any(least < kNear)) add_faint(s, ke, st);
      weights<kMask>(s, kw, kf, st, seen, ph, pl);
    };
    if (b * 32 + 32 <= all && cur.there[0] && cur.there[1]) {
      softmax(std::false_type{}, [](int, int) { return true; });
    } else {
      const int k0 = b * 32 + 4 * g;
      softmax(std::true_type{}, [&](int kt, int i) {
        return cur.there[kt] && k0 + 16 * kt + i < mine;
      });
    }
    uint32_t va[8], vb[8];  // dims 0-3 and 4-7 of the lane's eight, keys in slot order
#pragma unroll
    for (int kt = 0; kt < 2; kt++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        va[4 * kt + i] = cur.v[kt][i].x ^ 0x80808080u;
        vb[4 * kt + i] = cur.v[kt][i].y ^ 0x80808080u;
      }
    auto tile_e = [&](auto I, const uint32_t (&v)[8], v4f& o) {
      constexpr int i = decltype(I)::value;
      const v2h p0 = pair_of<i>(v[0], v[1]), p1 = pair_of<i>(v[2], v[3]);
      const v2h p2 = pair_of<i>(v[4], v[5]), p3 = pair_of<i>(v[6], v[7]);
      const v8h vv{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
      o = mma(vv, pl, o);
      o = mma(vv, ph, o);
    };
    tile_e(std::integral_constant<int, 0>{}, va, acc[0]);
    tile_e(std::integral_constant<int, 1>{}, va, acc[1]);
    tile_e(std::integral_constant<int, 2>{}, va, acc[2]);
    tile_e(std::integral_constant<int, 3>{}, va, acc[3]);
    tile_e(std::integral_constant<int, 0>{}, vb, acc[4]);
    tile_e(std::integral_constant<int, 1>{}, vb, acc[5]);
    tile_e(std::integral_constant<int, 2>{}, vb, acc[6]);
    tile_e(std::integral_constant<int, 3>{}, vb, acc[7]);
    cur = nxt;
  }

  // Join the waves: common maximum, then sums.
  __shared__ float2 ml[kFewWaves][kFewRows];
  __shared__ __attribute__((aligned(16))) float sums[kFewWaves][kFewRows][kFewStride];
  const float own = den_of(st.l, bad);
  if (g == 0) ml[w][r16] = float2{st.m, own};
#pragma unroll
  for (int i = 0; i < 4; i++) {  // dims 32 g + 8 i + e
    float* o = &sums[w][r16][32 * g + 8 * i];
    *reinterpret_cast<v4f*>(o) = v4f{acc[0][i], acc[1][i], acc[2][i], acc[3][i]};
    *reinterpret_cast<v4f*>(o + 4) = v4f{acc[4][i], acc[5][i], acc[6][i], acc[7][i]};
  }
  __syncthreads();
  constexpr int kPer = kFewRows * kHd / (64 * kFewWaves);  // dims a thread
  const int row = threadIdx.x * kPer / kHd, d0 = threadIdx.x * kPer % kHd;
  const int64_t r = t.r0 + row;
  if (r >= t.rows) return;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kFewWaves; i++) m = fmaxf(m, ml[i][row].x);
  const float ref = m == -INFINITY ? 0.f : m;
  float den = 0.f, o[kPer] = {};
#pragma unroll
  for (int i = 0; i < kFewWaves; i++) {
    const float f = __builtin_amdgcn_exp2f(ml[i][row].x - ref);
    den += times_exp2(ml[i][row].y, ml[i][row].x - ref);
#pragma unroll
    for (int d = 0; d < kPer; d++) o[d] = __builtin_fmaf(sums[i][row][d0 + d], f, o[d]);
  }
  float* dst;
  if (a.splits == 1) {
    const float f = den == 0.f ? 0.f : __builtin_ldexpf(1.f, e0 - kWeight) / den;
#pragma unroll
    for (int d = 0; d < kPer; d++) o[d] = o[d] * f;
    const int64_t tok = r / a.group;
    dst = a.out + (t.row0 + tok) * a.ldo +
          (int64_t)(h * a.group + (int)(r - tok * a.group)) * kHd + d0;
  } else {
    const int64_t at = (th * a.splits + z) * kFewRows + row;
    if (d0 == 0) a.part_ml[at] = float2{m, den};
    dst = a.part + at * kHd + d0;
  }
#pragma unroll
  for (int d = 0; d < kPer; d += 4)
    *reinterpret_cast<v4f*>(dst + d) = v4f{o[d], o[d + 1], o[d + 2], o[d + 3]};
}

// ---- joining the shares of cut keys: W waves a row ----
//
// A wave reads up to 8 shares of a row at a time, and its latency is that of its rounds
// and of finding its tile: more than 8 shares are divided over a row's W = 4 waves (64
// shares of 32 rows: 20 us with one, 6.6 with four). Few shares of many rows are bound by
// their bytes (7 of 18432 rows 17 us, 4.9 TB/s; four rows to a wave the same).

constexpr int kJoin = 8;  // shares that a wave reads at a time

template <int RT, int W>
__global__ void __launch_bounds__(256) kv_attn_join_kernel(Args a) {
  const int l = threadIdx.x & 63, w = uniform((int)threadIdx.x >> 6);
  const int64_t i = (int64_t)blockIdx.x * (4 / W) + w / W;
  const int64_t th = i / RT;
  const int row = (int)(i % RT), h = (int)(th % a.c.kv_heads);
  const Tile t = find_tile<RT>(a.c, a.group, a.tile0 + th / a.c.kv_heads);
  if (t.s < 0 || t.r0 + row >= t.rows) return;  // with W = 4 for the whole workgroup
  // lane z holds share z's maximum and denominator (splits <= 64)
  const int64_t at = th * a.splits * RT + row;
  const float2 ml = l < a.splits ? a.part_ml[at + (int64_t)l * RT] : float2{-INFINITY, 0.f};
  float m = ml.x;
#pragma unroll
  for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  const float d = ml.x - (m == -INFINITY ? 0.f : m);
  const float own = __builtin_amdgcn_exp2f(d);
  float den = times_exp2(ml.y, d);
#pragma unroll
  for (int o = 32; o; o >>= 1) den += __shfl_xor(den, o);
  float o0 = 0.f, o1 = 0.f;
  for (int z0 = kJoin * (w % W); z0 < a.splits; z0 += kJoin * W) {
    float2 v[kJoin];
#pragma unroll
    for (int k = 0; k < kJoin; k++)
      if (z0 + k < a.splits)
        v[k] = reinterpret_cast<const float2*>(a.part + (at + (int64_t)(z0 + k) * RT) * kHd)[l];
#pragma unroll
    for (int k = 0; k < kJoin; k++)
      if (z0 + k < a.splits) {
        const float f = __shfl(own, z0 + k);
        o0 = __builtin_fmaf(v[k].x, f, o0);
        o1 = __builtin_fmaf(v[k].y, f, o1);
      }
  }
  if (W > 1) {
    __shared__ float2 sums[W][64];
    sums[w][l] = float2{o0, o1};
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int k = 1; k < W; k++) {
      o0 += sums[k][l].x;
      o1 += sums[k][l].y;
    }
  }
  const float f =
      den == 0.f ? 0.f : __builtin_ldexpf(1.f, first_exp(a.c, t, h) - kWeight) / den;
  const int64_t r = t.r0 + row, tok = r / a.group;
  float* dst = a.out + (t.row0 + tok) * a.ldo +
               (int64_t)(h * a.group + (int)(r - tok * a.group)) * kHd;
  reinterpret_cast<float2*>(dst)[l] = float2{o0 * f, o1 * f};
}

// ---- chunks: NW waves of 16 QT rows over the same keys ----
//
// A block of 8 NW keys is loaded as codes, two blocks ahead, turned to fp16 once
// by the whole workgroup in the order of the MFMA operands and read by every
// wave from LDS (two buffers, one barrier a block). The first half of the waves
// turns its part before the block's products and the second half after them, so
// that the two waves of a SIMD meet less often in the same kind of work (768
// tokens x 28048 keys x 24 heads 605 -> 580 us, twice 4099 x 16411 2560 -> 2410;
// wave priorities around the products make no difference to either). A power of two for
// each query row, one more product a score, costs 2.5% and keeps rows independent.
// The operands of the next eight MFMAs are read from LDS before the eight at hand are
// issued, in an order that the compiler is held to (it reads each pair just before its
// use: 611 -> 576 and 2500 -> 2390 us). A wave's part of a block lies in one page, so its
// place is scalar arithmetic (a place a thread: 574 and 2363 us, then 548 and 2279 with the
// join). The flag of far value scales is read where the keys' terms are (at the block's start
// it waited for LDS: 1% and 1.5%).
//
// Bound: 4 MFMA products a score and value (two parts each), busy 46% of the cycles:
// 91% of the rate of a large library product for the first of these, 92% for the
// second. Tiles of 64 rows: 8 sequences of up to 100 tokens over up to 4099 keys, 24 heads,
// 90 us. What stands beside them does not disappear; at 611 us the first took 135 less
// without the softmax, 100 without turning keys, 100 without reading operands. Not
// faster: turns taken phase by phase (a barrier after each phase, the waves of a SIMD
// one phase apart), which does not fit the registers (1560 us); one sub-block's softmax
// between the next one's scores, with the queries' low parts in LDS to make room (640);
// four waves of 64 rows (2100, no room either).

template <int NW>
struct Block {
  static constexpr int kKeys = 8 * NW;
  static constexpr int kSubs = kKeys / 32;
  __attribute__((aligned(16))) char k[kSubs][2][4][1024];  // [sub][kt][kb][lane 16 B]
  __attribute__((aligned(16))) char v[kSubs][8][1024];     // [sub][e][lane 16 B]
  __attribute__((aligned(16))) float c[kKeys], e[kKeys], w[kKeys], f[kKeys];
  int far;  // a key has e < kNear
};

template <int NW, int QT>
__global__ void __launch_bounds__(64 * NW) kv_attn_chunk_kernel(Args a) {
  constexpr int kRows = 16 * QT * NW;
  using Blk = Block<NW>;
  constexpr int KB = Blk::kKeys;
  __shared__ Blk buf[2];
  const View& c = a.c;
  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, r16 = l & 15, g = l >> 4;
  const int z = (int)(blockIdx.x % a.splits);
  const int64_t th = blockIdx.x / a.splits;
  const int h = (int)(th % c.kv_heads);
  const Tile t = find_tile<kRows>(c, a.group, a.tile0 + th / c.kv_heads);
  if (t.s < 0) return;

  v8h qh[QT][4], ql[QT][4];
  int mine[QT];
  float qk[QT];
  bool bad[QT];
#pragma unroll
  for (int qt = 0; qt < QT; qt++) {
    const int64_t r = t.r0 + (w * QT + qt) * 16 + r16;
    float x[4][8];
    load_q(a, t, h, r, g, x);
    mine[qt] = keys_of(t, r, a.group, a.causal);
    const int qe = q_exp(clean(x, bad[qt]));
#pragma unroll
    for (int kb = 0; kb < 4; kb++) {
#pragma unroll
      for (int i = 0; i < 8; i++) x[kb][i] = __builtin_ldexpf(x[kb][i], qe);
      parts8(x[kb], qh[qt][kb], ql[qt][kb]);
    }
    qk[qt] = __builtin_ldexpf(a.scale2, -qe);
  }
  const int e0 = first_exp(c, t, h);
  const int keys = keys_of_rows(t, t.r0, kRows, a.group, a.causal);
  const int blocks = (keys + KB - 1) / KB;
  const int b0 = (int)((int64_t)blocks * z / a.splits);
  const int b1 = (int)((int64_t)blocks * (z + 1) / a.splits);
  // keys that the wave's rows see at most, and all of them see (the first row)
  const int64_t wr = t.r0 + w * QT * 16;
  const int wmost = wr < t.rows ? keys_of_rows(t, wr, QT * 16, a.group, a.causal) : 0;
  const int wall = keys_of(t, wr, a.group, a.causal);

  State st[QT];
  v4f acc[QT][8];
#pragma unroll
  for (int qt = 0; qt < QT; qt++) {
    st[qt] = State{-INFINITY, 0.f};
#pragma unroll
    for (int e = 0; e < 8; e++) acc[qt][e] = v4f{0.f, 0.f, 0.f, 0.f};
  }

  // The thread's part of a block: 16 dims of key (tid % 16) and 4 dims of four values'
  // rows, both of its wave's tile of 16 keys, which lies in one page; one key's scales
  // (the first KB threads).
  const int32_t* table = c.table + t.s * c.max_pages;
  const int k_j = (tid >> 4) & 7;                          // dims 16 k_j ..
  const int v_row = 4 * (tid >> 5), v_d = 4 * (tid & 31);  // keys of the block, dims
  const int wave_tile = uniform(v_row & ~15);
  uint4 kr;
  uint32_t vr[4];
  float ksr = 0.f, vsr = 0.f;
  bool ok = false;
  // Pages are looked up one block before the codes.
  auto page_of = [&](int p) { return p < keys ? table[p >> c.page_log2] : -1; };
  auto place = [&](int page, int p) -> int64_t {  // a page that is none: the first, masked
    return (((page >= 0 && page < c.pages ? page : 0) * (int64_t)c.kv_heads + h) << c.page_log2) +
           (p & ((1 << c.page_log2) - 1));
  };
  int wave_page = -1, one_page = -1;
  auto look = [&](int b) {
    wave_page = page_of(b * KB + wave_tile);
    if (tid < KB) one_page = page_of(b * KB + tid);
  };
  auto fetch = [&](int b) {
    const int64_t tile = place(uniform(wave_page), b * KB + wave_tile) * kHd;
    kr = *reinterpret_cast<const uint4*>(c.k + tile + (uint32_t)((tid & 15) * kHd + 16 * k_j));
#pragma unroll
    for (int i = 0; i < 4; i++)
      vr[i] = *reinterpret_cast<const uint32_t*>(
          c.v + tile + (uint32_t)(((v_row & 15) + i) * kHd + v_d));
    if (tid < KB) {
      const int64_t at = place(one_page, b * KB + tid);
      ksr = c.ks[at];
      vsr = c.vs[at];
      ok = one_page >= 0 && one_page < c.pages && b * KB + tid < t.len;
    }
    look(b + 1);
  };
  auto stage = [&](Blk& d) {
    const int kt = tid >> 7;  // 16-key tile of the block
    char* kd = d.k[kt >> 1][kt & 1][2 * (k_j >> 2)] + (16 * (k_j & 3) + (tid & 15)) * 16;
    *reinterpret_cast<v8h*>(kd) = codes8(kr.x, kr.y);
    *reinterpret_cast<v8h*>(kd + 1024) = codes8(kr.z, kr.w);
    uint32_t x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = vr[i] ^ 0x80808080u;
    // keys v_row .. + 3: tile (v_row / 16) % 2 of sub-block v_row / 32, lane group (v_row / 4) % 4
    char* vd = d.v[v_row >> 5][v_d & 7] + (16 * ((v_row >> 2) & 3) + (v_d >> 3)) * 16 +
               8 * ((v_row >> 4) & 1);
    auto put = [&](auto I) {
      constexpr int i = decltype(I)::value;
      const v2h p = pair_of<i>(x[0], x[1]), q = pair_of<i>(x[2], x[3]);
      typedef _Float16 v4h __attribute__((ext_vector_type(4)));
      *reinterpret_cast<v4h*>(vd + 1024 * i) = v4h{p[0], p[1], q[0], q[1]};
    };
    put(std::integral_constant<int, 0>{});
    put(std::integral_constant<int, 1>{});
    put(std::integral_constant<int, 2>{});
    put(std::integral_constant<int, 3>{});
    if (tid < KB) {
      const KeyTerms k = key_terms(ksr, vsr, ok, 1.f, e0);
      d.c[tid] = ok ? k.c : 0.f;
      d.e[tid] = ok ? k.e : -INFINITY;  // no key: its logit is -inf in every row
      d.w[tid] = k.w;
      d.f[tid] = k.f;
      const int far = __any(ok && k.e < kNear);  // the first wave holds all keys
      if (tid == 0) d.far = far;
    }
  };
  // MFMA operands of K (both key tiles of step kb) and V (dim tiles 2 p, 2 p + 1).
  auto load_k = [&](const Blk& d, int sub, int kb, v8h (&o)[2]) {
#pragma unroll
    for (int kt = 0; kt < 2; kt++) o[kt] = *reinterpret_cast<const v8h*>(d.k[sub][kt][kb] + l * 16);
  };
  auto load_v = [&](const Blk& d, int sub, int p, v8h (&o)[2]) {
#pragma unroll
    for (int j = 0; j < 2; j++) o[j] = *reinterpret_cast<const v8h*>(d.v[sub][2 * p + j] + l * 16);
  };
  auto compute = [&](const Blk& d, int b) {
    v8h op[2][2];
    load_k(d, 0, 0, op[0]);
#pragma unroll
    for (int sub = 0; sub < Blk::kSubs; sub++) {
      const int k0 = b * KB + 32 * sub;
      if (k0 >= wmost) break;
      v4f s[QT][2];
#pragma unroll
      for (int qt = 0; qt < QT; qt++) s[qt][0] = s[qt][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kb = 0; kb < 4; kb++) {
        if (kb < 3)
          load_k(d, sub, kb + 1, op[(kb + 1) & 1]);
        else
          load_v(d, sub, 0, op[0]);
        __builtin_amdgcn_sched_barrier(0);  // the reads stay ahead of the products
        const v8h(&ka)[2] = op[kb & 1];
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
          for (int qt = 0; qt < QT; qt++)
            s[qt][kt] = mma(ka[kt], ql[qt][kb], s[qt][kt]);
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
          for (int qt = 0; qt < QT; qt++)
            s[qt][kt] = mma(ka[kt], qh[qt][kb], s[qt][kt]);
        __builtin_amdgcn_sched_barrier(0);
      }
      const int at = 32 * sub + 4 * g;
      auto terms = [&](const float* p, v4f x[2]) {
        x[0] = *reinterpret_cast<const v4f*>(p + at);
        x[1] = *reinterpret_cast<const v4f*>(p + at + 16);
      };
      v8h ph[QT], pl[QT];
      auto softmax = [&](auto mask, auto seen) {
        constexpr bool kMask = decltype(mask)::value;
        v4f x[2], y[2];
        terms(d.c, x);
        terms(d.e, y);
        float mx[QT];
        bool up = false;
        const int far = d.far;
#pragma unroll
        for (int qt = 0; qt < QT; qt++) {
          // the key's scale first: the score alone may pass fp32's range
          const v4f cq[2] = {x[0] * qk[qt], x[1] * qk[qt]};
          mx[qt] = logits<kMask>(s[qt], cq, y, [&](int kt, int i) { return seen(qt, kt, i); });
          up |= rises(st[qt], mx[qt]);
        }
        if (__any(up)) {
#pragma unroll
          for (int qt = 0; qt < QT; qt++) raise(st[qt], mx[qt], acc[qt]);
        }
        if (uniform(far)) {
          terms(d.e, y);
#pragma unroll
          for (int qt = 0; qt < QT; qt++) add_faint(s[qt], y, st[qt]);
        }
        terms(d.w, x);
        terms(d.f, y);
#pragma unroll
        for (int qt = 0; qt < QT; qt++)
          weights<kMask>(s[qt], x, y, st[qt], [&](int kt, int i) { return seen(qt, kt, i); },
                         ph[qt], pl[qt]);
      };
      if (k0 + 32 <= wall) {
        softmax(std::false_type{}, [](int, int, int) { return true; });
      } else {
        const int kg = k0 + 4 * g;
        softmax(std::true_type{},
                [&](int qt, int kt, int i) { return kg + 16 * kt + i < mine[qt]; });
      }
#pragma unroll
      for (int p = 0; p < 4; p++) {
        if (p < 3)
          load_v(d, sub, p + 1, op[(p + 1) & 1]);
        else if (sub + 1 < Blk::kSubs)
          load_k(d, sub + 1, 0, op[0]);
        __builtin_amdgcn_sched_barrier(0);
        const v8h(&va)[2] = op[p & 1];
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int qt = 0; qt < QT; qt++) {
            v4f& o = acc[qt][2 * p + j];
            o = mma(va[j], pl[qt], o);
          }
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int qt = 0; qt < QT; qt++) {
            v4f& o = acc[qt][2 * p + j];
            o = mma(va[j], ph[qt], o);
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

  if (b0 < b1) {
    look(b0);
    fetch(b0);
    stage(buf[b0 & 1]);
    if (b0 + 1 < b1) fetch(b0 + 1);
    __syncthreads();
    const bool first = threadIdx.x < 32 * NW;
    for (int b = b0; b < b1; b++) {
      if (first) {
        if (b + 1 < b1) stage(buf[(b + 1) & 1]);
        if (b + 2 < b1) fetch(b + 2);
      }
      compute(buf[b & 1], b);
      if (!first) {
        if (b + 1 < b1) stage(buf[(b + 1) & 1]);
        if (b + 2 < b1) fetch(b + 2);
      }
      __syncthreads();
    }
  }

#pragma unroll
  for (int qt = 0; qt < QT; qt++) {
    const int row = (w * QT + qt) * 16 + r16;
    const int64_t r = t.r0 + row;
    if (r >= t.rows) continue;
    const float den = den_of(st[qt].l, bad[qt]);
    float f = 1.f;
    float* dst;
    if (a.splits == 1) {
      f = den == 0.f ? 0.f : __builtin_ldexpf(1.f, e0 - kWeight) / den;
      const int64_t tok = r / a.group;
      dst = a.out + (t.row0 + tok) * a.ldo +
            (int64_t)(h * a.group + (int)(r - tok * a.group)) * kHd + 32 * g;
    } else {
      const int64_t at = (th * a.splits + z) * kRows + row;
      if (g == 0) a.part_ml[at] = float2{st[qt].m, den};
      dst = a.part + at * kHd + 32 * g;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      *reinterpret_cast<v4f*>(dst + 8 * i) =
          v4f{acc[qt][0][i] * f, acc[qt][1][i] * f, acc[qt][2][i] * f, acc[qt][3][i] * f};
      *reinterpret_cast<v4f*>(dst + 8 * i + 4) =
          v4f{acc[qt][4][i] * f, acc[qt][5][i] * f, acc[qt][6][i] * f, acc[qt][7][i] * f};
    }
  }
}

template <int RT, class Launch>
hipError_t run(Args a, const kvplan::Plan& p, Launch launch, hipStream_t s) {
  // launches of as many tiles as a grid's 32-bit thread count takes
  for (int64_t tile = 0; tile < p.tiles; tile += p.tiles_per_launch) {
    const int64_t n = std::min(p.tiles_per_launch, p.tiles - tile) * a.c.kv_heads;
    a.tile0 = tile;
    launch(a, (unsigned)(n * p.splits));
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (p.splits > 1) {
      if (p.splits > kJoin)
        hipLaunchKernelGGL((kv_attn_join_kernel<RT, 4>), dim3((unsigned)(n * RT)), dim3(256), 0, s,
                           a);
      else
        hipLaunchKernelGGL((kv_attn_join_kernel<RT, 1>), dim3((unsigned)(n * RT / 4)), dim3(256), 0,
                           s, a);
      e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_kv_attn(const View& c, const float* q, int64_t ldq, float* out, int64_t ldo,
                          int heads, float scale, int causal, const kvplan::Plan& p,
                          void* scratch, hipStream_t s) {
  Args a{c, q, ldq, out, ldo, heads, heads / c.kv_heads, scale * 1.44269504088896341f, causal,
         p.splits, 0, nullptr, nullptr};
  if (p.splits > 1) {
    a.part = static_cast<float*>(scratch);
    a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(scratch) + p.part_bytes);
  }
  if (p.rows == kFewRows)
    return run<kFewRows>(a, p, [&](const Args& x, unsigned n) {
      hipLaunchKernelGGL(kv_attn_few_kernel, dim3(n), dim3(64 * kFewWaves), 0, s, x);
    }, s);
  if (p.rows == 64)
    return run<64>(a, p, [&](const Args& x, unsigned n) {
      hipLaunchKernelGGL((kv_attn_chunk_kernel<4, 1>), dim3(n), dim3(256), 0, s, x);
    }, s);
  return run<256>(a, p, [&](const Args& x, unsigned n) {
    hipLaunchKernelGGL((kv_attn_chunk_kernel<8, 2>), dim3(n), dim3(512), 0, s, x);
  }, s);
}

}  // namespace sdq
