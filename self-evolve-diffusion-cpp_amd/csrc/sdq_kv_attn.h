// Device code that the paged attention's kernels share: tiles of query rows, the two
// fp16 parts of an fp32 number, keys' terms and one query's softmax state. The numbers
// that stand here are derived at the head of sdq_kv_attn.hip.
#pragma once

#include "sdq_device.h"
#include "sdq_kv.h"

#pragma clang fp contract(off)

namespace sdq {
namespace kvattn {

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

// What the rows of a launch see, and where their sums go.
struct Own {  // a sequence's last tokens, its own keys
  static constexpr bool kFree = false, kGroups = false, kByRow = false, kStats = false,
                        kLogits = false, kRest = false;
};
struct Cross : Own {  // any rows, all keys of their sequence
  static constexpr bool kFree = true;
};
struct Counted : Own {  // rows' parts, maxima and denominators are kept
  static constexpr bool kStats = true;
};
struct Logits : Own {  // few rows' logits, maxima and denominators
  static constexpr bool kLogits = true;
};
struct Prefix : Cross {  // the rows of a run of sequences, the keys that those share
  static constexpr bool kGroups = true, kByRow = true;
};
struct Rest : Own {  // own keys behind shared ones
  static constexpr bool kByRow = true, kRest = true;
};

struct RowInfo {
  float qk, m, inv;
  int see;  // keys; 0: the row adds nothing
};
constexpr int kQTile = 8192;  // bytes of a tile's parts

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
  // kLogits: [row][head] maximum and reciprocal denominator (infinity and 0: adds nothing), and
  // [row][head][key] logits, `keys` of them a row
  float2* stats;
  float* logits;
  int64_t keys;
  // kStats: [cached head][tile of 16 rows] their parts, [hi, lo][kb][lane 16 B], and what else
  // their weights ask for. n16 numbers of tiles, as in find_tile.
  char* qparts;
  RowInfo* info;
  int64_t n16;
  // kByRow: cached heads h0 .. h0 + nh - 1 of this launch, shares z0 .. of `shares`; the
  // sums are [row][head of those][share][128]
  int h0, nh, z0, shares;
  int want;  // Prefix: workgroups that the shares are to make
  int least; // keys of a share
  kv::Shared pre;  // Prefix: c has its lens, table, max_pages and number of parts
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
  int part, part_len;  // Rest: the shared part (-1: none) and its tokens
  int tiles;           // Prefix: that hold rows, of all parts (0: not counted)
};
constexpr Tile kNoTile{-1, 0, 0, 0, 0, 0, -1, 0, 0};

// A row's token. Rows times heads are at most 2^31 (sdq_api.hip).
__device__ __forceinline__ int token_of(int64_t r, int group) {
  return (int)((uint32_t)r / (uint32_t)group);
}

// A lane's value that is the same in the whole wave, as a scalar.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Memory that no kernel of the launch writes, for loads through the scalar cache also where
// the kernel stores elsewhere.
template <class T>
__device__ __forceinline__ const __attribute__((address_space(4))) T* scalar_ptr(const T* p) {
  return (const __attribute__((address_space(4))) T*)(uintptr_t)p;
}

// The last of indexes 0 .. n - 1 whose f, which does not fall, is at most v; -1: none. By a
// search 64 ways at a time; f(n) may be asked for. The same in every wave.
template <class F>
__device__ __forceinline__ int last_upto(int most, F f, int64_t v) {
  const int l = threadIdx.x & 63;
  int lo = 0, n = most, step;
  do {
    step = (n + 63) / 64;
    const uint64_t upto = __ballot((int64_t)l * step < n && f(min(lo + l * step, most)) <= v);
    if (!upto) return -1;
    const int k = 63 - __builtin_clzll(upto);
    lo += k * step;
    n = min(step, n - k * step);
  } while (step > 1);
  return uniform(lo);
}

// The shared part that sequence s begins with, -1: none.
__device__ __forceinline__ int part_of(const kv::Shared& p, int s) {
  const int g = last_upto(p.n, [&](int i) { return (int64_t)p.seq_of(i); }, s);
  return g >= 0 && s < p.seq_of(g + 1) ? g : -1;
}
__device__ __forceinline__ int64_t length_of(const View& c, const kv::Shared& p, int g) {
  const int64_t n = p.lens[g], most = p.max_pages << c.page_log2;
  return n < 0 ? 0 : n > most ? most : n;
}
// Tile number `tile`. Sequence s, whose rows start at row a and end before row b of all
// (row: a token's head of the group), has the numbers from a / RT + s to b / RT + s, at
// least as many as it has tiles of RT rows: a number without a tile is none. So the
// sequence is found by search, with no sum over those before it
// (a scan over them took a fifth of a microsecond for each 64). The same in every wave.
//
// Fewer than 64 sequences: a lane each has its rows and length, loaded side by side (the
// search and what follows it would load one after the other).
template <class K, int RT>
__device__ __forceinline__ Tile find_tile(const Args& a, int64_t tile) {
  const View& c = a.c;
  const int group = a.group;
  Tile t = kNoTile;
  constexpr bool kParts = K::kRest;
  const bool near = c.nseq < 64 && (!K::kGroups || a.pre.nseq < 64) && (!kParts || a.pre.n < 64);
  int lo;
  int64_t tokens, at;
  if (near) {
    const int l = threadIdx.x & 63;
    int row = (int)kv::row_of(c, min(l, K::kGroups ? a.pre.nseq : c.nseq));
    const int len = (int)kv::length_of(c, min(l, c.nseq - 1));
    int part_at = 0, part_len = 0;
    if (kParts) {
      part_at = a.pre.seq_of(min(l, a.pre.n));
      part_len = (int)length_of(c, a.pre, min(l, a.pre.n - 1));
    }
    if (K::kGroups) row = __shfl(row, a.pre.seq_of(min(l, c.nseq)));
    const uint64_t upto = __ballot(l < c.nseq && (int64_t)row * group / RT + l <= tile);
    if (!upto) return t;
    lo = uniform(63 - __builtin_clzll(upto));
    t.row0 = __builtin_amdgcn_readlane(row, lo);
    tokens = __builtin_amdgcn_readlane(row, lo + 1) - t.row0;
    t.len = __builtin_amdgcn_readlane(len, lo);
    if (kParts) {
      const uint64_t begun = __ballot(l < a.pre.n && part_at <= lo);
      const int g = begun ? uniform(63 - __builtin_clzll(begun)) : -1;
      if (g >= 0 && lo < __builtin_amdgcn_readlane(part_at, g + 1)) {
        t.part = g;
        t.part_len = __builtin_amdgcn_readlane(part_len, g);
      }
    }
    if (K::kGroups) {
      const int n = __shfl_down(row, 1) - row;
      int tiles = l < c.nseq && n > 0 ? (int)(((int64_t)n * group + RT - 1) / RT) : 0;
#pragma unroll
      for (int o = 32; o; o >>= 1) tiles += __shfl_xor(tiles, o);
      t.tiles = uniform(tiles);
    }
    at = t.row0 * group / RT + lo;
  } else {
    auto row_of = [&](int s) { return kv::row_of(c, K::kGroups ? a.pre.seq_of(s) : s); };
    auto first = [&](int s) { return row_of(s) * group / RT + s; };
    lo = last_upto(c.nseq, first, tile);
    if (lo < 0) return t;
    t.row0 = row_of(lo);
    tokens = row_of(lo + 1) - t.row0;
    t.len = (int)kv::length_of(c, lo);
    if (kParts) {
      t.part = part_of(a.pre, lo);
      if (t.part >= 0) t.part_len = (int)length_of(c, a.pre, t.part);
    }
    at = first(lo);
  }
  t.r0 = (tile - at) * RT;
  t.rows = tokens > 0 ? tokens * group : 0;
  t.first = K::kFree ? 0 : t.len - (int)(tokens > 0 ? tokens : 0);
  if (t.r0 < t.rows) t.s = lo;
  return t;
}

// All rows of sequence s.
__device__ __forceinline__ Tile rows_of(const Args& a, int s) {
  Tile t = kNoTile;
  t.s = s;
  t.row0 = kv::row_of(a.c, s);
  const int64_t tokens = kv::row_of(a.c, s + 1) - t.row0;
  t.rows = tokens > 0 ? tokens * a.group : 0;
  t.len = (int)kv::length_of(a.c, s);
  t.first = t.len - (int)(tokens > 0 ? tokens : 0);
  return t;
}

// Row `row` of the call: its sequence (-1: none), that one's table row, length and shared part, and
// in `first` the row's own position.
__device__ __forceinline__ Tile find_row(const Args& a, int64_t row) {
  const View& c = a.c;
  Tile t = kNoTile;
  int s, end;
  if (c.nseq < 64 && a.pre.n < 64) {  // as in find_tile
    const int l = threadIdx.x & 63;
    const int at = (int)kv::row_of(c, min(l, c.nseq));
    const int len = (int)kv::length_of(c, min(l, c.nseq - 1));
    const int part_at = a.pre.seq_of(min(l, a.pre.n));
    const int part_len = (int)length_of(c, a.pre, min(l, a.pre.n - 1));
    const uint64_t upto = __ballot(l < c.nseq && at <= row);
    if (!upto) return t;
    s = uniform(63 - __builtin_clzll(upto));
    end = __builtin_amdgcn_readlane(at, s + 1);
    t.len = __builtin_amdgcn_readlane(len, s);
    const uint64_t begun = __ballot(l < a.pre.n && part_at <= s);
    const int g = begun ? uniform(63 - __builtin_clzll(begun)) : -1;
    if (g >= 0 && s < __builtin_amdgcn_readlane(part_at, g + 1)) {
      t.part = g;
      t.part_len = __builtin_amdgcn_readlane(part_len, g);
    }
  } else {
    s = last_upto(c.nseq, [&](int i) { return kv::row_of(c, i); }, row);
    if (s < 0) return t;
    end = (int)kv::row_of(c, s + 1);
    t.len = (int)kv::length_of(c, s);
    t.part = part_of(a.pre, s);
    if (t.part >= 0) t.part_len = (int)length_of(c, a.pre, t.part);
  }
  if (row >= end) return t;
  t.s = s;
  t.first = t.len - (int)(end - row);
  return t;
}

// Keys that row r sees (0: it has no position, or is none).
__device__ __forceinline__ int keys_of(const Tile& t, int64_t r, int group, int causal) {
  if (r >= t.rows) return 0;
  const int p = t.first + token_of(r, group);
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

// x - hi of either half of a pair of fp16, exact, in one operation. The factor is hidden from
// the compiler, which makes a conversion and a subtraction of the plain form. Written by hand the
// operation would not be seen as one that may not yet write over an operand of a matrix
// instruction.
__device__ __forceinline__ float minus_one() {
  float m = -1.f;
  asm("" : "+s"(m));
  return m;
}
__device__ __forceinline__ float less_low(v2h hi, float x) {
  return __builtin_fmaf((float)hi[0], minus_one(), x);
}
__device__ __forceinline__ float less_high(v2h hi, float x) {
  return __builtin_fmaf((float)hi[1], minus_one(), x);
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

// r[c] of the lanes g (l >> 4) of a row: that of lane c, r[g], comes to lane g in r[c].
__device__ __forceinline__ void swap_quads(v4f (&r)[4]) {
#pragma unroll
  for (int k = 0; k < 4; k++) {
    uint32_t x[4];
#pragma unroll
    for (int c = 0; c < 4; c++) x[c] = __float_as_uint(r[c][k]);
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const auto p = __builtin_amdgcn_permlane32_swap(x[c], x[c + 2], false, false);
      x[c] = p[0], x[c + 2] = p[1];
    }
#pragma unroll
    for (int c = 0; c < 4; c += 2) {
      const auto p = __builtin_amdgcn_permlane16_swap(x[c], x[c + 1], false, false);
      x[c] = p[0], x[c + 1] = p[1];
    }
#pragma unroll
    for (int c = 0; c < 4; c++) r[c][k] = __uint_as_float(x[c]);
  }
}

// The lane's slice of a query row (head of a token), zeros where it is none. Four lanes load 64
// bytes that lie side by side and exchange them for what each needs.
__device__ __forceinline__ void load_q(const Args& a, const Tile& t, int h, int64_t r, int g,
                                       float x[4][8]) {
  const bool ok = r < t.rows;
  const int64_t rr = ok ? r : 0;
  const int64_t tok = token_of(rr, a.group);
  const float* p =
      a.q + (t.row0 + tok) * a.ldq + (int64_t)(h * a.group + (int)(rr - tok * a.group)) * kHd + 4 * g;
#pragma unroll
  for (int half = 0; half < 2; half++) {
    v4f v[4];
#pragma unroll
    for (int c = 0; c < 4; c++)
      v[c] = ok ? *reinterpret_cast<const v4f*>(p + 64 * half + 16 * c) : v4f{0.f, 0.f, 0.f, 0.f};
    swap_quads(v);
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
      for (int i = 0; i < 4; i++) x[2 * half + (c >> 1)][4 * (c & 1) + i] = v[c][i];
  }
}
// A row's sums times f: the lane has dims 32 g + 8 i + e in acc[e][i]. As they were loaded, 64 bytes
// of a row by four lanes (a lane's own 16 bytes apart from the others' were partial lines).
__device__ __forceinline__ void store_row(float* row, const v4f acc[8], float f, int g, bool ok) {
#pragma unroll
  for (int u = 0; u < 2; u++) {
    v4f v[4];
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const int e = 4 * (c & 1), i = 2 * u + (c >> 1);
      v[c] = v4f{acc[e][i] * f, acc[e + 1][i] * f, acc[e + 2][i] * f, acc[e + 3][i] * f};
    }
    swap_quads(v);
    if (ok)
#pragma unroll
      for (int c = 0; c < 4; c++) *reinterpret_cast<v4f*>(row + 32 * c + 16 * u + 4 * g) = v[c];
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
// E0: the exponent of the sequence's first value scale (0: no value); from kLeast on, so that a
// first value of next to nothing leaves those after it their range.
__device__ __forceinline__ int exp_of(float v) {
  const int e = v != 0.f ? __builtin_amdgcn_frexp_expf(v) : 0;
  return e < kLeast ? kLeast : e;
}
// That scale: of the token that the first of `pages` begins with, 0 where there is none.
__device__ __forceinline__ float first_value(const View& c, const int32_t* pages, int64_t len, int h) {
  if (len <= 0) return 0.f;
  const int64_t page = *scalar_ptr(pages);
  return page >= 0 && page < c.pages ? *scalar_ptr(c.vs + ((page * c.kv_heads + h) << c.page_log2)) : 0.f;
}
// Of a tile's sequence: behind a shared part that part's first value, so that both passes' sums
// have the same units.
template <class K>
__device__ __forceinline__ float first_value(const Args& a, const Tile& t, int h) {
  if (K::kRest && t.part_len > 0)
    return first_value(a.c, a.pre.table + t.part * a.pre.max_pages, t.part_len, h);
  return first_value(a.c, a.c.table + t.s * a.c.max_pages, t.len, h);
}
template <class K>
__device__ __forceinline__ int first_exp(const Args& a, const Tile& t, int h) {
  return exp_of(first_value<K>(a, t, h));
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

// A row's entry of Args::stats.
__device__ __forceinline__ float2 stat_of(float m, float den) {
  return den > 0.f ? float2{m, 1.f / den} : float2{INFINITY, 0.f};
}

// The tile of 16 rows that row r (a multiple of 16 or within the tile) of t's sequence is in.
__device__ __forceinline__ int64_t tile16(const Args& a, const Tile& t, int h, int64_t r) {
  return h * a.n16 + t.row0 * a.group / 16 + t.s + (r >> 4);
}
__device__ __forceinline__ RowInfo info_of(const Args& a, const Tile& t, int64_t r, float qk, float m,
                                           float den) {
  const float2 st = stat_of(m, den);
  const int see = st.y > 0.f ? keys_of(t, r, a.group, a.causal) : 0;
  return RowInfo{qk, st.x, st.y, see};
}
// The wave's 16 rows from r0 on: their parts, as the lanes hold them.
__device__ __forceinline__ void keep_parts(const Args& a, const Tile& t, int h, int64_t r0,
                                           const v8h qh[4], const v8h ql[4]) {
  if (r0 >= t.rows) return;
  char* p = a.qparts + tile16(a, t, h, r0) * kQTile + (threadIdx.x & 63) * 16;
#pragma unroll
  for (int kb = 0; kb < 4; kb++) {
    *reinterpret_cast<v8h*>(p + 1024 * kb) = qh[kb];
    *reinterpret_cast<v8h*>(p + 4096 + 1024 * kb) = ql[kb];
  }
}

// Where a share of a tile's row keeps its sums (th: the workgroup's tile and head).
template <class K>
__device__ __forceinline__ int64_t share_at(const Args& a, const Tile& t, int64_t th, int h, int z,
                                            int rows, int row) {
  if (!K::kByRow) return (th * a.splits + z) * rows + row;
  const int64_t r = t.r0 + row, tok = token_of(r, a.group);
  const int64_t at = (t.row0 + tok) * (a.nh * a.group) + (h - a.h0) * a.group + (r - tok * a.group);
  return at * a.shares + a.z0 + z;
}

}  // namespace kvattn

// Keys as MFMA operands, of all sequences and heads (sdq_kv_packed.hip): once a call, then tiles
// of 256 rows in `grid` workgroups over them.
hipError_t launch_kv_pack(const kvattn::Args& a, void* packed, hipStream_t s);
template <class K>
hipError_t launch_kv_packed(const kvattn::Args& a, void* packed, unsigned grid, hipStream_t s);

}  // namespace sdq
