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

#include "sdq_kv_attn.h"
#include "sdq_kv_plan.h"

#pragma clang fp contract(off)

namespace sdq {
namespace {

using namespace kvattn;

// Shares that a tile's keys are cut into. A shared part's rows are known here alone: as many
// shares as make a.want workgroups of all parts' tiles. Where each has its own place among a
// row's (kByRow), a share has a.least keys at least; one that is left out says so.
template <class K>
__device__ __forceinline__ int shares_of(const Args& a, const Tile& t, int keys) {
  if (!K::kByRow) return a.splits;
  int n = a.splits;
  if (K::kGroups && t.tiles > 0) n = min(n, max(1, (int)((uint32_t)a.want / (uint32_t)(t.tiles * a.nh))));
  return min(n, max(1, (keys + a.least - 1) / a.least));
}
template <class K>
__device__ __forceinline__ void leave_out(const Args& a, const Tile& t, int64_t th, int h, int z, int rows) {
  if ((int)threadIdx.x < rows && t.r0 + threadIdx.x < t.rows)
    a.part_ml[share_at<K>(a, t, th, h, z, rows, threadIdx.x)] = float2{-INFINITY, 0.f};
}

// ---- few rows: a tile of 16, the workgroup's waves share out the keys ----
//
// Bound by the cache's bytes, 264 a key and cached head, each read once by the wave that uses
// it, straight into the MFMA operands' lanes, two blocks of 32 keys on their way (in turn: a
// wait for the older one leaves the other in flight). The keys' terms are worked out one key a
// lane and handed round in LDS. 1 token x 262145 keys, 8 cached heads, 103 us, 5.4 TB/s, the rate
// of a large copy. 8 tokens of ragged sequences up to 4099 keys, 24 heads: 27 us, 4.3 TB/s; there
// a wave has eight blocks at most, and every sequence has the same number of shares: the longest
// has shares of 1025 keys, where the mean is 652. Tiles of one sequence read its keys each (one of
// 131072 keys, 8 heads: 16 rows 50 us, 64 rows 150).

constexpr int kFewRows = kvplan::kFewRows;
constexpr int kFewWaves = kvplan::kFewWaves;
constexpr int kFewStride = kHd + 4;  // LDS row of a merged sum (bank spread)

template <class K>
__device__ __forceinline__ void few_rows(const Args& a, unsigned wg) {
  const View& c = a.c;
  const int nh = K::kByRow ? a.nh : c.kv_heads;
  const int w = uniform((int)threadIdx.x >> 6), l = threadIdx.x & 63, r16 = l & 15, g = l >> 4;
  const int z = (int)(wg % (unsigned)a.splits);
  const unsigned th = wg / (unsigned)a.splits;
  const int h = (K::kByRow ? a.h0 : 0) + (int)(th % (unsigned)nh);
  const Tile t = find_tile<K, kFewRows>(a, a.tile0 + th / (unsigned)nh);
  if (t.s < 0) return;

  const int keys = keys_of_rows(t, t.r0, kFewRows, a.group, a.causal);
  const int splits = shares_of<K>(a, t, keys);
  if (K::kByRow && z >= splits) {
    leave_out<K>(a, t, th, h, z, kFewRows);
    return;
  }
  const int blocks = (keys + 31) / 32;
  const int b0 = (int)((int64_t)blocks * z / splits);
  const int b1 = (int)((int64_t)blocks * (z + 1) / splits);
  // what this lane's row sees, and what every row of the tile does
  const int mine = keys_of(t, t.r0 + r16, a.group, a.causal);
  const int all = keys_of(t, t.r0, a.group, a.causal);  // the first row

  State st{-INFINITY, 0.f};
  v4f acc[8];
#pragma unroll
  for (int e = 0; e < 8; e++) acc[e] = v4f{0.f, 0.f, 0.f, 0.f};

  __shared__ v4f terms[kFewWaves][32];
  __shared__ float qks[kFewRows];
  float* row_logits = nullptr;  // of the lane's keys 4 g .. of a tile
  if (K::kLogits && t.r0 + r16 < t.rows) {
    const int64_t tok = token_of(t.r0 + r16, a.group);
    const int head = h * a.group + (int)(t.r0 + r16 - tok * a.group);
    row_logits = a.logits + ((t.row0 + tok) * a.heads + head) * a.keys + 4 * g;
  }
  // A block's codes and scales, loaded one block ahead, its pages another one. The first ones
  // and the first value's scale are on their way before the queries are made ready.
  struct Raw {
    uint4 k[2][2];
    uint2 v[2][4];
    float ks, vs;  // of key l % 32
    bool there[2];
  };
  // Every load is made whether or not there is a block (of the first page then): behind a branch
  // the compiler would wait for a block's loads in the round that issues them.
  const auto* table = scalar_ptr(c.table + t.s * c.max_pages);
  const int last = (keys - 1) >> c.page_log2;
  auto page_at = [&](int b, int kt) { return table[min((b * 32 + 16 * kt) >> c.page_log2, last)]; };
  auto load = [&](int b, const int pages[2], Raw& r) {
    int64_t at_of[2];
#pragma unroll
    for (int kt = 0; kt < 2; kt++) {
      const int p = b * 32 + 16 * kt;
      r.there[kt] = b < b1 && p < keys && pages[kt] >= 0 && pages[kt] < c.pages;
      const int64_t at = (((r.there[kt] ? pages[kt] : 0) * (int64_t)c.kv_heads + h)
                          << c.page_log2) + (p & ((1 << c.page_log2) - 1));
      const int8_t* kp = c.k + (at + r16) * kHd + 16 * g;
      r.k[kt][0] = *reinterpret_cast<const uint4*>(kp);
      r.k[kt][1] = *reinterpret_cast<const uint4*>(kp + 64);
#pragma unroll
      for (int i = 0; i < 4; i++)
        r.v[kt][i] = *reinterpret_cast<const uint2*>(c.v + (at + 4 * g + i) * kHd + 8 * r16);
      at_of[kt] = at;
    }
    const int64_t mine_at = (l & 16 ? at_of[1] : at_of[0]) + r16;
    r.ks = c.ks[mine_at];
    r.vs = c.vs[mine_at];
  };
  // Two blocks in turn, each loaded while the other is at work (a copy from one to the other
  // would wait for its loads).
  Raw raw[2];
  int pages[2];
  auto look = [&](int b) { pages[0] = page_at(b, 0), pages[1] = page_at(b, 1); };
  int b = b0 + w;
  if (b < b1) look(b);
  float x[4][8];
  load_q(a, t, h, t.r0 + r16, g, x);
  const float v0 = first_value<K>(a, t, h);
  if (b < b1) {
    load(b, pages, raw[0]);
    look(b + kFewWaves);
  }
  bool bad;
  const int qe = q_exp(clean(x, bad));
  v8h qh[4], ql[4];
#pragma unroll
  for (int kb = 0; kb < 4; kb++) {
#pragma unroll
    for (int i = 0; i < 8; i++) x[kb][i] = __builtin_ldexpf(x[kb][i], qe);
    parts8(x[kb], qh[kb], ql[kb]);
  }
  const float qk = bad ? 0.f : __builtin_ldexpf(a.scale2, -qe);
  const int e0 = exp_of(v0);
  if (K::kStats && z == 0 && w == 0) {
    keep_parts(a, t, h, t.r0, qh, ql);
    // a row that is none, or whose shares are joined later
    if (g == 0 && (a.splits > 1 || t.r0 + r16 >= t.rows))
      a.info[tile16(a, t, h, t.r0) * 16 + r16] = RowInfo{qk, INFINITY, 0.f, 0};
    if (g == 0) qks[r16] = qk;
  }

  auto block = [&](int b, const Raw& cur) {
    // Keys' terms: one key a lane, handed round in LDS (each lane for the eight keys that it needs
    // was a quarter of a block's operations).
    const KeyTerms own = key_terms(
        cur.ks, cur.vs, (l & 16 ? cur.there[1] : cur.there[0]) && b * 32 + (l & 31) < t.len, 1.f, e0);
    terms[w][l & 31] = v4f{own.c, own.e, own.w, own.f};
    const bool far = __any(own.e < kNear);
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
        const v4f k = terms[w][16 * kt + 4 * g + i];
        kc[kt][i] = k[0] * qk, ke[kt][i] = k[1], kw[kt][i] = k[2], kf[kt][i] = k[3];
      }
    }
    v8h ph, pl;
    auto softmax = [&](auto mask, auto seen) {
      constexpr bool kMask = decltype(mask)::value;
      const float mx = logits<kMask>(s, kc, ke, seen);
      if (K::kLogits && row_logits) {
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
          *reinterpret_cast<v4f*>(row_logits + b * 32 + 16 * kt) = s[kt];
      }
      if (__any(rises(st, mx))) raise(st, mx, acc);
      if (far) add_faint(s, ke, st);
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
  };
  for (; b < b1; b += 2 * kFewWaves) {
    load(b + kFewWaves, pages, raw[1]);
    look(b + 2 * kFewWaves);
    block(b, raw[0]);
    if (b + kFewWaves >= b1) break;
    load(b + 2 * kFewWaves, pages, raw[0]);
    look(b + 3 * kFewWaves);
    block(b + kFewWaves, raw[1]);
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
  if (!K::kByRow && a.splits == 1) {
    const float f = den == 0.f ? 0.f : __builtin_ldexpf(1.f, e0 - kWeight) / den;
#pragma unroll
    for (int d = 0; d < kPer; d++) o[d] = o[d] * f;
    const int64_t tok = token_of(r, a.group);
    const int head = h * a.group + (int)(r - tok * a.group);
    dst = a.out + (t.row0 + tok) * a.ldo + (int64_t)head * kHd + d0;
    if (K::kLogits && d0 == 0) a.stats[(t.row0 + tok) * a.heads + head] = stat_of(m, den);
    if (K::kStats && d0 == 0)
      a.info[tile16(a, t, h, t.r0) * 16 + row] = info_of(a, t, r, qks[row], m, den);
  } else {
    const int64_t at = share_at<K>(a, t, th, h, z, kFewRows, row);
    if (d0 == 0) a.part_ml[at] = float2{m, den};
    dst = a.part + at * kHd + d0;
  }
#pragma unroll
  for (int d = 0; d < kPer; d += 4)
    *reinterpret_cast<v4f*>(dst + d) = v4f{o[d], o[d + 1], o[d + 2], o[d + 3]};
}
template <class K>
__global__ void __launch_bounds__(64 * kFewWaves, 2) kv_attn_few_kernel(Args a) {
  few_rows<K>(a, blockIdx.x);
}

// ---- joining the shares of cut keys: W waves a row ----
//
// A wave reads up to 8 shares of a row at a time, and its latency is that of its rounds
// and of finding its tile: more than 8 shares are divided over a row's W = 4 waves (64
// shares of 32 rows: 20 us with one, 6.6 with four). Few shares of many rows are bound by
// their bytes (7 of 18432 rows 17 us, 4.9 TB/s; four rows to a wave the same).

constexpr int kJoin = 8;  // shares that a wave reads at a time

// A row's maximum and denominator out of its shares' (one a lane), and the lane's share's
// weight among them.
__device__ __forceinline__ float join_stats(float2 ml, float& m, float& den) {
  m = ml.x;
#pragma unroll
  for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  const float d = ml.x - (m == -INFINITY ? 0.f : m);
  den = times_exp2(ml.y, d);
#pragma unroll
  for (int o = 32; o; o >>= 1) den += __shfl_xor(den, o);
  return __builtin_amdgcn_exp2f(d);
}

// The sum of a row's shares, two dims a lane, at `at` + z * step of the shares z < n that
// `ml` (lane z's) holds: to out, unnormalized sums times 2^-kWeight 2^E0 / denominator. W waves
// a row; false: the wave has no part in what follows.
template <int W>
__device__ __forceinline__ bool join(const Args& a, float2 ml, int64_t at, int64_t step, int n, int w,
                                     float& m, float& den, float& o0, float& o1) {
  const int l = threadIdx.x & 63;
  const float own = join_stats(ml, m, den);
  o0 = 0.f, o1 = 0.f;
  for (int z0 = kJoin * (w % W); z0 < n; z0 += kJoin * W) {
    float2 v[kJoin];
#pragma unroll
    for (int k = 0; k < kJoin; k++)
      if (z0 + k < n)
        v[k] = reinterpret_cast<const float2*>(a.part + (at + (int64_t)(z0 + k) * step) * kHd)[l];
#pragma unroll
    for (int k = 0; k < kJoin; k++)
      if (z0 + k < n) {
        const float f = __shfl(own, z0 + k);
        o0 = __builtin_fmaf(v[k].x, f, o0);
        o1 = __builtin_fmaf(v[k].y, f, o1);
      }
  }
  if (W > 1) {
    __shared__ float2 sums[W][64];
    sums[w][l] = float2{o0, o1};
    __syncthreads();
    if (w) return false;
#pragma unroll
    for (int k = 1; k < W; k++) {
      o0 += sums[k][l].x;
      o1 += sums[k][l].y;
    }
  }
  return true;
}

template <class K, int RT, int W>
__device__ __forceinline__ void join_tiles(const Args& a) {
  const int l = threadIdx.x & 63, w = uniform((int)threadIdx.x >> 6);
  const int64_t i = (int64_t)blockIdx.x * (4 / W) + w / W;
  const int64_t th = i / RT;
  const int row = (int)(i % RT), h = (int)(th % a.c.kv_heads);
  const Tile t = find_tile<K, RT>(a, a.tile0 + th / a.c.kv_heads);
  if (t.s < 0 || t.r0 + row >= t.rows) return;  // with W = 4 for the whole workgroup
  const float v0 = first_value<K>(a, t, h);
  // lane z holds share z's maximum and denominator (splits <= 64)
  const int64_t at = th * a.splits * RT + row;
  const float2 ml = l < a.splits ? a.part_ml[at + (int64_t)l * RT] : float2{-INFINITY, 0.f};
  float m, den, o0, o1;
  if (!join<W>(a, ml, at, RT, a.splits, w, m, den, o0, o1)) return;
  const float f =
      den == 0.f ? 0.f : __builtin_ldexpf(1.f, exp_of(v0) - kWeight) / den;
  const int64_t r = t.r0 + row, tok = token_of(r, a.group);
  const int head = h * a.group + (int)(r - tok * a.group);
  reinterpret_cast<float2*>(a.out + (t.row0 + tok) * a.ldo + (int64_t)head * kHd)[l] =
      float2{o0 * f, o1 * f};
  if (K::kStats && l == 0) {
    RowInfo& info = a.info[tile16(a, t, h, r) * 16 + (r & 15)];
    info = info_of(a, t, r, info.qk, m, den);
  }
}

template <class K, int RT, int W>
__global__ void __launch_bounds__(256) kv_attn_join_kernel(Args a) {
  join_tiles<K, RT, W>(a);
}

// ---- few rows: what each key was given ----
//
// The few-row form leaves its logits, t_rj of row r and key j; per key and cached head this
// adds up   sum_r 2^(t_rj - m_r - e_j) / d_r   (sdq_kv_weights.hip forms the logits again where
// rows are many). A thread has four keys, a row of logits is read once, and maxima and
// denominators come from the shares themselves, so that the join of the outputs is the same
// launch: its workgroups are the first `joins`. 8 tokens over up to 4099 keys, 24 heads: 7.4 us beside
// the attention's 29; one over 131073 keys, 32 heads on 8, 14 beside 64. Both wait for the logits, 4
// bytes a row and key. From 33 rows on the chunks and sdq_kv_weights.hip are faster (one sequence
// over 4099 keys, 24 heads: 32 rows 47 us for 48, 64 rows 72 for 49).

constexpr int kCountKeys = 1024;  // of a workgroup
constexpr int kCountRows = 64;    // whose statistics LDS holds

template <int W>
__global__ void __launch_bounds__(256) kv_counts_kernel(Args a, float* __restrict__ sums,
                                                        unsigned joins, int across) {
  if (blockIdx.x < joins) {
    join_tiles<Own, kFewRows, W>(a);
    return;
  }
  __shared__ float2 stats[kCountRows];
  __shared__ int sees[kCountRows];
  const View& c = a.c;
  const int tid = threadIdx.x, l = tid & 63, w = uniform(tid >> 6);
  const unsigned i = blockIdx.x - joins;
  const int sh = (int)(i / across);
  const int h = sh % c.kv_heads, s = sh / c.kv_heads;
  const Tile t = rows_of(a, s);
  const int e0 = first_exp<Own>(a, t, h);
  const int64_t tile0 = t.row0 * a.group / kFewRows + s;  // numbers as in find_tile
  for (int k0 = (int)(i % across) * kCountKeys; k0 < t.len; k0 += across * kCountKeys) {
    const int p = k0 + 4 * tid;
    const int64_t at = p < t.len ? kv::place_of(c, s, p, h) : -1;
    v4f e = v4f{0.f, 0.f, 0.f, 0.f}, sum = e;
    if (at >= 0) {
      const v4f vs = *reinterpret_cast<const v4f_any*>(c.vs + at);
#pragma unroll
      for (int j = 0; j < 4; j++) e[j] = key_terms(0.f, vs[j], p + j < t.len, 0.f, e0).e;
    }
    for (int64_t r0 = 0; r0 < t.rows; r0 += kCountRows) {
      const int n = (int)(t.rows - r0 < kCountRows ? t.rows - r0 : kCountRows);
      __syncthreads();  // the last rows' statistics are read
      for (int r = w; r < n; r += 4) {
        const int64_t row = r0 + r, tok = row / a.group;
        float2 st;
        if (a.splits == 1) {
          st = a.stats[(t.row0 + tok) * a.heads + h * a.group + (row - tok * a.group)];
        } else {
          const int64_t th = (tile0 + row / kFewRows) * c.kv_heads + h;
          const float2 ml = l < a.splits ? a.part_ml[(th * a.splits + l) * kFewRows + row % kFewRows]
                                         : float2{-INFINITY, 0.f};
          float m, den;
          join_stats(ml, m, den);
          st = stat_of(m, den);
        }
        if (l == 0) {
          stats[r] = st;
          sees[r] = st.y > 0.f ? keys_of(t, row, a.group, a.causal) : 0;
        }
      }
      __syncthreads();
      if (at >= 0) {
        int64_t tok = r0 / a.group;
        int qh = (int)(r0 - tok * a.group);
        for (int r = 0; r < n; r++) {
          const int see = sees[r];
          if (p < see) {
            const float2 st = stats[r];
            const v4f x = *reinterpret_cast<const v4f*>(
                a.logits + ((t.row0 + tok) * a.heads + h * a.group + qh) * a.keys + p);
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const float y = p + j < see ? x[j] - st.x - e[j] : -INFINITY;
              sum[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(y), st.y, sum[j]);
            }
          }
          if (++qh == a.group) qh = 0, tok++;
        }
      }
    }
    if (at < 0 || t.rows == 0) continue;
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (p + j < t.len) sums[at + j] = p + j < t.first ? sums[at + j] + sum[j] : sum[j];
  }
}

// The same for rows behind a shared part, whose shares lie side by side: z < z0 are the part's, the
// others the row's own, up to 128 of them, two a lane. Those that were left out are not read.
template <int W>
__global__ void __launch_bounds__(256) kv_attn_join_rows_kernel(Args a, int64_t i0) {
  const int l = threadIdx.x & 63, w = uniform((int)threadIdx.x >> 6);
  const int64_t i = i0 + (int64_t)blockIdx.x * (4 / W) + w / W;
  const int per = a.nh * a.group;
  const int64_t row = i / per;
  if (row >= a.c.T) return;
  const int head = (int)(i - row * per);
  const int64_t at = i * a.shares;
  float2 ml[2];
#pragma unroll
  for (int j = 0; j < 2; j++)
    ml[j] = l + 64 * j < a.shares ? a.part_ml[at + l + 64 * j] : float2{-INFINITY, 0.f};
  const Tile t = find_row(a, row);
  if (t.s < 0) return;
  const float v0 = first_value<Rest>(a, t, a.h0 + head / a.group);
  // a row without a position sees nothing; a sequence without a shared part has none of its shares
#pragma unroll
  for (int j = 0; j < 2; j++)
    if (t.first < 0 || (t.part < 0 && l + 64 * j < a.z0)) ml[j] = float2{-INFINITY, 0.f};
  float m = fmaxf(ml[0].x, ml[1].x);
#pragma unroll
  for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  const float ref = m == -INFINITY ? 0.f : m;
  float own[2], den = 0.f;
  uint64_t live[2];
#pragma unroll
  for (int j = 0; j < 2; j++) {
    // a share whose only keys have logits of NaN has no maximum, but a denominator
    const bool has = ml[j].x != -INFINITY || ml[j].y != 0.f;
    live[j] = __ballot(has);
    own[j] = __builtin_amdgcn_exp2f(ml[j].x - ref);
    den += has ? times_exp2(ml[j].y, ml[j].x - ref) : 0.f;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) den += __shfl_xor(den, o);
  const float2* part = reinterpret_cast<const float2*>(a.part + at * kHd) + l;
  float o0 = 0.f, o1 = 0.f;
#pragma unroll
  for (int j = 0; j < 2; j++) {
    // wave w of the row takes every W-th of the live ones, kJoin of them at a time
    uint64_t rest = live[j];
    while (rest) {
      float2 v[kJoin];
      int z[kJoin];
#pragma unroll
      for (int k = 0; k < kJoin; k++) {
        z[k] = -1;
#pragma unroll
        for (int u = 0; u < W; u++) {
          const int n = rest ? __builtin_ctzll(rest) : -1;
          rest &= rest - 1;
          if (u == w % W) z[k] = n;
        }
        if (z[k] >= 0) v[k] = part[(int64_t)(z[k] + 64 * j) * 64];
      }
#pragma unroll
      for (int k = 0; k < kJoin; k++)
        if (z[k] >= 0) {
          const float f = __shfl(own[j], z[k]);
          o0 = __builtin_fmaf(v[k].x, f, o0);
          o1 = __builtin_fmaf(v[k].y, f, o1);
        }
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
  const float f = den == 0.f ? 0.f : __builtin_ldexpf(1.f, exp_of(v0) - kWeight) / den;
  reinterpret_cast<float2*>(a.out + row * a.ldo + (int64_t)(a.h0 * a.group + head) * kHd)[l] =
      float2{o0 * f, o1 * f};
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

template <class K, int NW, int QT>
__device__ __forceinline__ void chunk_rows(const Args& a, unsigned wg) {
  constexpr int kRows = 16 * QT * NW;
  using Blk = Block<NW>;
  constexpr int KB = Blk::kKeys;
  __shared__ Blk buf[2];
  const View& c = a.c;
  const int nh = K::kByRow ? a.nh : c.kv_heads;
  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, r16 = l & 15, g = l >> 4;
  const int z = (int)(wg % (unsigned)a.splits);
  const unsigned th = wg / (unsigned)a.splits;
  const int h = (K::kByRow ? a.h0 : 0) + (int)(th % (unsigned)nh);
  const Tile t = find_tile<K, kRows>(a, a.tile0 + th / (unsigned)nh);
  if (t.s < 0) return;

  const int keys = keys_of_rows(t, t.r0, kRows, a.group, a.causal);
  const int splits = shares_of<K>(a, t, keys);
  if (K::kByRow && z >= splits) {
    leave_out<K>(a, t, th, h, z, kRows);
    return;
  }
  const float v0 = first_value<K>(a, t, h);
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
    qk[qt] = bad[qt] ? 0.f : __builtin_ldexpf(a.scale2, -qe);
    if (K::kStats && z == 0) {
      keep_parts(a, t, h, t.r0 + (w * QT + qt) * 16, qh[qt], ql[qt]);
      const int64_t r0 = t.r0 + (w * QT + qt) * 16;
      if (g == 0 && r0 < t.rows && (a.splits > 1 || r >= t.rows))
        a.info[tile16(a, t, h, r0) * 16 + r16] = RowInfo{qk[qt], INFINITY, 0.f, 0};
    }
  }
  const int e0 = exp_of(v0);
  const int blocks = (keys + KB - 1) / KB;
  const int b0 = (int)((int64_t)blocks * z / splits);
  const int b1 = (int)((int64_t)blocks * (z + 1) / splits);
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
    const bool ok = r < t.rows;
    const float den = den_of(st[qt].l, bad[qt]);
    float f = 1.f;
    float* dst = a.out;
    if (!ok) {
      // its lanes take part in the exchange below
    } else if (!K::kByRow && a.splits == 1) {
      f = den == 0.f ? 0.f : __builtin_ldexpf(1.f, e0 - kWeight) / den;
      const int64_t tok = token_of(r, a.group);
      const int head = h * a.group + (int)(r - tok * a.group);
      dst = a.out + (t.row0 + tok) * a.ldo + (int64_t)head * kHd;
      if (K::kStats && g == 0)
        a.info[tile16(a, t, h, r) * 16 + r16] = info_of(a, t, r, qk[qt], st[qt].m, den);
    } else {
      const int64_t at = share_at<K>(a, t, th, h, z, kRows, row);
      if (g == 0) a.part_ml[at] = float2{st[qt].m, den};
      dst = a.part + at * kHd;
    }
    store_row(dst, acc[qt], f, g, ok);
  }
}

template <class K, int NW, int QT>
__global__ void __launch_bounds__(64 * NW, NW == 4 && QT == 2 ? 2 : 1) kv_attn_chunk_kernel(Args a) {
  // causal: the last rows, which see most, first (4099 rows over themselves, 24 heads on 8: 329 us
  // the other way round, 252 so)
  chunk_rows<K, NW, QT>(a, a.causal ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

template <class K, int ROWS>
__device__ __forceinline__ void tile_rows(const Args& a, unsigned wg) {
  if constexpr (ROWS == kFewRows)
    few_rows<K>(a, wg);
  else
    chunk_rows<K, 4, ROWS / 64>(a, wg);
}
// Shared parts and own keys in one launch, the parts' `shared` workgroups first: the own keys'
// are short and fill what those leave (16 tokens of 24 heads behind 4099 shared keys 20 us, two
// launches 16 + 9; 297 rows behind 8209 and 5026 125, 123 + 20). 128 rows a part and head:
// 131073 keys x 8 heads 183 us of 116 at a large library product's rate. Vector operations take 57% of
// the cycles (the softmax, turning the keys), the products 39%; waves wait for a counter or barrier 30%
// of their life; turning the keys to fp16 is shared by half as many rows as in the chunks
// of 256. Blocks on their way in LDS by LDS-DMA, four of them, made it slower (220 us): what they
// cost in LDS reads is more than the loads' latency.
template <int PR, int OR>
__global__ void __launch_bounds__(256, 2) kv_attn_shared_kernel(Args pre, Args own, unsigned shared) {
  if (blockIdx.x < shared)
    tile_rows<Prefix, PR>(pre, blockIdx.x);
  else
    tile_rows<Rest, OR>(own, blockIdx.x - shared);
}

// Workgroups for n tiles (from a.tile0 on) of nh heads.
template <class K>
hipError_t launch_tiles(const Args& a, const kvplan::Plan& p, int64_t n, int nh, hipStream_t s) {
  const dim3 grid((unsigned)(n * nh * p.splits));
  if (p.rows == kFewRows)
    hipLaunchKernelGGL(kv_attn_few_kernel<K>, grid, dim3(64 * kFewWaves), 0, s, a);
  else if (p.rows == 64)
    hipLaunchKernelGGL((kv_attn_chunk_kernel<K, 4, 1>), grid, dim3(256), 0, s, a);
  else if constexpr (K::kGroups)  // rows of a part are 128 at most
    hipLaunchKernelGGL((kv_attn_chunk_kernel<K, 4, 2>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((kv_attn_chunk_kernel<K, 8, 2>), grid, dim3(512), 0, s, a);
  return hipGetLastError();
}

template <class K, int RT>
hipError_t launch_join(const Args& a, int64_t n, hipStream_t s) {
  if (a.splits > kJoin)
    hipLaunchKernelGGL((kv_attn_join_kernel<K, RT, 4>), dim3((unsigned)(n * RT)), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((kv_attn_join_kernel<K, RT, 1>), dim3((unsigned)(n * RT / 4)), dim3(256), 0, s,
                       a);
  return hipGetLastError();
}

template <class K>
hipError_t run(Args a, const kvplan::Plan& p, void* packed, hipStream_t s) {
  a.splits = p.splits;
  // sdq_kv_attention goes without: it has to run where scratch cannot be had
  constexpr bool kPacks = !std::is_same<K, Own>::value;
  if (kPacks && packed) {
    const hipError_t e = launch_kv_pack(a, packed, s);
    if (e != hipSuccess) return e;
  }
  // launches of as many tiles as a grid's 32-bit thread count takes
  for (int64_t tile = 0; tile < p.tiles; tile += p.tiles_per_launch) {
    const int64_t n = std::min(p.tiles_per_launch, p.tiles - tile);
    a.tile0 = tile;
    hipError_t e;
    if constexpr (kPacks)
      e = packed ? launch_kv_packed<K>(a, packed, (unsigned)(n * a.c.kv_heads * p.splits), s)
                 : launch_tiles<K>(a, p, n, a.c.kv_heads, s);
    else
      e = launch_tiles<K>(a, p, n, a.c.kv_heads, s);
    if (e != hipSuccess) return e;
    if (p.splits > 1) {
      e = p.rows == kFewRows ? launch_join<K, kFewRows>(a, n * a.c.kv_heads, s)
          : p.rows == 64     ? launch_join<K, 64>(a, n * a.c.kv_heads, s)
                             : launch_join<K, 256>(a, n * a.c.kv_heads, s);
      if (e != hipSuccess) return e;
    }
  }
  return hipSuccess;
}

Args args_of(const View& c, const KvRows& r, void* scratch, int64_t part_bytes) {
  Args a{};
  a.c = c;
  a.q = r.q, a.ldq = r.ldq, a.out = r.out, a.ldo = r.ldo;
  a.heads = r.heads, a.group = r.heads / c.kv_heads;
  a.scale2 = r.scale * 1.44269504088896341f;
  a.causal = r.causal;
  a.part = static_cast<float*>(scratch);
  a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(scratch) + part_bytes);
  return a;
}

}  // namespace

hipError_t launch_kv_attn(const View& c, const KvRows& r, const kvplan::Plan& p, void* scratch,
                          hipStream_t s) {
  return run<Own>(args_of(c, r, scratch, p.part_bytes), p, nullptr, s);
}

hipError_t launch_kv_cross(const View& c, const KvRows& r, const kvplan::Plan& p, void* scratch,
                           void* packed, hipStream_t s) {
  return run<Cross>(args_of(c, r, scratch, p.part_bytes), p, packed, s);
}

hipError_t launch_kv_counted(const View& c, const KvRows& r, const kvplan::Plan& p, void* scratch,
                             const kvplan::WeightsPlan& wp, void* kept, void* packed, hipStream_t s) {
  Args a = args_of(c, r, scratch, p.part_bytes);
  a.qparts = static_cast<char*>(kept);
  a.info = reinterpret_cast<RowInfo*>(a.qparts + wp.n16 * c.kv_heads * kQTile);
  a.n16 = wp.n16;
  return run<Counted>(a, p, packed, s);
}

int64_t kv_logit_keys(const View& c) { return round_up(std::max<int64_t>(c.max_pages << c.page_log2, 1), 32); }

hipError_t launch_kv_counted_few(const View& c, const KvRows& r, const kvplan::Plan& p, void* scratch,
                                 float2* stats, float* logits, float* sums, int cu_count,
                                 hipStream_t s) {
  Args a = args_of(c, r, scratch, p.part_bytes);
  a.stats = stats, a.logits = logits, a.keys = kv_logit_keys(c);
  a.splits = p.splits;
  hipError_t e;
  for (int64_t tile = 0; tile < p.tiles; tile += p.tiles_per_launch) {
    a.tile0 = tile;
    const int64_t n = std::min(p.tiles_per_launch, p.tiles - tile) * c.kv_heads * p.splits;
    hipLaunchKernelGGL(kv_attn_few_kernel<Logits>, dim3((unsigned)n), dim3(64 * kFewWaves), 0, s, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  // with shares, all tiles are one launch's: so is their join
  a.tile0 = 0;
  const int64_t rows = p.tiles * c.kv_heads * kFewRows;
  const unsigned joins = p.splits == 1 ? 0 : (unsigned)(p.splits > kJoin ? rows : rows / 4);
  const int64_t pairs = (int64_t)c.nseq * c.kv_heads;
  const int64_t across = std::min(ceil_div(std::max<int64_t>(c.max_pages << c.page_log2, 1), kCountKeys),
                                  ceil_div(4 * (int64_t)cu_count, pairs));
  const dim3 grid((unsigned)(joins + across * pairs));
  if (p.splits > kJoin)
    hipLaunchKernelGGL((kv_counts_kernel<4>), grid, dim3(256), 0, s, a, sums, joins, (int)across);
  else
    hipLaunchKernelGGL((kv_counts_kernel<1>), grid, dim3(256), 0, s, a, sums, joins, (int)across);
  return hipGetLastError();
}

template <int PR>
void launch_both(const Args& pre, const Args& own, int own_rows, unsigned shared, unsigned all,
                 hipStream_t s) {
  if (own_rows == kFewRows)
    hipLaunchKernelGGL((kv_attn_shared_kernel<PR, kFewRows>), dim3(all), dim3(256), 0, s, pre, own,
                       shared);
  else
    hipLaunchKernelGGL((kv_attn_shared_kernel<PR, 64>), dim3(all), dim3(256), 0, s, pre, own, shared);
}

hipError_t launch_kv_shared(const View& c, const kv::Shared& parts, const KvRows& r,
                            const kvplan::SharedPlan& p, void* scratch, hipStream_t s) {
  Args own = args_of(c, r, scratch, p.part_bytes);
  own.pre = parts;
  own.shares = p.pre.splits + p.own.splits;
  Args pre = own;
  own.z0 = p.pre.splits, own.splits = p.own.splits, own.least = p.own_least;
  pre.z0 = 0, pre.splits = p.pre.splits, pre.least = p.pre_least, pre.want = p.want, pre.causal = 0;
  pre.c.lens = parts.lens, pre.c.table = parts.table;
  pre.c.nseq = parts.n, pre.c.max_pages = parts.max_pages;
  for (int h0 = 0; h0 < c.kv_heads; h0 += p.heads) {
    own.h0 = pre.h0 = h0;
    own.nh = pre.nh = std::min(p.heads, c.kv_heads - h0);
    hipError_t e;
    if (p.own.rows <= 64 && p.pre.tiles <= p.pre.tiles_per_launch && p.own.tiles <= p.own.tiles_per_launch) {
      own.tile0 = pre.tile0 = 0;
      const unsigned shared = (unsigned)(p.pre.tiles * own.nh * p.pre.splits);
      const unsigned all = shared + (unsigned)(p.own.tiles * own.nh * p.own.splits);
      if (p.pre.rows == kFewRows)
        launch_both<kFewRows>(pre, own, p.own.rows, shared, all, s);
      else if (p.pre.rows == 64)
        launch_both<64>(pre, own, p.own.rows, shared, all, s);
      else
        launch_both<128>(pre, own, p.own.rows, shared, all, s);
      if ((e = hipGetLastError()) != hipSuccess) return e;
    } else {
      for (int64_t t = 0; t < p.pre.tiles; t += p.pre.tiles_per_launch) {
        pre.tile0 = t;
        e = launch_tiles<Prefix>(pre, p.pre, std::min(p.pre.tiles_per_launch, p.pre.tiles - t), own.nh, s);
        if (e != hipSuccess) return e;
      }
      for (int64_t t = 0; t < p.own.tiles; t += p.own.tiles_per_launch) {
        own.tile0 = t;
        e = launch_tiles<Rest>(own, p.own, std::min(p.own.tiles_per_launch, p.own.tiles - t), own.nh, s);
        if (e != hipSuccess) return e;
      }
    }
    // rows a launch: a grid's threads are a 32-bit number
    const int64_t rows = c.T * own.nh * own.group, most = int64_t(1) << 22;
    for (int64_t i = 0; i < rows; i += most) {
      const int64_t n = std::min(most, rows - i);
      // 16 rows of 113 shares 12 us with four waves a row, 15 with one; 1120 of 70 14.5 and 12.8
      if (own.shares > 4 * kJoin && rows < 1024)
        hipLaunchKernelGGL((kv_attn_join_rows_kernel<4>), dim3((unsigned)n), dim3(256), 0, s, own, i);
      else
        hipLaunchKernelGGL((kv_attn_join_rows_kernel<1>), dim3((unsigned)ceil_div(n, 4)), dim3(256),
                           0, s, own, i);
      if ((e = hipGetLastError()) != hipSuccess) return e;
    }
  }
  return hipSuccess;
}

}  // namespace sdq
