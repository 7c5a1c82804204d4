// Attention of many rows over the paged int8 cache, its keys turned to MFMA operands once
// (gfx950). The same numbers as sdq_kv_attn.hip's chunks, bit for bit.
//
// The chunks' kernel turns a block's codes to fp16 for every 256 rows, and its waves do so
// between their products. Where a sequence has thousands of rows, one pass does it for all
// (pack: 264 bytes a key and cached head read, 528 written), in the order that the products
// read, so that LDS-DMA moves the blocks as they are. The loop then holds MFMAs, LDS reads and
// the softmax only, and there is room to put a block's exponentials beside the next block's
// scores, and the next block's logits beside this one's sums: neither waits for the other.
//
// 24 heads: 27280 rows over 512 keys 419 us (8 of them the pass), 509 in chunks, in turn on one card
// (385 to 422 on others); 2048 rows over 4099 254 and 288, 8192 over 4099 709 and 720, 1024 over
// 4099 162 and 158, over 512 39 and 45: taken from 1024 rows a sequence on. Bound by the matrix
// units and the softmax beside them: 8192 rows over as many keys at 1.17 PFLOP/s, the rate of a
// large library product. Over 512 keys the matrix units are busy 42% of the cycles and the vector
// units 49%, waves wait for a counter or barrier 29% of their life and for their turn to issue 33%;
// what stands beside the loop, 670 MB of queries and output, is not overlapped with it. A tile is
// two workgroups of four waves, two workgroups a CU: eight waves at one ring were slower.
#include <algorithm>

#include "sdq_kv_attn.h"
#include "sdq_kv_plan.h"

#pragma clang fp contract(off)

namespace sdq {
namespace {

using namespace kvattn;

constexpr int kWaves = 4;
constexpr int QT = 2;                  // tiles of 16 rows a wave
constexpr int kRows = 256;             // of a tile, two workgroups
constexpr int kHalf = 16 * QT * kWaves;
constexpr int kRing = 4;               // blocks of 32 keys in LDS
constexpr int kDma = 5;                // a wave's, a block: four of codes, one of terms

// 32 keys: K [kt][kb][lane 16 B], V [e][lane 16 B], and their terms.
struct Packed {
  char k[2][4][1024];
  char v[8][1024];
  float c[32], e[32], w[32], f[32];
};
static_assert(sizeof(Packed) == 16896);

struct Pack {
  Packed* blocks;  // [sequence, cached head][block]
  int* far;        // [sequence, cached head][two blocks]: a key has e < kNear
  int64_t most;    // pairs of blocks that a sequence has at most
};

// One workgroup per 64 keys of a sequence and head.
__global__ void __launch_bounds__(512) kv_pack_kernel(Args a, Pack pk) {
  __shared__ __attribute__((aligned(16))) Packed buf[2];
  const View& c = a.c;
  const int tid = threadIdx.x;
  const int b = (int)(blockIdx.x % pk.most);
  const int64_t sh = blockIdx.x / pk.most;
  const int h = (int)(sh % c.kv_heads), s = (int)(sh / c.kv_heads);
  const int len = (int)kv::length_of(c, s);
  if (b * 64 >= len) return;
  const int32_t* table = c.table + s * c.max_pages;
  const int e0 = exp_of(first_value(c, table, len, h));
  auto place = [&](int p, bool& ok) -> int64_t {
    const int page = p < len ? table[p >> c.page_log2] : -1;
    ok = page >= 0 && page < c.pages;
    return (((ok ? page : 0) * (int64_t)c.kv_heads + h) << c.page_log2) + (p & ((1 << c.page_log2) - 1));
  };
  const int k_j = (tid >> 4) & 7, v_row = 4 * (tid >> 5), v_d = 4 * (tid & 31);
  bool ok;
  const int64_t tile = place(b * 64 + (v_row & ~15), ok) * kHd;
  const uint4 kr = *reinterpret_cast<const uint4*>(c.k + tile + (tid & 15) * kHd + 16 * k_j);
  uint32_t x[4];
#pragma unroll
  for (int i = 0; i < 4; i++)
    x[i] = *reinterpret_cast<const uint32_t*>(c.v + tile + ((v_row & 15) + i) * kHd + v_d) ^ 0x80808080u;
  {
    const int kt = tid >> 7;
    char* kd = buf[kt >> 1].k[kt & 1][2 * (k_j >> 2)] + (16 * (k_j & 3) + (tid & 15)) * 16;
    *reinterpret_cast<v8h*>(kd) = codes8(kr.x, kr.y);
    *reinterpret_cast<v8h*>(kd + 1024) = codes8(kr.z, kr.w);
    char* vd = buf[v_row >> 5].v[v_d & 7] + (16 * ((v_row >> 2) & 3) + (v_d >> 3)) * 16 +
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
  }
  if (tid < 64) {
    const int64_t at = place(b * 64 + tid, ok);
    const KeyTerms k = key_terms(c.ks[at], c.vs[at], ok, 1.f, e0);
    Packed& d = buf[tid >> 5];
    d.c[tid & 31] = ok ? k.c : 0.f;
    d.e[tid & 31] = ok ? k.e : -INFINITY;  // no key: its logit is -inf in every row
    d.w[tid & 31] = k.w;
    d.f[tid & 31] = k.f;
    const int far = __any(ok && k.e < kNear);
    if (tid == 0) pk.far[sh * pk.most + b] = far;
  }
  __syncthreads();
  const uint4* from = reinterpret_cast<const uint4*>(buf);
  uint4* to = reinterpret_cast<uint4*>(pk.blocks + (sh * pk.most + b) * 2);
  for (int i = tid; i < (int)(2 * sizeof(Packed) / 16); i += 512) to[i] = from[i];
}

template <class K>
__global__ void __launch_bounds__(64 * kWaves, 2) kv_attn_packed_kernel(Args a, Pack pk) {
  __shared__ __attribute__((aligned(16))) Packed ring[kRing];
  const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, r16 = l & 15, g = l >> 4;
  const unsigned wg = a.causal ? gridDim.x - 1 - blockIdx.x : blockIdx.x;  // as the chunks
  const int nh = a.c.kv_heads;
  const unsigned both = (unsigned)(nh * a.splits);  // a half of a tile, then the other
  const unsigned half = wg / both % 2, th = (wg / (2 * both) * both + wg % both) / (unsigned)a.splits;
  const int z = (int)(wg % both % (unsigned)a.splits);
  const int h = (int)(th % (unsigned)nh);
  const Tile t = find_tile<K, kRows>(a, a.tile0 + th / (unsigned)nh);
  const int r_half = (int)half * kHalf;
  if (t.s < 0 || t.r0 + r_half >= t.rows) return;

  // shares of 64 keys' blocks, as the chunks cut them
  const int keys = keys_of_rows(t, t.r0, kRows, a.group, a.causal);
  const int pairs = (keys + 63) / 64;
  const int b0 = 2 * (int)((int64_t)pairs * z / a.splits);
  const int b1 = 2 * (int)((int64_t)pairs * (z + 1) / a.splits);
  // of those, what the half's rows see
  const int n = max(0, min(b1, (keys_of_rows(t, t.r0 + r_half, kHalf, a.group, a.causal) + 31) / 32) - b0);
  const int64_t rec = ((int64_t)t.s * nh + h) * pk.most;
  const Packed* blocks = pk.blocks + rec * 2;
  // the flags of 64 pairs of blocks, one a lane
  const int* fars = pk.far + rec;
  int far = 0;
  auto flags = [&](int pair) { far = pair + l < pairs ? fars[pair + l] : 0; };
  const uint32_t lds = uniform((int)dev::lds_addr32(ring));

  // The wave's part of block b0 + i (of the last one behind it) into slot i % kRing.
  auto issue = [&](int i) {
    const dev::v4u from = dev::raw_rsrc(blocks + min(b0 + i, b1 - 1), (uint32_t)sizeof(Packed));
    const uint32_t to = lds + (uint32_t)(i & (kRing - 1)) * (uint32_t)sizeof(Packed);
#pragma unroll
    for (int k = 0; k < 4; k++)
      dev::dma16<4>(from, l * 16, w * 4096 + k * 1024, to + w * 4096 + k * 1024);
    if (l < 8) dev::dma16<4>(from, l * 16, 16384 + w * 128, to + 16384 + w * 128);
  };

  const float v0 = first_value<K>(a, t, h);
  v8h qh[QT][4], ql[QT][4];
  int mine[QT];
  float qk[QT];
  bool bad[QT];
#pragma unroll
  for (int qt = 0; qt < QT; qt++) {
    const int64_t r = t.r0 + r_half + (w * QT + qt) * 16 + r16;
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
      keep_parts(a, t, h, t.r0 + r_half + (w * QT + qt) * 16, qh[qt], ql[qt]);
      const int64_t r0 = t.r0 + r_half + (w * QT + qt) * 16;
      if (g == 0 && r0 < t.rows && (a.splits > 1 || r >= t.rows))
        a.info[tile16(a, t, h, r0) * 16 + r16] = RowInfo{qk[qt], INFINITY, 0.f, 0};
    }
  }
  const int e0 = exp_of(v0);
  // blocks that the wave's rows see at most, and those that all of them see whole
  const int64_t wr = t.r0 + r_half + w * QT * 16;
  const int wmost = wr < t.rows ? keys_of_rows(t, wr, QT * 16, a.group, a.causal) : 0;
  const int wall = keys_of(t, wr, a.group, a.causal);
  const int seen = min(n, (wmost + 31) / 32 - b0), whole = wall / 32 - b0;

  State st[QT];
  v4f acc[QT][8];
#pragma unroll
  for (int qt = 0; qt < QT; qt++) {
    st[qt] = State{-INFINITY, 0.f};
#pragma unroll
    for (int e = 0; e < 8; e++) acc[qt][e] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  // a block's logits (its scores first), two key tiles of each row tile
  struct Logits32 {
    v4f s[QT][2];
  };
  auto terms = [&](const float* p, v4f x[2]) {
    x[0] = *reinterpret_cast<const v4f*>(p + 4 * g);
    x[1] = *reinterpret_cast<const v4f*>(p + 4 * g + 16);
  };
  // What follows from block i's logits before its weights: masks, the largest, the reference.
  auto settle = [&](const Packed& d, int i, Logits32& x) {
    float mx[QT];
    bool up = false;
    if (i >= whole) {
#pragma unroll
      for (int qt = 0; qt < QT; qt++)
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (32 * (b0 + i) + 16 * (j >> 2) + 4 * g + (j & 3) >= mine[qt])
            x.s[qt][j >> 2][j & 3] = -INFINITY;
    }
#pragma unroll
    for (int qt = 0; qt < QT; qt++) {
      float m = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; j++) m = fmaxf(m, x.s[qt][j >> 2][j & 3]);
      mx[qt] = quad_max(m);
      up |= rises(st[qt], mx[qt]);
    }
    if (__any(up)) {
#pragma unroll
      for (int qt = 0; qt < QT; qt++) raise(st[qt], mx[qt], acc[qt]);
    }
    const int pair = (i >> 1) & 63;
    if ((i & 127) == 0 && i) flags((b0 + i) >> 1);
    if (__builtin_amdgcn_readlane(far, pair)) {
      v4f y[2];
      terms(d.e, y);
#pragma unroll
      for (int qt = 0; qt < QT; qt++) add_faint(x.s[qt], y, st[qt]);
    }
  };
  // Block i, whose logits are settled: the next one's scores beside its exponentials, its sums
  // beside the next one's logits.
  auto step = [&](int i, const Logits32& x, Logits32& nx, auto mask) {
    constexpr bool kMask = decltype(mask)::value;
    const Packed &d = ring[i & (kRing - 1)], &e = ring[(i + 1) & (kRing - 1)];
    v8h ph[QT], pl[QT];
    float sum[QT], ref[QT];
#pragma unroll
    for (int qt = 0; qt < QT; qt++) sum[qt] = 0.f, ref[qt] = st[qt].m == -INFINITY ? 0.f : st[qt].m;
    // What a group of eight products and the work beside it read from LDS, one group ahead: two
    // operands, and the terms of elements 2 j, 2 j + 1 (two keys side by side).
    struct Group {
      v8h op[2];
      float2 a, b;
    } grp[2];
    auto two = [&](const float* p, int j) {
      return *reinterpret_cast<const float2*>(p + 4 * g + 16 * (j >> 1) + 2 * (j & 1));
    };
    auto load_k = [&](int kb, Group& o) {
#pragma unroll
      for (int kt = 0; kt < 2; kt++) o.op[kt] = *reinterpret_cast<const v8h*>(e.k[kt][kb] + l * 16);
      o.a = two(d.w, kb), o.b = two(d.f, kb);
    };
    auto load_v = [&](int p, Group& o) {
#pragma unroll
      for (int j = 0; j < 2; j++) o.op[j] = *reinterpret_cast<const v8h*>(d.v[2 * p + j] + l * 16);
      o.a = two(e.c, p), o.b = two(e.e, p);
    };
    load_k(0, grp[0]);
#pragma unroll
    for (int kb = 0; kb < 4; kb++) {
      if (kb < 3)
        load_k(kb + 1, grp[(kb + 1) & 1]);
      else
        load_v(0, grp[0]);
      __builtin_amdgcn_sched_barrier(0);
      const Group& o = grp[kb & 1];
#pragma unroll
      for (int kt = 0; kt < 2; kt++)
#pragma unroll
        for (int qt = 0; qt < QT; qt++)
          nx.s[qt][kt] = mma(o.op[kt], ql[qt][kb], kb ? nx.s[qt][kt] : v4f{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int kt = 0; kt < 2; kt++)
#pragma unroll
        for (int qt = 0; qt < QT; qt++) nx.s[qt][kt] = mma(o.op[kt], qh[qt][kb], nx.s[qt][kt]);
      // weights of elements 2 kb, 2 kb + 1 (weights() of sdq_kv_attn.h, spread out)
#pragma unroll
      for (int qt = 0; qt < QT; qt++) {
        float p[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const int j = 2 * kb + u;
          const float v = __builtin_amdgcn_exp2f(x.s[qt][j >> 2][j & 3] - ref[qt]);
          sum[qt] = __builtin_fmaf(v, u ? o.a.y : o.a.x, sum[qt]);
          p[u] = v * (u ? o.b.y : o.b.x);
          if (kMask && 32 * (b0 + i) + 16 * (j >> 2) + 4 * g + (j & 3) >= mine[qt])
            p[u] = 0.f;  // its scale may be NaN
        }
        const v2h hi = rounded(p[0], p[1]);
        const v2h lo = rounded(less_low(hi, p[0]), less_high(hi, p[1]));
        ph[qt][2 * kb] = hi[0], ph[qt][2 * kb + 1] = hi[1];
        pl[qt][2 * kb] = lo[0], pl[qt][2 * kb + 1] = lo[1];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int qt = 0; qt < QT; qt++) st[qt].l += sum[qt];
#pragma unroll
    for (int p = 0; p < 4; p++) {
      if (p < 3) load_v(p + 1, grp[(p + 1) & 1]);
      __builtin_amdgcn_sched_barrier(0);
      const Group& o = grp[p & 1];
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int qt = 0; qt < QT; qt++) acc[qt][2 * p + j] = mma(o.op[j], pl[qt], acc[qt][2 * p + j]);
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int qt = 0; qt < QT; qt++) acc[qt][2 * p + j] = mma(o.op[j], ph[qt], acc[qt][2 * p + j]);
      // logits of elements 2 p, 2 p + 1: the key's scale first, the score alone may pass fp32's range
#pragma unroll
      for (int qt = 0; qt < QT; qt++)
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const int j = 2 * p + u;
          v4f& s = nx.s[qt][j >> 2];
          s[j & 3] = __builtin_fmaf(s[j & 3], (u ? o.a.y : o.a.x) * qk[qt], u ? o.b.y : o.b.x);
        }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  if (n > 0) {
    flags(b0 >> 1);
    issue(0), issue(1), issue(2);
    __builtin_amdgcn_s_waitcnt(dev::waitcnt_vm(2 * kDma));
    asm volatile("s_barrier" ::: "memory");
    Logits32 x;
    if (seen > 0) {
      v4f tc[2], te[2];
#pragma unroll
      for (int qt = 0; qt < QT; qt++) x.s[qt][0] = x.s[qt][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kb = 0; kb < 4; kb++)
#pragma unroll
        for (int kt = 0; kt < 2; kt++) {
          const v8h k = *reinterpret_cast<const v8h*>(ring[0].k[kt][kb] + l * 16);
#pragma unroll
          for (int qt = 0; qt < QT; qt++) {
            x.s[qt][kt] = mma(k, ql[qt][kb], x.s[qt][kt]);
            x.s[qt][kt] = mma(k, qh[qt][kb], x.s[qt][kt]);
          }
        }
      terms(ring[0].c, tc);
      terms(ring[0].e, te);
#pragma unroll
      for (int qt = 0; qt < QT; qt++)
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
          for (int j = 0; j < 4; j++)
            x.s[qt][kt][j] = __builtin_fmaf(x.s[qt][kt][j], tc[kt][j] * qk[qt], te[kt][j]);
      settle(ring[0], 0, x);
    }
    // whole blocks, then those with keys that rows do not see (two loops: in one the compiler takes
    // what the two forms of a block have in common out of the order that it is given)
    auto run = [&](int i, int end, auto mask) {
      for (; i < end; i++) {
        // block i + 1 has landed in every wave, and block i - 1 is done with
        __builtin_amdgcn_s_waitcnt(dev::waitcnt_vm(kDma));
        asm volatile("s_barrier" ::: "memory");
        issue(i + 3);
        if (i >= seen) continue;
        Logits32 y;
        step(i, x, y, mask);
        x = y;
        if (i + 1 < seen) settle(ring[(i + 1) & (kRing - 1)], i + 1, x);
      }
    };
    const int first = max(0, min(whole, n));
    run(0, first, std::false_type{});
    run(first, n, std::true_type{});
    __builtin_amdgcn_s_waitcnt(dev::waitcnt_vm(0));
  }

#pragma unroll
  for (int qt = 0; qt < QT; qt++) {
    const int row = r_half + (w * QT + qt) * 16 + r16;
    const int64_t r = t.r0 + row;
    const bool ok = r < t.rows;
    const float den = den_of(st[qt].l, bad[qt]);
    float f = 1.f;
    float* dst = a.out;
    if (!ok) {
      // its lanes take part in the exchange below
    } else if (a.splits == 1) {
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

Pack pack_of(const View& c, void* packed) {
  Pack pk;
  pk.most = ceil_div(c.max_pages << c.page_log2, 64);
  pk.blocks = static_cast<Packed*>(packed);
  pk.far = reinterpret_cast<int*>(pk.blocks + 2 * pk.most * c.nseq * c.kv_heads);
  return pk;
}

}  // namespace

// Rows enough that turning the keys to operands once costs less than for every 256 of them, and
// operands within bounds. 0: not so.
int64_t kv_packed_bytes(const View& c, int group, const kvplan::Plan& p) {
  const int64_t most = ceil_div(c.max_pages << c.page_log2, 64), pairs = (int64_t)c.nseq * c.kv_heads;
  if (p.rows != kRows || most == 0 || c.T * group / c.nseq < 4 * kRows) return 0;
  const int64_t each = 2 * (int64_t)sizeof(Packed) + 4;
  if (pairs > kvplan::kMaxScratch / each / most) return 0;
  return round_up(pairs * most * each, 16);
}

hipError_t launch_kv_pack(const Args& a, void* packed, hipStream_t s) {
  const Pack pk = pack_of(a.c, packed);
  hipLaunchKernelGGL(kv_pack_kernel, dim3((unsigned)(pk.most * a.c.nseq * a.c.kv_heads)), dim3(512), 0, s,
                     a, pk);
  return hipGetLastError();
}
template <class K>
hipError_t launch_kv_packed(const Args& a, void* packed, unsigned grid, hipStream_t s) {
  hipLaunchKernelGGL(kv_attn_packed_kernel<K>, dim3(2 * grid), dim3(64 * kWaves), 0, s, a,
                     pack_of(a.c, packed));
  return hipGetLastError();
}
template hipError_t launch_kv_packed<Cross>(const Args&, void*, unsigned, hipStream_t);
template hipError_t launch_kv_packed<Counted>(const Args&, void*, unsigned, hipStream_t);

}  // namespace sdq
