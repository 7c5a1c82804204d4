// The softmax weights that each cached key was given, summed over a call's rows (gfx950).
//
// Per key j and cached head, over the call's rows r of the head's group that see it, with
// t_rj = scale log2(e) q_r . k_j + e_j, row r's maximum m_r of t and denominator d_r as the
// attention left them (e_j: the exponent of the key's value scale, see sdq_kv_attn.hip):
//   sum_r 2^(t_rj - m_r - e_j) / d_r.
//
// The logits are formed again, bit for bit as the attention forms them (a row's weights then
// sum to 1 however large they are), two MFMA products each: half of the attention's. That
// left the rows' two fp16 parts in the order of the MFMA operands, so that this kernel moves
// them by LDS-DMA and its loop holds MFMAs, LDS reads and exponentials only.
// A wave keeps 64 keys in registers, the workgroup 512, and the rows pass by in LDS, 64 at a
// time in a ring of three; a lane sums the weights of 16 of its keys for one row of 16, the
// lanes' sums are joined once a block of keys. The products of the next 16 rows stand beside
// the exponentials of the last ones. Few blocks of many rows are cut into ranges of
// rows, whose sums a second kernel adds up in order: no atomics, the same bits every time.
//
// 4099 rows over themselves, 24 heads on 8: 139 us and 4.6 of the join, where the products are 87
// at a large library product's rate; the exponentials beside them and the diagonal's half-used
// blocks are the rest (CUs busy 85% of the time, the matrix units 42% of that, waves waiting for a
// counter or barrier 38% of their life).
#include <algorithm>

#include "sdq_kv_attn.h"
#include "sdq_kv_plan.h"

#pragma clang fp contract(off)

namespace sdq {
namespace {

using namespace kvattn;

constexpr int kWaves = 8;
constexpr int kTiles = 4;                     // of 16 keys, a wave
constexpr int kBlock = 16 * kTiles * kWaves;  // keys of a workgroup
constexpr int kRows = 64;                     // of a stage in LDS
constexpr int kRing = 3;
static_assert(kBlock == kvplan::kCountBlock && kQTile + 16 * sizeof(RowInfo) == kvplan::kCountKept);
constexpr int kLeastLog = 10;                 // of a range's rows (2^8 157 us, 2^12 223, see above)
constexpr int kShortLog = 7;                  // the same where there are workgroups to spare
constexpr int kDma = 5;                       // a wave's, a stage: 4 of the parts, one of the rest

struct Stage {
  __attribute__((aligned(16))) char q[kRows / 16][kQTile];
  RowInfo row[kRows];
};

struct Work {
  float* sums;
  float* part;  // [sequence, head][block, range][kBlock] where rows are cut
  int across;   // workgroups of a sequence and head
  int cut;      // rows may be cut
  int s0;       // the launch's first sequence
};

// How the blocks of keys of a sequence and head, and ranges of 2^log of its rows, are shared out.
struct Cut {
  int blocks, ranges, log;
};
__device__ __forceinline__ Cut cut_of(const Tile& t, const Work& wk) {
  Cut c{(t.len + kBlock - 1) / kBlock, 1, 40};
  if (wk.cut && c.blocks > 0) {
    // up to 4 items a workgroup: a pair's items are fewer than 8 * across
    const int64_t want = (4 * wk.across + c.blocks - 1) / c.blocks;
    // one a CU (half of across) of short ranges, if there are no more: 1100 keys, 8 heads, 1000 rows
    // 111 -> 78 us of the call
    c.log = kShortLog;
    while (c.log < kLeastLog &&
           2 * ((t.rows + (int64_t(1) << c.log) - 1) >> c.log) * c.blocks > wk.across)
      c.log++;
    while ((t.rows + (int64_t(1) << c.log) - 1) >> c.log > want) c.log++;
    c.ranges = (int)((t.rows + (int64_t(1) << c.log) - 1) >> c.log);
  }
  return c;
}
// First row that sees a key of block b, rounded down to a stage's.
__device__ __forceinline__ int64_t first_row(const Args& a, const Tile& t, int b) {
  const int64_t tok = a.causal ? b * kBlock - t.first : 0;
  return tok > 0 ? tok * a.group / kRows * kRows : 0;
}
__global__ void __launch_bounds__(64 * kWaves) kv_weights_kernel(Args a, Work wk) {
  __shared__ Stage ring[kRing];
  __shared__ __attribute__((aligned(16))) float terms[kWaves][2][64];
  const View& c = a.c;
  const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, r16 = l & 15, g = l >> 4;
  const int x = (int)(blockIdx.x % wk.across);
  const int64_t sh = blockIdx.x / wk.across;
  const int h = (int)(sh % c.kv_heads), s = (int)(sh / c.kv_heads);
  const Tile t = rows_of(a, s);
  if (t.rows == 0) return;
  const Cut cut = cut_of(t, wk);
  const auto* table = scalar_ptr(c.table + s * c.max_pages);
  const int e0 = first_exp<Own>(a, t, h);
  const int64_t tile0 = h * a.n16 + t.row0 * a.group / 16 + wk.s0 + s;
  const uint32_t lds = uniform((int)dev::lds_addr32(ring));

  // Items (block, range) in order, those that no row sees left out: every across-th is ours.
  const bool whole = cut.ranges == 1;
  int skip = whole ? 0 : x;
  for (int b = whole ? x : 0; b < cut.blocks; b += whole ? wk.across : 1) {
    const int64_t lead = first_row(a, t, b);
    const int z0 = (int)(lead >> cut.log);
    const int n = lead < t.rows ? cut.ranges - z0 : 0;
    if (skip >= n) {
      if (!whole) skip -= n;
      continue;
    }
    // the wave's keys as MFMA operands and their scales
    const int k0 = b * kBlock + 16 * kTiles * w;
    v8h key[kTiles][4];
    v4f kc[kTiles], ke[kTiles];
    int page[kTiles];
#pragma unroll
    for (int kt = 0; kt < kTiles; kt++) page[kt] = table[min(k0 + 16 * kt, t.len - 1) >> c.page_log2];
    int64_t at[kTiles];
    uint4 raw[kTiles][2];
#pragma unroll
    for (int kt = 0; kt < kTiles; kt++) {  // of the first page where there is none
      if (k0 + 16 * kt >= t.len || page[kt] >= c.pages) page[kt] = -1;
      at[kt] = (((page[kt] < 0 ? 0 : page[kt]) * (int64_t)c.kv_heads + h) << c.page_log2) +
               ((k0 + 16 * kt) & ((1 << c.page_log2) - 1));
      const int8_t* kp = c.k + (at[kt] + r16) * kHd + 16 * g;
      raw[kt][0] = *reinterpret_cast<const uint4*>(kp);
      raw[kt][1] = *reinterpret_cast<const uint4*>(kp + 64);
    }
    // scales: a key a lane, what follows from them handed round in LDS
    const int64_t own = (g == 0 ? at[0] : g == 1 ? at[1] : g == 2 ? at[2] : at[3]) + r16;
    const int own_page = g == 0 ? page[0] : g == 1 ? page[1] : g == 2 ? page[2] : page[3];
    const float ks = c.ks[own], vs = c.vs[own];
    const KeyTerms k = key_terms(ks, vs, own_page >= 0 && k0 + l < t.len, 1.f, e0);
    terms[w][0][l] = k.c, terms[w][1][l] = k.e;
    const bool any_far = __any(k.e < kNear);
#pragma unroll
    for (int kt = 0; kt < kTiles; kt++) {
#pragma unroll
      for (int j = 0; j < 2; j++) {
        key[kt][2 * j] = codes8(raw[kt][j].x, raw[kt][j].y);
        key[kt][2 * j + 1] = codes8(raw[kt][j].z, raw[kt][j].w);
      }
      kc[kt] = *reinterpret_cast<const v4f*>(&terms[w][0][16 * kt + 4 * g]);
      ke[kt] = *reinterpret_cast<const v4f*>(&terms[w][1][16 * kt + 4 * g]);
    }

    for (; skip < n; skip += wk.across) {
      const int z = z0 + skip;
      const int64_t begin = lead > (int64_t)z << cut.log ? lead : (int64_t)z << cut.log;
      const int64_t end = (int64_t)(z + 1) << cut.log < t.rows ? (int64_t)(z + 1) << cut.log : t.rows;
      v4f sum[kTiles];
#pragma unroll
      for (int kt = 0; kt < kTiles; kt++) sum[kt] = v4f{0.f, 0.f, 0.f, 0.f};

      // Stages of 64 rows from `begin` (a multiple of 64); behind the last tile that one again. A
      // wave moves half a tile of parts and an eighth of the rest.
      const int tiles = (int)((end - begin + 15) >> 4), stages = (tiles + 3) >> 2;
      const int64_t first = tile0 + (begin >> 4);
      auto issue = [&](int i, int slot) {
        const uint32_t to = lds + (uint32_t)slot * (uint32_t)sizeof(Stage);
        const int64_t tile = first + min(4 * i + (w >> 1), tiles - 1);
        const dev::v4u parts = dev::raw_rsrc(a.qparts + tile * kQTile, kQTile);
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const uint32_t at = (uint32_t)(w & 1) * 4096 + 1024 * k;
          dev::dma16<4>(parts, l * 16, at, to + (w >> 1) * kQTile + at);
        }
        if (l < 8) {
          const uint32_t at = (uint32_t)(w & 1) * 128;
          dev::dma16<4>(dev::raw_rsrc(a.info + tile * 16, 256), l * 16, at,
                        to + 4 * kQTile + (w >> 1) * 256 + at);
        }
      };
      // Of tiles in order, the first that sees any of the wave's keys and the first that sees all.
      auto from = [&](int key) {
        const int64_t r = a.causal ? (int64_t)(key - t.first) * a.group - begin : 0;
        return r;  // the first row that sees the key
      };
      const int64_t some = from(k0) >> 4, every = (from(k0 + 16 * kTiles - 1) + 15) >> 4;
      struct Scores {
        v4f s[kTiles];
        RowInfo ri;
      };
      // The scores of tile `nx` beside the weights of the tile ahead of it.
      v8h op[2][2];
      auto step = [&](const Stage& d, int nx, bool live, Scores& to, const Scores& of, auto faint,
                      auto mask) {
        constexpr bool kFaint = decltype(faint)::value, kMask = decltype(mask)::value;
        // operands are read a step of eight products ahead, the next tile's first ones too
        auto read = [&](int tile, int kb) {
#pragma unroll
          for (int part = 0; part < 2; part++)
            op[kb & 1][part] = *reinterpret_cast<const v8h*>(d.q[tile] + 4096 * part + 1024 * kb + l * 16);
        };
        to.ri = d.row[16 * nx + r16];
        if (!live) to.ri.m = INFINITY, to.ri.inv = 0.f, to.ri.see = 0;
        // A row that adds nothing: its logits are formed as 0, since one past fp32's range, less the
        // infinite maximum, would be NaN.
        if (to.ri.inv == 0.f) to.ri.qk = 0.f;
        if (kMask || nx == 0) read(nx, 0);  // masked tiles may be left out
#pragma unroll
        for (int kb = 0; kb < 4; kb++) {
          if (kb < 3)
            read(nx, kb + 1);
          else if (!kMask && nx < 3)
            read(nx + 1, 0);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int part = 1; part >= 0; part--)
#pragma unroll
            for (int kt = 0; kt < kTiles; kt++)
              to.s[kt] = mma(key[kt][kb], op[kb & 1][part],
                             kb == 0 && part == 1 ? v4f{0.f, 0.f, 0.f, 0.f} : to.s[kt]);
          const v4f ck = kc[kb] * of.ri.qk;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            float y = __builtin_fmaf(of.s[kb][i], ck[i], ke[kb][i]) - of.ri.m;
            if (kFaint) y -= ke[kb][i];
            if (kMask) y = k0 + 16 * kb + 4 * g + i < of.ri.see ? y : -INFINITY;
            sum[kb][i] = __builtin_fmaf(__builtin_amdgcn_exp2f(y), of.ri.inv, sum[kb][i]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      auto pass = [&](auto faint) {
        Scores sc[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {  // before the first tile: adds nothing
          sc[j].ri = RowInfo{0.f, INFINITY, 0.f, 0};
#pragma unroll
          for (int kt = 0; kt < kTiles; kt++) sc[j].s[kt] = v4f{0.f, 0.f, 0.f, 0.f};
        }
        // tile 4 i + nx, and the weights of the one ahead of it
        auto one = [&](const Stage& d, int i, int nx, Scores& to, const Scores& of, auto mask) {
          if (4 * i + nx >= some) step(d, nx, 4 * i + nx < tiles, to, of, faint, mask);
        };
        __builtin_amdgcn_s_waitcnt(dev::waitcnt_vm(0));
        asm volatile("s_barrier" ::: "memory");  // the last item's rows are read
        issue(0, 0), issue(1, 1);
        int slot = 0, ahead = 2;
        auto run = [&](int i, int to, auto mask) {
          for (; i < to; i++) {
            __builtin_amdgcn_s_waitcnt(dev::waitcnt_vm(kDma));
            asm volatile("s_barrier" ::: "memory");
            issue(i + 2, ahead);
            const Stage& d = ring[slot];
            one(d, i, 0, sc[1], sc[0], mask);
            one(d, i, 1, sc[0], sc[1], mask);
            one(d, i, 2, sc[1], sc[0], mask);
            one(d, i, 3, sc[0], sc[1], mask);
            slot = slot == kRing - 1 ? 0 : slot + 1;
            ahead = ahead == kRing - 1 ? 0 : ahead + 1;
          }
        };
        // Stages whose rows may not see all of the wave's keys, then the others (a row that adds
        // nothing has finite logits and an infinite maximum: only keys ahead of a row are masked).
        const int first = (int)max((int64_t)0, min((int64_t)stages, (every + 4) >> 2));
        run(0, first, std::true_type{});
        run(first, stages, std::false_type{});
        one(ring[0], stages, 0, sc[1], sc[0], std::true_type{});  // the last tile's weights
      };
      if (any_far)
        pass(std::true_type{});
      else
        pass(std::false_type{});

      // the 16 rows' sums of a key lie in 16 lanes; lane r16 then keeps key 4 g + r16 % 4 of tile
      // r16 / 4
      float mine = 0.f;
#pragma unroll
      for (int kt = 0; kt < kTiles; kt++) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float v = any_far ? sum[kt][i] : __builtin_ldexpf(sum[kt][i], -(int)ke[kt][i]);
          // A row that sees a scale of infinity or NaN gives it no weight or has none itself, but
          // makes a NaN here.
          if (!(fabsf(kc[kt][i]) <= 3.402823466e38f)) v = 0.f;
#pragma unroll
          for (int o = 8; o; o >>= 1) v += __shfl_xor(v, o);
          mine = r16 == 4 * kt + i ? v : mine;
        }
      }
      const int p = 16 * kTiles * w + 16 * (r16 >> 2) + 4 * g + (r16 & 3);  // in the block
      if (cut.ranges > 1)
        wk.part[(sh * 8 * wk.across + (int64_t)b * cut.ranges + z) * kBlock + p] = mine;
      else if (b * kBlock + p < t.len) {
        const int64_t at = kv::place_of(c, s, b * kBlock + p, h);
        if (at >= 0) wk.sums[at] = b * kBlock + p < t.first ? wk.sums[at] + mine : mine;
      }
    }
    skip = whole ? 0 : skip - n;
  }
  __builtin_amdgcn_s_waitcnt(dev::waitcnt_vm(0));
}

// Where rows were cut: the ranges' sums of a key, in order, to its place.
__global__ void __launch_bounds__(kBlock) kv_weights_join_kernel(Args a, Work wk) {
  const int64_t sh = blockIdx.x / wk.across;
  const int h = (int)(sh % a.c.kv_heads), s = (int)(sh / a.c.kv_heads);
  const Tile t = rows_of(a, s);
  const Cut cut = cut_of(t, wk);
  if (t.rows == 0 || cut.ranges == 1) return;
  for (int b = (int)(blockIdx.x % wk.across); b < cut.blocks; b += wk.across) {
    const int p = b * kBlock + threadIdx.x;
    const int64_t lead = first_row(a, t, b);
    if (p >= t.len || lead >= t.rows) continue;
    const int64_t at = kv::place_of(a.c, s, p, h);
    if (at < 0) continue;
    float v = p < t.first ? wk.sums[at] : 0.f;
    const float* part = wk.part + (sh * 8 * wk.across + (int64_t)b * cut.ranges) * kBlock + threadIdx.x;
#pragma unroll 4
    for (int z = (int)(lead >> cut.log); z < cut.ranges; z++) v += part[(int64_t)z * kBlock];
    wk.sums[at] = v;
  }
}

}  // namespace

hipError_t launch_kv_weights(const View& c, const KvRows& r, const kvplan::WeightsPlan& p, void* kept, float* w,
                             void* scratch, hipStream_t s) {
  Args a{};
  a.heads = r.heads, a.group = r.heads / c.kv_heads;
  a.causal = r.causal;
  a.qparts = static_cast<char*>(kept);
  a.info = reinterpret_cast<RowInfo*>(a.qparts + p.n16 * c.kv_heads * kQTile);
  a.n16 = p.n16;
  Work wk{w, static_cast<float*>(scratch), p.across, p.cut, 0};
  for (int s0 = 0; s0 < c.nseq; s0 += p.seqs) {
    a.c = c;
    a.c.q_start += s0, a.c.lens += s0, a.c.table += s0 * c.max_pages;
    a.c.nseq = std::min(p.seqs, c.nseq - s0);
    wk.s0 = s0;
    const dim3 grid((unsigned)((int64_t)p.across * a.c.nseq * c.kv_heads));
    hipLaunchKernelGGL(kv_weights_kernel, grid, dim3(64 * kWaves), 0, s, a, wk);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (!p.cut) continue;
    hipLaunchKernelGGL(kv_weights_join_kernel, grid, dim3(kBlock), 0, s, a, wk);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace sdq
