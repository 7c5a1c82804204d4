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

constexpr int kWaves = 8;
constexpr int kTiles = 4;                     // of 16 keys, a wave
constexpr int kBlock = 16 * kTiles * kWaves;  // keys of a workgroup
constexpr int kRows = 32;                     // in LDS
constexpr int kLeastLog = 8;                  // of a range's rows

struct RowInfo {
  float qk, m, inv;
  int see;  // keys; 0: the row adds nothing
};
struct Stage {
  __attribute__((aligned(16))) char q[2][kRows / 16][4][1024];  // [hi, lo][tile][kb][lane 16 B]
  RowInfo row[kRows];
};

struct Work {
  float* sums;
  float* part;  // [sequence, head][block, range][kBlock] where rows are cut
  int across;   // workgroups of a sequence and head
  int cut;      // rows may be cut
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
    c.log = kLeastLog;
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
  __shared__ Stage buf[2];
  const View& c = a.c;
  const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, r16 = l & 15, g = l >> 4;
  const int x = (int)(blockIdx.x % wk.across);
  const int64_t sh = blockIdx.x / wk.across;
  const int h = (int)(sh % c.kv_heads), s = (int)(sh / c.kv_heads);
  const Tile t = rows_of(a, s);
  if (t.rows == 0) return;
  const Cut cut = cut_of(t, wk);
  const int32_t* table = c.table + s * c.max_pages;
  const int e0 = first_exp<Own>(a, t, h);
  const int step_tok = kRows / a.group, step_qh = kRows % a.group;

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
    bool far = false;
#pragma unroll
    for (int kt = 0; kt < kTiles; kt++) {
      const int p = k0 + 16 * kt;
      const int page = p < t.len ? table[p >> c.page_log2] : -1;
      const bool there = page >= 0 && page < c.pages;
      const int64_t at = (((there ? page : 0) * (int64_t)c.kv_heads + h) << c.page_log2) +
                         (p & ((1 << c.page_log2) - 1));
      const int8_t* kp = c.k + (at + r16) * kHd + 16 * g;
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const uint4 r = *reinterpret_cast<const uint4*>(kp + 64 * j);
        key[kt][2 * j] = codes8(r.x, r.y);
        key[kt][2 * j + 1] = codes8(r.z, r.w);
      }
      const v4f ks = *reinterpret_cast<const v4f_any*>(c.ks + at + 4 * g);
      const v4f vs = *reinterpret_cast<const v4f_any*>(c.vs + at + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const KeyTerms k =
            key_terms(ks[i], vs[i], there && p + 4 * g + i < t.len, 1.f, e0);
        kc[kt][i] = k.c, ke[kt][i] = k.e;
        far |= k.e < kNear;
      }
    }
    const bool any_far = __any(far);

    for (; skip < n; skip += wk.across) {
      const int64_t z = z0 + skip;
      const int64_t begin = lead > z << cut.log ? lead : z << cut.log;
      const int64_t end = (z + 1) << cut.log < t.rows ? (z + 1) << cut.log : t.rows;
      v4f sum[kTiles];
#pragma unroll
      for (int kt = 0; kt < kTiles; kt++) sum[kt] = v4f{0.f, 0.f, 0.f, 0.f};

      // A stage's rows: 8 dims a thread, loaded one stage ahead of their turn to fp16. The row's
      // token and query head go on by what kRows rows are.
      const int row = tid >> 4, j = tid & 15;
      int tok = (int)((begin + row) / a.group), qh = (int)(begin + row - (int64_t)tok * a.group);
      const int rows = (int)(end - begin);
      v4f raw[2];
      float2 st;
      int see;
      auto load = [&](int r0) {
        const bool ok = r0 + row < rows;
        const int64_t at = t.row0 + (ok ? tok : 0);
        const int head = h * a.group + (ok ? qh : 0);
        const float* q = a.q + at * a.ldq + (int64_t)head * kHd + 8 * j;
#pragma unroll
        for (int i = 0; i < 2; i++) raw[i] = *reinterpret_cast<const v4f*>(q + 4 * i);
        st = a.stats[at * a.heads + head];
        const int p = t.first + tok;
        see = !ok || p < 0 ? 0 : a.causal && p < t.len ? p + 1 : t.len;
        tok += step_tok, qh += step_qh;
        if (qh >= a.group) qh -= a.group, tok++;
      };
      auto stage = [&](Stage& d) {
        float v[8], mx = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float f = raw[i >> 2][i & 3];
          v[i] = fabsf(f) <= 3.402823466e38f ? f : 0.f;
          mx = fmaxf(mx, fabsf(v[i]));
        }
#pragma unroll
        for (int o = 8; o; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        const int e = q_exp(mx);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __builtin_ldexpf(v[i], e);
        // dims 8 j ..: k slots 8 (j / 2 % 4) + i of step 2 (j / 8) + j % 2
        v8h hi, lo;
        parts8(v, hi, lo);
        const int off = (16 * ((j >> 1) & 3) + (row & 15)) * 16, kb = 2 * (j >> 3) + (j & 1);
        *reinterpret_cast<v8h*>(d.q[0][row >> 4][kb] + off) = hi;
        *reinterpret_cast<v8h*>(d.q[1][row >> 4][kb] + off) = lo;
        if (j == 0)
          d.row[row] = RowInfo{__builtin_ldexpf(a.scale2, -e), st.x, st.y, st.y > 0.f ? see : 0};
      };
      auto compute = [&](const Stage& d, auto faint) {
        constexpr bool kFaint = decltype(faint)::value;
        constexpr int kRt = kRows / 16;
        RowInfo ri[kRt];
        bool some = false, every = true;
#pragma unroll
        for (int rt = 0; rt < kRt; rt++) {
          ri[rt] = d.row[16 * rt + r16];
          some |= ri[rt].see > k0;
          every &= ri[rt].see >= k0 + 16 * kTiles;
        }
        if (!__any(some)) return;
        v4f sc[kRt][kTiles];
#pragma unroll
        for (int rt = 0; rt < kRt; rt++)
#pragma unroll
          for (int kt = 0; kt < kTiles; kt++) sc[rt][kt] = v4f{0.f, 0.f, 0.f, 0.f};
        // a step's operands are read before the products of the step ahead of it
        v8h op[2][2][kRt];
        auto read = [&](int kb) {
#pragma unroll
          for (int part = 0; part < 2; part++)
#pragma unroll
            for (int rt = 0; rt < kRt; rt++)
              op[kb & 1][part][rt] = *reinterpret_cast<const v8h*>(d.q[part][rt][kb] + l * 16);
        };
        read(0);
#pragma unroll
        for (int kb = 0; kb < 4; kb++) {
          if (kb < 3) read(kb + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int part = 1; part >= 0; part--)
#pragma unroll
            for (int rt = 0; rt < kRt; rt++)
#pragma unroll
              for (int kt = 0; kt < kTiles; kt++)
                sc[rt][kt] = mma(key[kt][kb], op[kb & 1][part][rt], sc[rt][kt]);
          __builtin_amdgcn_sched_barrier(0);
        }
        auto add = [&](auto mask) {
#pragma unroll
          for (int rt = 0; rt < kRt; rt++)
#pragma unroll
            for (int kt = 0; kt < kTiles; kt++) {
              const v4f ck = kc[kt] * ri[rt].qk;
#pragma unroll
              for (int i = 0; i < 4; i++) {
                float y = __builtin_fmaf(sc[rt][kt][i], ck[i], ke[kt][i]) - ri[rt].m;
                if (kFaint) y -= ke[kt][i];
                if (decltype(mask)::value) y = k0 + 16 * kt + 4 * g + i < ri[rt].see ? y : -INFINITY;
                sum[kt][i] = __builtin_fmaf(__builtin_amdgcn_exp2f(y), ri[rt].inv, sum[kt][i]);
              }
            }
        };
        if (__all(every))
          add(std::false_type{});
        else
          add(std::true_type{});
      };
      auto pass = [&](auto faint) {
        load(0);
        __syncthreads();  // the last item's rows are read
        stage(buf[0]);
        load(kRows);
        __syncthreads();
        int n = 0;
        for (int r0 = 0; r0 < rows; r0 += kRows, n ^= 1) {
          if (r0 + kRows < rows) {
            stage(buf[n ^ 1]);
            load(r0 + 2 * kRows);
          }
          compute(buf[n], faint);
          __syncthreads();
        }
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

KvWeightsPlan plan_kv_weights(int64_t T, int nseq, int group, int kv_heads, int64_t most, int cu_count) {
  KvWeightsPlan p{};
  // One workgroup to a CU at once, four rounds of them.
  const int64_t pairs = (int64_t)nseq * kv_heads, want = 4 * (int64_t)cu_count;
  p.cut = T * group / nseq >= 128;
  const int64_t blocks = ceil_div(std::max<int64_t>(most, 1), kBlock);
  p.across = (int)std::max<int64_t>(1, std::min(p.cut ? want : blocks, ceil_div(want, pairs)));
  // sequences at a time that a grid's 32-bit thread count takes
  p.seqs = (int)std::min<int64_t>(nseq, std::max<int64_t>(1, (int64_t(1) << 22) / ((int64_t)p.across * kv_heads)));
  if (p.cut) p.scratch_bytes = (int64_t)p.seqs * kv_heads * 8 * p.across * kBlock * 4;
  return p;
}

hipError_t launch_kv_weights(const View& c, const KvRows& r, const float2* stats, float* w,
                             const KvWeightsPlan& p, void* scratch, hipStream_t s) {
  Args a{};
  a.c = c;
  a.q = r.q, a.ldq = r.ldq;
  a.heads = r.heads, a.group = r.heads / c.kv_heads;
  a.scale2 = r.scale * 1.44269504088896341f;
  a.causal = r.causal;
  a.stats = const_cast<float2*>(stats);
  const Work wk{w, static_cast<float*>(scratch), p.across, p.cut};
  for (int s0 = 0; s0 < c.nseq; s0 += p.seqs) {
    a.c = c;
    a.c.q_start += s0, a.c.lens += s0, a.c.table += s0 * c.max_pages;
    a.c.nseq = std::min(p.seqs, c.nseq - s0);
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
