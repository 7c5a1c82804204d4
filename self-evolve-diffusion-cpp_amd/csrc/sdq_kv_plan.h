// Host arithmetic of the paged attention, of the sums of its weights and of eviction: tile height,
// share count and scratch of a call, from sizes alone (plain C++, no device code).
#pragma once

#include <algorithm>
#include <cstdint>
#include <initializer_list>

namespace sdq {
namespace kvplan {

constexpr int kFewRows = 16;  // rows of a tile of the few-row form
constexpr int kFewWaves = 4;
constexpr int64_t kMaxScratch = int64_t(1) << 29;
constexpr int kMaxSplits = 64;

struct Plan {
  int rows;                  // of a tile: 16 (few rows), 64 or 256 (chunks)
  int splits;                // shares that the keys are cut into
  int64_t tiles;             // numbers of tiles, over all sequences
  int64_t tiles_per_launch;
  int64_t part_bytes;        // partial sums; maxima and denominators follow
  int64_t scratch_bytes;     // 0: none
};

// Whose plan: a sequence's last tokens over its own keys; rows over other keys; shared parts'
// rows over those, and over the keys behind them.
enum Kind { kOwn, kCross, kPart, kRest };
constexpr int kWhole = 768;  // keys that cross attention's few rows take in one share

// T rows of nseq sequences, group query heads to each of kv_heads cached ones,
// most: the keys a sequence can have.
inline Plan plan(int64_t T, int nseq, int group, int kv_heads, int64_t most, int cu_count,
                 Kind kind = kOwn) {
  Plan p{};
  const int64_t rows = T * group;
  // Rows of a sequence, on average: only their sum is known here. Any choice is
  // right for any lengths (us, four sequences over 4099 keys): 24 cached heads, 32 rows 47 with
  // 16 and 68 with 64, 48 rows 63 and 76, 96 rows 99, 114 with 64 and 117 with 256, 160 rows 131,
  // 151 and 165, 256 rows 184, 209 and 185; 8 cached heads, 24 rows 26 and 39, 48 rows 33 and 41,
  // 72 rows 39 and 42, 144 rows 61, 68 and 48.
  const int64_t mean = (rows + nseq - 1) / nseq;
  p.rows = mean <= 32 ? kFewRows : mean <= 128 ? 64 : 256;
  // parts of 32768 keys, 24 heads, 64 rows 91 with 64 and 119 with 128, 96 rows 171 and 126
  if (mean > 64 && kind == kPart) p.rows = 128;
  // Few rows' tiles have the shorter way from a call to its result, and one for each 16 rows has
  // more of the CUs (us, cross attention): 512 keys, 8 cached heads, one sequence of 256 rows 11.6
  // for 26.8 with 64 and 38.9 with 256; 24 heads, four of 128 rows 23.7, 33.2 and 31.2, but
  // sixteen of 64 rows 42.9, 37.2 and 58.7. 4099 keys: 24 heads, four of 96 rows 100, 115, 121;
  // sixteen 303, 434, 411; 8 heads, four of 128 rows 44.3, 44.2, 43.8, one of 256 rows 33, 36 and
  // 48. Shared parts of 8209 keys, 8 heads: 256 rows 47 for 57 with 128, 512 rows 78 for 77; 300 keys
  // behind them, four of 48 rows 42 for 48 with 64. Each tile reads its keys, which over long ones
  // is what it waits for: shared parts of 8 heads, 64 rows over 32768 keys 46 for 52 with 64, over
  // 131072 137 for 116, 128 rows 250 for 169 with 128. From 1024 rows on cross attention's chunks have
  // an order of their own (sdq_kv_packed.hip). Own keys keep the heights above, and their bits.
  const int64_t few = (mean + kFewRows - 1) / kFewRows * nseq * kv_heads;  // workgroups
  const bool whole = kind == kCross && most <= kWhole;
  const bool small = mean <= 256 && few <= cu_count / 2 && few * most <= int64_t(1) << 21;
  if (whole ? mean < 1024 && few <= 4 * cu_count : (kind == kCross && mean <= 96) || (kind != kOwn && small))
    p.rows = kFewRows;
  // Numbers of tiles: rows / height and one a sequence (csrc/sdq_kv_attn.hip); those that
  // hold one are at most the sum of ceil(rows_s / height) over the sequences that have any.
  p.tiles = rows / p.rows + nseq;
  const int64_t groups =  // workgroups without a cut
      (rows + std::min<int64_t>(nseq, T) * (p.rows - 1)) / p.rows * kv_heads;
  // Enough workgroups for every CU. A few-row one is four waves that wait for memory, and
  // two fit a CU at once: three to a CU (8 ragged sequences x 24 heads up to 4099 keys: two 36
  // us, three 27, four 29, six 32). A chunk's of 256 rows takes a CU's registers, and the
  // second round evens out what the first leaves idle.
  const int64_t want = (p.rows == kFewRows ? 3 : p.rows == 64 ? 4 : 2) * (int64_t)cu_count;
  const int64_t least = p.rows == kFewRows ? 256 : 512;  // keys of a share
  int64_t s = std::min<int64_t>(want / std::max<int64_t>(groups, 1), most / least);
  s = std::max<int64_t>(1, std::min<int64_t>(s, kMaxSplits));
  // Joining costs a launch, 3 us and more: 512 keys 12.6 us for 15.9 in two shares (8 rows, 24
  // heads), 700 keys 15.0 for 16.9, 1024 keys 17.7 for 21.5, but 17.3 for 15.8 of 4 rows.
  if (p.rows == kFewRows && whole) s = 1;
  const int64_t per = (int64_t)kv_heads * p.rows * (128 + 2) * 4;  // bytes a tile and share
  while (s > 1 && p.tiles * per * s > kMaxScratch) s--;
  p.splits = (int)s;
  // a launch's threads (the join has up to 256 a row) stay under 2^31
  const int64_t threads = (int64_t)kv_heads * std::max<int64_t>(512 * s, 256 * p.rows);
  p.tiles_per_launch = std::max<int64_t>(1, ((int64_t(1) << 31) - 1) / threads);
  if (s > 1) p.tiles_per_launch = std::max(p.tiles_per_launch, p.tiles);
  if (s > 1) {
    p.part_bytes = p.tiles * kv_heads * s * p.rows * 128 * 4;
    p.scratch_bytes = p.part_bytes / 128 * 130;
  }
  return p;
}

// Attention over shared parts and own keys: their shares' sums one beside the other for every
// row, cached heads at a time that the scratch takes.
struct SharedPlan {
  Plan pre, own;
  int want;                 // workgroups that the parts' shares are to make
  int pre_least, own_least; // keys of a share
  int heads;                // cached heads at a time
  int64_t part_bytes;       // partial sums; maxima and denominators follow
  int64_t scratch_bytes;
};
constexpr int kMaxShares = 128, kMaxOwnShares = 16;

// n shared parts of up to most_pre tokens.
inline SharedPlan shared_plan(int64_t T, int nseq, int n, int group, int kv_heads, int64_t most,
                              int64_t most_pre, int cu_count) {
  SharedPlan p{};
  p.own = plan(T, nseq, group, kv_heads, most, cu_count, kRest);
  p.own.splits = std::min(p.own.splits, kMaxOwnShares);
  p.pre = plan(T, n, group, kv_heads, most_pre, cu_count, kPart);
  // How many tiles the parts' rows make is known on the device, which cuts their keys into that
  // many shares that two workgroups a CU are at work; here the most that can be. Rows of no
  // sequence, and tiles that a part does not fill, leave room for one more than the rows say.
  p.want = 2 * cu_count;
  p.pre_least = p.own_least = 256;
  const int64_t tiles = std::max<int64_t>(1, T * group / p.pre.rows);
  const int64_t s = std::min<int64_t>(p.want / std::max<int64_t>(tiles * kv_heads, 1), most_pre / p.pre_least);
  p.pre.splits = (int)std::max<int64_t>(1, std::min<int64_t>(s, kMaxShares - kMaxOwnShares));
  const int shares = p.own.splits + p.pre.splits;
  const int64_t head = T * group * shares * (128 + 2) * 4;
  p.heads = (int)std::max<int64_t>(1, std::min<int64_t>(kv_heads, kMaxScratch / std::max<int64_t>(head, 1)));
  for (Plan* q : {&p.pre, &p.own})
    q->tiles_per_launch = std::max<int64_t>(
        1, ((int64_t(1) << 30) - 1) / ((int64_t)p.heads * q->splits * 512));
  p.part_bytes = T * group * p.heads * shares * 128 * 4;
  p.scratch_bytes = p.part_bytes / 128 * 130;
  return p;
}

// The sums of weights by key that form the logits again (sdq_kv_weights.hip).
constexpr int kCountBlock = 512;            // keys of a workgroup
constexpr int kCountKept = 8192 + 16 * 16;  // bytes that the attention leaves of a tile of 16 rows
struct WeightsPlan {
  int across;   // workgroups of a sequence and head
  int cut;      // its rows may be cut into ranges
  int seqs;     // sequences at a time
  int64_t n16;  // numbers of tiles of 16 rows
  int64_t kept_bytes, scratch_bytes;
};
inline WeightsPlan weights_plan(int64_t T, int nseq, int group, int kv_heads, int64_t most, int cu_count) {
  WeightsPlan p{};
  p.n16 = T * group / 16 + nseq;
  p.kept_bytes = p.n16 * kv_heads * kCountKept;
  // One workgroup to a CU at once, two rounds of them.
  const int64_t pairs = (int64_t)nseq * kv_heads, want = 2 * (int64_t)cu_count;
  const int64_t many = (want + pairs - 1) / pairs;
  // sequences at a time that a grid's 32-bit thread count takes, and 512 MiB of ranges' sums
  const int64_t ranges = kMaxScratch / (8 * kCountBlock * 4);
  p.cut = T * group / nseq >= 128 && many * kv_heads <= ranges;
  const int64_t blocks = (std::max<int64_t>(most, 1) + kCountBlock - 1) / kCountBlock;
  p.across = (int)std::max<int64_t>(1, std::min(p.cut ? want : blocks, many));
  p.seqs = (int)std::min<int64_t>(
      nseq, std::max<int64_t>(1, (p.cut ? ranges : int64_t(1) << 22) / ((int64_t)p.across * kv_heads)));
  if (p.cut) p.scratch_bytes = (int64_t)p.seqs * kv_heads * 8 * p.across * kCountBlock * 4;
  return p;
}

// Eviction (sdq_kv_evict.hip). Tables longer than a workgroup's registers: chunks of whole times
// 16384 tokens, at most 64 of them, and fewer where the cached heads are so many that a sequence's
// counts would pass 256 MiB (from 171 heads on; one chunk has 24.1 KiB a head).
constexpr int kEvictRegisters = 16384;  // tokens
constexpr int64_t kEvictCounts = 3 * 2048 * 4, kEvictFound = 3 * 32, kEvictScratch = int64_t(1) << 28;
struct EvictPlan {
  int seqs;       // sequences at a time
  int chunks;     // of a sequence, 0: it fits a workgroup
  int64_t chunk;  // tokens
  int64_t scratch_bytes;
};
inline EvictPlan evict_plan(int nseq, int kv_heads, int64_t most) {
  EvictPlan p{};
  p.seqs = std::max(1, (1 << 21) / kv_heads);  // a grid's threads are a 32-bit number
  if (most > kEvictRegisters) {
    const int64_t fit = (kEvictScratch / kv_heads - kEvictFound) / kEvictCounts;
    const int64_t chunks =
        std::max<int64_t>(1, std::min<int64_t>({64, (1 << 20) / kv_heads, fit}));
    p.chunk = ((most + chunks - 1) / chunks + kEvictRegisters - 1) / kEvictRegisters * kEvictRegisters;
    p.chunks = (int)((most + p.chunk - 1) / p.chunk);
    const int64_t pair = p.chunks * kEvictCounts + kEvictFound;
    p.seqs = (int)std::max<int64_t>(1, std::min<int64_t>(kEvictScratch / (pair * kv_heads),
                                                         (1 << 20) / ((int64_t)p.chunks * kv_heads)));
    p.seqs = std::min(p.seqs, nseq);
    p.scratch_bytes = pair * kv_heads * p.seqs;
  }
  return p;
}

}  // namespace kvplan
}  // namespace sdq
