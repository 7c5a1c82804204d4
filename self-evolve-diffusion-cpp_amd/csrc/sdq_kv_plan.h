// Host arithmetic of the paged attention: tile height, share count and scratch
// of a call, from sizes alone (plain C++, no device code).
#pragma once

#include <algorithm>
#include <cstdint>

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

// T rows of nseq sequences, group query heads to each of kv_heads cached ones,
// most: the keys a sequence can have.
inline Plan plan(int64_t T, int nseq, int group, int kv_heads, int64_t most, int cu_count) {
  Plan p{};
  const int64_t rows = T * group;
  // Rows of a sequence, on average: only their sum is known here. Any choice is
  // right for any lengths. Where the taller tile is faster (us, four sequences over 4099
  // keys): 24 cached heads, 32 rows 54 with 16 and 68 with 64, 48 rows 78 and 77, 96 rows 115
  // with 64 and 121 with 256, 160 rows 156 and 169, 256 rows 209 and 189; 8 cached heads, 24
  // rows 30 and 39, 48 rows 38 and 40, 72 rows 42 and 41, 144 rows 68 and 49.
  const int64_t mean = (rows + nseq - 1) / nseq;
  p.rows = mean <= 32 ? kFewRows : mean <= 128 ? 64 : 256;
  // Numbers of tiles: rows / height and one a sequence (csrc/sdq_kv_attn.hip); those that
  // hold one are at most the sum of ceil(rows_s / height) over the sequences that have any.
  p.tiles = rows / p.rows + nseq;
  const int64_t groups =  // workgroups without a cut
      (rows + std::min<int64_t>(nseq, T) * (p.rows - 1)) / p.rows * kv_heads;
  // Enough workgroups for every CU. A few-row one is four waves that wait for memory, and
  // two fit a CU at once: three to a CU (8 sequences x 24 heads x 4099 keys: two 52 us,
  // three 42, four 45, six 47). A chunk's of 256 rows takes a CU's registers, and the
  // second round evens out what the first leaves idle.
  const int64_t want = (p.rows == kFewRows ? 3 : p.rows == 64 ? 4 : 2) * (int64_t)cu_count;
  const int64_t least = p.rows == kFewRows ? 256 : 512;  // keys of a share
  int64_t s = std::min<int64_t>(want / std::max<int64_t>(groups, 1), most / least);
  s = std::max<int64_t>(1, std::min<int64_t>(s, kMaxSplits));
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

}  // namespace kvplan
}  // namespace sdq
