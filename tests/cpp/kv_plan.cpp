// Sweeps the paged attention's plan (csrc/sdq_kv_plan.h): every launch's grid and every
// tile's scratch within bounds, whatever the lengths of the sequences.
#include <cstdio>
#include <random>

#include "sdq_kv_plan.h"

namespace kp = sdq::kvplan;

#define REQUIRE(c)                                                                     \
  if (!(c)) {                                                                          \
    std::printf("T=%lld nseq=%d group=%d kvh=%d most=%lld: %s\n", (long long)T, nseq,  \
                group, kvh, (long long)most, #c);                                      \
    return 1;                                                                          \
  }

int main() {
  std::mt19937_64 rng(1);
  auto log_size = [&](int bits) {
    const int64_t top = int64_t(1) << (rng() % (bits + 1));
    return 1 + (int64_t)(rng() % top);
  };
  for (int i = 0; i < 200000; i++) {
    const int kvh = (int)log_size(i % 3 ? 6 : 15);
    const int group = (int)std::min<int64_t>(log_size(6), 65535 / kvh);
    if (group < 1) continue;
    const int64_t T = std::min(log_size(30), (int64_t(1) << 33) / kvh);
    const int nseq = (int)std::min<int64_t>(log_size(16), 65535);
    const int64_t most = i % 50 ? log_size(30) : 0;
    const kp::Plan p = kp::plan(T, nseq, group, kvh, most, 256);
    REQUIRE(p.rows == 16 || p.rows == 64 || p.rows == 256);
    REQUIRE(p.splits >= 1 && p.splits <= kp::kMaxSplits);
    // ragged sequences: each has as many numbers as tiles, the last one within the plan's
    int64_t at = 0;
    const int seqs = std::min(nseq, 40);
    for (int s = 0; s < seqs; s++) {
      const int64_t end = s == nseq - 1 || rng() % 8 == 0 ? T : at + (int64_t)(rng() % (T - at + 1));
      const int64_t first = at * group / p.rows + s, next = end * group / p.rows + s + 1;
      REQUIRE(next - first >= ((end - at) * group + p.rows - 1) / p.rows);
      REQUIRE(next <= p.tiles);
      at = end;
    }
    REQUIRE(p.tiles_per_launch >= 1);
    const int64_t n = std::min(p.tiles, p.tiles_per_launch) * kvh;
    const int64_t block = p.rows == 16 ? 64 * kp::kFewWaves : p.rows == 64 ? 256 : 512;
    REQUIRE(n * p.splits <= 0xffffffffll && n * p.splits * block <= 0xffffffffll);
    if (p.splits > 1) {
      REQUIRE(p.tiles_per_launch >= p.tiles);  // shares are numbered over one launch
      REQUIRE(n * p.rows * 256 <= 0xffffffffll);
      REQUIRE(p.part_bytes == n * p.splits * p.rows * 128 * 4);
      REQUIRE(p.scratch_bytes >= p.part_bytes + n * p.splits * p.rows * 8);
      REQUIRE(p.scratch_bytes <= kp::kMaxScratch);
    } else {
      REQUIRE(p.scratch_bytes == 0);
    }
  }
  return 0;
}
