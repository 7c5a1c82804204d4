// Sweeps the plans of attention over shared parts and of cross attention (csrc/sdq_kv_plan.h):
// every launch's grid and the scratch within bounds, and the shares of a row as many as a wave's
// lanes take.
#include <cstdio>
#include <random>

#include "sdq_kv_plan.h"

namespace kp = sdq::kvplan;

#define REQUIRE(c)                                                                           \
  if (!(c)) {                                                                                \
    std::printf("T=%lld nseq=%d n=%d group=%d kvh=%d most=%lld %lld: %s\n", (long long)T, nseq, \
                n, group, kvh, (long long)most, (long long)pre, #c);                         \
    return 1;                                                                                \
  }

int main() {
  std::mt19937_64 rng(2);
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
    const int n = (int)std::min<int64_t>(log_size(i % 2 ? 3 : 16), 65535);
    const int64_t most = i % 50 ? log_size(30) : 0, pre = i % 49 ? log_size(30) : 0;
    const kp::SharedPlan p = kp::shared_plan(T, nseq, n, group, kvh, most, pre, 256);
    const int shares = p.pre.splits + p.own.splits;
    REQUIRE(p.pre.splits >= 1 && p.own.splits >= 1 && shares <= kp::kMaxShares);
    REQUIRE(p.heads >= 1 && p.heads <= kvh);
    REQUIRE(p.part_bytes == T * group * p.heads * shares * 512);
    REQUIRE(p.scratch_bytes >= p.part_bytes + T * group * p.heads * shares * 8);
    REQUIRE(p.scratch_bytes <= kp::kMaxScratch || p.heads == 1);
    for (const kp::Plan* q : {&p.pre, &p.own}) {
      const int64_t at_once = std::min(q->tiles, q->tiles_per_launch);
      const int64_t block = q->rows == 16 ? 64 * kp::kFewWaves : q->rows == 64 ? 256 : 512;
      REQUIRE(q->tiles_per_launch >= 1);
      REQUIRE(at_once * p.heads * q->splits * block <= 0xffffffffll);
      REQUIRE(q->tiles >= T * group / q->rows);
    }
    const kp::Plan c = kp::plan(T, nseq, group, kvh, most, 256, kp::kCross);
    const int64_t at_once = std::min(c.tiles, c.tiles_per_launch) * kvh * c.splits;
    REQUIRE(c.rows == 16 || c.rows == 64 || c.rows == 256);
    REQUIRE(c.splits >= 1 && c.splits <= kp::kMaxSplits && c.tiles_per_launch >= 1);
    REQUIRE(c.tiles >= T * group / c.rows + nseq);
    REQUIRE(at_once * 512 <= 0xffffffffll && c.scratch_bytes <= kp::kMaxScratch);
    REQUIRE(c.splits == 1 || (c.tiles_per_launch >= c.tiles && c.scratch_bytes > c.part_bytes));
    REQUIRE(c.splits == 1 || at_once / c.splits * c.rows * 256 <= 0xffffffffll);
  }
  return 0;
}
