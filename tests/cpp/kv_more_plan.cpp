// Sweeps the plans of the weights' sums and of eviction (csrc/sdq_kv_plan.h): every launch's grid
// and the scratch within bounds, and chunks that cover their table.
#include <cstdio>
#include <random>

#include "sdq_kv_plan.h"

namespace kp = sdq::kvplan;

#define REQUIRE(c)                                                                           \
  if (!(c)) {                                                                                \
    std::printf("T=%lld nseq=%d group=%d kvh=%d most=%lld: %s\n", (long long)T, nseq, group, \
                kvh, (long long)most, #c);                                                   \
    return 1;                                                                                \
  }

int main() {
  std::mt19937_64 rng(3);
  auto log_size = [&](int bits) {
    const int64_t top = int64_t(1) << (rng() % (bits + 1));
    return 1 + (int64_t)(rng() % top);
  };
  for (int i = 0; i < 400000; i++) {
    const int kvh = (int)std::min<int64_t>(log_size(i % 3 ? 8 : 16), 65535);
    const int group = (int)std::min<int64_t>(log_size(6), std::max(1, 65535 / kvh));
    const int64_t T = std::min(log_size(30), (int64_t(1) << 31) / ((int64_t)kvh * group));
    if (T < 1) continue;
    const int nseq = (int)std::min<int64_t>(log_size(16), 65535);
    const int64_t most = i % 50 ? log_size(30) : 0;

    const kp::WeightsPlan w = kp::weights_plan(T, nseq, group, kvh, most, 256);
    REQUIRE(w.across >= 1 && w.seqs >= 1 && w.seqs <= nseq);
    REQUIRE((int64_t)w.seqs * kvh * w.across * kp::kCountBlock <= 0xffffffffll);
    REQUIRE(w.n16 >= T * group / 16 + nseq && w.kept_bytes >= w.n16 * kvh * kp::kCountKept);
    REQUIRE(w.scratch_bytes <= kp::kMaxScratch);
    // fewer than 8 * across ranges' sums of a sequence and head (cut_of in sdq_kv_weights.hip)
    REQUIRE(!w.cut || w.scratch_bytes >= (int64_t)w.seqs * kvh * 8 * w.across * kp::kCountBlock * 4);

    const kp::EvictPlan e = kp::evict_plan(nseq, kvh, most);
    REQUIRE(e.seqs >= 1);
    const int64_t pairs = (int64_t)std::min(e.seqs, nseq) * kvh;
    if (most <= kp::kEvictRegisters) {
      REQUIRE(e.chunks == 0 && e.scratch_bytes == 0 && pairs * 1024 <= 0xffffffffll);
      continue;
    }
    REQUIRE(e.chunks >= 1 && e.chunk % kp::kEvictRegisters == 0 && e.chunks * e.chunk >= most);
    REQUIRE((e.chunks - 1) * e.chunk < most);
    REQUIRE(pairs * e.chunks * 1024 <= 0xffffffffll);
    REQUIRE(e.scratch_bytes >= pairs * (e.chunks * kp::kEvictCounts + kp::kEvictFound));
    REQUIRE(e.scratch_bytes <= kp::kEvictScratch ||
            (e.chunks == 1 && e.seqs == 1 && e.scratch_bytes <= kvh * (kp::kEvictCounts + kp::kEvictFound)));
    // as many chunks as there were without the bound, where it does not bind
    REQUIRE(kvh > 170 || e.chunk < most / 64 + kp::kEvictRegisters + 1);
  }
  return 0;
}
