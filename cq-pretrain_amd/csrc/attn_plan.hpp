// How a call of the attention over the 4-bit pages runs (host code; internal to libcqgdn).
#pragma once
#include <stdint.h>

#include <algorithm>

namespace cqgdn {

constexpr int kWaves = 4;         // of a workgroup; they take its steps in turn
constexpr int kStep = 64;         // positions of a wave's step
constexpr int kMaxSplits = 512;   // parts of a call by either kernel, which the join holds the weights of
// Rows of a request and key head above which its positions are converted once for all of them (attn_tile.hip)
// and not once for every 16: over up to 2000 positions of 64 requests (D = 128) 36 rows take 27 us here and 35 there, 64
// rows 31 and 38, 128 rows 55 and 47; with D = 64 64 rows 26 and 27, 128 rows 39 and 36.
constexpr int kFewRows = 48;
// Positions of a request that can be seen: limits are 32-bit, and a step may begin behind the last position and ask
// for the one after it.
constexpr int kAttendRoom = INT32_MAX - 1024;

// How a call runs: by which kernel, and in how many parts of the positions, of `per` steps each (decode).
struct AttendPlan {
  bool tiles;
  int splits, per;
};
// `capacity` positions a table row holds, of which kAttendRoom can be seen: (splits - 1) per kStep < that, so a part's
// first position needs no more than 32 bits.  With a window a row sees no more of them than it, and never more parts.
inline AttendPlan attend_plan(int64_t N, int kv_heads, int group, int D, int max_queries, int64_t capacity, int window) {
  const int64_t rows = (int64_t)max_queries * group;
  capacity = std::min<int64_t>(capacity, kAttendRoom);
  int64_t seen = window > 0 ? std::min(capacity, (int64_t)window + max_queries + kStep) : capacity;
  if (rows > kFewRows) {
    // as many parts as give the CUs the workgroups that their registers hold, each of at least 512 positions
    const int64_t blocks = N * kv_heads * ((rows + 127) / 128), fit = D == 256 ? 256 : D == 64 ? 768 : 512;
    if (window > 0) seen = std::min<int64_t>(capacity, (int64_t)window + 128 / group + 64);
    const int64_t most = std::min<int64_t>(kMaxSplits, fit / std::max<int64_t>(blocks, 1));
    return {true, (int)std::max<int64_t>(1, std::min<int64_t>(seen / 512, most)), 0};
  }
  const int64_t resident = D == 256 ? 512 : D == 128 ? 768 : 1024;
  constexpr int64_t kLeast = kWaves * kStep;
  // Parts of the same length, so that ragged requests load the CUs alike: a step a wave at the least, and as long
  // as keep the launch within one and a half times the workgroups that are resident at once, were every request to
  // fill its table row (five ragged documents of 65536 positions, D = 256: 768 workgroups 36 us, 1024 42, 512 42; 64
  // requests of 8192, D = 128: 1024 46 us, 768 50, 2048 49); three steps a wave where every CU still has a workgroup
  // (one request of 65536: 21 us, with one step 30).  One part where it is short, because the join is a launch more:
  // 8 requests of 450 positions 9.6 us, in two parts 13.1, of 1000 12.3 and 13.8; and where the workgroups fill the
  // CUs already, 128 of 1700 22.6 and 26.7.
  const auto parts = [D](int64_t positions, int64_t most, int64_t blocks, int64_t& times) {
    const int64_t least = (positions + kLeast - 1) / kLeast;
    if (least <= (blocks >= 256 && D < 256 ? 8 : blocks >= 32 ? 5 : 3)) {
      times = std::max<int64_t>(1, least);
      return (int64_t)1;
    }
    times = std::max({(int64_t)1, (least + most - 1) / most, std::min<int64_t>(3, least * blocks / 256)});
    return std::max<int64_t>(1, (least + times - 1) / times);
  };
  const int64_t blocks = std::max<int64_t>(1, N * kv_heads * ((rows + 15) / 16));
  int64_t times, splits = parts(capacity, std::min<int64_t>(kMaxSplits, std::max<int64_t>(1, resident * 3 / 2 / blocks)), blocks, times);
  if (window > 0) splits = parts(seen, splits, blocks, times);
  return {false, (int)splits, (int)(times * kWaves)};
}

}  // namespace cqgdn
