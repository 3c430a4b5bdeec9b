// The plan of a qk_kv_weigh call: which kernel, how its keys and rows are shared
// out, and the workspace that takes. Plain C++, so that the same code is tested on the
// host.
#pragma once

#include <cstddef>
#include <cstdint>

#include "kv_index.hpp"

namespace qk {

struct WeighPlan {
  bool few;           // kv_weigh_few_kernel: 16 rows a tile and keys streamed; else keys held and rows streamed
  int32_t key_parts;  // workgroups along a sequence's keys
  int32_t part_keys;  // keys of each
  int32_t row_parts;  // of the latter: workgroups along the rows, their sums joined
  size_t bytes;       // workspace: [row_parts x sequences x kv_heads x key_parts * part_keys] sums
};

namespace weigh {

constexpr int64_t kUnits = 256;      // the card's compute units
constexpr int64_t kHeldKeys = 256;   // keys that a workgroup of the kernel for many rows holds
constexpr int64_t kMostBytes = int64_t{1} << 31;

inline int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace weigh

inline WeighPlan plan_weigh(int64_t tokens, int64_t sequences, int64_t q_heads, int64_t kv_heads, int64_t max_context) {
  using namespace weigh;
  WeighPlan p{};
  if (tokens == 0 || sequences == 0) return p;
  max_context = max_context < 1 ? 1 : max_context < kMostPositions ? max_context : int64_t{kMostPositions};
  const int64_t rows = tokens * (q_heads / kv_heads), units = sequences * kv_heads;
  // By the mean, as lengths are on the device. One sequence of many rows among ones of
  // few takes its tiles one after another then, and is better off in a call of its own (us,
  // 64 single tokens over up to 8192 keys and a chunk over 8192, in one call and in two: a chunk
  // of 64 tokens 234 and 89, of 128 424 and 101, of 512 1571 and 168, of 900 2743 and 240).
  p.few = rows <= 64 * sequences;
  p.row_parts = 1;
  if (p.few) {
    // Sixteen workgroups for each compute unit where contexts are many and uneven (us:
    // 64 sequences of up to 8192 keys and 8 heads in Q4_1 75, by four each 100; 32 of them 46 and 52, in
    // F16 76 and 90). Four each for few, where a start costs more than it balances (8 of
    // 8192 22 by sixteen and 19, in F16 27 and 21; one of 131072 43 and 38.5). 128 keys are one block
    // for each of four waves.
    int64_t parts = up((units > kUnits / 4 ? 16 : 4) * kUnits, units);
    if (parts > up(max_context, 128)) parts = up(max_context, 128);
    p.part_keys = static_cast<int32_t>(up(up(max_context, parts), 128) * 128);
    p.key_parts = static_cast<int32_t>(up(max_context, p.part_keys));
    return p;
  }
  p.part_keys = kHeldKeys;
  p.key_parts = static_cast<int32_t>(up(max_context, kHeldKeys));
  // Rows are shared out where keys alone do not occupy the card, eight tiles of 32 rows
  // at least. A prompt has few blocks of keys, and the first ones are seen by the most rows
  // (us: two prompts of up to 2047, 28 heads over 4: 43 to 49, undivided 532). Where keys
  // are many, rows stay whole (63 new tokens over 32768: 1024 workgroups, 49 to 57).
  int64_t parts = up(8 * kUnits, units * p.key_parts);
  const int64_t most = up(rows, 256 * sequences), each = units * p.key_parts * kHeldKeys * static_cast<int64_t>(sizeof(float));
  if (parts > most) parts = most;
  if (parts * each > kMostBytes) parts = kMostBytes / each;
  if (parts > 1) {
    p.row_parts = static_cast<int32_t>(parts);
    p.bytes = static_cast<size_t>(parts * each);
  }
  return p;
}

// Whether the call's launches fit a grid, which has fewer than 2^32 threads.
inline bool weigh_fits(const WeighPlan& p, int64_t sequences, int64_t kv_heads) {
  return sequences * kv_heads * p.key_parts <= (int64_t{UINT32_MAX} / 256) / p.row_parts;
}

}  // namespace qk
