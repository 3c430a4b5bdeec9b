// The plan of a paged attention call: which kernel, how many tiles, how many
// workgroups share a tile's keys, and the workspace that takes. Plain C++, so
// that the same code is tested on the host.
#pragma once

#include <cstddef>
#include <cstdint>

#include "kv_index.hpp"
#include "qk_abi.h"

namespace qk {

constexpr int kGoodPartKeys = 2048;  // see plan_attention
constexpr int kOrdered = 128;        // most sequences that are taken by length

// How a call is laid out, from host values alone.
struct AttentionPlan {
  bool few;              // 16-row tiles (paged_attention_few*.hip; of Q4_1 also 8), else 256 to 32 (paged_attention_many.hip)
  int key_groups;        // of the latter: 1, or 2 or 4 waves that share 32 rows, each with a part of the keys
  int rows;              // rows of a tile: (new token, query head of the key/value head)
  int32_t tiles;         // at most so many tiles
  int32_t splits;        // workgroups that may share a tile's keys
  int32_t fill;          // so many of them fill the card
  int32_t pairs;         // see AttentionArgs
  size_t sums_at, parts_at, bytes;  // workspace; 0 bytes without splits
};
// Waves of a workgroup of paged_attention_many.hip, 32 rows each: eight, but
// four with 512 registers each where F32 q meets a BF16 cache (three parts).
constexpr int attention_many_waves(bool bf16, bool q32) { return bf16 && q32 ? 4 : 8; }

// Lengths of any size that callers give for "all" (INT64_MAX among them) as ones
// that sums and the kernels' 32 bits hold: positions are below kMostPositions, so
// a window that reaches over all of them is none.
constexpr int64_t bounded_window(int64_t window) { return window < kMostPositions ? window : 0; }
constexpr int64_t bounded_context(int64_t max_context) {
  return max_context < 1 ? 1 : max_context < kMostPositions ? max_context : int64_t{kMostPositions};
}

namespace plan {

// The card's compute units: a plan, and with it a workspace's size, is the
// same with and without a device at hand.
constexpr int64_t kUnits = 256;
// Single tokens: where there are more (tile, head) units than compute units the
// contexts stay whole and are taken by length (us: 40 sequences of up to 4000
// keys 89, cut in two 103). Else they are cut, into parts of kGoodPart keys, or
// as short as it takes for two workgroups a unit. Longer parts leave a batch of
// uneven contexts unbalanced (16 of up to 32768 keys: parts of 8192 237, of 2048
// 187), shorter ones pay for their joining (one of 131072: parts of 2048 102, of
// 512 136).
// So are contexts that a sequence's several tiles keep from being taken by length (24
// sequences of up to 10 new tokens and 10000 keys: whole 186, in parts 125; of up
// to 4000 103 and 75).
constexpr int64_t kGoodPart = kGoodPartKeys;
// Up to four 16-row tiles a sequence, HBM and the joining still bound the
// kernel for few rows, and it is ahead of the other with its large tiles (us, 16
// new tokens of 32 heads over 8: 4000 keys 24.5 and 29.6, three such sequences 27.6
// and 44.6; a bfloat16 cache, 12 of them, 62 and 107); but with q of the cache's type the
// other one's products cost half, and more than a few sequences occupy the card in it
// (12 of up to 30 tokens and 4000 keys: 73 and 62).
constexpr int64_t kAlone = 4;
// Ranking the contexts by length costs a few microseconds: from this many keys on.
constexpr int64_t kOrderedKeys = 1024;
// Keys are shared out only while a plan has fewer (tile, head) units than this,
// so the counters of every plan fit one fixed region at the workspace's start:
// no call's parts lie where a call of another batch keeps its counters.
constexpr int64_t kMostUnits = 2 * kUnits;
// Over Q4_1 blocks the kernel cuts contexts into even shares of all keys, for two
// workgroups a compute unit (its registers hold no more), parts of 256 keys, two turns of
// four waves, at least. The plan's part is the grid, of four workgroups a compute unit: it
// bounds into how many shares the longest contexts go; workgroups without one end at once
// (us). A grid half as large: 32 sequences of up to 8192 keys 95
// and 109, three of up to 131072 83 to 86 and 93, but 16 of up to 8192 54 and 50.
// Parts of 512 keys: one sequence of 1000 16 and 17, of 2000 18.2 and 20.8, of 4096 15.6 and 17.6.
constexpr int kLeastPartQ4 = 256, kSlotsQ4 = 1024;
constexpr size_t kCounterBytes = kMostUnits * sizeof(uint32_t);

inline int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Many rows: waves to a row (its keys shared among them, in tiles of 256, 128 or
// 64 rows; half as many with q in three parts) and workgroups to a tile's keys. Each
// has its price, so the pair is taken whose estimated time is least:
//   - the compute units' work, in keys: the longest workgroup's, or all of it
//     spread evenly, or as many of the shortest as one unit gets;
//   - times a tile's time a key, which a smaller tile has less than its
//     share of; and each workgroup's start;
//   - the parts' way through memory, and the launch that joins them.
// The constants order the pairs rather than tell the time. They are fitted to 368
// calls (20 to 12000 keys, 64 to 4095 new tokens a sequence, 1 to 12
// sequences, windows, all types, both head dimensions) with up to 28 pairs each: the
// pair taken is 1.8% behind the best one in the mean; the largest tiles that
// occupy the card, sharing keys up to 2048 keys, and else as many parts as run at
// once, were 7.5% behind (1500 tokens with a window of 1000: 95 us and now 72; 1373
// over 2380 keys, 28 heads over 4: 126 and 103).
struct ManyRows {
  int64_t rows, tokens, sequences, kv_heads, group, window, max_context;
  int tile_rows, head_dim, parts;

  // half a tile a sequence is nearer to what there will be than a whole one
  int64_t likely_units(int64_t of_rows) const { return (up(rows, of_rows) + (sequences - 1) / 2) * kv_heads; }
  double time(int key_groups, int64_t splits) const {
    const int64_t of_rows = tile_rows / key_groups, seen = window + of_rows / group + 1;
    const bool bounded = window > 0 && max_context > seen;
    const int64_t most = bounded ? seen : max_context, early = max_context - up(tokens, sequences);
    const int64_t least = bounded ? seen : early < 64 ? 64 : early;
    const auto of_part = [&](int64_t keys) {
      const int64_t step = splits > 1 ? 256 : key_groups == 4 ? 128 : 64;
      return static_cast<double>(up(up(keys, splits), step) * step);
    };
    const int64_t units = likely_units(of_rows) * splits;
    const double even = 1.03 * units / kUnits * (of_part(most) + of_part(least)) / 2;
    double keys = of_part(most);
    if (keys < even) keys = even;
    if (keys < up(units, kUnits) * of_part(least)) keys = up(units, kUnits) * of_part(least);
    const double share = key_groups == 1 ? 1.0 : key_groups == 2 ? (parts == 3 ? 0.71 : 0.76) : parts == 3 ? 0.53 : 0.49;
    const double key = (parts == 3 ? 0.09 : 0.04) * (head_dim == 128 ? 1.0 : 0.64) * share;
    const double rounds = units > kUnits ? 1.0 * units / kUnits : 1.0;
    return key * keys + 1.5 * rounds + (splits > 1 ? 6.5 + 2.2e-6 * units * of_rows * head_dim : 0.0);
  }
  void choose(int& key_groups, int64_t& splits) const {
    double best = 1e30;
    for (int groups = 1; groups <= 4; groups *= 2)
      for (int64_t parts_of = 1; parts_of <= 24 && (parts_of == 1 || parts_of <= up(max_context, 256)); ++parts_of) {
        const double t = time(groups, parts_of);
        if (t >= best) continue;
        best = t;
        key_groups = groups;
        splits = parts_of;
      }
  }
};

}  // namespace plan

inline AttentionPlan plan_attention(int64_t tokens, int64_t sequences, int64_t q_heads, int64_t kv_heads, int head_dim,
                                    int type, int q_type, int64_t window, int64_t max_context) {
  using namespace plan;
  AttentionPlan p{};
  window = bounded_window(window);
  max_context = bounded_context(max_context);
  if (tokens == 0 || sequences == 0) return p;
  const int64_t group = q_heads / kv_heads, rows = tokens * group;
  p.few = rows <= (q_type == QK_TYPE_F32 || sequences <= kAlone ? 64 : 32) * sequences;
  const int waves_rows = 32 * attention_many_waves(type == QK_TYPE_BF16, q_type == QK_TYPE_F32);
  // every sequence may end in a part of a tile, and none has a tile without a row
  const auto tiles_of = [&](int64_t tile_rows) {
    int64_t tiles = (rows + sequences * (tile_rows - 1)) / tile_rows;
    if (tiles > rows) tiles = rows;
    if (group <= tile_rows && tiles > tokens) tiles = tokens;
    return tiles;
  };
  int64_t keys = max_context;
  if (window > 0 && keys > window + waves_rows) keys = window + waves_rows;
  p.key_groups = 1;
  int64_t splits = 1;
  if (!p.few)
    ManyRows{rows, tokens, sequences, kv_heads, group, window, max_context, waves_rows, head_dim,
             q_type == QK_TYPE_F32 ? (type == QK_TYPE_BF16 ? 3 : 2) : 1}
        .choose(p.key_groups, splits);
  // Over Q4_1 blocks a tile of up to 8 rows leaves the matrix core's other columns to
  // other keys (us; single tokens of 32 heads over 8: one over 131072 77, in 16 rows 82, over 4096
  // 15.6 and 18.0; 16 over up to 8192 53.7 and 56.3; 64, where memory bounds it, 114 and 115).
  const int few_rows = type != QK_TYPE_Q4_1 || rows > 8 * sequences ? 16 : 8;
  const int tile_rows = p.few ? few_rows : waves_rows / p.key_groups;
  p.rows = tile_rows;
  const int64_t tiles = tiles_of(tile_rows);
  p.tiles = static_cast<int32_t>(tiles);
  const int64_t units = tiles * kv_heads;
  const bool whole = p.few && keys >= kOrderedKeys && units > kUnits;
  const bool ordered = whole && rows <= tile_rows * sequences && sequences <= kOrdered;  // else some sequence has two tiles
  if (p.few) splits = whole ? 1 : up(kMostUnits, units);
  p.fill = static_cast<int32_t>(splits);
  if (p.few && !ordered && units <= kMostUnits && splits < up(keys, kGoodPart)) {
    const int64_t most = up(4 * kMostUnits, units);
    splits = up(keys, kGoodPart) < most ? up(keys, kGoodPart) : most;
  }
  if (p.few && type == QK_TYPE_Q4_1) {
    // the kernel cuts contexts into even shares of all keys
    splits = whole || units > kMostUnits ? 1 : up(kSlotsQ4, units);
    if (splits > up(keys, kLeastPartQ4)) splits = up(keys, kLeastPartQ4);
  }
  const int64_t least = p.few ? 128 : 256;
  if (splits > up(keys, least)) splits = up(keys, least);
  p.splits = static_cast<int32_t>(splits);
  if (ordered && splits == 1) p.pairs = static_cast<int32_t>(up(kUnits, kv_heads));
  if (splits > 1) {
    const size_t parts = static_cast<size_t>(units * splits * tile_rows);
    p.sums_at = kCounterBytes;
    p.parts_at = p.sums_at + ((parts * 2 * sizeof(float) + 255) & ~size_t{255});
    p.bytes = p.parts_at + parts * head_dim * sizeof(float);
  }
  return p;
}

// Whether the call's launches fit a grid, which has fewer than 2^32 threads.
inline bool plan_fits(const AttentionPlan& p, int64_t kv_heads, int type, int q_type) {
  const int64_t units = p.tiles * kv_heads, waves = attention_many_waves(type == QK_TYPE_BF16, q_type == QK_TYPE_F32);
  const int64_t threads = units * p.splits * (p.few ? 256 : 64 * waves);
  const int64_t joining = p.few || p.splits == 1 ? 0 : units * (p.rows / 32) * 256;
  return threads <= UINT32_MAX && joining <= UINT32_MAX;
}

}  // namespace qk
