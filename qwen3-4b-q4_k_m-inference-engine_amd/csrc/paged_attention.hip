// The plan of a paged attention call: which kernel, how many tiles, how many
// workgroups share a tile's keys, and the workspace that takes.
#include "paged_attention.hpp"

namespace qk {
namespace {

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
// Many rows: the largest tiles that occupy the compute units, 256 rows, or 128 or
// 64 whose waves share the keys, but that only up to kPartedKeys keys: then
// 256-row tiles whose keys workgroups share are faster (us: 512 tokens of 32
// heads over 2048 keys 48 against 50, over 4096 keys 91 against 82; 12 ragged
// prompts of up to 300, 28 heads, 128-row tiles 32, 64-row ones 36). 128-row tiles
// also where 256-row ones would be one uneven round: 2048 tokens of a prompt,
// 256 tiles, 107 against 90; not at 4000 with a window of 1000, 500 tiles, 93
// against 116.
constexpr int64_t kPartedKeys = 2048;
constexpr size_t kCounterBytes = kMostUnits * sizeof(uint32_t);

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace

AttentionPlan plan_attention(int64_t tokens, int64_t sequences, int64_t q_heads, int64_t kv_heads, int head_dim, int type,
                             int q_type, int64_t window, int64_t max_context) {
  AttentionPlan p{};
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
  // half a tile a sequence is nearer to what there will be
  const auto likely_units = [&](int64_t tile_rows) { return (up(rows, tile_rows) + (sequences - 1) / 2) * kv_heads; };
  int64_t keys = max_context < 1 ? 1 : max_context;
  if (window > 0 && keys > window + waves_rows) keys = window + waves_rows;
  p.key_groups = 1;
  if (!p.few && keys <= kPartedKeys && likely_units(waves_rows) < kUnits * 3 / 2)
    p.key_groups = likely_units(waves_rows / 2) < kUnits * 5 / 8 ? 4 : 2;
  const int tile_rows = p.few ? 16 : waves_rows / p.key_groups;
  p.rows = tile_rows;
  const int64_t tiles = tiles_of(tile_rows);
  p.tiles = static_cast<int32_t>(tiles);
  const int64_t units = tiles * kv_heads;
  // many rows: as many parts as run at once, or a little over (600 tokens over
  // 4096 keys in three parts 91 us, in four, a second round, 120)
  const bool whole = p.few && keys >= kOrderedKeys && units > kUnits;
  const bool ordered = whole && rows <= 16 * sequences && sequences <= kOrdered;  // else some sequence has two tiles
  int64_t splits = whole ? 1 : up(kMostUnits, units);
  if (!p.few) {
    splits = (10 * kUnits + 3 * likely_units(tile_rows)) / (10 * likely_units(tile_rows));
    if (splits < 1) splits = 1;
  }
  p.fill = static_cast<int32_t>(splits);
  if (p.few && !ordered && units <= kMostUnits && splits < up(keys, kGoodPart)) {
    const int64_t most = up(4 * kMostUnits, units);
    splits = up(keys, kGoodPart) < most ? up(keys, kGoodPart) : most;
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

hipError_t launch_paged_attention(AttentionArgs a, const AttentionPlan& plan, int type, int head_dim, int q_type,
                                  void* workspace, hipStream_t stream) {
  a.tiles = plan.tiles;
  a.splits = plan.splits;
  a.fill = plan.fill;
  a.pairs = plan.pairs;
  char* ws = static_cast<char*>(workspace);
  a.arrived = reinterpret_cast<uint32_t*>(ws);
  a.sums = reinterpret_cast<float*>(ws + plan.sums_at);
  a.parts = reinterpret_cast<float*>(ws + plan.parts_at);
  return plan.few ? launch_attention_few(a, type, head_dim, q_type, stream)
                  : launch_attention_many(a, plan.key_groups, type, head_dim, q_type, stream);
}

}  // namespace qk
