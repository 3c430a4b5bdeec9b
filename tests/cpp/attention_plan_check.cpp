// csrc/attention_plan.hpp on the host: for lengths of any size, plans whose
// workspace holds what their tiles and parts write, with nothing overflowing on
// the way. Built with the address and undefined-behaviour sanitizers.
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <random>

#include "attention_plan.hpp"

#define CHECK(c) \
  do { \
    if (!(c)) { \
      std::printf("FAILED %s:%d %s\n", __FILE__, __LINE__, #c); \
      std::exit(1); \
    } \
  } while (0)

namespace {

struct Call {
  int64_t tokens, sequences, kv_heads, group;
  int head_dim, type, q_type;
  qk::AttentionPlan plan(int64_t window, int64_t max_context) const {
    return qk::plan_attention(tokens, sequences, kv_heads * group, kv_heads, head_dim, type, q_type, window, max_context);
  }
};

bool same(const qk::AttentionPlan& a, const qk::AttentionPlan& b) {
  return a.few == b.few && a.key_groups == b.key_groups && a.rows == b.rows && a.tiles == b.tiles && a.splits == b.splits &&
         a.fill == b.fill && a.pairs == b.pairs && a.sums_at == b.sums_at && a.parts_at == b.parts_at && a.bytes == b.bytes;
}

void sound(const Call& c, const qk::AttentionPlan& p) {
  if (c.tokens * c.kv_heads * c.group <= 1 << 23) CHECK(qk::plan_fits(p, c.kv_heads, c.type, c.q_type));
  CHECK(p.tiles >= 1 && p.splits >= 1);
  CHECK(p.rows >= 16 && p.key_groups >= 1);
  // every row has a tile, whichever sequences have them
  CHECK(int64_t{p.tiles} * p.rows >= c.tokens * c.group || p.tiles >= c.tokens);
  if (p.splits == 1) {
    CHECK(p.bytes == 0);
    return;
  }
  const size_t units = static_cast<size_t>(p.tiles) * c.kv_heads, rows = units * p.splits * p.rows;
  if (p.few) CHECK(units * sizeof(uint32_t) <= p.sums_at);
  CHECK(p.parts_at >= p.sums_at + rows * 2 * sizeof(float));
  CHECK(p.bytes >= p.parts_at + rows * c.head_dim * sizeof(float));
}

}  // namespace

int main() {
  std::mt19937 rng(7);
  auto draw = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  const int64_t lengths[] = {0, 1, 2, 100, 1000, 4096, 131072, INT32_MAX - 300, INT32_MAX - 1, INT32_MAX, int64_t{INT32_MAX} + 1,
                             int64_t{1} << 40, INT64_MAX - 300, INT64_MAX - 200, INT64_MAX - 1, INT64_MAX};
  for (int round = 0; round < 3000; ++round) {
    Call c;
    c.sequences = draw(0, 2) ? draw(1, 12) : draw(1, 3000);
    c.tokens = c.sequences + (draw(0, 1) ? 0 : draw(0, 5000));
    c.kv_heads = draw(1, 16);
    c.group = draw(1, 9);
    c.head_dim = draw(0, 1) ? 128 : 64;
    c.type = draw(0, 1) ? QK_TYPE_BF16 : QK_TYPE_F16;
    c.q_type = draw(0, 1) ? QK_TYPE_F32 : c.type;
    for (int64_t window : lengths)
      for (int64_t max_context : lengths) sound(c, c.plan(window, max_context));
    const int64_t context = lengths[draw(0, 6)];
    // a window over every position is none, a bound beyond the last position is that one
    for (int64_t all : {int64_t{INT32_MAX}, int64_t{1} << 40, INT64_MAX - 255, INT64_MAX})
      CHECK(same(c.plan(all, context), c.plan(0, context)));
    CHECK(same(c.plan(context, INT64_MAX), c.plan(context, INT32_MAX)));
  }
  std::printf("all checks passed\n");
  return 0;
}
