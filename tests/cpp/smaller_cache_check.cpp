// The plans of attention over Q4_1 blocks and of qk_kv_weigh, and the division by a
// page's size, over lengths of any size.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#include "attention_plan.hpp"
#include "weigh_plan.hpp"

#define CHECK(x)                                                       \
  do {                                                                 \
    if (!(x)) {                                                        \
      std::printf("%s:%d: %s\n", __FILE__, __LINE__, #x);              \
      std::exit(1);                                                    \
    }                                                                  \
  } while (0)

using namespace qk;

static void divisions() {
  const int32_t edge = kMostPositions - 1;
  for (int32_t size = 1; size <= 65536; size += size < 300 ? 1 : size % 97 + 1) {
    const PageDivision d = page_division(size);
    for (int32_t k = 0; k < 200; ++k) {
      const int32_t near = edge / size * size;
      for (int32_t key : {k, k * size, k * size + size - 1, edge - k, near - k, near + k, k * 5368709})
        if (key >= 0 && key <= edge) CHECK(page_entry(d, key) == key / size);
    }
  }
}

static void attention() {
  for (int64_t sequences : {1, 3, 16, 64, 129, 65535})
    for (int64_t each : {1, 2, 5, 17, 300})
      for (int64_t heads : {1, 2, 8, 4096})
        for (int64_t group : {1, 4, 7, 16, 64})
          for (int64_t context : {int64_t{0}, int64_t{1}, int64_t{1000}, int64_t{131072}, int64_t{1} << 30, INT64_MAX})
            for (int64_t window : {int64_t{0}, int64_t{100}, INT64_MAX})
              for (int q_type : {QK_TYPE_F32, QK_TYPE_F16})
                for (int dim : {64, 128}) {
                  const int64_t tokens = sequences * each;
                  if (tokens * heads * group > (int64_t{1} << 28)) continue;
                  const AttentionPlan p = plan_attention(tokens, sequences, heads * group, heads, dim, QK_TYPE_Q4_1, q_type, window, context);
                  CHECK(p.tiles >= 1 && p.splits >= 1);
                  if (!p.few) continue;
                  CHECK(p.rows == 8 || p.rows == 16);
                  // enough tiles for any way that the rows fall to sequences
                  CHECK(p.tiles >= (tokens * group + p.rows - 1) / p.rows);
                  if (p.splits > 1) {
                    const int64_t units = p.tiles * heads, parts = units * p.splits * p.rows;
                    CHECK(units <= plan::kMostUnits);  // its counters
                    CHECK(p.sums_at >= static_cast<size_t>(units) * 4);
                    CHECK(p.parts_at >= p.sums_at + static_cast<size_t>(parts) * 8);
                    CHECK(p.bytes >= p.parts_at + static_cast<size_t>(parts) * dim * 4);
                  } else {
                    CHECK(p.bytes == 0);
                  }
                }
}

static void weights() {
  for (int64_t sequences : {1, 3, 64, 65535})
    for (int64_t each : {1, 2, 20, 2047, 100000})
      for (int64_t heads : {1, 8, 4096})
        for (int64_t group : {1, 4, 64})
          for (int64_t context : {int64_t{0}, int64_t{1}, int64_t{127}, int64_t{8192}, int64_t{1000003}, int64_t{1} << 30, INT64_MAX}) {
            const int64_t tokens = sequences * each;
            if (tokens >= kMostTokens || tokens * heads * group > (int64_t{1} << 28)) continue;
            const WeighPlan p = plan_weigh(tokens, sequences, heads * group, heads, context);
            const int64_t most = context < 1 ? 1 : context < kMostPositions ? context : kMostPositions;
            CHECK(p.key_parts >= 1 && p.row_parts >= 1 && p.part_keys >= 1);
            CHECK(int64_t{p.key_parts} * p.part_keys >= most);         // every key has a workgroup
            CHECK(int64_t{p.key_parts} * p.part_keys <= INT32_MAX);    // and fits the kernels' 32 bits
            CHECK(p.part_keys % 32 == 0);
            if (p.row_parts > 1)
              CHECK(p.bytes == static_cast<size_t>(p.row_parts * sequences * heads * p.key_parts * p.part_keys * 4));
            else
              CHECK(p.bytes == 0);
            CHECK(p.bytes <= static_cast<size_t>(weigh::kMostBytes));
            if (weigh_fits(p, sequences, heads))
              CHECK(sequences * heads * p.key_parts * p.row_parts * 256 <= int64_t{UINT32_MAX});
          }
  CHECK(plan_weigh(0, 3, 8, 8, 100).bytes == 0 && plan_weigh(3, 0, 8, 8, 100).bytes == 0);
}

int main() {
  divisions();
  attention();
  weights();
  std::printf("all checks passed\n");
}
