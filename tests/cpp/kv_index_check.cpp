// csrc/kv_index.hpp on the host: whatever token_start, context and page_table
// hold, every row, position and place that it yields lies inside the buffers,
// and sound batches get exactly the rows, positions and places of their
// definition. Built with the address and undefined-behaviour sanitizers.
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "kv_index.hpp"

#define CHECK(c) \
  do { \
    if (!(c)) { \
      std::printf("FAILED %s:%d %s\n", __FILE__, __LINE__, #c); \
      std::exit(1); \
    } \
  } while (0)

namespace {

struct Batch {
  std::vector<int32_t> start, context, table;
  qk::KvArgs a{};
  void link() {
    a.token_start = start.data();
    a.context = context.data();
    a.page_table = table.data();
  }
};

void in_bounds(const Batch& b) {
  const qk::KvArgs& a = b.a;
  for (int s = 0; s < a.sequences; ++s) {
    const qk::KvSequence q = qk::kv_sequence(a, s);
    CHECK(q.count >= 0 && q.row >= 0);
    CHECK(q.count == 0 || q.row + q.count <= a.tokens);
    const int last = q.count > 0 ? q.first + q.count - 1 : -1;  // must not overflow
    CHECK(last < INT_MAX);
    for (int32_t entry : {-1, 0, 1, a.table_pages - 1, a.table_pages, last / a.page_size, INT_MAX, INT_MIN}) {
      const int32_t page = qk::kv_page(a, s, entry);
      CHECK(page >= -1 && page < a.pages);
    }
  }
  for (int row = 0; row < a.tokens; ++row) {
    const int s = qk::kv_find_sequence(a, row);
    CHECK(s >= 0 && s < a.sequences);
  }
}

}  // namespace

int main() {
  std::mt19937 rng(20261206);
  auto draw = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  for (int round = 0; round < 4000; ++round) {
    Batch b;
    qk::KvArgs& a = b.a;
    a.sequences = draw(1, 9);
    a.pages = draw(1, 12);
    a.page_size = draw(1, 20);
    a.kv_heads = draw(1, 4);
    a.head_stride = 64;
    a.token_stride = 64 * a.kv_heads;
    a.page_stride = int64_t{a.token_stride} * a.page_size;
    a.table_pages = draw(1, 6);
    a.table_stride = a.table_pages + draw(0, 2);
    // a sound batch, empty sequences and unowned rows at both ends among it
    b.start.push_back(draw(0, 2));
    for (int s = 0; s < a.sequences; ++s) {
      const int n = draw(0, 5);
      b.start.push_back(b.start.back() + n);
      b.context.push_back(n + draw(0, 30));
      for (int64_t e = 0; e < a.table_stride; ++e) b.table.push_back(draw(0, a.pages - 1));
    }
    a.tokens = b.start.back() + draw(0, 2);
    b.link();
    for (int s = 0; s < a.sequences; ++s) {
      const qk::KvSequence q = qk::kv_sequence(a, s);
      const int n = b.start[s + 1] - b.start[s];
      CHECK(!q.fault && q.count == n && (n == 0 || (q.row == b.start[s] && q.first == b.context[s] - n)));
      for (int i = 0; i < n; ++i) CHECK(qk::kv_find_sequence(a, q.row + i) == s);
      for (int e = 0; e < a.table_pages; ++e) CHECK(qk::kv_page(a, s, e) == b.table[s * a.table_stride + e]);
    }
    const int64_t end = qk::kv_place(a, a.pages - 1, a.page_size - 1, a.kv_heads - 1) + 64;
    CHECK(end == a.page_stride * a.pages);
    in_bounds(b);
    // the same with spoiled entries
    const int32_t odd[] = {INT_MIN, INT_MIN + 1, -1, 0, 1, a.pages - 1, a.pages, a.tokens, a.tokens + 1, INT_MAX - 1, INT_MAX};
    for (int i = 0; i < 4; ++i) {
      b.start[draw(0, a.sequences)] = odd[draw(0, 10)];
      b.context[draw(0, a.sequences - 1)] = odd[draw(0, 10)];
      b.table[draw(0, static_cast<int>(b.table.size()) - 1)] = odd[draw(0, 10)];
      in_bounds(b);
    }
  }
  std::printf("all checks passed\n");
  return 0;
}
