// The keys of attention tiles and of the workgroups that share them
// (csrc/kv_index.hpp) on the host: parts that cover a tile's keys once, within
// the page table, whatever token_start and context hold, with nothing overflowing
// on the way. Built with the address and undefined-behaviour sanitizers.
#include <algorithm>
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

int main() {
  std::mt19937 rng(11);
  auto draw = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  const int odd[] = {INT_MIN, INT_MIN + 1, -(1 << 24), -1, 0, 1, 1000, (1 << 24) - 1, (1 << 30) - 1, 1 << 30, (1 << 30) + 1,
                     (1 << 30) + 1000, 1500000000, INT_MAX - 200, INT_MAX - 1, INT_MAX};
  const int windows[] = {0, 0, 1, 100, 5000, (1 << 30) - 1};
  int walked = 0, cut = 0;
  for (int round = 0; round < 5000; ++round) {
    qk::KvArgs a{};
    a.sequences = draw(1, 6);
    a.page_size = draw(0, 1) ? draw(1, 300) : 65536;
    a.table_pages = draw(0, 2) ? draw(1, 40) : INT_MAX;
    const int64_t room = int64_t{a.table_pages} * a.page_size;
    std::vector<int32_t> start{draw(0, 3)}, context;
    for (int s = 0; s < a.sequences; ++s) {
      const int n = draw(0, 2) ? draw(0, 5) : draw(0, 3000);
      start.push_back(start.back() + n);
      context.push_back(draw(0, 3) ? static_cast<int>(std::min<int64_t>(n + draw(0, 9000), std::max<int64_t>(room, n))) : odd[draw(0, 15)]);
    }
    a.tokens = start.back() + draw(0, 2);
    if (draw(0, 3) == 0) start[draw(0, a.sequences)] = odd[draw(0, 15)];
    a.token_start = start.data();
    a.context = context.data();
    const int group = draw(1, 9), window = windows[draw(0, 5)], tile_rows = 16 << draw(0, 4);
    for (int s = 0; s < a.sequences; ++s) {
      const qk::KvSequence q = qk::kv_sequence(a, s);
      CHECK(q.beyond == (context[s] > (1 << 30) || context[s] > room));
      // a negative context keeps its rows, none of which has a position
      const bool owned = start[s] >= 0 && start[s + 1] >= start[s] && start[s + 1] <= a.tokens;
      if (owned) CHECK(q.row == start[s] && q.count == start[s + 1] - start[s]);
      if (!owned || context[s] < q.count) CHECK(q.fault);
      if (context[s] < 0) CHECK(q.fault && q.first + q.count <= 0);
      const int seen = qk::kv_keys(q);
      CHECK(seen >= 0 && seen <= room && seen <= 1 << 30);
      for (int begin = 0; begin < q.count * group; begin += tile_rows) {
        qk::AttentionTile t{};
        t.s = s;
        t.row = q.row;
        t.count = q.count;
        t.first = q.first;
        t.beyond = q.beyond;
        t.begin = begin;
        qk::tile_keys(group, window, tile_rows, t);
        CHECK(0 <= t.key_lo && t.key_lo <= t.key_hi);
        CHECK(t.key_lo == t.key_hi || t.key_hi <= seen);
        if (q.beyond) CHECK(t.key_lo == t.key_hi);
        // the rows' own ends
        for (int row : {begin, std::min(begin + tile_rows, t.rows) - 1}) {
          const int position = q.first + row / group, from = window > 0 ? position - window + 1 : 0;
          if (!q.beyond && position >= 0) CHECK(position < t.key_hi && std::max(from, 0) >= t.key_lo);
        }
        cut += q.beyond;
        for (int splits : {1, 2, 7, 24, 256, 2048})
          for (int step : {64, 128})
            for (int least : {128, 256, 2048, seen / splits}) {
              int at = t.key_lo;
              const qk::KeyChunk first = qk::key_chunk(t, 0, splits, step, least < 128 ? 128 : least);
              CHECK(first.used >= 1 && first.used <= splits);
              for (int split : {0, 1, first.used - 2, first.used - 1, first.used, splits - 1}) {
                if (split < 0 || split >= splits) continue;
                const qk::KeyChunk c = qk::key_chunk(t, split, splits, step, least < 128 ? 128 : least);
                CHECK(c.used == first.used && c.lo <= c.hi && c.lo >= t.key_lo && c.hi <= t.key_hi);
                CHECK((split < c.used && t.key_lo < t.key_hi) == (c.lo < c.hi));
                CHECK(c.hi <= INT_MAX - 4096);  // look-ups run up to five tiles ahead
                if (split == 0) CHECK(c.lo == t.key_lo);
                if (split == c.used - 1) CHECK(c.hi == t.key_hi);
                if (split == 1 && c.used > 1) CHECK(c.lo == at);
                if (split == 0) at = c.hi;
                walked += c.hi > c.lo;
              }
            }
      }
    }
  }
  CHECK(walked > 30000 && cut > 300);
  std::printf("all checks passed\n");
  return 0;
}
