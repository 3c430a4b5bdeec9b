// Which rows, positions and places in a paged cache a kernel may touch: all
// that is read from the device arrays of a batch (token_start, context,
// page_table) becomes an index here and nowhere else, cut to the buffers.
// Plain C++, so that the same code is tested on the host.
#pragma once

#include <cstdint>

#ifdef __HIP__
#define QK_HD __host__ __device__ __forceinline__
#else
#define QK_HD inline
#endif

namespace qk {

// Contexts are no longer than this: positions, and what the kernels add to them,
// stay within 32 bits.
constexpr int32_t kMostPositions = 1 << 30;
constexpr int32_t kMostTokens = 1 << 24;  // new tokens of a batch are fewer

// A cache and a batch as the kernels take them.
struct KvArgs {
  uint16_t* k;
  uint16_t* v;
  int64_t page_stride;                // elements
  int32_t token_stride, head_stride;  // elements
  int32_t pages, page_size;
  int32_t kv_heads;
  int32_t sequences, tokens;
  int32_t table_pages;  // entries of a table row
  int64_t table_stride;
  const int32_t* token_start;
  const int32_t* context;
  const int32_t* page_table;
  uint32_t* fault;
};

// A sequence's new rows and the position of the first of them. Lengths that do
// not fit (fault) are cut: row .. row + count lies in [0, tokens], positions are below
// 2^31 (negative ones see nothing). beyond: the last of them has no place in the
// page table, or lies past kMostPositions.
struct KvSequence {
  int32_t row, count, first;
  bool fault, beyond;
};
QK_HD KvSequence kv_sequence(const KvArgs& a, int s) {
  const int32_t lo = a.token_start[s], hi = a.token_start[s + 1], context = a.context[s];
  KvSequence q;
  q.row = lo < 0 ? 0 : lo;
  const int32_t end = hi < a.tokens ? hi : a.tokens;
  q.count = hi >= lo && end > q.row ? end - q.row : 0;
  q.fault = lo < 0 || hi > a.tokens || hi < lo || context < 0 || context < static_cast<int64_t>(hi) - lo;
  // hi >= q.row >= 0 wherever count > 0, so this does not exceed context; count is
  // below kMostTokens, so positions cut at its negative stay negative
  const int64_t first = q.count > 0 ? static_cast<int64_t>(context) - (hi - q.row) : 0;
  q.first = first < -kMostTokens ? -kMostTokens : static_cast<int32_t>(first);
  const int64_t room = static_cast<int64_t>(a.table_pages) * a.page_size;
  q.beyond = context > kMostPositions || context > room;
  return q;
}

// The keys that a sequence's new tokens see without a window.
QK_HD int32_t kv_keys(const KvSequence& q) {
  return q.count > 0 && !q.beyond && q.first + q.count > 0 ? q.first + q.count : 0;
}

// The sequence that owns `row`: the last whose token_start is <= row (empty
// sequences share their start with the next one).
QK_HD int kv_find_sequence(const KvArgs& a, int row) {
  int lo = 0, hi = a.sequences - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.token_start[mid] <= row)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// Where the page table holds entry `entry` of sequence s, or 0 (a place that
// every table has) with ok cleared.
QK_HD int64_t kv_table_at(const KvArgs& a, int s, int32_t entry, bool& ok) {
  ok = entry >= 0 && entry < a.table_pages;
  return ok ? s * a.table_stride + entry : 0;
}

// The page that holds entry `entry` of sequence s, or -1 if the table has no
// such entry or the entry no such page.
QK_HD int32_t kv_page(const KvArgs& a, int s, int32_t entry) {
  bool ok;
  const int32_t page = a.page_table[kv_table_at(a, s, entry, ok)];
  return ok && page >= 0 && page < a.pages ? page : -1;
}

// key / page_size of keys below 2^30 as the high half of a product: with 2^l the least
// power of two that page_size does not exceed, ceil(2^(30 + l) / page_size) is below 2^31
// and gives the quotient in its bits from 30 + l on; doubled, from 31 + l on.
struct PageDivision {
  uint32_t factor;
  int32_t shift;  // below the high half; -1: pages of one token
};
QK_HD PageDivision page_division(int32_t page_size) {
  int bits = 0;
  while ((int64_t{1} << bits) < page_size) ++bits;
  return {static_cast<uint32_t>(2 * (((uint64_t{1} << (30 + bits)) + page_size - 1) / page_size)), bits - 1};
}
QK_HD int32_t page_entry(const PageDivision& d, int32_t key) {
  const uint32_t high = static_cast<uint32_t>(static_cast<uint64_t>(static_cast<uint32_t>(key)) * d.factor >> 32);
  return d.shift < 0 ? key : static_cast<int32_t>(high >> d.shift);
}

// Element offset of (page, slot, head); page in [0, pages), slot in [0, page_size).
QK_HD int64_t kv_place(const KvArgs& a, int32_t page, int32_t slot, int32_t head) {
  return page * a.page_stride + static_cast<int64_t>(slot) * a.token_stride + static_cast<int64_t>(head) * a.head_stride;
}

// An attention workgroup's tile.
struct AttentionTile {
  int s;               // sequence; -1: the workgroup has no tile
  int row, count;      // first new row and new rows of the sequence
  int first;           // position of its first new row
  int begin, rows;     // first row of the tile among the sequence's, rows of the sequence (count * group)
  int key_lo, key_hi;  // keys that any row of the tile sees
  bool beyond;         // of the sequence
};

// The rest of a tile, from its sequence and first row. A context that is beyond its
// page table has no keys: none is walked before that is reported.
QK_HD void tile_keys(int group, int window, int tile_rows, AttentionTile& t) {
  t.rows = t.count * group;
  if (t.beyond) {
    t.key_lo = t.key_hi = 0;
    return;
  }
  const int end = t.begin + tile_rows < t.rows ? t.begin + tile_rows : t.rows;
  t.key_hi = t.first + (end - 1) / group + 1;
  const int lowest = window > 0 ? t.first + t.begin / group - window + 1 : 0;
  t.key_lo = lowest > 0 ? lowest : 0;
  if (t.key_hi < t.key_lo) t.key_hi = t.key_lo;  // positions before 0 see nothing
}

// A tile's keys over its workgroups: chunks of `chunk` keys, but long enough that
// `splits` of them suffice, in multiples of `step`; `used` of them are not empty
// (one at least).
struct KeyChunk {
  int lo, hi, used;
};
QK_HD KeyChunk key_chunk(const AttentionTile& t, int split, int splits, int step, int chunk) {
  const int keys = t.key_hi - t.key_lo;
  const int least = (keys + splits - 1) / splits;
  chunk = chunk < least ? least : chunk;
  chunk = (chunk + step - 1) / step * step;
  KeyChunk c;
  c.used = keys > 0 ? (keys - 1) / chunk + 1 : 1;
  c.lo = split < c.used ? t.key_lo + split * chunk : t.key_hi;
  c.hi = t.key_hi - c.lo > chunk ? c.lo + chunk : t.key_hi;
  return c;
}

}  // namespace qk
