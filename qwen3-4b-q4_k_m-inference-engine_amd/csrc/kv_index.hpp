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
// not fit are cut: row .. row + count lies in [0, tokens], positions are below
// 2^31 (negative ones see nothing).
struct KvSequence {
  int32_t row, count, first;
  bool fault;
};
QK_HD KvSequence kv_sequence(const KvArgs& a, int s) {
  const int32_t lo = a.token_start[s], hi = a.token_start[s + 1], context = a.context[s];
  KvSequence q;
  q.row = lo < 0 ? 0 : lo;
  const int32_t end = hi < a.tokens ? hi : a.tokens;
  const bool ordered = hi >= lo && context >= 0;
  q.count = ordered && end > q.row ? end - q.row : 0;
  q.fault = lo < 0 || hi > a.tokens || !ordered || context < static_cast<int64_t>(hi) - lo;
  // hi >= q.row >= 0 wherever count > 0, so this neither overflows nor exceeds context
  q.first = q.count > 0 ? context - (hi - q.row) : 0;
  return q;
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

// Element offset of (page, slot, head); page in [0, pages), slot in [0, page_size).
QK_HD int64_t kv_place(const KvArgs& a, int32_t page, int32_t slot, int32_t head) {
  return page * a.page_stride + static_cast<int64_t>(slot) * a.token_stride + static_cast<int64_t>(head) * a.head_stride;
}

}  // namespace qk
