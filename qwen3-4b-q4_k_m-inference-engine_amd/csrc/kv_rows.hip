// Cached rows of the new tokens out of their pages, as values: what a caller keeps
// of a sequence elsewhere, hands to another cache, or compares. D/8 lanes a row, as in
// the append; a workgroup takes one token and up to 16 (D = 128) or 32 (D = 64) of
// its rows. What bounds it is the way to a row, not memory: each workgroup searches its
// token's sequence and looks up its page before the one load that a lane has in flight
// (8192 tokens of 2 x 8 heads of 128 out of Q4_1 blocks, 44 MB, 13.7 us, 3.2 TB/s, where a
// copy reaches 5.1). A call of few tokens is the launch.
#include <type_traits>

#include "q4_1.hpp"
#include "qk_device.hpp"
#include "qk_launch.hpp"
#include "serving.hpp"

namespace qk {
namespace {

// KIND: the cache's type.
template <int D, int KIND, bool OUT32>
__global__ __launch_bounds__(256) void kv_rows_kernel(const RowsArgs a) {
  constexpr bool BF16 = KIND == QK_TYPE_BF16, Q4 = KIND == QK_TYPE_Q4_1;
  constexpr int L = D / 8;  // lanes a row
  const int tid = static_cast<int>(threadIdx.x);
  const int token = static_cast<int>(blockIdx.x);
  const int row = static_cast<int>(blockIdx.y) * (256 / L) + tid / L;
  const int u = tid % L;
  if (blockIdx.x == 0 && blockIdx.y == 0)  // lengths that do not fit, of sequences without rows too
    for (int i = tid; i < a.kv.sequences; i += 256)
      if (kv_sequence(a.kv, i).fault) kv_fault(a.kv, QK_KV_FAULT_LENGTH);
  const int s = kv_find_sequence(a.kv, token);
  const KvSequence seq = kv_sequence(a.kv, s);
  if (token < seq.row || token >= seq.row + seq.count) return;  // no sequence owns this row
  if (row >= 2 * a.kv.kv_heads) return;
  const bool is_k = row < a.kv.kv_heads;
  const int head = is_k ? row : row - a.kv.kv_heads;
  void* out = is_k ? a.k_out : a.v_out;
  if (!out) return;
  const int position = seq.first + (token - seq.row);
  const int entry = position < 0 ? -1 : position / a.kv.page_size;
  const int page = kv_page(a.kv, s, entry);
  u32x4 x;  // eight 16-bit values
  if (page < 0) {
    if (u == 0) kv_fault(a.kv, position < 0 ? QK_KV_FAULT_LENGTH : QK_KV_FAULT_PAGE);
    x = u32x4{0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu};  // NaN in either type
  } else {
    const int64_t place = kv_place(a.kv, page, position - entry * a.kv.page_size, head);
    const uint16_t* pool = is_k ? a.kv.k : a.kv.v;
    if constexpr (Q4) {
      // values 8 u .. of the row: the low or the high halves of a piece's codes
      u32x4 low, high;
      q4_values(q4_load(reinterpret_cast<const uint8_t*>(pool) + q4_bytes(place), (u >> 2) * 2 + (u & 1)), low, high);
      x = u & 2 ? high : low;
    } else {
      x = load16(pool + place + 8 * u);
    }
  }
  const int64_t at = (static_cast<int64_t>(token) * a.kv.kv_heads + head) * D + 8 * u;
  if constexpr (!OUT32) {
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(out) + at) = x;
  } else {
    f32x4 y[2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t bits = x[i / 2] >> 16 * (i & 1) & 0xFFFFu;
      y[i / 4][i % 4] = BF16 ? __builtin_bit_cast(float, bits << 16) : half_bits_to_float(bits);
    }
    f32x4* to = reinterpret_cast<f32x4*>(static_cast<float*>(out) + at);
    to[0] = y[0];
    to[1] = y[1];
  }
}

}  // namespace

hipError_t launch_kv_rows(const RowsArgs& a, int type, int head_dim, int out_type, hipStream_t stream) {
  const int per = 256 / (head_dim / 8);
  const dim3 grid(static_cast<uint32_t>(a.kv.tokens), static_cast<uint32_t>((2 * a.kv.kv_heads + per - 1) / per));
  const bool wide = out_type == QK_TYPE_F32;
  auto go = [&](auto kernel) { kernel<<<grid, 256, 0, stream>>>(a); };
  auto by_type = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    if (type == QK_TYPE_BF16)
      wide ? go(kv_rows_kernel<D, QK_TYPE_BF16, true>) : go(kv_rows_kernel<D, QK_TYPE_BF16, false>);
    else if (type == QK_TYPE_Q4_1)
      wide ? go(kv_rows_kernel<D, QK_TYPE_Q4_1, true>) : go(kv_rows_kernel<D, QK_TYPE_Q4_1, false>);
    else
      wide ? go(kv_rows_kernel<D, QK_TYPE_F16, true>) : go(kv_rows_kernel<D, QK_TYPE_F16, false>);
  };
  head_dim == 128 ? by_type(std::integral_constant<int, 128>{}) : by_type(std::integral_constant<int, 64>{});
  note("kv_rows_kernel", static_cast<int64_t>(grid.x) * grid.y, head_dim, type, wide);
  return hipGetLastError();
}

}  // namespace qk
