// Attention of new tokens over a paged cache: one wave per (token, query head),
// 64 keys at a time, one pass with a running maximum and sum.
#include "qk_device.hpp"
#include "qk_launch.hpp"
#include "serving.hpp"

namespace qk {
namespace {

template <bool BF16>
__device__ __forceinline__ float widen(uint16_t b) {
  if constexpr (BF16)
    return __builtin_bit_cast(float, static_cast<uint32_t>(b) << 16);
  else
    return half_bits_to_float(b);
}
template <bool BF16>
__device__ __forceinline__ uint16_t narrow(float v) {
  if constexpr (BF16)
    return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
  else
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}
__device__ __forceinline__ float wave_max_any(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off));
  return v;
}

template <int D, bool BF16, bool Q32>
__global__ __launch_bounds__(64) void attention_row_kernel(const AttentionArgs a) {
  __shared__ float qs[D], ps[64];
  __shared__ int64_t at[64];
  const int lane = static_cast<int>(threadIdx.x);
  const int token = static_cast<int>(blockIdx.x), h = static_cast<int>(blockIdx.y);
  const int s = kv_find_sequence(a.kv, token);
  const KvSequence seq = kv_sequence(a.kv, s);
  if (seq.fault && lane == 0) kv_fault(a.kv, QK_KV_FAULT_LENGTH);
  if (token < seq.row || token >= seq.row + seq.count) return;
  const int position = seq.first + (token - seq.row);
  const int64_t q_at = token * a.q_stride + static_cast<int64_t>(h) * D;
  for (int i = lane; i < D; i += 64)
    qs[i] = Q32 ? static_cast<const float*>(a.q)[q_at + i] : widen<BF16>(static_cast<const uint16_t*>(a.q)[q_at + i]);
  __syncthreads();
  float top = -__builtin_inff(), total = 0.0f, o[D / 64] = {};
  bool bad = false;
  const int begin = a.window > 0 && position >= a.window ? position - a.window + 1 : 0;
  for (int base = begin; base <= position; base += 64) {
    const int j = base + lane;
    float score = -__builtin_inff();
    int64_t place = 0;
    if (j <= position) {
      const int entry = j / a.kv.page_size;
      const int page = kv_page(a.kv, s, entry);
      if (page < 0) {
        bad = true;
      } else {
        place = kv_place(a.kv, page, j - entry * a.kv.page_size, h / a.group);
        float dot = 0.0f;
        for (int i = 0; i < D; i += 8) {
          const u16x8 k = *reinterpret_cast<const u16x8*>(a.kv.k + place + i);
#pragma unroll
          for (int e = 0; e < 8; ++e) dot = __builtin_fmaf(qs[i + e], widen<BF16>(k[e]), dot);
        }
        score = dot * a.scale;
      }
    }
    const float peak = fmaxf(top, wave_max_any(score));
    const float rescale = peak == -__builtin_inff() ? 1.0f : expf(top - peak);
    const float p = score == -__builtin_inff() ? 0.0f : expf(score - peak);
    total = total * rescale + row_lanes_sum<64>(p);
    top = peak;
    ps[lane] = p;
    at[lane] = place;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < D / 64; ++c) o[c] *= rescale;
    for (int i = 0; i < 64 && base + i <= position; ++i)
#pragma unroll
      for (int c = 0; c < D / 64; ++c) o[c] = __builtin_fmaf(ps[i], widen<BF16>(a.kv.v[at[i] + c * 64 + lane]), o[c]);
    __syncthreads();
  }
  bad = __any(bad);
  if (bad && lane == 0) kv_fault(a.kv, QK_KV_FAULT_PAGE);
  const int64_t out_at = (static_cast<int64_t>(token) * a.q_heads + h) * D;
  for (int c = 0; c < D / 64; ++c) {
    const float y = bad ? __builtin_nanf("") : total > 0.0f ? o[c] / total : total == 0.0f ? 0.0f : total;
    if (Q32)
      static_cast<float*>(a.out)[out_at + c * 64 + lane] = y;
    else
      static_cast<uint16_t*>(a.out)[out_at + c * 64 + lane] = narrow<BF16>(y);
  }
  if (a.lse && lane == 0)
    a.lse[static_cast<int64_t>(token) * a.q_heads + h] = bad ? __builtin_nanf("") : top + logf(total);
}

}  // namespace

size_t paged_attention_workspace(int64_t, int64_t, int64_t, int64_t, int, int, int, int64_t, int64_t) { return 0; }

hipError_t launch_paged_attention(const AttentionArgs& a, int type, int head_dim, int q_type, int64_t, void*,
                                  hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(a.kv.tokens), static_cast<uint32_t>(a.q_heads));
  const bool bf16 = type == QK_TYPE_BF16, q32 = q_type == QK_TYPE_F32;
  auto go = [&](auto kernel) { kernel<<<grid, 64, 0, stream>>>(a); };
  if (head_dim == 128)
    bf16 ? (q32 ? go(attention_row_kernel<128, true, true>) : go(attention_row_kernel<128, true, false>))
         : (q32 ? go(attention_row_kernel<128, false, true>) : go(attention_row_kernel<128, false, false>));
  else
    bf16 ? (q32 ? go(attention_row_kernel<64, true, true>) : go(attention_row_kernel<64, true, false>))
         : (q32 ? go(attention_row_kernel<64, false, true>) : go(attention_row_kernel<64, false, false>));
  note("attention_row_kernel", static_cast<int64_t>(grid.x) * grid.y, head_dim, bf16, q32);
  return hipGetLastError();
}

}  // namespace qk
