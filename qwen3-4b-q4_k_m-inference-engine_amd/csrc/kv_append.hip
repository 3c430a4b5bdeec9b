// New tokens' keys and values into their cache pages, with the head RMSNorm and
// the rotary positions of q and k on the way, and the rotated q: one launch.
//
// A head's row is D/8 lanes of 8 values each (two 16-byte loads). Lane u of a
// row holds the two quads that rotate with each other: values 4u .. 4u+3 and
// dims/2 + 4u .. (split halves), or 8u .. 8u+7 (neighbouring pairs, and the
// values past `dims`, which stay), so a rotation needs no other lane and the
// norm one sum over the row's lanes. A workgroup takes one token and up to 16
// (D = 128) or 32 (D = 64) of its rows; its first D/2 threads form the token's
// dims/2 angles once, through LDS.
//
// Angles: a far position loses its angle in fp32 (position 10^5: 6e-3 of a
// radian), so position * base^(-2j/dims) / 2pi is formed in 64 bits and cut to
// its fraction of a turn before the fp32 sine and cosine.
//
// Memory bounds long prompts: 4096 tokens of 32 + 2 x 8 heads of 128, 184 MB, 38 us
// (4.8 TB/s, a copy's rate); launch and three dependent reads (lengths, page id,
// values) a decode step: one token 2.7 us, 64 3.9.
#include "qk_device.hpp"
#include "qk_launch.hpp"
#include "serving.hpp"

namespace qk {
namespace {

template <bool BF16>
__device__ __forceinline__ uint16_t narrow(float v) {
  if constexpr (BF16)
    return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
  else
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}

template <int D, bool BF16, bool Q32>
__global__ __launch_bounds__(256) void kv_append_kernel(const AppendArgs a) {
  constexpr int L = D / 8;  // lanes a row
  __shared__ float cosine[D / 2], sine[D / 2];
  const int tid = static_cast<int>(threadIdx.x);
  const int token = static_cast<int>(blockIdx.x);
  const int row = static_cast<int>(blockIdx.y) * (256 / L) + tid / L;
  const int rows = a.q_heads + 2 * a.kv.kv_heads;
  const int u = tid % L;
  const bool is_q = row < a.q_heads, is_k = !is_q && row < a.q_heads + a.kv.kv_heads;
  const int dims = is_q || is_k ? a.dims : 0;

  // where the lane's two quads lie in the row
  const bool split = 8 * u < dims && !a.interleaved;
  const int first = split ? 4 * u : 8 * u, second = split ? dims / 2 + 4 * u : 8 * u + 4;
  f32x4 x0 = {}, x1 = {};
  int head = 0;
  if (row < rows) {
    head = is_q ? row : is_k ? row - a.q_heads : row - a.q_heads - a.kv.kv_heads;
    const float* src = is_q ? a.q + token * a.q_stride : is_k ? a.k + token * a.k_stride : a.v + token * a.v_stride;
    src += head * D;
    x0 = *reinterpret_cast<const f32x4_a4*>(src + first);
    x1 = *reinterpret_cast<const f32x4_a4*>(src + second);
  }
  const int s = kv_find_sequence(a.kv, token);
  const KvSequence seq = kv_sequence(a.kv, s);
  if (blockIdx.x == 0 && blockIdx.y == 0)  // lengths that do not fit, of sequences without rows too
    for (int i = tid; i < a.kv.sequences; i += 256)
      if (kv_sequence(a.kv, i).fault) kv_fault(a.kv, QK_KV_FAULT_LENGTH);
  if (token < seq.row || token >= seq.row + seq.count) return;  // no sequence owns this row
  const int position = seq.first + (token - seq.row);
  if (tid < a.dims / 2) {
    const double turns = position * (exp2(a.turns_log2 * tid) * 0.15915494309189535);
    const float part = static_cast<float>(turns - floor(turns));
    float sn, cs;
    sincospif(2.0f * part, &sn, &cs);
    cosine[tid] = cs;
    sine[tid] = sn;
  }
  __syncthreads();
  if (row >= rows) return;

  const float* norm = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
  if (norm) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = __builtin_fmaf(x0[i], x0[i], __builtin_fmaf(x1[i], x1[i], sum));
    sum = row_lanes_sum<L>(sum);
    const float inv = rsqrtf(sum * (1.0f / D) + a.eps);
    x0 = x0 * inv * *reinterpret_cast<const f32x4_a4*>(norm + first);
    x1 = x1 * inv * *reinterpret_cast<const f32x4_a4*>(norm + second);
  }
  if (8 * u < dims) {
    if (split) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float c = cosine[4 * u + i], n = sine[4 * u + i], b = x0[i];
        x0[i] = b * c - x1[i] * n;
        x1[i] = x1[i] * c + b * n;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float c0 = cosine[4 * u + i], n0 = sine[4 * u + i], b0 = x0[2 * i];
        const float c1 = cosine[4 * u + 2 + i], n1 = sine[4 * u + 2 + i], b1 = x1[2 * i];
        x0[2 * i] = b0 * c0 - x0[2 * i + 1] * n0;
        x0[2 * i + 1] = x0[2 * i + 1] * c0 + b0 * n0;
        x1[2 * i] = b1 * c1 - x1[2 * i + 1] * n1;
        x1[2 * i + 1] = x1[2 * i + 1] * c1 + b1 * n1;
      }
    }
  }
  if (is_q && Q32) {
    float* out = static_cast<float*>(a.q_out) + (static_cast<int64_t>(token) * a.q_heads + head) * D;
    *reinterpret_cast<f32x4*>(out + first) = x0;
    *reinterpret_cast<f32x4*>(out + second) = x1;
    return;
  }
  uint16_t* out;
  if (is_q) {
    out = static_cast<uint16_t*>(a.q_out) + (static_cast<int64_t>(token) * a.q_heads + head) * D;
  } else {
    const int entry = position < 0 ? -1 : position / a.kv.page_size;
    const int page = kv_page(a.kv, s, entry);
    if (page < 0) {
      if (u == 0) kv_fault(a.kv, position < 0 ? QK_KV_FAULT_LENGTH : QK_KV_FAULT_PAGE);
      return;
    }
    out = (is_k ? a.kv.k : a.kv.v) + kv_place(a.kv, page, position - entry * a.kv.page_size, head);
  }
  typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
  u16x4 y0, y1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y0[i] = narrow<BF16>(x0[i]);
    y1[i] = narrow<BF16>(x1[i]);
  }
  *reinterpret_cast<u16x4*>(out + first) = y0;
  *reinterpret_cast<u16x4*>(out + second) = y1;
}

__global__ void kv_fault_clear_kernel(uint32_t* word, uint32_t bits) { atomicAnd(word, ~bits); }

}  // namespace

hipError_t launch_kv_fault_clear(uint32_t* word, uint32_t bits, hipStream_t stream) {
  kv_fault_clear_kernel<<<1, 1, 0, stream>>>(word, bits);
  return hipGetLastError();
}

hipError_t launch_kv_append(const AppendArgs& a, int type, int head_dim, int q_type, hipStream_t stream) {
  const int rows = a.q_heads + 2 * a.kv.kv_heads, per = 256 / (head_dim / 8);
  const dim3 grid(static_cast<uint32_t>(a.kv.tokens), static_cast<uint32_t>((rows + per - 1) / per));
  const bool bf16 = type == QK_TYPE_BF16, q32 = q_type == QK_TYPE_F32;
  auto go = [&](auto kernel) { kernel<<<grid, 256, 0, stream>>>(a); };
  if (head_dim == 128)
    bf16 ? (q32 ? go(kv_append_kernel<128, true, true>) : go(kv_append_kernel<128, true, false>))
         : (q32 ? go(kv_append_kernel<128, false, true>) : go(kv_append_kernel<128, false, false>));
  else
    bf16 ? (q32 ? go(kv_append_kernel<64, true, true>) : go(kv_append_kernel<64, true, false>))
         : (q32 ? go(kv_append_kernel<64, false, true>) : go(kv_append_kernel<64, false, false>));
  note("kv_append_kernel", static_cast<int64_t>(grid.x) * grid.y, head_dim, bf16, q32);
  return hipGetLastError();
}

}  // namespace qk
