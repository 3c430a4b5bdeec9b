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
//
// Q4_1 caches: a finished row goes through LDS, from where each lane takes four
// values and the four 16 further on, the codes of one dword, four lanes a block. The norm's
// sum of squares and the sine and cosine are formed in 64 bits there and rounded once, so
// that codes do not depend on the order of a sum; the inverse root, the scaling and the
// rotation (products rounded each) are fp32. Of 4.2 million keys' codes two differ from
// those of other fp32 steps, at borders between codes. 4096 tokens, 173 MB with the
// rotated q: 32 us (5.3 TB/s).
#include "q4_1.hpp"
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

// a c + b n. EACH: every product rounded by itself, so that the codes of a Q4_1 cache do
// not depend on which of them the compiler fuses.
template <bool EACH>
__device__ __forceinline__ float turned(float a, float c, float b, float n) {
  if constexpr (EACH) {
#pragma clang fp contract(off)
    return a * c + b * n;
  }
  return a * c + b * n;
}

// A row's lane of a Q4_1 cache: x0 its values 4 u .. of block `u / 4`, x1 the ones 16
// on, u = lane of the block. The block's d and m are rounded first (d towards zero,
// so that no value leaves F16), and the codes go by them. fp32, as the row is: a value
// that near a border between two codes may come out as the other one.
__device__ __forceinline__ void store_q4(uint8_t* row, int u, f32x4 x0, f32x4 x1) {
  float low = fminf(fminf(fminf(x0[0], x0[1]), fminf(x0[2], x0[3])), fminf(fminf(x1[0], x1[1]), fminf(x1[2], x1[3])));
  float high = fmaxf(fmaxf(fmaxf(x0[0], x0[1]), fmaxf(x0[2], x0[3])), fmaxf(fmaxf(x1[0], x1[1]), fmaxf(x1[2], x1[3])));
  float zeros = 0.0f;  // or NaN, if a value is NaN or infinite
#pragma unroll
  for (int i = 0; i < 4; ++i) zeros += 0.0f * x0[i] + 0.0f * x1[i];
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    low = fminf(low, __shfl_xor(low, off));
    high = fmaxf(high, __shfl_xor(high, off));
    zeros += __shfl_xor(zeros, off);
  }
  const _Float16 m = static_cast<_Float16>(low);
  const float base = static_cast<float>(m), span = fmaxf(high - base, 0.0f) / 15.0f;
  _Float16 d = static_cast<_Float16>(span);
  uint32_t d_bits = __builtin_bit_cast(uint16_t, d);
  if (static_cast<float>(d) > span) --d_bits;
  const float step = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(d_bits)));
  const float inverse = step == 0.0f ? 0.0f : 1.0f / step;
  const float top = static_cast<float>(static_cast<_Float16>(high));
  const bool broken = !(zeros == 0.0f) || fabsf(base) == __builtin_inff() || fabsf(top) == __builtin_inff();
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = static_cast<uint32_t>(fminf(fmaxf(rintf((x0[i] - base) * inverse), 0.0f), 15.0f));
    const uint32_t hi = static_cast<uint32_t>(fminf(fmaxf(rintf((x1[i] - base) * inverse), 0.0f), 15.0f));
    codes |= (lo | hi << 4) << (8 * i);
  }
  uint8_t* block = row + (u >> 2) * kQ4Bytes;
  *reinterpret_cast<uint32_t*>(block + 4 + 4 * (u & 3)) = broken ? 0u : codes;
  if ((u & 3) == 0)
    *reinterpret_cast<uint32_t*>(block) = broken ? 0x7E007E00u : d_bits | static_cast<uint32_t>(__builtin_bit_cast(uint16_t, m)) << 16;
}

template <int D, bool BF16, bool Q32, bool Q4>
__global__ __launch_bounds__(256) void kv_append_kernel(const AppendArgs a) {
  constexpr int L = D / 8;  // lanes a row
  __shared__ float cosine[D / 2], sine[D / 2];
  __shared__ __attribute__((aligned(16))) float finished[Q4 ? 256 * 8 : 4];  // a Q4_1 cache's rows
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
    // where tokens were evicted, a token's position is not its place in the cache
    const int64_t angle = a.seen ? static_cast<int64_t>(a.seen[s]) - a.kv.context[s] + position : position;
    const double turns = static_cast<double>(angle) * (exp2(a.turns_log2 * tid) * 0.15915494309189535);
    if constexpr (Q4) {  // codes are decided by the last bits of what is stored
      double sn, cs;
      sincospi(2.0 * (turns - floor(turns)), &sn, &cs);
      cosine[tid] = static_cast<float>(cs);
      sine[tid] = static_cast<float>(sn);
    } else {
      const float part = static_cast<float>(turns - floor(turns));
      float sn, cs;
      sincospif(2.0f * part, &sn, &cs);
      cosine[tid] = cs;
      sine[tid] = sn;
    }
  }
  __syncthreads();
  if (row >= rows) return;

  const float* norm = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
  if (norm) {
    float sum = 0.0f;
    if constexpr (Q4) {
      double squares = 0.0;
#pragma unroll
      for (int i = 0; i < 4; ++i) squares += static_cast<double>(x0[i]) * x0[i] + static_cast<double>(x1[i]) * x1[i];
#pragma unroll
      for (int off = 1; off < L; off <<= 1) squares += __shfl_xor(squares, off);
      sum = static_cast<float>(squares);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) sum = __builtin_fmaf(x0[i], x0[i], __builtin_fmaf(x1[i], x1[i], sum));
      sum = row_lanes_sum<L>(sum);
    }
    const float inv = rsqrtf(sum * (1.0f / D) + a.eps);
    x0 = x0 * inv * *reinterpret_cast<const f32x4_a4*>(norm + first);
    x1 = x1 * inv * *reinterpret_cast<const f32x4_a4*>(norm + second);
  }
  if (8 * u < dims) {
    if (split) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float c = cosine[4 * u + i], n = sine[4 * u + i], b = x0[i];
        x0[i] = turned<Q4>(b, c, x1[i], -n);
        x1[i] = turned<Q4>(x1[i], c, b, n);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float c0 = cosine[4 * u + i], n0 = sine[4 * u + i], b0 = x0[2 * i];
        const float c1 = cosine[4 * u + 2 + i], n1 = sine[4 * u + 2 + i], b1 = x1[2 * i];
        x0[2 * i] = turned<Q4>(b0, c0, x0[2 * i + 1], -n0);
        x0[2 * i + 1] = turned<Q4>(x0[2 * i + 1], c0, b0, n0);
        x1[2 * i] = turned<Q4>(b1, c1, x1[2 * i + 1], -n1);
        x1[2 * i + 1] = turned<Q4>(x1[2 * i + 1], c1, b1, n1);
      }
    }
  }
  if (is_q && Q32) {
    float* out = static_cast<float*>(a.q_out) + (static_cast<int64_t>(token) * a.q_heads + head) * D;
    *reinterpret_cast<f32x4*>(out + first) = x0;
    *reinterpret_cast<f32x4*>(out + second) = x1;
    return;
  }
  uint16_t* out = nullptr;
  int64_t place = 0;
  if (is_q) {
    out = static_cast<uint16_t*>(a.q_out) + (static_cast<int64_t>(token) * a.q_heads + head) * D;
  } else {
    const int entry = position < 0 ? -1 : position / a.kv.page_size;
    const int page = kv_page(a.kv, s, entry);
    if (page < 0) {
      if (u == 0) kv_fault(a.kv, position < 0 ? QK_KV_FAULT_LENGTH : QK_KV_FAULT_PAGE);
      return;
    }
    place = kv_place(a.kv, page, position - entry * a.kv.page_size, head);
    out = (is_k ? a.kv.k : a.kv.v) + place;
  }
  if constexpr (Q4) {
    if (!is_q) {  // all of a row's lanes, which lie in one wave, come here
      float* row_values = finished + tid / L * D;
      *reinterpret_cast<f32x4*>(row_values + first) = x0;
      *reinterpret_cast<f32x4*>(row_values + second) = x1;
      __builtin_amdgcn_wave_barrier();
      const int at = (u >> 2) * kQ4Values + 4 * (u & 3);
      x0 = *reinterpret_cast<const f32x4*>(row_values + at);
      x1 = *reinterpret_cast<const f32x4*>(row_values + at + 16);
      store_q4(reinterpret_cast<uint8_t*>(is_k ? a.kv.k : a.kv.v) + q4_bytes(place), u, x0, x1);
      return;
    }
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
  const bool q4 = type == QK_TYPE_Q4_1;
  if (head_dim == 128)
    bf16 ? (q32 ? go(kv_append_kernel<128, true, true, false>) : go(kv_append_kernel<128, true, false, false>))
    : q4 ? (q32 ? go(kv_append_kernel<128, false, true, true>) : go(kv_append_kernel<128, false, false, true>))
         : (q32 ? go(kv_append_kernel<128, false, true, false>) : go(kv_append_kernel<128, false, false, false>));
  else
    bf16 ? (q32 ? go(kv_append_kernel<64, true, true, false>) : go(kv_append_kernel<64, true, false, false>))
    : q4 ? (q32 ? go(kv_append_kernel<64, false, true, true>) : go(kv_append_kernel<64, false, false, true>))
         : (q32 ? go(kv_append_kernel<64, false, true, false>) : go(kv_append_kernel<64, false, false, false>));
  note("kv_append_kernel", static_cast<int64_t>(grid.x) * grid.y, head_dim, bf16, q32, q4);
  return hipGetLastError();
}

}  // namespace qk
