// What the two paged attention kernels share: number types, the split of a
// value into 16-bit parts, a workgroup's tile, and the join of a tile's parts.
//
// A tile is a run of rows of one sequence and one key/value head; row r of the
// sequence is (new token r / group, query head r % group of the head). Both
// kernels form S^T = K Q^T and O^T = V^T P^T on the matrix cores: the query is
// the column of every accumulator, so a row's maximum, sum and rescaling are
// values of the lane itself, and the accumulator registers of S^T, narrowed,
// are the B operand of the second product as they stand (its k index runs over
// the keys in the order that the registers hold them, and V is read in the same
// order, transposed, by ds_read_b64_tr_b16).
//
// Softmax in base 2: weights are 2^(x - M + kLift), x = scale log2(e) q.k. M
// follows the running maximum only when that grows by more than kSlack
// (weights stay below 2^(kLift + kSlack) = 2^14, within fp16), which spares
// nearly all rescalings of the output; kLift keeps weights down to 2^-22 of
// the largest out of fp16's subnormals. Both cancel in the division by the sum.
#pragma once

#include "qk_device.hpp"
#include "qk_launch.hpp"
#include "serving.hpp"

namespace qk {

constexpr float kLift = 8.0f, kSlack = 6.0f;
constexpr float kNoMax = -3.4028234e38f;  // the maximum of no score: no finite score is below it
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <bool BF16>
struct Num;
template <>
struct Num<false> {
  typedef _Float16 T;
  typedef _Float16 V8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mfma16(V8 a, V8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  template <class F>
  static __device__ __forceinline__ F mfma32(V8 a, V8 b, F c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static constexpr uint32_t kExponent = 0x7C007C00u, kCarry = 0x04000400u, kOne = 0x7C00u;
};
template <>
struct Num<true> {
  typedef __bf16 T;
  typedef __bf16 V8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mfma16(V8 a, V8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  template <class F>
  static __device__ __forceinline__ F mfma32(V8 a, V8 b, F c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static constexpr uint32_t kExponent = 0x7F807F80u, kCarry = 0x00800080u, kOne = 0x7F80u;
};

template <bool BF16>
__device__ __forceinline__ uint32_t infinite_halves(uint32_t two) {  // bits 15 and 31: exponent all ones
  return ((two & Num<BF16>::kExponent) + Num<BF16>::kCarry) & 0x80008000u;
}
template <bool BF16>
__device__ __forceinline__ bool any_infinite(u32x4 v) {
  return (infinite_halves<BF16>(v.x) | infinite_halves<BF16>(v.y) | infinite_halves<BF16>(v.z) |
          infinite_halves<BF16>(v.w)) != 0;
}
// v with its infinities and NaN as zeros.
template <bool BF16>
__device__ __forceinline__ u32x4 only_finite(u32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((v[i] & Num<BF16>::kOne) == Num<BF16>::kOne) v[i] &= 0xFFFF0000u;
    if ((v[i] >> 16 & Num<BF16>::kOne) == Num<BF16>::kOne) v[i] &= 0x0000FFFFu;
  }
  return v;
}

// Parts of an fp32 value: 16-bit q is its own only part; F32 is two fp16 parts
// (22 bits; q rows are first scaled by a power of two into fp16's upper range,
// so that the second part stays normal) or three bf16 parts (24 bits).
template <bool BF16, bool Q32>
constexpr int kParts = Q32 ? (BF16 ? 3 : 2) : 1;

template <bool BF16, int NP>
__device__ __forceinline__ void split8(const float (&x)[8], typename Num<BF16>::V8 (&out)[NP]) {
  typedef typename Num<BF16>::T T;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float rest = x[i];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const T part = static_cast<T>(rest);
      out[p][i] = part;
      rest -= static_cast<float>(part);
    }
  }
}

__device__ __forceinline__ float swap16_max(float v) {
  const auto t = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false,
                                                  false);
  const unsigned a = t[0], b = t[1];
  return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float swap32_max(float v) {
  const auto t = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false,
                                                  false);
  const unsigned a = t[0], b = t[1];
  return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

// Sequence by sequence, ceil(rows / tile_rows) tiles each: wave-parallel running
// sums of the tile counts until they pass `tile`. Where `report`, lengths that do
// not fit are reported, of all sequences: one without rows has no tile.
__device__ __forceinline__ AttentionTile find_tile(const AttentionArgs& a, int tile, int tile_rows, bool report) {
  const int lane = static_cast<int>(threadIdx.x & 63);
  AttentionTile t;
  t.s = -1;
  int before = 0;
  for (int base = 0; base < a.kv.sequences; base += 64) {
    const int s = base + lane;
    int mine = 0;
    KvSequence q{};
    if (s < a.kv.sequences) {
      q = kv_sequence(a.kv, s);
      mine = (q.count * a.group + tile_rows - 1) / tile_rows;
    }
    if (report && q.fault) kv_fault(a.kv, QK_KV_FAULT_LENGTH);
    if (t.s >= 0) continue;
    int run = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int other = __shfl_up(run, off);
      if (lane >= off) run += other;
    }
    const uint64_t past = __ballot(before + run > tile);
    if (past) {
      const int at = __builtin_ctzll(past);
      t.s = base + at;
      t.row = __builtin_amdgcn_readlane(q.row, at);
      t.count = __builtin_amdgcn_readlane(q.count, at);
      t.first = __builtin_amdgcn_readlane(q.first, at);
      t.beyond = __builtin_amdgcn_readlane(q.beyond ? 1 : 0, at) != 0;
      t.begin = (tile - before - __builtin_amdgcn_readlane(run - mine, at)) * tile_rows;
      if (!report) break;
    }
    before += __builtin_amdgcn_readlane(run, 63);
  }
  if (t.s >= 0) tile_keys(a.group, a.window, tile_rows, t);
  return t;
}

// The most keys that a row of any sequence sees.
__device__ __forceinline__ int longest_context(const AttentionArgs& a) {
  const int lane = static_cast<int>(threadIdx.x & 63);
  int most = 0;
  for (int s = lane; s < a.kv.sequences; s += 64) {
    const KvSequence q = kv_sequence(a.kv, s);
    const int keys = kv_keys(q);
    most = keys > most ? keys : most;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const int other = __shfl_xor(most, off);
    most = other > most ? other : most;
  }
  return __builtin_amdgcn_readfirstlane(a.window > 0 && most > a.window ? a.window : most);
}

// Values that another workgroup of the launch reads: coherent at agent scope,
// past this XCD's L2 (a release fence there would write all of it back).
__device__ __forceinline__ void put(float* p, float x, float y) {
  const uint64_t v = static_cast<uint64_t>(__builtin_bit_cast(uint32_t, y)) << 32 | __builtin_bit_cast(uint32_t, x);
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void get(const float* p, float& x, float& y) {
  const uint64_t v =
      __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  x = __builtin_bit_cast(float, static_cast<uint32_t>(v));
  y = __builtin_bit_cast(float, static_cast<uint32_t>(v >> 32));
}

// After a workgroup has put its part: true in the workgroup that is the last
// of `used` to get here (all parts are visible to it), which also leaves the
// counter at zero for the next call.
__device__ __forceinline__ bool last_to_arrive(uint32_t* counter, int used, uint32_t& shared_word) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the thread's stores have reached memory
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t n = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (n + 1 == static_cast<uint32_t>(used))
      __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    shared_word = n;
  }
  __syncthreads();
  return shared_word + 1 == static_cast<uint32_t>(used);
}

// Four values of a row's result in q's type.
template <bool BF16, bool Q32>
__device__ __forceinline__ void store_row(void* out, int64_t at, f32x4 y) {
  if constexpr (Q32) {
    *reinterpret_cast<f32x4*>(static_cast<float*>(out) + at) = y;
  } else {
    typedef typename Num<BF16>::T T;
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 z;
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = static_cast<T>(y[e]);
    *reinterpret_cast<T4*>(static_cast<T*>(out) + at) = z;
  }
}

// A row's sum and maximum as its log of the sum of exp.
__device__ __forceinline__ float row_lse(float top, float sum) {
  return sum == 0.0f ? -__builtin_inff() : (top - kLift) * kLn2 + logf(sum);
}

}  // namespace qk
