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
// Softmax in base 2: weights are 2^(x - M + kLift), x = scale log2(e) q.k. M, the
// row's reference, follows the running maximum only when that grows by more than
// kSlack (weights stay below 2^(kLift + kSlack), within fp16), which spares
// nearly all rescalings of the output. Both cancel in the division by the sum.
//
// fp16 holds a weight to its last bit down to 2^-14, in two parts to 2^-20 of
// itself down to 2^-5 (kReach below M), and smaller ones to 2^-25. That is far
// below what counts in most rows, but not where the large weights' values are near
// zero, as those of a first token that takes most of the mass are. So where a
// block of keys over an F16 cache holds smaller weights, and a row's output does not
// yet outweigh what they may lack (kSound), M sinks and what they lack is
// added: sums and outputs are fp32 and have the range for it, down to weights of
// 2^-100 of the row's sum. bf16 has that range itself.
#pragma once

#include "qk_device.hpp"
#include "qk_launch.hpp"
#include "serving.hpp"

namespace qk {

template <bool BF16>
constexpr float kLift = BF16 ? 8.0f : 9.0f;
constexpr float kSlack = 6.0f;
template <int NP>  // F16, weights in NP parts
constexpr float kReach = kLift<false> + (NP > 1 ? 5.0f : 14.0f);
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
  if constexpr (!BF16) {  // 0 times each: zeros, or a NaN
    typedef _Float16 H2 __attribute__((ext_vector_type(2)));
    H2 sum = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t two = v[i];
      sum = __builtin_elementwise_fma(__builtin_bit_cast(H2, two), H2{}, sum);
    }
    return (__builtin_bit_cast(uint32_t, sum) & 0x7FFF7FFFu) != 0;
  }
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

// The reference of a row over an F16 cache that has to rise to `most`. Whole numbers,
// so that rescaling is exact; weights in two parts leave half of the room above
// for later, larger ones, as more of the smaller ones fit below.
template <int NP>
__device__ __forceinline__ float risen(float top, float most) {
  return most > top + kSlack ? ceilf(most - (NP > 1 ? kSlack / 2 : 0.0f)) : top;
}
// What weights of NP fp16 parts lack is at most 2^-25 each where it counts. A
// row's output outweighs it from kSound times the largest value v on: were all of
// 2^13 smaller weights short by that, and their values alike, it would be 2^-19
// (two parts) or 2^-12 of the output.
template <int NP>
constexpr float kSound = NP > 1 ? 0x1p7f : 1.0f;
// Up to which reference a row is sound whose output is `size` at `top`.
template <int NP>
__device__ __forceinline__ float sound_to(float top, float size, float largest) {
  const int spare = __builtin_amdgcn_frexp_expf(size) - 1 - __builtin_amdgcn_frexp_expf(kSound<NP> * largest);
  return largest == 0.0f ? __builtin_inff() : size == 0.0f ? -__builtin_inff() : top + static_cast<float>(spare);
}
// How far the reference of a row sinks that is not sound, its output at most `size`
// and its sum `sum`: to where it may be, but no further than that what the weights
// lack (2^-22 or 2^-11 of them) stays within fp16, nor at all beyond 2^112, so that
// neither later blocks nor the join of 2048 parts leave fp32.
template <int NP>
__device__ __forceinline__ int sinking(float size, float sum, float largest) {
  constexpr int kMost = NP > 1 ? 20 : 12;
  const int lacks = __builtin_amdgcn_frexp_expf(kSound<NP> * largest) - __builtin_amdgcn_frexp_expf(size) + 3;
  const int by = size == 0.0f || lacks > kMost ? kMost : lacks < 1 ? 1 : lacks;
  return by + __builtin_amdgcn_frexp_expf(fmaxf(size, sum)) > 112 ? 0 : by;
}
// The larger of two pairs of fp16 values by their sizes, both finite.
__device__ __forceinline__ uint32_t larger_sizes(uint32_t x, uint32_t y) {
  typedef uint16_t U2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(U2, x & 0x7FFF7FFFu),
                                                                 __builtin_bit_cast(U2, y & 0x7FFF7FFFu)));
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

// A row's sum and reference as its log of the sum of exp.
template <bool BF16>
__device__ __forceinline__ float row_lse(float top, float sum) {
  return sum == 0.0f ? -__builtin_inff() : (top - kLift<BF16>) * kLn2 + logf(sum);
}

}  // namespace qk
