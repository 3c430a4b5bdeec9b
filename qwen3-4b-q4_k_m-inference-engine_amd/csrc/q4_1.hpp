// Cached rows in Q4_1 blocks (GGUF type 3): 32 values in 20 bytes, a 16-bit scale
// d and lowest value m, then 16 bytes of codes, byte j with value j in its low
// half and value j + 16 in its high one. A code c stands for d c + m, rounded
// once to F16: what attention multiplies is then an F16 cache's row, and the
// rounding (2^-12 of the value) is far below the code's own (1/30 of a block's range).
//
// The codes become F16 without a conversion: a nibble under the exponent of 1024
// (bits 0 .. 3) or of 64 (bits 4 .. 7) is 1024 + c or 64 + c, less that is c,
// exactly, and one packed fma gives the value: 14 instructions for eight values in
// their order, 13 in any.
#pragma once

#include "qk_device.hpp"

namespace qk {

constexpr int kQ4Values = 32, kQ4Bytes = 20;

// Byte offset of a row from its offset in values (a multiple of 32).
__host__ __device__ __forceinline__ int64_t q4_bytes(int64_t values) { return (values >> 5) * kQ4Bytes; }

typedef uint32_t u32x2_q4 __attribute__((ext_vector_type(2)));
typedef u32x2_q4 u32x2_a4 __attribute__((aligned(4)));

// Half of a block's codes: values 8 half .. 8 half + 7 in the low halves of its
// bytes, 16 + 8 half .. in the high ones; and the block's d and m.
struct Q4Piece {
  u32x2_q4 codes;
  uint32_t dm;
};
// Piece `unit` of a row: block unit / 2, half unit % 2.
__device__ __forceinline__ Q4Piece q4_load(const uint8_t* row, int unit) {
  const uint8_t* block = row + (unit >> 1) * kQ4Bytes;
  return {*reinterpret_cast<const u32x2_a4*>(block + 4 + 8 * (unit & 1)), *reinterpret_cast<const uint32_t*>(block)};
}
// Where its values lie in a row, in chunks of eight: this one, and two on.
__device__ __forceinline__ int q4_chunk(int unit) { return 4 * (unit >> 1) + (unit & 1); }

typedef _Float16 half2_q4 __attribute__((ext_vector_type(2)));

// Codes as F16: `two` holds one in bits 0 .. 3 of each half, or in bits 4 .. 7. The
// exponents come from a register that the compiler does not see through: with two
// constants an and and an or would be two instructions.
struct Q4Exponents {
  uint32_t low = 0x64006400u, high = 0x54005400u;  // of 1024 and of 64
  __device__ __forceinline__ Q4Exponents() { asm("" : "+v"(low), "+v"(high)); }
};
__device__ __forceinline__ half2_q4 q4_low(uint32_t two, const Q4Exponents& e) {
  return __builtin_bit_cast(half2_q4, (two & 0x000F000Fu) | e.low) +
         half2_q4{static_cast<_Float16>(-1024.0f), static_cast<_Float16>(-1024.0f)};
}
__device__ __forceinline__ half2_q4 q4_high(uint32_t two, const Q4Exponents& e) {
  return __builtin_bit_cast(half2_q4, (two & 0x00F000F0u) | e.high) +
         half2_q4{static_cast<_Float16>(-64.0f), static_cast<_Float16>(-64.0f)};
}

// Eight values of a dword of codes as four pairs, of bytes 0 and 2 and then 1 and 3, low
// halves first: values 0 2 16 18 1 3 17 19 from the dword's first on.
__device__ __forceinline__ void q4_pairs(uint32_t codes, half2_q4 d, half2_q4 m, const Q4Exponents& e, half2_q4 (&out)[4]) {
  out[0] = __builtin_elementwise_fma(q4_low(codes, e), d, m);
  out[1] = __builtin_elementwise_fma(q4_high(codes, e), d, m);
  out[2] = __builtin_elementwise_fma(q4_low(codes >> 8, e), d, m);
  out[3] = __builtin_elementwise_fma(q4_high(codes >> 8, e), d, m);
}
// Where the i-th of those lies.
__host__ __device__ constexpr int q4_pair_value(int i) { return 2 * (i & 1) + (i & 2 ? 16 : 0) + (i >> 2); }

// A lane's share of a row that four lanes load: a quarter of its codes, KS = D / 32
// dwords of one block, and that block's d and m.
template <int KS>
struct Q4Quarter {
  typedef uint32_t Codes __attribute__((ext_vector_type(KS)));
  Codes codes;
  uint32_t dm;
};
template <int KS>
__device__ __forceinline__ int q4_quarter_block(int quarter) {
  return KS == 4 ? quarter : quarter >> 1;
}
template <int KS>
__device__ __forceinline__ Q4Quarter<KS> q4_load_quarter(const uint8_t* row, int quarter) {
  typedef typename Q4Quarter<KS>::Codes Codes_a4 __attribute__((aligned(4)));
  const uint8_t* block = row + q4_quarter_block<KS>(quarter) * kQ4Bytes;
  return {*reinterpret_cast<const Codes_a4*>(block + 4 + (KS == 4 ? 0 : 8 * (quarter & 1))),
          *reinterpret_cast<const uint32_t*>(block)};
}
// Where the values of its dword s begin in the row.
template <int KS>
__device__ __forceinline__ int q4_quarter_value(int quarter, int s) {
  return (KS == 4 ? 32 * quarter : 32 * (quarter >> 1) + 8 * (quarter & 1)) + 4 * s;
}

// Eight values of four bytes of codes: their low halves' to `low`, their high halves' to `high`.
__device__ __forceinline__ void q4_values4(uint32_t codes, half2_q4 d, half2_q4 m, const Q4Exponents& e, uint32_t (&low)[2],
                                           uint32_t (&high)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t two = __builtin_amdgcn_perm(0u, codes, i == 0 ? 0x0C010C00u : 0x0C030C02u);  // bytes 2 i and 2 i + 1
    low[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(q4_low(two, e), d, m));
    high[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(q4_high(two, e), d, m));
  }
}
// The sixteen values of a piece: chunks q4_chunk(unit) and q4_chunk(unit) + 2.
__device__ __forceinline__ void q4_values(const Q4Piece& p, u32x4& low, u32x4& high) {
  const half2_q4 dm = __builtin_bit_cast(half2_q4, p.dm);
  const half2_q4 d = {dm.x, dm.x}, m = {dm.y, dm.y};
  const Q4Exponents e;
  uint32_t l[2], h[2];
  q4_values4(p.codes.x, d, m, e, l, h);
  low.x = l[0], low.y = l[1], high.x = h[0], high.y = h[1];
  q4_values4(p.codes.y, d, m, e, l, h);
  low.z = l[0], low.w = l[1], high.z = h[0], high.w = h[1];
}
// Value i of a row.
__device__ __forceinline__ _Float16 q4_value(const uint8_t* row, int i) {
  const uint8_t* block = row + (i >> 5) * kQ4Bytes;
  const half2_q4 dm = __builtin_bit_cast(half2_q4, *reinterpret_cast<const uint32_t*>(block));
  const int code = block[4 + (i & 15)] >> (i & 16 ? 4 : 0) & 15;
  return __builtin_fmaf16(static_cast<_Float16>(code), dm.x, dm.y);
}

}  // namespace qk
