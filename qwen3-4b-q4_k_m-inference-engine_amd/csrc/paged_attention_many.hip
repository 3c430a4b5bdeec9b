// Paged attention for many rows a sequence: prompts and chunks of prompts. The
// matrix cores bound it.
//
// A workgroup's waves hold 32 rows each, as the columns of 32x32x16 MFMAs, and
// share tiles of 64 keys in LDS. Eight waves, two on a SIMD, so that one's
// softmax runs under the other's products; within a wave too the scores of the
// next 32 keys are formed next to the softmax of these (four waves where
// three parts of an F32 q leave no registers for that). A tile's loads are
// issued a tile ahead and written to LDS half a tile before its first use,
// one barrier a tile; three tiles lie in LDS, as the slowest wave may still read
// the one before while the fastest writes the one after.
// For calls of few rows KG waves share 32 rows instead, 32 keys each of a tile of
// 64 (KG = 2) or 128 (KG = 4, in two buffers, without the look ahead); their parts
// are joined in LDS. Fewer rows a workgroup, but no part in memory where the
// others need it (plan_attention has the figures).
// Rows of 2 D bytes are stored with their 16-byte chunks permuted by the key
// (tile_chunk), which keeps both the row reads of K and the transposing reads
// of V off each other's banks.
#include <type_traits>

#include "paged_attention.hpp"

namespace qk {
namespace {

constexpr int kChunkStep = 64, kLeastChunk = 256;  // of the keys that workgroups share out
typedef float f32x16 __attribute__((ext_vector_type(16)));

// The 16-byte chunk of a row is XORed so that 16 consecutive keys (a K read)
// and 4 keys x 64 bytes (a V read) each cover all banks.
template <int D>
__device__ __forceinline__ int tile_swizzle(int key) {
  return D == 128 ? (key & 3) << 2 | (key >> 2 & 3) : (key >> 1 & 1) << 2 | (key >> 2 & 3);
}
template <int D>
__device__ __forceinline__ int tile_chunk(int key, int chunk) {
  return key * (2 * D) + ((chunk ^ tile_swizzle<D>(key)) << 4);
}

template <int D, bool BF16, bool Q32, int KG>
__global__ __launch_bounds__(64 * attention_many_waves(BF16, Q32), attention_many_waves(BF16, Q32) / 4) void
attention_many_kernel(const AttentionArgs a) {
  typedef Num<BF16> N;
  typedef typename N::T T;
  typedef typename N::V8 V8;
  constexpr int kWaves = attention_many_waves(BF16, Q32);
  constexpr int NP = kParts<BF16, Q32>;
  constexpr int kRows = 32 * kWaves / KG;   // rows of a tile
  constexpr int kKeys = KG == 1 ? 64 : 32 * KG;  // keys of a tile in LDS
  constexpr int kBuffers = KG == 4 ? 2 : 3;
  constexpr int KS = D / 16, DT = D / 32;   // k steps of q.k, 32-wide tiles of the output
  constexpr int LPK = D / 8;                // lanes that load one key
  constexpr int KPL = 64 * kWaves / LPK;    // keys a load of the workgroup
  constexpr int NL = kKeys / KPL;           // such loads a tile
  constexpr int kTile = kKeys * 2 * D;      // bytes of a tile's keys, or values
  constexpr int kRing = KG == 4 ? 4 : 8;    // tiles whose places are kept
  struct Shared {
    union {
      struct {
        uint8_t k[kBuffers][kTile];
        uint8_t v[kBuffers][kTile];
      };
      float o[KG == 1 ? 1 : kWaves][KG == 1 ? 1 : 32 * D];
    };
    int64_t place[kRing][kKeys];
    float top[kWaves][32], sum[kWaves][32];
    uint32_t odd[4], bad;
  };
  __shared__ __attribute__((aligned(16))) Shared sh;

  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int head = static_cast<int>(blockIdx.x) % a.kv.kv_heads, unit = static_cast<int>(blockIdx.x) / a.kv.kv_heads;
  const int tile = a.tiles - 1 - unit / a.splits, split = unit % a.splits;  // long tiles first
  const AttentionTile t = find_tile(a, tile, kRows, blockIdx.x == 0);
  if (t.s < 0) return;
  const KeyChunk c = key_chunk(t, split, a.splits, kChunkStep, kLeastChunk);
  if (split >= c.used) return;
  if (tid == 0) sh.bad = t.beyond, sh.odd[0] = sh.odd[1] = 0;  // odd[n & 3] is cleared while tile n - 2 runs
  if (t.beyond && tid == 0) kv_fault(a.kv, QK_KV_FAULT_PAGE);

  // the lane's row
  const int col = lane & 31, half = lane >> 5;
  const int group = wave / KG, part = wave % KG;  // of rows; of a tile's keys
  const int wave_row = t.begin + group * 32;
  const int row = wave_row + col;
  const bool live = row < t.rows;
  const int token = t.row + (live ? row / a.group : 0), h = head * a.group + (live ? row % a.group : 0);
  const int position = t.first + (token - t.row);
  const int last = live ? min(position, c.hi - 1) : -1;
  const int from = a.window > 0 ? position - a.window + 1 : 0;
  const int64_t out_at = live ? static_cast<int64_t>(token) * a.q_heads + h : -1;
  V8 q[KS][NP];
  float factor = fabsf(a.scale) * kLog2e;  // a negative scale's sign goes into q, so that the largest score is the largest q.k
  {
    const int64_t at = token * a.q_stride + static_cast<int64_t>(h) * D + 8 * half;
    if constexpr (Q32) {
      const float sign = a.scale < 0.0f ? -1.0f : 1.0f;
      float x[KS][8];
      float most = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const f32x4 v = *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.q) + at + 16 * s + e);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[s][e + j] = live ? v[j] * sign : 0.0f;
            most = fmaxf(most, fabsf(x[s][e + j]));
          }
        }
      if constexpr (!BF16) {
        most = swap32_max(most);
        const bool scaled = most > 0.0f && most < __builtin_inff();
        const int e = scaled ? 14 - __builtin_amdgcn_frexp_expf(most) : 0;  // the row's largest in [2^13, 2^14)
        factor = ldexpf(factor, -e);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int j = 0; j < 8; ++j) x[s][j] = ldexpf(x[s][j], e);
      }
#pragma unroll
      for (int s = 0; s < KS; ++s) split8<BF16, NP>(x[s], q[s]);
    } else {
      const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const u32x4 v = load16(static_cast<const uint16_t*>(a.q) + at + 16 * s) ^ sign;
        q[s][0] = __builtin_bit_cast(V8, live ? v : u32x4{});
      }
    }
  }
  // a factor of nothing would turn the -inf of masked scores into NaN
  factor = fmaxf(factor, 0x1p-126f);
  // all rows of the wave / of the workgroup see the keys of [.._from, .._last]
  const int wave_end = min(wave_row + 32, t.rows), tile_end = min(t.begin + kRows, t.rows);
  const int wave_last = t.first + wave_row / a.group, tile_last = t.first + t.begin / a.group;
  const int wave_from = a.window > 0 ? t.first + (wave_end - 1) / a.group - a.window + 1 : 0;
  const int tile_from = a.window > 0 ? t.first + (tile_end - 1) / a.group - a.window + 1 : 0;
  // and no row of the wave sees a key past any_last
  const int any_last = wave_row < t.rows ? min(t.first + (wave_end - 1) / a.group, c.hi - 1) : -1;

  // tiles of keys: page ids (a lane a key) four ahead, places three, loads two
  const int count = (c.hi - c.lo + kKeys - 1) / kKeys;
  int32_t page = 0;
  bool listed = true, bad = false;
  const bool looks = wave < kKeys / 64;
  const auto key_of = [&](int n) __attribute__((always_inline)) { return min(c.lo + n * kKeys + tid, c.hi - 1); };
  const auto look_up = [&](int n) __attribute__((always_inline)) {
    if (n < count) page = a.kv.page_table[kv_table_at(a.kv, t.s, key_of(n) / a.kv.page_size, listed)];
  };
  const auto settle = [&](int n) __attribute__((always_inline)) {
    if (n >= count) return;
    const bool ok = listed && page >= 0 && page < a.kv.pages;
    bad |= !ok;
    sh.place[n & (kRing - 1)][tid] = kv_place(a.kv, ok ? page : 0, key_of(n) % a.kv.page_size, head);
  };
  u32x4 kreg[NL], vreg[NL];
  const auto load = [&](int n) __attribute__((always_inline)) {
    if (n >= count) return;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int64_t at = sh.place[n & (kRing - 1)][KPL * i + tid / LPK] + 8 * (tid % LPK);
      kreg[i] = load16(a.kv.k + at);
      vreg[i] = load16(a.kv.v + at);
    }
  };
  // registers -> LDS; values of keys past the end become zeros, and where some
  // row does not see some key, or a weight's parts may be of either sign, or
  // none, so do infinite ones (odd)
  const auto store = [&](int n, int buffer) __attribute__((always_inline)) {
    if (n >= count) return;
    const int key0 = c.lo + n * kKeys;
    const bool edge = !(key0 + kKeys - 1 <= tile_last && key0 + kKeys <= c.hi && key0 >= tile_from);
    if (edge) {
#pragma unroll
      for (int i = 0; i < NL; ++i)
        if (key0 + KPL * i + tid / LPK >= c.hi) vreg[i] = u32x4{};
    }
    if (edge || NP > 1 || !BF16) {
      bool odd = false;
#pragma unroll
      for (int i = 0; i < NL; ++i) odd |= any_infinite<BF16>(vreg[i]);
      if (odd) {
#pragma unroll
        for (int i = 0; i < NL; ++i) vreg[i] = only_finite<BF16>(vreg[i]);
        sh.odd[n & 3] = 1;
      }
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int at = buffer * kTile + tile_chunk<D>(KPL * i + tid / LPK, tid % LPK);
      *reinterpret_cast<u32x4*>(sh.k[0] + at) = kreg[i];
      *reinterpret_cast<u32x4*>(sh.v[0] + at) = vreg[i];
    }
  };

  f32x16 o[DT] = {};
  float top = kNoMax, sum = 0.0f;
  // LDS addresses. K: key col, chunk 2 s + half. V: key 4 half + (lane & 15) / 4,
  // then 8 on, chunk 4 d + 2 (lane >> 4 & 1) + (lane >> 1 & 1). Kept as they
  // are (opaque), so that buffer and block are constants of the instructions.
  typedef short i16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) i16x4* LdsQuad;
  typedef __attribute__((address_space(3))) u32x4* LdsChunk;
  typedef __attribute__((address_space(3))) uint8_t* LdsByte;
  uint32_t k_at[KS], v_at[DT][2];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    k_at[s] = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((LdsByte)sh.k[0])) +
              part * (32 * 2 * D) + tile_chunk<D>(col, 2 * s + half);
    asm("" : "+v"(k_at[s]));
  }
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v_at[d][i] = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((LdsByte)sh.v[0])) +
                   part * (32 * 2 * D) +
                   tile_chunk<D>(4 * half + (lane >> 2 & 3) + 8 * i, 4 * d + 2 * (lane >> 4 & 1) + (lane >> 1 & 1)) + (lane & 1) * 8;
      asm("" : "+v"(v_at[d][i]));
    }

  const auto rescale = [&](float to) __attribute__((always_inline)) {
    const float f = __builtin_amdgcn_exp2f(top - to);
    top = to;
    sum *= f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = o[d] * f;
  };
  // blocks of 32 keys; `at`: of the block in sh.k and sh.v
  const auto scores = [&](int at, f32x16& x) __attribute__((always_inline)) {
    x = f32x16{};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const V8 k = __builtin_bit_cast(V8, *(LdsChunk)(uintptr_t)(k_at[s] + at));
#pragma unroll
      for (int p = 0; p < NP; ++p) x = N::mfma32(k, q[s][p], x);
    }
  };
  // Registers 8 g + 4 e + r of a block's scores hold key 16 g + 8 e + 4 half + r.
  // No short circuit: a select, not a branch.
  const auto sees = [&](int key0, int r) __attribute__((always_inline)) {
    const int key = key0 + (r >> 3) * 16 + (r >> 2 & 1) * 8 + 4 * half + (r & 3);
    return static_cast<bool>(static_cast<int>(key <= last) & static_cast<int>(key >= from));
  };
  const auto add_values = [&](int at, const V8 (&w)[2][NP]) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const int row = at + 16 * g * 2 * D;
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad)(uintptr_t)(v_at[d][0] + row));
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad)(uintptr_t)(v_at[d][1] + row));
        const V8 v = __builtin_bit_cast(V8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int p = 0; p < NP; ++p) o[d] = N::mfma32(v, w[g][p], o[d]);
      }
  };
  float sound = -__builtin_inff();  // the reference up to which the row is sound
  const auto least_full = [&]() __attribute__((always_inline)) {  // scores below have weights that lack bits that count
    return top > sound ? top - kReach<NP> : -__builtin_inff();
  };
  // The softmax step of the block whose q.k are in x and the product with its
  // values; between the two, next to the exponentials, the scores of the next
  // block into y. True where weights may lack bits that count (see correct).
  const auto attend = [&](int key0, int at, f32x16& x, int next_at, f32x16* y) __attribute__((always_inline)) {
    float most = -__builtin_inff(), least = __builtin_inff();
    if (key0 + 31 <= wave_last && key0 + 32 <= c.hi && key0 >= wave_from) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        most = fmaxf(most, x[r]);
        if constexpr (!BF16) least = fminf(least, x[r]);
      }
    } else {  // some row does not see some key
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const bool in = sees(key0, r);
        if constexpr (!BF16) least = fminf(least, in ? x[r] : __builtin_inff());
        x[r] = in ? x[r] : -__builtin_inff();
        most = fmaxf(most, x[r]);
      }
    }
    most *= factor;
    if (__any(most > top + kSlack)) {
      most = swap32_max(most);
      if constexpr (BF16) {
        rescale(fmaxf(top, most));
      } else {
        rescale(risen<NP>(top, most));
      }
    }
    const bool lacks = !BF16 && __any(least * factor < least_full());
    if (y) scores(next_at, *y);
    const float base = kLift<BF16> - top;
    V8 w[2][NP];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * g + e], factor, base));
        sum += p[e];
      }
      split8<BF16, NP>(p, w[g]);
    }
    add_values(at, w);
    return lacks;
  };
  // Adds what the weights of a block lack to rows that are not sound, in steps of a
  // sinking reference. Scores and weights are formed anew, the same bits: registers
  // to keep them are not to be had. Looking for such weights costs nothing that
  // shows, this 2 to 5% where scores have a spread of 1.5 (512 tokens over 4096 keys,
  // F32 q: 83 to 87 us), a quarter at twice that (105) and with a first token that
  // takes nearly all of the mass (99). In the same place, without asking whether
  // a row is sound: 277 and 109.
  const auto correct = [&](int key0, int at) __attribute__((always_inline)) {
    uint32_t sizes = 0;
#pragma unroll
    for (int i = 0; i < 32 * 2 * D / 1024; ++i) {
      const u32x4 v = load16(sh.v[0] + part * (32 * 2 * D) + at + i * 1024 + lane * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) sizes = larger_sizes(sizes, v[e]);
    }
    sizes = sizes > sizes << 16 ? sizes >> 16 : sizes & 0xFFFFu;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t other = __shfl_xor(sizes, off);
      sizes = other > sizes ? other : sizes;
    }
    const float largest = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(sizes)));
    float size;
    const auto judge = [&]() __attribute__((always_inline)) {
      size = 0.0f;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) size = fmaxf(size, fabsf(o[d][r]) < __builtin_inff() ? fabsf(o[d][r]) : 0.0f);
      size = swap32_max(size);
      sound = sound_to<NP>(top, size, largest);
    };
    judge();
    if (!__any(top > sound)) return;
    f32x16 x;
    scores(at, x);
    const float base = kLift<BF16> - top, low = least_full();
    float p[2][8];
    bool lacks = false;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const bool in = sees(key0, r);
      lacks |= in && x[r] * factor < low;
      p[r / 8][r % 8] = in ? __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], factor, base)) : 0.0f;
    }
    lacks = swap32_max(lacks ? 1.0f : 0.0f) > 0.0f;
    V8 w[2][NP];
#pragma unroll
    for (int g = 0; g < 2; ++g) split8<BF16, NP>(p[g], w[g]);
    for (int step = 0; step < 8; ++step) {
      const int by = lacks && top > sound ? sinking<NP>(size, swap32_max(sum), largest) : 0;
      if (!__any(by > 0)) break;
      rescale(top - static_cast<float>(by));
#pragma unroll
      for (int g = 0; g < 2; ++g) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
#pragma unroll
          for (int n = 0; n < NP; ++n) p[g][e] -= static_cast<float>(w[g][n][e]);
          p[g][e] = by > 0 ? ldexpf(p[g][e], by) : 0.0f;
        }
        split8<BF16, NP>(p[g], w[g]);
      }
      add_values(at, w);
      judge();
    }
  };
  // infinite or NaN values went into the product as zeros (0 times them is no
  // zero); the rows that see them get them here
  const auto add_infinite = [&](int n) __attribute__((always_inline)) {
    for (int m = 0; m < kKeys / KG; ++m) {
      const int key = c.lo + n * kKeys + part * 32 + m;
      if (key >= c.hi) break;
      const uint16_t* v = a.kv.v + sh.place[n & (kRing - 1)][part * 32 + m] + 4 * half;
      const bool sees = key <= last && key >= from;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float e = static_cast<float>(__builtin_bit_cast(T, v[32 * d + (r >> 2) * 8 + (r & 3)]));
          if (sees && !(fabsf(e) < __builtin_inff())) o[d][r] += e;
        }
    }
  };
  // tile n + 1 into LDS, the loads and look-ups after it; then all may read it
  const auto advance = [&](int n, int next) __attribute__((always_inline)) {
    if constexpr (KG == 4) __syncthreads();  // tile n is there, and all are done with tile n - 1
    store(n + 1, next);
    load(n + 2);
    if (looks) {
      settle(n + 3);
      look_up(n + 4);
    }
    if (tid == 0) sh.odd[(n + 2) & 3] = 0;  // read last before the barrier of tile n - 1, set next after the next one
    if constexpr (KG != 4) __syncthreads();
  };

  int n = 0;
  if (count > 0) {
    if (looks) {
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        look_up(i);
        settle(i);
      }
      look_up(3);
    }
    __syncthreads();
    load(0);
    store(0, 0);
    load(1);
    // through the tiles that no row of the wave sees it only helps to load
    const int end = any_last < c.lo + 32 * part ? 0 : min((any_last - c.lo - 32 * part) / kKeys + 1, count);
    if constexpr (KG == 1) {
      __syncthreads();
      if (end > 0) {
        f32x16 x0, x1;
        scores(0, x0);
        // tile n in buffer n % 3; past the last tile the scores are of no tile, and not used
        const auto both = [&](auto buffer) __attribute__((always_inline)) {
          constexpr int at = decltype(buffer)::value * kTile, next = (decltype(buffer)::value + 1) % 3;
          const int key0 = c.lo + n * kKeys;
          const bool lacks0 = attend(key0, at, x0, at + 32 * 2 * D, &x1);
          if (__builtin_expect(lacks0, 0)) correct(key0, at);
          advance(n, next);
          const bool lacks1 = attend(key0 + 32, at + 32 * 2 * D, x1, next * kTile, &x0);
          if (__builtin_expect(lacks1, 0)) correct(key0 + 32, at + 32 * 2 * D);
          if (sh.odd[n & 3]) add_infinite(n);
          return ++n < end;
        };
        while (both(std::integral_constant<int, 0>{}) && both(std::integral_constant<int, 1>{}) &&
               both(std::integral_constant<int, 2>{})) {
        }
      }
      for (; n < count; ++n) advance(n, (n + 1) % 3);
    } else if constexpr (KG == 2) {
      __syncthreads();
      if (end > 0) {
        f32x16 x0, x1;
        scores(0, x0);
        const auto one = [&](auto buffer, f32x16& x, f32x16& y) __attribute__((always_inline)) {
          constexpr int at = decltype(buffer)::value * kTile, next = (decltype(buffer)::value + 1) % 3;
          advance(n, next);
          const bool lacks = attend(c.lo + n * kKeys + 32 * part, at, x, next * kTile, &y);
          if (__builtin_expect(lacks, 0)) correct(c.lo + n * kKeys + 32 * part, at);
          if (sh.odd[n & 3]) add_infinite(n);
          return ++n < end;
        };
        while (one(std::integral_constant<int, 0>{}, x0, x1) && one(std::integral_constant<int, 1>{}, x1, x0) &&
               one(std::integral_constant<int, 2>{}, x0, x1) && one(std::integral_constant<int, 0>{}, x1, x0) &&
               one(std::integral_constant<int, 1>{}, x0, x1) && one(std::integral_constant<int, 2>{}, x1, x0)) {
        }
      }
      for (; n < count; ++n) advance(n, (n + 1) % 3);
    } else {
      // tile n in buffer n % 2
      const auto one = [&](auto buffer) __attribute__((always_inline)) {
        constexpr int at = decltype(buffer)::value * kTile;
        advance(n, decltype(buffer)::value ^ 1);
        f32x16 x;
        scores(at, x);
        const bool lacks = attend(c.lo + n * kKeys + 32 * part, at, x, 0, nullptr);
        if (__builtin_expect(lacks, 0)) correct(c.lo + n * kKeys + 32 * part, at);
        if (sh.odd[n & 3]) add_infinite(n);
        return ++n < end;
      };
      if (end > 0)
        while (one(std::integral_constant<int, 0>{}) && one(std::integral_constant<int, 1>{})) {
        }
      for (; n < count; ++n) advance(n, (n + 1) % 2);
    }
  }

  if (looks && __any(bad) && lane == 0) {
    sh.bad = 1;
    kv_fault(a.kv, QK_KV_FAULT_PAGE);
  }
  __syncthreads();
  sum = swap32_sum(sum);
  if (sh.bad) sum = __builtin_nanf("");
  // The accumulators as QUADS of four values a lane: quad q holds values
  // 8 q + 4 half .. of the row. With keys in parts, each of the waves that share
  // rows takes an equal run of quads of their joined result.
  constexpr int kQuads = DT * 4 / KG;
  f32x4 y[kQuads];
  if constexpr (KG == 1) {
#pragma unroll
    for (int q = 0; q < kQuads; ++q)
      y[q] = f32x4{o[q / 4][q % 4 * 4], o[q / 4][q % 4 * 4 + 1], o[q / 4][q % 4 * 4 + 2], o[q / 4][q % 4 * 4 + 3]};
  } else {
    // the tiles in LDS are done with since the barrier above
#pragma unroll
    for (int q = 0; q < DT * 4; ++q)
      *reinterpret_cast<f32x4*>(&sh.o[wave][q * 256 + lane * 4]) =
          f32x4{o[q / 4][q % 4 * 4], o[q / 4][q % 4 * 4 + 1], o[q / 4][q % 4 * 4 + 2], o[q / 4][q % 4 * 4 + 3]};
    if (half == 0) {
      sh.top[wave][col] = top;
      sh.sum[wave][col] = sum;
    }
    __syncthreads();
    float all = kNoMax, total = 0.0f;
#pragma unroll
    for (int k = 0; k < KG; ++k) all = fmaxf(all, sh.top[group * KG + k][col]);
#pragma unroll
    for (int q = 0; q < kQuads; ++q) y[q] = f32x4{};
#pragma unroll
    for (int k = 0; k < KG; ++k) {
      const int other = group * KG + k;
      const float f = __builtin_amdgcn_exp2f(sh.top[other][col] - all);
      total += f * sh.sum[other][col];
#pragma unroll
      for (int q = 0; q < kQuads; ++q)
        y[q] += f * *reinterpret_cast<const f32x4*>(&sh.o[other][(part * kQuads + q) * 256 + lane * 4]);
    }
    top = all;
    sum = total;
  }
  if (c.used > 1) {  // for attention_join_kernel: [group of rows][quad][lane]
    constexpr int kGroups = kWaves / KG;
    const int64_t at = (((static_cast<int64_t>(tile) * a.kv.kv_heads + head) * a.splits + split) * kGroups + group) * 32;
    if (wave_row >= t.rows) return;
    if (half == 0 && part == 0) {
      a.sums[2 * (at + col)] = top;
      a.sums[2 * (at + col) + 1] = sum;
    }
    float* out = a.parts + at * D + part * kQuads * 256 + 4 * lane;
#pragma unroll
    for (int q = 0; q < kQuads; ++q) *reinterpret_cast<f32x4*>(out + q * 256) = y[q];
    return;
  }
  if (out_at < 0) return;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int q = 0; q < kQuads; ++q) {
    const int64_t at = out_at * D + (part * kQuads + q) * 8 + 4 * half;
    store_row<BF16, Q32>(a.out, at, y[q] * inv);
  }
  if (a.lse && half == 0 && part == 0) a.lse[out_at] = row_lse<BF16>(top, sum);
}

// Joins the parts of rows whose keys several workgroups took, 32 rows a
// workgroup, a quarter of their values a wave. A launch of its own: it reads the
// parts at the whole card's rate. 512 tokens over 4096 keys, 33 MB of parts: 11 of
// 85 us, 8 less in all than with the joining left to each tile's last workgroup,
// which reads half a megabyte alone.
template <int D, bool BF16, bool Q32>
__global__ __launch_bounds__(256) void attention_join_kernel(const AttentionArgs a, int tile_rows) {
  constexpr int kQuads = D / 32;  // of a wave: four values a lane each, as the parts hold them
  const int lane = static_cast<int>(threadIdx.x) & 63, wave = static_cast<int>(threadIdx.x) >> 6;
  const int groups = tile_rows / 32, group = static_cast<int>(blockIdx.x) % groups, unit = static_cast<int>(blockIdx.x) / groups;
  const int tile = unit / a.kv.kv_heads, head = unit % a.kv.kv_heads;
  const AttentionTile t = find_tile(a, tile, tile_rows, false);
  if (t.s < 0) return;
  const int used = key_chunk(t, 0, a.splits, kChunkStep, kLeastChunk).used;
  const int col = lane & 31, half = lane >> 5, row = t.begin + group * 32 + col;
  if (used == 1 || row >= t.rows) return;
  const int64_t first = (static_cast<int64_t>(unit) * a.splits * groups + group) * 32, step = int64_t{32} * groups;
  float all = kNoMax, total = 0.0f;
  for (int k = 0; k < used; ++k) all = fmaxf(all, a.sums[2 * (first + k * step + col)]);
  f32x4 y[kQuads] = {};
#pragma unroll 4
  for (int k = 0; k < used; ++k) {
    const int64_t at = first + k * step;
    const float f = __builtin_amdgcn_exp2f(a.sums[2 * (at + col)] - all);
    total += f * a.sums[2 * (at + col) + 1];
    const float* part = a.parts + at * D + wave * kQuads * 256 + 4 * lane;
#pragma unroll
    for (int q = 0; q < kQuads; ++q) y[q] += f * *reinterpret_cast<const f32x4*>(part + q * 256);
  }
  const int64_t out_at = static_cast<int64_t>(t.row + row / a.group) * a.q_heads + head * a.group + row % a.group;
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int q = 0; q < kQuads; ++q) store_row<BF16, Q32>(a.out, out_at * D + (wave * kQuads + q) * 8 + 4 * half, y[q] * inv);
  if (a.lse && half == 0 && wave == 0) a.lse[out_at] = row_lse<BF16>(all, total);
}

template <int D>
hipError_t launch_join(const AttentionArgs& a, int tile_rows, bool bf16, bool q32, hipStream_t stream) {
  const uint32_t grid = static_cast<uint32_t>(a.tiles) * a.kv.kv_heads * (tile_rows / 32);
  auto go = [&](auto kernel) { kernel<<<grid, 256, 0, stream>>>(a, tile_rows); };
  bf16 ? (q32 ? go(attention_join_kernel<D, true, true>) : go(attention_join_kernel<D, true, false>))
       : (q32 ? go(attention_join_kernel<D, false, true>) : go(attention_join_kernel<D, false, false>));
  return hipGetLastError();
}

template <int KG>
hipError_t launch_groups(const AttentionArgs& a, int type, int head_dim, int q_type, hipStream_t stream) {
  const uint32_t grid = static_cast<uint32_t>(a.tiles) * a.splits * a.kv.kv_heads;
  const bool bf16 = type == QK_TYPE_BF16, q32 = q_type == QK_TYPE_F32;
  const int threads = 64 * attention_many_waves(bf16, q32);
  auto go = [&](auto kernel) { kernel<<<grid, threads, 0, stream>>>(a); };
  if (head_dim == 128)
    bf16 ? (q32 ? go(attention_many_kernel<128, true, true, KG>) : go(attention_many_kernel<128, true, false, KG>))
         : (q32 ? go(attention_many_kernel<128, false, true, KG>) : go(attention_many_kernel<128, false, false, KG>));
  else
    bf16 ? (q32 ? go(attention_many_kernel<64, true, true, KG>) : go(attention_many_kernel<64, true, false, KG>))
         : (q32 ? go(attention_many_kernel<64, false, true, KG>) : go(attention_many_kernel<64, false, false, KG>));
  note("attention_many_kernel", grid, head_dim, bf16, q32, KG, a.splits > 1);
  const hipError_t error = hipGetLastError();
  if (error != hipSuccess || a.splits == 1) return error;
  return head_dim == 128 ? launch_join<128>(a, threads / 2 / KG, bf16, q32, stream)
                         : launch_join<64>(a, threads / 2 / KG, bf16, q32, stream);
}

}  // namespace

hipError_t launch_attention_many(const AttentionArgs& a, int key_groups, int type, int head_dim, int q_type,
                                 hipStream_t stream) {
  return key_groups == 1   ? launch_groups<1>(a, type, head_dim, q_type, stream)
         : key_groups == 2 ? launch_groups<2>(a, type, head_dim, q_type, stream)
                           : launch_groups<4>(a, type, head_dim, q_type, stream);
}

}  // namespace qk
