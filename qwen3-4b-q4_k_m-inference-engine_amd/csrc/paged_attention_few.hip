// Paged attention for few rows a sequence: the single tokens of a decode step,
// drafted tokens. HBM bounds it: every key and value is read once for a tile
// of 16 rows, which one 16x16x32 MFMA takes as its columns.
//
// The four waves of a workgroup share nothing while they run: wave w takes
// blocks w, w + 4, .. of 32 keys and holds keys and values in 16 KB of LDS of its
// own; keys are read from there as the A operand, values by
// ds_read_b64_tr_b16, four keys of a column at a time. No barrier in the loop.
// Each block's loads are issued one block ahead, its page ids two, so 16 KB a
// wave are in flight under the arithmetic.
// Loads take whole rows (256 bytes a key, 16 lanes) and are marked as not used
// again: this card's plain reads reach 6.4 TB/s, those 7.2. 64 sequences of up to
// 8192 keys, 1.06 GB: 175 us (6.1 TB/s), 3 of 131072: 156 (5.6); before the
// sequences were taken by length 225, and 263 with keys loaded straight into the
// operand's layout (64 bytes of a row an instruction).
#include "paged_attention_few.hpp"

namespace qk {
namespace {

constexpr int kRows = 16, kWaves = 4, kStep = kBlock * kWaves;

// 16-byte chunks of V rows in LDS are permuted so that the eight keys which one
// pass of a transposing read touches lie in different banks.
template <int D>
__device__ __forceinline__ int v_chunk(int key, int chunk) {
  const int f = D == 128 ? (key & 7) << 1 : (key >> 1 & 3) << 1;
  return key * (2 * D) + ((chunk ^ f) << 4);
}

// And of K rows, so that 16 keys' same chunk lie in different banks.
template <int D>
__device__ __forceinline__ int k_chunk(int key, int chunk) {
  return key * (2 * D) + ((chunk ^ (D == 128 ? key & 15 : key >> 1 & 7)) << 4);
}

template <int D, bool BF16, bool Q32>
__global__ __launch_bounds__(256, 2) void attention_few_kernel(const AttentionArgs a) {
  typedef Num<BF16> N;
  typedef typename N::T T;
  typedef typename N::V8 V8;
  constexpr int NP = kParts<BF16, Q32>;
  // Parts of a weight: two with 16-bit q as well, as the matrix cores are idle nine
  // tenths of the time (three contexts of 131072, BF16: 153 and 156 us, error of the
  // result 2.3e-3 and 1.6e-3, half a step).
  constexpr int NW = NP > 1 ? NP : 2;
  constexpr int KS = D / 32, DT = D / 16;    // k steps of q.k, 16-wide tiles of the output
  constexpr int LPK = D / 8;                 // lanes that load one key's values
  constexpr int VL = kBlock * LPK / 64;      // loads of a block's values
  constexpr int KPL = 64 / LPK;              // keys a load
  struct Shared : FewShared {
    union {
      struct {
        uint8_t k[kWaves][kBlock * 2 * D];
        uint8_t v[kWaves][kBlock * 2 * D];
      };
      float o[kWaves][kRows][D];
    };
    int64_t place[kWaves][2][kBlock];
    float top[kWaves][kRows], sum[kWaves][kRows];
  };
  __shared__ __attribute__((aligned(16))) Shared sh;

  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int head = static_cast<int>(blockIdx.x) % a.kv.kv_heads, unit = static_cast<int>(blockIdx.x) / a.kv.kv_heads;
  const int tile = unit / a.splits, split = unit % a.splits;
  const AttentionTile t = few_tile<kRows>(a, tile, sh);
  if (t.s < 0) return;
  // chunks of one length for all sequences, so that a batch's longest does not outlast the rest
  int chunk = kStep;
  if (a.splits > 1) {
    const int longest = longest_context(a), filled = longest / a.fill;
    chunk = filled < kGoodPartKeys ? filled : kGoodPartKeys;
    chunk = chunk < longest / a.splits ? longest / a.splits : chunk;
    chunk = chunk < kStep ? kStep : chunk;
  }
  const KeyChunk c = key_chunk(t, split, a.splits, kStep, chunk);
  if (split >= c.used) return;
  if (tid == 0) sh.bad = t.beyond;
  __syncthreads();

  // the lane's row: column of every accumulator
  const int col = lane & 15, grp = lane >> 4;
  const int row = t.begin + col;
  const bool live = row < t.rows;
  const int token = t.row + (live ? row / a.group : 0), h = head * a.group + (live ? row % a.group : 0);
  const int position = t.first + (token - t.row);
  const int last = live ? (position < c.hi - 1 ? position : c.hi - 1) : -1;  // keys that the row sees here: from .. last
  const int from = a.window > 0 ? position - a.window + 1 : 0;
  // every row sees all keys of [all_from, all_last]
  const int all_last = t.first + t.begin / a.group;
  const int end_row = t.begin + kRows < t.rows ? t.begin + kRows : t.rows;
  const int all_from = a.window > 0 ? t.first + (end_row - 1) / a.group - a.window + 1 : 0;

  // page ids two blocks ahead, places one ahead
  const int blocks = (c.hi - c.lo + kBlock - 1) / kBlock;
  int32_t page = 0;
  bool listed = true, bad = false;
  const auto key_of = [&](int b) {  // the lane's key of block b; keys past the end stand in for by the last one
    const int key = c.lo + b * kBlock + (lane & 31);
    return key < c.hi ? key : c.hi - 1;
  };
  const auto look_up = [&](int b) {
    page = a.kv.page_table[kv_table_at(a.kv, t.s, key_of(b) / a.kv.page_size, listed)];
  };
  u32x4 kreg[VL], vreg[VL];
  const auto settle = [&](int b) {  // page id -> place of block b
    const int key = key_of(b);
    const bool ok = listed && page >= 0 && page < a.kv.pages;
    bad |= !ok;
    sh.place[wave][b / kWaves & 1][lane & 31] = kv_place(a.kv, ok ? page : 0, key % a.kv.page_size, head);
    __builtin_amdgcn_wave_barrier();
  };
  const auto load_k = [&](int b) {
#pragma unroll
    for (int i = 0; i < VL; ++i)
      kreg[i] = stream_load16(a.kv.k + sh.place[wave][b / kWaves & 1][KPL * i + lane / LPK] + 8 * (lane % LPK));
  };
  const auto load_v = [&](int b) {
#pragma unroll
    for (int i = 0; i < VL; ++i)
      vreg[i] = stream_load16(a.kv.v + sh.place[wave][b / kWaves & 1][KPL * i + lane / LPK] + 8 * (lane % LPK));
  };
  if (wave < blocks) {
    look_up(wave);
    settle(wave);
    look_up(wave + kWaves);
    load_k(wave);
    load_v(wave);
  }

  // q, in parts
  V8 q[KS][NP];
  float factor = a.scale * kLog2e;
  {
    const int64_t at = token * a.q_stride + static_cast<int64_t>(h) * D + 8 * grp;
    if constexpr (Q32) {
      float x[KS][8];
      float most = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const f32x4 v = *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.q) + at + 32 * s + i);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[s][i + j] = live ? v[j] : 0.0f;
            most = fmaxf(most, fabsf(x[s][i + j]));
          }
        }
      if constexpr (!BF16) {
        most = swap32_max(swap16_max(most));
        // 2^(14 - exponent): the row's largest value in [2^13, 2^14)
        const bool scaled = most > 0.0f && most < __builtin_inff();
        const int e = scaled ? 14 - __builtin_amdgcn_frexp_expf(most) : 0;
        factor = ldexpf(factor, -e);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int i = 0; i < 8; ++i) x[s][i] = ldexpf(x[s][i], e);
      }
#pragma unroll
      for (int s = 0; s < KS; ++s) split8<BF16, NP>(x[s], q[s]);
    } else {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const u32x4 v = load16(static_cast<const uint16_t*>(a.q) + at + 32 * s);
        q[s][0] = __builtin_bit_cast(V8, live ? v : u32x4{});
      }
    }
  }

  f32x4 o[DT] = {};
  float top = kNoMax, sum = 0.0f;
  // the lane's part of a transposing read: key 4 grp + col / 4, and 16 on
  const int tr_key = 4 * grp + (col >> 2);
  const int tr_at = v_chunk<D>(tr_key, col >> 1 & 1) + (col & 1) * 8;
  uint8_t* const vs = sh.v[wave];
  uint8_t* const ks = sh.k[wave];
  typedef short i16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) i16x4* LdsRow;

  const auto rescale = [&](float to) {
    const float f = __builtin_amdgcn_exp2f(top - to);
    top = to;
    sum *= f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = o[d] * f;
  };
  float sound = -__builtin_inff();  // the reference up to which the row is sound
  const auto least_full = [&]() __attribute__((always_inline)) {  // scores below have weights that lack bits that count
    return top > sound ? top - kReach<NW> : -__builtin_inff();
  };
  // q.k of the block in ks, scaled: by products of their own, so that weights formed
  // of them twice are the same bits
  const auto scores = [&](f32x4 (&x)[2]) __attribute__((always_inline)) {
#pragma clang fp contract(off)
    x[0] = x[1] = f32x4{};
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const V8 k = __builtin_bit_cast(V8, load16(ks + i * (16 * 2 * D) + k_chunk<D>(col, 4 * s + grp)));
#pragma unroll
        for (int p = 0; p < NP; ++p) x[i] = N::mfma16(k, q[s][p], x[i]);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = x[i] * factor;
  };
  // No short circuit: a select, not a branch.
  const auto sees = [&](int key0, int i, int r) __attribute__((always_inline)) {
    const int key = key0 + 16 * i + 4 * grp + r;
    return static_cast<bool>(static_cast<int>(key <= last) & static_cast<int>(key >= from));
  };
  const auto add_values = [&](const V8 (&w)[NW]) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      uint8_t* const at = vs + (tr_at ^ (d << 5));
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsRow)(at));
      const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsRow)(at + 16 * 2 * D));
      const auto both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int n = 0; n < NW; ++n) o[d] = N::mfma16(__builtin_bit_cast(V8, both), w[n], o[d]);
    }
  };
  // Adds what the weights of the block in ks and vs lack to rows that are not sound,
  // in steps of a sinking reference. Scores and weights are formed anew, the same bits.
  const auto correct = [&](int key0) __attribute__((always_inline)) {
    uint32_t sizes = 0;
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      const u32x4 v = load16(vs + i * 1024 + lane * 16);
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
        for (int r = 0; r < 4; ++r) size = fmaxf(size, fabsf(o[d][r]) < __builtin_inff() ? fabsf(o[d][r]) : 0.0f);
      size = swap32_max(swap16_max(size));
      sound = sound_to<NW>(top, size, largest);
    };
    judge();
    if (!__any(top > sound)) return;
    f32x4 x[2];
    scores(x);
    const float low = least_full();
    float p[8];
    bool lacks = false;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool in = sees(key0, i, r);
        lacks |= in && x[i][r] < low;
        p[4 * i + r] = in ? __builtin_amdgcn_exp2f(x[i][r] - (top - kLift<BF16>)) : 0.0f;
      }
    lacks = swap32_max(swap16_max(lacks ? 1.0f : 0.0f)) > 0.0f;
    V8 w[NW];
    split8<BF16, NW>(p, w);
    for (int step = 0; step < 8; ++step) {
      const int by = lacks && top > sound ? sinking<NW>(size, swap32_max(swap16_max(sum)), largest) : 0;
      if (!__any(by > 0)) break;
      rescale(top - static_cast<float>(by));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int n = 0; n < NW; ++n) p[e] -= static_cast<float>(w[n][e]);
        p[e] = by > 0 ? ldexpf(p[e], by) : 0.0f;
      }
      split8<BF16, NW>(p, w);
      add_values(w);
      judge();
    }
  };

  for (int b = wave; b < blocks; b += kWaves) {
    const int key0 = c.lo + b * kBlock;
#pragma unroll
    for (int i = 0; i < VL; ++i) *reinterpret_cast<u32x4*>(ks + k_chunk<D>(KPL * i + lane / LPK, lane % LPK)) = kreg[i];
    // loads past the last block are of its last key: a branch here would make
    // every wait one for all loads in flight
    const int next = b + kWaves;
    settle(next);
    load_k(next);
    look_up(next + kWaves);
    f32x4 x[2];
    scores(x);
    const bool whole = key0 + kBlock - 1 <= all_last && key0 + kBlock <= c.hi && key0 >= all_from;
    // values into LDS; those of keys past the end as zeros (their weight is 0), and
    // where a weight may be 0, or its parts of either sign, infinite ones too
    bool odd = false;
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      if (key0 + KPL * i + lane / LPK >= c.hi) vreg[i] = u32x4{};
      odd |= any_infinite<BF16>(vreg[i]);
    }
    odd = __any(odd);
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      const int key = KPL * i + lane / LPK;
      *reinterpret_cast<u32x4*>(vs + v_chunk<D>(key, lane % LPK)) = odd ? only_finite<BF16>(vreg[i]) : vreg[i];
    }
    load_v(next);
    __builtin_amdgcn_wave_barrier();
    // softmax of 32 keys: registers r of tile i hold key 16 i + 4 grp + r
    float most = -__builtin_inff(), least = __builtin_inff();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (!whole) {
          const bool in = sees(key0, i, r);
          if constexpr (!BF16) least = fminf(least, in ? x[i][r] : __builtin_inff());
          x[i][r] = in ? x[i][r] : -__builtin_inff();
        } else if constexpr (!BF16) {
          least = fminf(least, x[i][r]);
        }
        most = fmaxf(most, x[i][r]);
      }
    if (__any(most > top + kSlack)) {
      most = swap32_max(swap16_max(most));
      if constexpr (BF16) {
        rescale(fmaxf(top, most));
      } else {
        rescale(risen<NW>(top, most));
      }
    }
    float p[8];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[4 * i + r] = __builtin_amdgcn_exp2f(x[i][r] - (top - kLift<BF16>));
        sum += p[4 * i + r];
      }
    V8 w[NW];
    split8<BF16, NW>(p, w);
    add_values(w);
    if constexpr (!BF16)
      if (__builtin_expect(__any(least < least_full()), 0)) correct(key0);
    __builtin_amdgcn_wave_barrier();
    if (odd) {
      // infinite or NaN values of keys that some rows do not see: 0 times them
      // is no zero, so they went into the product as zeros and are added here
      // to the rows that do see them (any weight times them is themselves)
      for (int j = 0; j < kBlock && key0 + j < c.hi; ++j) {
        const bool sees = key0 + j <= last && key0 + j >= from;
        const uint16_t* v = a.kv.v + sh.place[wave][b / kWaves & 1][j] + 4 * grp;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float e = static_cast<float>(__builtin_bit_cast(T, v[16 * d + r]));
            if (sees && !(fabsf(e) < __builtin_inff())) o[d][r] += e;
          }
      }
    }
  }

  // the four waves' parts
  if (__any(bad) && lane == 0) sh.bad = 1;
  sum = swap32_sum(swap16_sum(sum));
  if (grp == 0) {
    sh.top[wave][col] = top;
    sh.sum[wave][col] = sum;
  }
  __syncthreads();  // every wave is done with its values
#pragma unroll
  for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(&sh.o[wave][col][16 * d + 4 * grp]) = o[d];
  __syncthreads();
  constexpr int E = D / 16;  // values a thread: 16 threads a row, pairs 32 apart, so that a row's threads read and write 128 bytes in one
  const int r = tid >> 4, e0 = (tid & 15) * 2;
  const auto pair = [&](int i) { return e0 + 16 * i; };  // of values i and i + 1
  const bool mine = t.begin + r < t.rows;
  float all, total, y[E];
  const auto gather = [&](int waves) {
    all = kNoMax;
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) y[i] = 0.0f;
    for (int w = 0; w < waves; ++w) all = fmaxf(all, sh.top[w][r]);
    for (int w = 0; w < waves; ++w) {
      const float f = __builtin_amdgcn_exp2f(sh.top[w][r] - all);
      total += f * sh.sum[w][r];
#pragma unroll
      for (int i = 0; i < E; ++i) y[i] += f * sh.o[w][r][pair(i & ~1) + (i & 1)];
    }
  };
  gather(kWaves);
  if (sh.bad) {
    total = __builtin_nanf("");
    if (tid == 0) kv_fault(a.kv, QK_KV_FAULT_PAGE);
  }
  if (c.used > 1) {
    const int64_t slot = (static_cast<int64_t>(tile) * a.kv.kv_heads + head) * a.splits;
    if (mine) {
      const int64_t at = (slot + split) * kRows + r;
      if ((tid & 15) == 0) put(a.sums + 2 * at, all, total);
#pragma unroll
      for (int i = 0; i < E; i += 2) put(a.parts + at * D + pair(i), y[i], y[i + 1]);
    }
    if (!last_to_arrive(a.arrived + static_cast<int64_t>(tile) * a.kv.kv_heads + head, c.used, sh.arrived)) return;
    // Waves without a row of their own take a share of the parts, where there are
    // more than one step's eight: of a single token's four rows a quarter each
    // (7200 keys, 57 parts: 20.3 us instead of 23.1; 1000, eight parts: 13.1
    // instead of 11.8).
    const int live = min(kRows, t.rows - t.begin), ways = live > 8 || c.used <= 8 ? 1 : live > 4 ? 2 : 4;
    const int share = wave & (ways - 1), r = wave / ways * 4 + (lane >> 4);
    const int per = (c.used + ways - 1) / ways, lo = share * per, hi = min(c.used, lo + per);
    all = kNoMax;
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) y[i] = 0.0f;
    if (r < live && lo < hi) {
      // lane j of a row's 16 has the sums of parts j, j + 16, .. of each 64
      const int j = tid & 15;
      float next[8][E];
      const auto fetch = [&](int k0) {  // eight parts; past the last that one again, not added
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float* part = a.parts + ((slot + min(k0 + k, hi - 1)) * kRows + r) * D;
#pragma unroll
          for (int i = 0; i < E; i += 2) get(part + pair(i), next[k][i], next[k][i + 1]);
        }
      };
      for (int base = lo; base < hi; base += 64) {
        float m[4], l[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) get(a.sums + 2 * ((slot + min(base + 16 * n + j, hi - 1)) * kRows + r), m[n], l[n]);
        fetch(base);
        float to = all;
#pragma unroll
        for (int n = 0; n < 4; ++n) to = fmaxf(to, m[n]);
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) to = fmaxf(to, __shfl_xor(to, off));
        const float f = __builtin_amdgcn_exp2f(all - to);
        all = to;
        total *= f;
#pragma unroll
        for (int i = 0; i < E; ++i) y[i] *= f;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          m[n] = __builtin_amdgcn_exp2f(m[n] - all);
          total += base + 16 * n + j < hi ? m[n] * l[n] : 0.0f;
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const int k0 = base + 8 * n;
          if (k0 >= hi) break;
          float part[8][E];
#pragma unroll
          for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int i = 0; i < E; ++i) part[k][i] = next[k][i];
          if (n < 7 && k0 + 8 < hi) fetch(k0 + 8);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float g = __shfl(m[n / 2], (tid & 48) + 8 * (n & 1) + k);
#pragma unroll
            for (int i = 0; i < E; ++i) y[i] += k0 + k < hi ? g * part[k][i] : 0.0f;
          }
        }
      }
#pragma unroll
      for (int off = 1; off < 16; off <<= 1) total += __shfl_xor(total, off);
    }
    if (ways > 1) {
      if (r < live) {
        if ((tid & 15) == 0) {
          sh.top[share][r] = all;
          sh.sum[share][r] = total;
        }
#pragma unroll
        for (int i = 0; i < E; ++i) sh.o[share][r][pair(i & ~1) + (i & 1)] = y[i];
      }
      __syncthreads();
      gather(ways);
    }
  }
  if (!mine) return;
  const int out_row = t.begin + r;
  const int64_t at = static_cast<int64_t>(t.row + out_row / a.group) * a.q_heads + head * a.group + out_row % a.group;
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  if constexpr (Q32) {
    typedef float F2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < E; i += 2)
      *reinterpret_cast<F2*>(static_cast<float*>(a.out) + at * D + pair(i)) = F2{y[i] * inv, y[i + 1] * inv};
  } else {
    typedef T T2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < E; i += 2)
      *reinterpret_cast<T2*>(static_cast<T*>(a.out) + at * D + pair(i)) =
          T2{static_cast<T>(y[i] * inv), static_cast<T>(y[i + 1] * inv)};
  }
  if (a.lse && (tid & 15) == 0) a.lse[at] = row_lse<BF16>(all, total);
}

}  // namespace

hipError_t launch_attention_few(const AttentionArgs& a, int type, int head_dim, int q_type, hipStream_t stream) {
  const uint32_t grid = static_cast<uint32_t>(a.tiles) * a.splits * a.kv.kv_heads;
  const bool bf16 = type == QK_TYPE_BF16, q32 = q_type == QK_TYPE_F32;
  auto go = [&](auto kernel) { kernel<<<grid, 64 * kWaves, 0, stream>>>(a); };
  if (head_dim == 128)
    bf16 ? (q32 ? go(attention_few_kernel<128, true, true>) : go(attention_few_kernel<128, true, false>))
         : (q32 ? go(attention_few_kernel<128, false, true>) : go(attention_few_kernel<128, false, false>));
  else
    bf16 ? (q32 ? go(attention_few_kernel<64, true, true>) : go(attention_few_kernel<64, true, false>))
         : (q32 ? go(attention_few_kernel<64, false, true>) : go(attention_few_kernel<64, false, false>));
  note("attention_few_kernel", grid, head_dim, bf16, q32, a.splits > 1);
  return hipGetLastError();
}

}  // namespace qk
