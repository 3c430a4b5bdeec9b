// Paged attention for few rows a sequence over Q4_1 blocks: a third of an F16
// cache's bytes, and the unpacking that comes with them.
//
// As in paged_attention_few.hip the four waves of a workgroup share nothing while
// they run and take blocks of 32 keys in turn, here two a turn. Codes stay packed up to
// the registers that the matrix cores read:
// - A key's row goes straight into the lanes that need it. Lane (key, grp) of the A
//   operand takes the grp-th quarter of the row, so that the 20 bytes it loads are one
//   block of 32 values (D = 128; half a block at D = 64) with its d and m, and step s of
//   q.k is dword s of them, in the order in which unpacking yields its eight values. q
//   is read in that order too.
// - V is needed by columns. Its blocks go through LDS as they are, 2.5 KB of 32 keys;
//   lane (column i, grp) reads dword i of eight keys' codes: eight columns of each,
//   which are rows i of eight tiles of the output. Two keys' halves are joined before
//   the codes are unpacked, as the operand holds keys in pairs. What lies in LDS is
//   80 bytes a key, 64 of codes, then d and m: keys of the four groups of lanes
//   lie in different banks.
// A value is one packed fma of an exact code: the F16 number that the block stands
// for, so all of the F16 kernel's arithmetic holds as it is there.
// Rows of K and page ids are loaded a turn ahead, V's at the turn's start, under the
// products of q.k. No load is marked as not used again: where a token's heads lie side
// by side a head's 80 bytes are part of a line whose rest another workgroup reads (64
// tokens over up to 8192: 327 us so marked, 205 without). For the same reason the heads of
// a tile run in the same XCD where contexts are whole.
// What a rare row needs (a score that is no number, weights below what fp16 holds)
// is in careful(), which fetches its operands again: kept in registers for it they
// spill. Registers, not waves, are short: 4 waves of up to 256.
//
// 64 tokens over up to 8192: 112 us, of that the F16 cache takes 175; codes unpacked
// into LDS first took 190. Three over up to 131072 (F16 q): 83 to 87, and 156. The kernel then
// reads 3 TB/s, 5 in the middle of long parts. Its 320 to 410 vector operations a block of 32
// keys, a third of them the unpacking, are 45 of the 112 us if spread over the whole card, its
// bytes 65 at a copy's rate: with two waves a SIMD it reaches neither, with one of them alone
// where a compute unit's shorter context has ended.
#include <type_traits>

#include "paged_attention_few.hpp"

namespace qk {
namespace {

constexpr int kWaves = 4, kStep = kBlock * kWaves;

// The column that row i of output tile d is: nibble d of the lane's dword (with
// D = 64 columns i and i + 8 share one), bytes from the low halves' first on.
template <int D>
__device__ __forceinline__ int few_q4_dim(int d, int i) {
  return D == 128 ? 32 * (i >> 2) + 4 * (i & 3) + (d >> 1) + 16 * (d & 1)
                  : 32 * (i >> 2 & 1) + 4 * (i & 3) + 2 * (i >> 3) + (d >> 1) + 16 * (d & 1);
}

// R rows a tile; the 16 columns of a product are 16 / R groups of them, each with
// every 16 / R-th block of keys of its own. q is in all groups; a block's weights are
// zero in the others'. Groups share nothing: each is a row of its own until the end.
template <int D, bool Q32, int R>
__global__ __launch_bounds__(64 * kWaves, 2) void attention_few_q4_kernel(const AttentionArgs a) {
  typedef Num<false> N;
  typedef typename N::V8 V8;
  constexpr int NP = kParts<false, Q32>;
  constexpr int NW = 2;                     // parts of a weight, as over an F16 cache
  constexpr int KS = D / 32, DT = D / 16;   // k steps of q.k (dwords of codes a lane and key), 16-wide tiles of the output
  constexpr int kGroups = 16 / R;
  constexpr int NB = 2, kSets = NB / kGroups;  // blocks a wave and turn, a group and turn
  static_assert(NB * kBlock == 64, "a turn's keys are looked up a lane each");
  constexpr int kRow = D / 8 + D / 32;      // dwords of a row in LDS: codes, then d and m of each block
  typedef Q4Quarter<KS> Piece;  // of one key
  struct Shared : FewShared {
    union {
      uint32_t v[kWaves][NB][kBlock * kRow];
      float o[kWaves * 16][D];  // of a wave's part p (one a group) and row r: (wave kGroups + p) R + r
    };
    int64_t place[kWaves][2][NB * kBlock];  // bytes
    float top[kWaves * 16], sum[kWaves * 16];
  };
  __shared__ __attribute__((aligned(16))) Shared sh;

  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Workgroups go to the eight XCDs in turn. Where tokens lie outside heads (rows of
  // 80 bytes in lines of 128), the heads of a tile to the same one, which has the shared
  // lines in its cache: 64 sequences of up to 8192 keys 112 us, by head 123. In parts the
  // tiles' uneven numbers of them would load the XCDs unevenly: by head, first parts first.
  const int heads = a.kv.kv_heads, block = static_cast<int>(blockIdx.x);
  const bool shared = a.splits == 1 && a.kv.head_stride < a.kv.token_stride;
  const int eight = block / (8 * heads), within = block - eight * 8 * heads, side = min(8, a.tiles - 8 * eight);
  const int head = shared ? within / side : block % heads, unit = shared ? 8 * eight + within - head * side : block / heads;
  const int split = unit / a.tiles, tile = unit - split * a.tiles;
  const AttentionTile t = few_tile<R>(a, tile, sh);
  if (t.s < 0) return;
  // Parts of one length for all sequences, as long as it takes for all of them to run
  // at once: an even share of all keys for each workgroup that the card holds, less the
  // half part that each tile ends in.
  int chunk = kStep;
  if (a.splits > 1) {
    const KeyCounts keys = count_keys(a, R);
    const int held = plan::kMostUnits / a.kv.kv_heads, parts = held - keys.tiles / 2 > 1 ? held - keys.tiles / 2 : 1;
    const int64_t share = (keys.all + parts - 1) / parts;
    chunk = share < keys.longest ? static_cast<int>(share) : keys.longest;
    chunk = chunk < plan::kLeastPartQ4 ? plan::kLeastPartQ4 : chunk;
  }
  const KeyChunk c = key_chunk(t, split, a.splits, kStep, chunk);
  if (split >= c.used) return;
  if (tid == 0) sh.bad = t.beyond;
  __syncthreads();

  // the lane's row, and its group of keys: column of every accumulator
  const int col = lane & 15, grp = lane >> 4, mine = col / R;
  const int row = t.begin + col % R;
  const bool live = row < t.rows;
  const int token = t.row + (live ? row / a.group : 0), h = head * a.group + (live ? row % a.group : 0);
  const int position = t.first + (token - t.row);
  const int last = live ? (position < c.hi - 1 ? position : c.hi - 1) : -1;  // keys that the row sees here: from .. last
  const int from = a.window > 0 ? position - a.window + 1 : 0;
  // every row sees all keys of [all_from, all_last]
  const int all_last = t.first + t.begin / a.group;
  const int end_row = t.begin + R < t.rows ? t.begin + R : t.rows;
  const int all_from = a.window > 0 ? t.first + (end_row - 1) / a.group - a.window + 1 : 0;

  // Block n of turn i is block (i NB + n) kWaves + wave of the chunk.
  const int blocks = (c.hi - c.lo + kBlock - 1) / kBlock;
  const auto block_of = [&](int turn, int n) { return (turn * NB + n) * kWaves + wave; };
  const auto key0_of = [&](int turn, int n) { return c.lo + block_of(turn, n) * kBlock; };
  int32_t page = 0, entry = 0;
  bool listed = true, bad = false;
  const auto key_of = [&](int turn) {  // the lane's key of a turn; keys past the end stand in for by the last one
    const int key = key0_of(turn, lane / kBlock) + lane % kBlock;
    return key < c.hi ? key : c.hi - 1;
  };
  const auto look_up = [&](int turn) {
    entry = page_entry(a.pages, key_of(turn));
    page = a.kv.page_table[kv_table_at(a.kv, t.s, entry, listed)];
  };
  const auto settle = [&](int turn) {  // page ids -> places
    const bool ok = listed && page >= 0 && page < a.kv.pages;
    bad |= !ok;
    const int slot = key_of(turn) - entry * a.kv.page_size;
    sh.place[wave][turn & 1][lane] = q4_bytes(kv_place(a.kv, ok ? page : 0, slot, head));
    __builtin_amdgcn_wave_barrier();
  };
  Piece kreg[NB][2], vreg[NB][2];  // [block][key / 16]
  const auto load = [&](const uint16_t* pool, int turn, int n, Piece (&to)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint8_t* at = reinterpret_cast<const uint8_t*>(pool) + sh.place[wave][turn & 1][n * kBlock + 16 * i + col];
      to[i] = q4_load_quarter<KS>(at, grp);
    }
  };
  // q as it lies in memory: of step s the dword's low halves' values, and its high halves'
  typedef std::conditional_t<Q32, float, _Float16> Q;
  typedef Q Q4 __attribute__((ext_vector_type(4)));
  Q4 q_low[KS], q_high[KS];
  if (wave < blocks) look_up(0);
  {
    const Q* from_q = static_cast<const Q*>(a.q) + token * a.q_stride + static_cast<int64_t>(h) * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      q_low[s] = *reinterpret_cast<const Q4*>(from_q + q4_quarter_value<KS>(grp, s));
      q_high[s] = *reinterpret_cast<const Q4*>(from_q + q4_quarter_value<KS>(grp, s) + 16);
    }
  }
  if (wave < blocks) {
    settle(0);
    look_up(1);
#pragma unroll
    for (int n = 0; n < NB; ++n) load(a.kv.k, 0, n, kreg[n]);
  }

  // q, in parts: eight values of step s in the order of a dword's unpacked codes
  V8 q[KS][NP];
  float factor = a.scale * kLog2e;
  {
    const auto in_order = [&](int s, int i) { return live ? (i & 2 ? q_high : q_low)[s][q4_pair_value(i) & 15] : static_cast<Q>(0.0f); };
    if constexpr (Q32) {
      float most = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(in_order(s, i)));
      most = swap32_max(swap16_max(most));
      // 2^(14 - exponent): the row's largest value in [2^13, 2^14)
      const bool scaled = most > 0.0f && most < __builtin_inff();
      const int e = scaled ? 14 - __builtin_amdgcn_frexp_expf(most) : 0;
      factor = ldexpf(factor, -e);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = ldexpf(in_order(s, i), e);
        split8<false, NP>(x, q[s]);
      }
    } else {
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) q[s][0][i] = in_order(s, i);
    }
  }

  f32x4 o[DT] = {};
  float top = kNoMax, sum = 0.0f;
  // where the lane's pieces go in LDS, and the dword that it reads of each key's codes
  const int v_to = D == 128 ? 4 * grp : 2 * grp, v_dm = D / 8 + (D == 128 ? grp : grp >> 1);
  const int v_from = 4 * grp * kRow + (D == 128 ? col : col & 7), v_dm_from = 4 * grp * kRow + D / 8 + (D == 128 ? col >> 2 : (col & 7) >> 2);
  const uint32_t halves = D == 128 || col < 8 ? 0x05040100u : 0x07060302u;  // D = 64: columns i and i + 8 have one dword

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
  const Q4Exponents exponents;
  // Block n's codes out of LDS, two keys' of a dword together, with their d and m.
  struct Block {
    uint32_t two[4][DT / 4];
    half2_q4 d[4], m[4];
  };
  const auto fetch = [&](int n) __attribute__((always_inline)) {
    Block b;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t* const at = sh.v[wave][n] + (16 * (j >> 1) + 2 * (j & 1)) * kRow;
      const uint32_t w0 = at[v_from], w1 = at[v_from + kRow], dm0 = at[v_dm_from], dm1 = at[v_dm_from + kRow];
      b.d[j] = __builtin_bit_cast(half2_q4, __builtin_amdgcn_perm(dm1, dm0, 0x05040100u));
      b.m[j] = __builtin_bit_cast(half2_q4, __builtin_amdgcn_perm(dm1, dm0, 0x07060302u));
#pragma unroll
      for (int i = 0; i < DT / 4; ++i) b.two[j][i] = __builtin_amdgcn_perm(w1, w0, i == 0 ? halves : 0x07060302u);
    }
    return b;
  };
  // Its values of output tile d, in pairs of keys.
  const auto tile_of = [&](const Block& b, int d) __attribute__((always_inline)) {
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t two = b.two[j][d >> 2] >> (d & 2 ? 8 : 0);
      const half2_q4 code = d & 1 ? q4_high(two, exponents) : q4_low(two, exponents);
      v[j] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(code, b.d[j], b.m[j]));
    }
    return v;
  };
  // w: the weights of the block's group, and of others, that do not count. FINITE: all
  // values are; else those that are not go in as zeros (0 times them is none, and a
  // weight's parts may be of either sign).
  const auto add_values = [&](int n, const Block& b, const V8 (&w)[NW], auto finite) __attribute__((always_inline)) {
    constexpr bool FINITE = decltype(finite)::value;
    V8 of_group[NW];
#pragma unroll
    for (int p = 0; p < NW; ++p) of_group[p] = kGroups == 1 || mine == n % kGroups ? w[p] : V8{};
#pragma unroll
    for (int d = 0; d < DT; ++d) {  // a tile's products run under the next one's unpacking
      u32x4 v = tile_of(b, d);
      if constexpr (!FINITE) v = only_finite<false>(v);
#pragma unroll
      for (int p = 0; p < NW; ++p) o[d] = N::mfma16(__builtin_bit_cast(V8, v), of_group[p], o[d]);
    }
  };
  // Scores q.k of the 32 keys of a block, of which `k` holds the lane's pieces.
  const auto scores = [&](const Piece (&k)[2], f32x4 (&y)[2]) __attribute__((always_inline)) {
    y[0] = y[1] = f32x4{};
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const half2_q4 dm = __builtin_bit_cast(half2_q4, k[i].dm);
        const half2_q4 d = {dm.x, dm.x}, m = {dm.y, dm.y};
        half2_q4 k4[4];
        q4_pairs(k[i].codes[s], d, m, exponents, k4);
        const V8 key = __builtin_bit_cast(V8, k4);
#pragma unroll
        for (int p = 0; p < NP; ++p) y[i] = N::mfma16(key, q[s][p], y[i]);
      }
  };
  // A score of register r of half i of a block that begins at key0, -inf where the row does not see the key.
  const auto masked = [&](float x, int key0, int i, int r) __attribute__((always_inline)) {
    const int key = key0 + 16 * i + 4 * grp + r;
    return static_cast<int>(key <= last) & static_cast<int>(key >= from) ? x : -__builtin_inff();
  };
  // The size of the lane's row of the output, and the reference up to which that
  // makes it sound beside values of the turn's size (a bound, from the blocks' d and m).
  const auto judge = [&](float largest) __attribute__((always_inline)) {
    float size = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) size = fmaxf(size, fabsf(o[d][r]) < __builtin_inff() ? fabsf(o[d][r]) : 0.0f);
    size = swap32_max(swap16_max(size));
    sound = sound_to<NW>(top, size, largest);
    return size;
  };
  const auto largest_value = [&]() __attribute__((always_inline)) {
    float most = 0.0f;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const half2_q4 dm = __builtin_bit_cast(half2_q4, sh.v[wave][n][(16 * i + col) * kRow + v_dm]);
        const float d = fabsf(static_cast<float>(dm.x)), low = fabsf(static_cast<float>(dm.y));
        // in fp32: where code 15 leaves F16, lower codes may stand for any value of it
        const float high = fminf(fabsf(__builtin_fmaf(15.0f, static_cast<float>(dm.x), static_cast<float>(dm.y))), 65504.0f);
        const bool any = d < __builtin_inff() && low < __builtin_inff();  // else no value of the block is finite
        most = fmaxf(most, any ? fmaxf(low, high) : 0.0f);
      }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) most = fmaxf(most, __shfl_xor(most, off));
    return most;
  };
  // A turn with values that are not finite, or with weights that lack bits that count:
  // block by block, keys loaded again and values from LDS, in the registers that the
  // other turns' loads need.
  const auto careful = [&](int turn) __attribute__((always_inline)) {
#pragma clang fp contract(off)
    const auto fetch_anew = [&](int n) __attribute__((always_inline)) {  // or unpacked values would stay in registers in between
      asm volatile("" ::: "memory");
      return fetch(n);
    };
    const float largest = largest_value();
#pragma unroll 1
    for (int n = 0; n < NB; ++n) {
      if (block_of(turn, n) >= blocks) break;
      Piece k[2];
      load(a.kv.k, turn, n, k);
      f32x4 x[2];
      scores(k, x);
      const int key0 = key0_of(turn, n);
      float p[8];
      float least = __builtin_inff(), most = -__builtin_inff();
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = mine == n % kGroups ? masked(x[e / 4][e % 4] * factor, key0, e / 4, e % 4) : -__builtin_inff();
        if (p[e] > -__builtin_inff()) least = fminf(least, p[e]);
        most = fmaxf(most, p[e]);
      }
      if (__any(most > top + kSlack)) {  // the block before may have lowered it
        most = swap32_max(swap16_max(most));
        rescale(risen<NW>(top, most));
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(p[e] - (top - kLift<false>));
        sum += p[e];
      }
      V8 w[NW];
      split8<false, NW>(p, w);
      add_values(n, fetch_anew(n), w, std::false_type{});
      // what the weights of rows that are not sound lack, in steps of a sinking reference
      float size = judge(largest);
      const bool lacks = swap32_max(swap16_max(least < least_full() ? 1.0f : 0.0f)) > 0.0f;
      for (int step = 0; step < 8; ++step) {
        const int by = lacks && top > sound ? sinking<NW>(size, swap32_max(swap16_max(sum)), largest) : 0;
        if (!__any(by > 0)) break;
        rescale(top - static_cast<float>(by));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
#pragma unroll
          for (int i = 0; i < NW; ++i) p[e] -= static_cast<float>(w[i][e]);
          p[e] = by > 0 ? ldexpf(p[e], by) : 0.0f;
        }
        split8<false, NW>(p, w);
        add_values(n, fetch_anew(n), w, std::false_type{});
        size = judge(largest);
      }
      // Values that are not finite, to the rows that see them (any weight times them is
      // themselves): a product of which kinds there are, 1 for an infinity, 2^6 for a
      // negative one, 2^12 for a NaN, none of which 32 keys carry over, with ones.
      V8 seen;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        seen[e] = static_cast<_Float16>(mine == n % kGroups && masked(0.0f, key0, e / 4, e % 4) == 0.0f ? 1.0f : 0.0f);
      const Block b = fetch_anew(n);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const u32x4 v = tile_of(b, d);
        V8 kinds;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t bits = v[e >> 1] >> 16 * (e & 1) & 0xFFFFu, size = bits & 0x7FFFu;
          const float kind = size < 0x7C00u ? 0.0f : size > 0x7C00u ? 0x1p12f : bits >> 15 ? 0x1p6f : 1.0f;
          kinds[e] = static_cast<_Float16>(kind);
        }
        const f32x4 all = N::mfma16(kinds, seen, f32x4{});
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int of = static_cast<int>(all[r]);
          const float both = (of & 63 ? __builtin_inff() : 0.0f) + (of >> 6 & 63 ? -__builtin_inff() : 0.0f);
          if (of) o[d][r] += of >> 12 ? __builtin_nanf("") : both;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

  for (int turn = 0; block_of(turn, 0) < blocks; ++turn) {
#pragma clang fp contract(off)
    // Loads are issued whether or not there are blocks to come, past the last one of its
    // last key: a path around them would make every wait one for all loads in flight.
#pragma unroll
    for (int n = 0; n < NB; ++n) load(a.kv.v, turn, n, vreg[n]);
    settle(turn + 1);
    look_up(turn + 2);
    // scores: registers r of half i hold key 16 i + 4 grp + r of a block
    f32x4 x[kSets][2] = {};
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      if (n == 0 || block_of(turn, n) < blocks) {
        f32x4 y[2];
        scores(kreg[n], y);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            x[n / kGroups][i][r] = n % kGroups == 0 || mine == n % kGroups ? y[i][r] : x[n / kGroups][i][r];
      }
      load(a.kv.k, turn + 1, n, kreg[n]);
    }
    // softmax
    const bool whole = key0_of(turn, NB - 1) + kBlock - 1 <= all_last && key0_of(turn, NB - 1) + kBlock <= c.hi &&
                       key0_of(turn, 0) >= all_from;
    float most = -__builtin_inff(), least = __builtin_inff();
#pragma unroll
    for (int s = 0; s < kSets; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[s][i] = x[s][i] * factor;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (!whole) {
            x[s][i][r] = masked(x[s][i][r], key0_of(turn, s * kGroups + mine), i, r);
            least = fminf(least, x[s][i][r] > -__builtin_inff() ? x[s][i][r] : __builtin_inff());
          } else {
            least = fminf(least, x[s][i][r]);
          }
          most = fmaxf(most, x[s][i][r]);
        }
      }
    if (__any(most > top + kSlack)) {
      most = swap32_max(swap16_max(most));
      rescale(risen<NW>(top, most));
    }
    _Float16 zeros = 0.0f;  // or NaN
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t* const to = sh.v[wave][n] + (16 * i + col) * kRow;
        *reinterpret_cast<typename Piece::Codes*>(to + v_to) = vreg[n][i].codes;
        to[v_dm] = vreg[n][i].dm;  // of D = 64 two lanes write the same
        const half2_q4 dm = __builtin_bit_cast(half2_q4, vreg[n][i].dm);
        zeros = __builtin_fmaf16(dm.y, 0.0f, zeros);  // values lie between m and 15 d + m
        zeros = __builtin_fmaf16(__builtin_fmaf16(15.0f, dm.x, dm.y), 0.0f, zeros);
      }
    __builtin_amdgcn_wave_barrier();
    bool care = __any(!(zeros == static_cast<_Float16>(0.0f)));
    if (__builtin_expect(__any(least < least_full()), 0)) {
      judge(largest_value());
      care |= __any(least < least_full());
    }
    if (__builtin_expect(care, 0)) {
      careful(turn);
#pragma unroll
      for (int n = 0; n < NB; ++n) load(a.kv.k, turn + 1, n, kreg[n]);
      continue;
    }
    V8 w[kSets][NW];
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(x[s][e / 4][e % 4] - (top - kLift<false>));
        sum += p[e];
      }
      split8<false, NW>(p, w[s]);
    }
#pragma unroll
    for (int n = 0; n < NB; ++n)
      if (n == 0 || block_of(turn, n) < blocks) add_values(n, fetch(n), w[n / kGroups], std::true_type{});
    __builtin_amdgcn_wave_barrier();
  }

  // the waves' parts, one a group
  if (__any(bad) && lane == 0) sh.bad = 1;
  sum = swap32_sum(swap16_sum(sum));
  if (grp == 0) {
    sh.top[wave * 16 + col] = top;
    sh.sum[wave * 16 + col] = sum;
  }
  __syncthreads();  // every wave is done with its values
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) sh.o[wave * 16 + col][few_q4_dim<D>(d, 4 * grp + r)] = o[d][r];
  __syncthreads();
  // their join: D / 2 lanes a row, two values each
  typedef float F2 __attribute__((ext_vector_type(2)));
  constexpr int kLanes = D / 2, kSlots = 64 * kWaves / kLanes;
  const int slot = tid / kLanes, at = tid % kLanes * 2, rows = min(R, t.rows - t.begin);
  float all, total;
  F2 y;
  const auto gather = [&](int r, int parts) __attribute__((always_inline)) {
    all = kNoMax;
    total = 0.0f;
    y = F2{};
    for (int p = 0; p < parts; ++p) all = fmaxf(all, sh.top[p * R + r]);
    for (int p = 0; p < parts; ++p) {
      const float f = __builtin_amdgcn_exp2f(sh.top[p * R + r] - all);
      total += f * sh.sum[p * R + r];
      y += f * *reinterpret_cast<const F2*>(&sh.o[p * R + r][at]);
    }
  };
  const auto store = [&](int r) __attribute__((always_inline)) {
    const int of = t.begin + r;
    const int64_t to = static_cast<int64_t>(t.row + of / a.group) * a.q_heads + head * a.group + of % a.group;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    if constexpr (Q32) {
      *reinterpret_cast<F2*>(static_cast<float*>(a.out) + to * D + at) = y * inv;
    } else {
      *reinterpret_cast<half2_q4*>(static_cast<_Float16*>(a.out) + to * D + at) =
          half2_q4{static_cast<_Float16>(y.x * inv), static_cast<_Float16>(y.y * inv)};
    }
    if (a.lse && at == 0) a.lse[to] = row_lse<false>(all, total);
  };
  const bool broken = sh.bad != 0;
  if (broken && tid == 0) kv_fault(a.kv, QK_KV_FAULT_PAGE);
  const int64_t first_part = (static_cast<int64_t>(tile) * a.kv.kv_heads + head) * a.splits;
  for (int r = slot; r < rows; r += kSlots) {
    gather(r, kWaves * kGroups);
    if (broken) total = __builtin_nanf("");
    if (c.used == 1) {
      store(r);
    } else {
      const int64_t part = (first_part + split) * R + r;
      if (at == 0) put(a.sums + 2 * part, all, total);
      put(a.parts + part * D + at, y.x, y.y);
    }
  }
  if (c.used == 1) return;
  if (!last_to_arrive(a.arrived + static_cast<int64_t>(tile) * a.kv.kv_heads + head, c.used, sh.arrived)) return;
  // Of the workgroups' parts. Slots without a row of their own take a share of another's parts.
  constexpr int kMostWays = kWaves * 16 / R < kSlots ? kWaves * 16 / R : kSlots;
  int ways = 1;
  while (2 * ways <= kMostWays && 2 * ways * rows <= kSlots) ways *= 2;
  const int share = slot % ways, per = (c.used + ways - 1) / ways, lo = share * per, hi = min(c.used, lo + per);
  for (int r0 = 0; r0 < rows; r0 += kSlots / ways) {
    const int r = r0 + slot / ways;
    all = kNoMax;
    total = 0.0f;
    y = F2{};
    if (r < rows) {
      for (int base = lo; base < hi; base += kLanes) {  // a lane a part, then its sums to all lanes
        constexpr int kAhead = 8;
        const int mine_at = base + tid % kLanes;
        float m, l;
        get(a.sums + 2 * ((first_part + min(mine_at, hi - 1)) * R + r), m, l);
        F2 next[kAhead];
        const auto fetch_parts = [&](int k0) {  // past the last that one again, not added
#pragma unroll
          for (int k = 0; k < kAhead; ++k) {
            float x0, x1;
            get(a.parts + ((first_part + min(k0 + k, hi - 1)) * R + r) * D + at, x0, x1);
            next[k] = F2{x0, x1};
          }
        };
        fetch_parts(base);
        float to = fmaxf(all, m);
#pragma unroll
        for (int off = 1; off < kLanes; off <<= 1) to = fmaxf(to, __shfl_xor(to, off));
        const float f = __builtin_amdgcn_exp2f(all - to);
        all = to;
        m = mine_at < hi ? __builtin_amdgcn_exp2f(m - all) : 0.0f;
        l = mine_at < hi ? m * l : 0.0f;
#pragma unroll
        for (int off = 1; off < kLanes; off <<= 1) l += __shfl_xor(l, off);
        total = total * f + l;
        y *= f;
        for (int k0 = base; k0 < min(hi, base + kLanes); k0 += kAhead) {
          F2 now[kAhead];
#pragma unroll
          for (int k = 0; k < kAhead; ++k) now[k] = next[k];
          if (k0 + kAhead < min(hi, base + kLanes)) fetch_parts(k0 + kAhead);
#pragma unroll
          for (int k = 0; k < kAhead; ++k) {
            const float g = __shfl(m, (lane & ~(kLanes - 1)) + (k0 - base) + k);
            if (k0 + k < hi) y += g * now[k];
          }
        }
      }
    }
    if (ways > 1) {  // then one round does all rows
      __syncthreads();
      if (r < rows) {
        if (at == 0) {
          sh.top[share * R + r] = all;
          sh.sum[share * R + r] = total;
        }
        *reinterpret_cast<F2*>(&sh.o[share * R + r][at]) = y;
      }
      __syncthreads();
      if (slot >= rows) return;
      gather(slot, ways);
      store(slot);
      return;
    }
    if (r < rows) store(r);
  }
}

}  // namespace

hipError_t launch_attention_few_q4(const AttentionArgs& a, int tile_rows, int head_dim, int q_type, hipStream_t stream) {
  const uint32_t grid = static_cast<uint32_t>(a.tiles) * a.splits * a.kv.kv_heads;
  const bool q32 = q_type == QK_TYPE_F32;
  auto go = [&](auto kernel) { kernel<<<grid, 64 * kWaves, 0, stream>>>(a); };
  auto by_rows = [&](auto rows) {
    constexpr int R = decltype(rows)::value;
    if (head_dim == 128)
      q32 ? go(attention_few_q4_kernel<128, true, R>) : go(attention_few_q4_kernel<128, false, R>);
    else
      q32 ? go(attention_few_q4_kernel<64, true, R>) : go(attention_few_q4_kernel<64, false, R>);
  };
  if (tile_rows == 8)
    by_rows(std::integral_constant<int, 8>{});
  else
    by_rows(std::integral_constant<int, 16>{});
  note("attention_few_q4_kernel", grid, head_dim, q32, tile_rows, a.splits > 1);
  return hipGetLastError();
}

}  // namespace qk
