// What cached tokens get of the attention of the new ones, added up a key/value head:
//   weight[j] += sum over new tokens i >= j and query heads of exp2(f q_i.k_j - l_i),
// f = scale log2(e), l_i the row's log of the sum of exp in base 2. A workgroup owns its
// keys, so no atomics: the sums' order is the plan's.
//
// Few rows (a decode step): keys are streamed, once, as in paged_attention_few.hip:
// four waves take blocks of 32 keys in turn, each through 8 KB of LDS of its own,
// as the columns of 16x16x32 products whose rows are the queries; a key's sum is that of
// a lane's registers and of four lanes. Q4_1 rows come straight from their codes, as in
// paged_attention_few_q4.hip. One token over 1000 keys: 7.4 us, the call. 64 tokens
// over up to 8192 in Q4_1: 74 us, 2.5 TB/s of keys and weights read and weights written;
// vector operations bound it, 270 a block of keys: unpacking, places (divisions by the
// page's size), and eight exponentials, each behind a branch on its mask and taken for a
// tile's rows that are none as well (12 of 16, with one token and four heads a group).
// A workgroup takes its sequence's tiles of 16 rows one after another, keys anew for each:
// a call lasts as long as that of a chunk among single tokens (weigh_plan.hpp).
//
// Many rows (a prompt's): each of four waves holds 64 keys in registers, as the
// columns of 32x32x16 products, and all walk the same tiles of 32 rows, in LDS, split in
// parts there and loaded a tile ahead. The exponentials and the conversion of F32 q, which
// every workgroup does anew, bound it (105 of 245 vector operations a tile). Where keys are too few
// to occupy the card the rows are shared out too, and a second launch adds up the parts.
// 63 new tokens over 32768 keys in F16, F32 q: 49 to 57 us. Two prompts of up to 2047 in BF16, 28
// heads over 4: 43 to 49, of which exponentials and sums are 11 if spread over the card; there
// each of 1856 workgroups gathers 256 keys for 14 tiles at most, uneven numbers of them.
//
// F32 q and 16-bit keys meet as in the attention: two fp16 parts of q (22 bits, after
// scaling each row by a power of two) or three bf16 ones.
#include <type_traits>

#include "paged_attention.hpp"

namespace qk {
namespace {

// A row's log of the sum of exp in base 2, for weights exp2(x - it): infinite, so that
// they are nothing, for rows that are none, see nothing or have no number there.
__device__ __forceinline__ float row_log2(const WeighArgs& a, int64_t row_at, bool live) {
  const float log = live ? a.lse[row_at] : -__builtin_inff();
  return log > -__builtin_inff() ? log * kLog2e : __builtin_inff();
}
// A weight; one that is NaN (of a score or a log that is) counts for nothing.
__device__ __forceinline__ float weight_of(float x, float factor, float log2_sum) {
  return fmaxf(__builtin_amdgcn_exp2f(__builtin_fmaf(x, factor, -log2_sum)), 0.0f);
}

// Where a key's weight lies, -1 if its page is none.
__device__ __forceinline__ int64_t weight_place(const WeighArgs& a, int page, int slot, int head) {
  return page < 0 ? -1 : (static_cast<int64_t>(page) * a.kv.kv_heads + head) * a.kv.page_size + slot;
}
__device__ __forceinline__ int64_t weight_of_key(const WeighArgs& a, int s, int key, int head) {
  const int entry = key / a.kv.page_size;
  return weight_place(a, kv_page(a.kv, s, entry), key - entry * a.kv.page_size, head);
}
// What a new token's slot held before is of another token: its weight begins here.
__device__ __forceinline__ void add_weight(const WeighArgs& a, const KvSequence& q, int s, int key, int64_t at, float old,
                                           float sum, bool first_time) {
  const bool is_new = key >= q.first;
  a.weight[at] = (is_new && first_time ? 0.0f : old) + sum;
  if (is_new && first_time) a.position[at] = (a.seen ? a.seen[s] - a.kv.context[s] : 0) + key;
}

// The sequence's lengths; false (and reported) where it has no key to weigh or no room.
__device__ __forceinline__ bool weigh_keys(const WeighArgs& a, int s, bool report, KvSequence& q, int& keys) {
  q = kv_sequence(a.kv, s);
  keys = kv_keys(q);
  const bool longer = keys > a.most_keys;
  if (report && threadIdx.x == 0) {
    if (q.fault || longer) kv_fault(a.kv, QK_KV_FAULT_LENGTH);
    if (q.beyond) kv_fault(a.kv, QK_KV_FAULT_PAGE);
  }
  return keys > 0 && !longer;
}

// ------------------------------------------------------------- few rows --

constexpr int kBlock = 32, kWaves = 4;

// Chunks of 16 bytes of a row in LDS, so that 16 keys' same chunk lie in different banks.
template <int D>
__device__ __forceinline__ int k_chunk(int key, int chunk) {
  return key * (2 * D) + ((chunk ^ (D == 128 ? key & 15 : key >> 1 & 7)) << 4);
}

template <int D, int KIND, bool Q32>
__global__ __launch_bounds__(64 * kWaves, KIND != QK_TYPE_Q4_1 && Q32 && D == 128 ? 3 : 4) void kv_weigh_few_kernel(const WeighArgs a) {
  constexpr bool BF16 = KIND == QK_TYPE_BF16, Q4 = KIND == QK_TYPE_Q4_1;
  typedef Num<BF16> N;
  typedef typename N::V8 V8;
  constexpr int NP = kParts<BF16, Q32>, KS = D / 32;
  constexpr int LPK = D / 8, KPL = 64 / LPK, NL = Q4 ? 2 : kBlock / KPL;  // lanes a key, keys a load, loads a block
  __shared__ __attribute__((aligned(16))) uint8_t k_lds[kWaves][Q4 ? 16 : kBlock * 2 * D];
  __shared__ int64_t place[kWaves][2][kBlock];
  __shared__ __attribute__((aligned(16))) float factors[kWaves][16], logs[kWaves][16];

  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Workgroups go to the eight XCDs in turn. Where there are many, the first parts of all
  // contexts come first, as later ones are empty where contexts are short, and the
  // heads of one whose Q4_1 rows share lines of memory go to the same XCD: 64 sequences
  // of up to 8192 keys 75 us, a context and head at a time 85; 16 of them 36 and 26.
  const int heads = a.kv.kv_heads, block = static_cast<int>(blockIdx.x);
  const bool many = a.kv.sequences * heads > static_cast<int>(weigh::kUnits);
  const bool shared = Q4 && many && a.kv.head_stride < a.kv.token_stride;
  const int eight = block / (8 * heads), within = block - eight * 8 * heads, side = min(8, a.kv.sequences * a.key_parts - 8 * eight);
  const int head = shared ? within / side : block % heads, unit = shared ? 8 * eight + within - head * side : block / heads;
  const int s = many ? unit % a.kv.sequences : unit / a.key_parts, part = many ? unit / a.kv.sequences : unit % a.key_parts;
  KvSequence seq;
  int keys;
  if (!weigh_keys(a, s, head == 0 && part == 0, seq, keys)) return;
  const int lo = part * a.part_keys, hi = keys - lo < a.part_keys ? keys : lo + a.part_keys;
  const int blocks = hi > lo ? (hi - lo + kBlock - 1) / kBlock : 0;
  if (wave >= blocks) return;  // waves share nothing
  const int rows = seq.count * a.group, col = lane & 15, grp = lane >> 4;
  bool bad = false;

  for (int begin = 0; begin < rows; begin += 16) {
    int32_t page = 0;
    bool listed = true;
    const auto key_of = [&](int b) {  // the lane's key of block b; keys past the end stand in for by the last one
      const int key = lo + b * kBlock + (lane & 31);
      return key < hi ? key : hi - 1;
    };
    const auto look_up = [&](int b) {
      page = a.kv.page_table[kv_table_at(a.kv, s, key_of(b) / a.kv.page_size, listed)];
    };
    // Of the lane's key's weight, and what is there. That is loaded with the block's keys,
    // before them: a load at the end of a block would have to wait for the next one's.
    int64_t at = 0, next_at = 0;
    float old = 0.0f, next_old = 0.0f;
    const auto settle = [&](int b) {
      const bool ok = listed && page >= 0 && page < a.kv.pages;
      bad |= !ok;
      const int slot = key_of(b) % a.kv.page_size;
      next_at = weight_place(a, ok ? page : -1, slot, head);
      next_old = a.weight[next_at < 0 ? 0 : next_at];
      const int64_t to = kv_place(a.kv, ok ? page : 0, slot, head);
      place[wave][b / kWaves & 1][lane & 31] = Q4 ? q4_bytes(to) : to;
      __builtin_amdgcn_wave_barrier();
    };
    // 16-bit rows as whole rows, through LDS; of Q4_1 ones each lane takes the quarter that it multiplies
    std::conditional_t<Q4, Q4Quarter<KS>, u32x4> reg[NL];
    const auto load = [&](int b) {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        if constexpr (Q4)
          reg[i] = q4_load_quarter<KS>(reinterpret_cast<const uint8_t*>(a.kv.k) + place[wave][b / kWaves & 1][16 * i + col], grp);
        else
          reg[i] = stream_load16(a.kv.k + place[wave][b / kWaves & 1][KPL * i + lane / LPK] + 8 * (lane % LPK));
      }
    };
    look_up(wave);
    settle(wave);
    look_up(wave + kWaves);
    load(wave);

    // the queries as rows of the product: lane (row, grp), and for the sums of registers
    // 4 grp .. of a result that row's factor and log
    V8 q[KS][NP];
    {
      const int row = begin + col;
      const bool live = row < rows;
      const int token = seq.row + (live ? row / a.group : 0), h = head * a.group + (live ? row % a.group : 0);
      float factor = a.scale * kLog2e;
      const int64_t from = token * a.q_stride + static_cast<int64_t>(h) * D;
      // the first of step k's values 4 i .. 4 i + 3
      const auto quad_at = [&](int k, int i) { return Q4 ? q4_quarter_value<KS>(grp, k) + 16 * i : 32 * k + 8 * grp + 4 * i; };
      // which of those is its e-th
      const auto value_at = [](int e) { return Q4 ? q4_pair_value(e) % 16 + (e & 2 ? 4 : 0) : e; };
      if constexpr (Q32) {
        float x[KS][8];
        float most = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.q) + from + quad_at(k, i));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              x[k][4 * i + j] = live ? v[j] : 0.0f;
              most = fmaxf(most, fabsf(x[k][4 * i + j]));
            }
          }
        int e = 0;
        if constexpr (!BF16) {
          most = swap32_max(swap16_max(most));
          const bool scaled = most > 0.0f && most < __builtin_inff();
          e = scaled ? 14 - __builtin_amdgcn_frexp_expf(most) : 0;  // the row's largest in [2^13, 2^14)
          factor = ldexpf(factor, -e);
        }
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          float y[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = ldexpf(x[k][value_at(i)], e);
          split8<BF16, NP>(y, q[k]);
        }
      } else {
        typedef typename N::T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          T4 v[2];
#pragma unroll
          for (int i = 0; i < 2; ++i)
            v[i] = *reinterpret_cast<const T4*>(static_cast<const typename N::T*>(a.q) + from + quad_at(k, i));
#pragma unroll
          for (int i = 0; i < 8; ++i) q[k][0][i] = live ? v[value_at(i) / 4][value_at(i) % 4] : static_cast<typename N::T>(0.0f);
        }
      }
      if (grp == 0) {
        factors[wave][col] = factor;
        logs[wave][col] = row_log2(a, static_cast<int64_t>(token) * a.q_heads + h, live);
      }
      __builtin_amdgcn_wave_barrier();
    }
    const f32x4 factor = *reinterpret_cast<const f32x4*>(&factors[wave][4 * grp]);
    const f32x4 log2_sum = *reinterpret_cast<const f32x4*>(&logs[wave][4 * grp]);
    const int end_row = begin + 16 < rows ? begin + 16 : rows;
    const int all_see = seq.first + begin / a.group;  // keys up to here all rows see
    const int any_sees = seq.first + (end_row - 1) / a.group;

    uint8_t* const ks = k_lds[wave];
    const Q4Exponents exponents;
    for (int b = wave; b < blocks; b += kWaves) {
      const int key0 = lo + b * kBlock;
      f32x4 x[2] = {};
      if constexpr (Q4) {
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const half2_q4 dm = __builtin_bit_cast(half2_q4, reg[i].dm);
            half2_q4 pairs[4];
            q4_pairs(reg[i].codes[k], half2_q4{dm.x, dm.x}, half2_q4{dm.y, dm.y}, exponents, pairs);
#pragma unroll
            for (int p = 0; p < NP; ++p) x[i] = N::mfma16(q[k][p], __builtin_bit_cast(V8, pairs), x[i]);
          }
      } else {
#pragma unroll
        for (int i = 0; i < NL; ++i) *reinterpret_cast<u32x4*>(ks + k_chunk<D>(KPL * i + lane / LPK, lane % LPK)) = reg[i];
      }
      at = next_at;
      old = next_old;
      // past the last block loads are of its last key: a path around them would make every wait one for all loads
      settle(b + kWaves);
      load(b + kWaves);
      look_up(b + 2 * kWaves);
      __builtin_amdgcn_wave_barrier();
      if constexpr (!Q4) {
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const V8 key = __builtin_bit_cast(V8, load16(ks + i * (16 * 2 * D) + k_chunk<D>(col, 4 * k + grp)));
#pragma unroll
            for (int p = 0; p < NP; ++p) x[i] = N::mfma16(q[k][p], key, x[i]);
          }
      }
      float sum[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = key0 + 16 * i + col;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float w = weight_of(x[i][r], factor[r], log2_sum[r]);
          // row 4 grp + r sees the key if its position is no smaller
          sum[i] += key0 + kBlock - 1 <= all_see || seq.first + (begin + 4 * grp + r) / a.group >= key ? w : 0.0f;
        }
        sum[i] = swap32_sum(swap16_sum(sum[i]));
      }
      const int key = key0 + lane;
      if (lane < kBlock && key < hi && at >= 0 && (key <= any_sees || begin == 0))
        add_weight(a, seq, s, key, at, old, lane < 16 ? sum[0] : sum[1], begin == 0);
      __builtin_amdgcn_wave_barrier();
    }
  }
  if (__any(bad) && lane == 0) kv_fault(a.kv, QK_KV_FAULT_PAGE);
}

// ------------------------------------------------------------ many rows --

constexpr int kTileRows = 32, kKeysAWave = 64;

// A row's chunk in LDS, so that 32 rows' same chunk lie in different banks.
template <int D>
__device__ __forceinline__ int q_chunk(int row, int chunk) {
  return row * (2 * D) + ((chunk ^ (row & (D / 8 - 1))) << 4);
}

template <int D, int KIND, bool Q32>
__global__ __launch_bounds__(64 * kWaves, 3) void kv_weigh_many_kernel(const WeighArgs a) {
  constexpr bool BF16 = KIND == QK_TYPE_BF16, Q4 = KIND == QK_TYPE_Q4_1;
  typedef Num<BF16> N;
  typedef typename N::V8 V8;
  typedef float f32x16 __attribute__((ext_vector_type(16)));
  constexpr int NP = kParts<BF16, Q32>, KS = D / 16;
  constexpr int E = D / 8;  // values of a row that a thread brings, eight threads a row
  static_assert(64 * kWaves == 8 * kTileRows, "eight threads a row");
  __shared__ __attribute__((aligned(16))) uint8_t q_lds[2][NP][kTileRows * 2 * D];
  __shared__ __attribute__((aligned(16))) float factors[2][kTileRows], logs[2][kTileRows];

  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int head = static_cast<int>(blockIdx.x) % a.kv.kv_heads;
  int unit = static_cast<int>(blockIdx.x) / a.kv.kv_heads;
  const int row_part = unit % a.row_parts;
  unit /= a.row_parts;
  const int s = unit % a.kv.sequences, part = unit / a.kv.sequences;  // keys that many rows see first
  KvSequence seq;
  int keys;
  if (!weigh_keys(a, s, head == 0 && part == 0 && row_part == 0, seq, keys)) return;
  const int lo = part * a.part_keys, rows = seq.count * a.group;
  if (lo >= keys) return;
  // tiles of rows that see any of these keys, this workgroup's share of them
  const int first_row = lo > seq.first ? (lo - seq.first) * a.group / kTileRows : 0;
  const int tiles = (rows + kTileRows - 1) / kTileRows - first_row, share = (tiles + a.row_parts - 1) / a.row_parts;
  const int from = first_row + row_part * share, to = min(first_row + tiles, from + share);

  // the wave's keys: lane (key, half) of group g
  const int col = lane & 31, half = lane >> 5, key0 = lo + wave * kKeysAWave;
  bool bad = false;
  V8 k[2][KS];
  int least_row[2];  // the first row that sees the lane's key
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int key = min(key0 + 32 * g + col, keys - 1), entry = key / a.kv.page_size;
    const int page = kv_page(a.kv, s, entry);
    bad |= page < 0;
    const int64_t place = kv_place(a.kv, page < 0 ? 0 : page, key - entry * a.kv.page_size, head);
    least_row[g] = key0 + 32 * g + col > seq.first ? (key0 + 32 * g + col - seq.first) * a.group : 0;
    if constexpr (Q4) {
#pragma unroll
      for (int i = 0; i < KS / 2; ++i) {
        u32x4 low, high;
        q4_values(q4_load(reinterpret_cast<const uint8_t*>(a.kv.k) + q4_bytes(place), 2 * i + half), low, high);
        k[g][2 * i] = __builtin_bit_cast(V8, low);
        k[g][2 * i + 1] = __builtin_bit_cast(V8, high);
      }
    } else {
#pragma unroll
      for (int i = 0; i < KS; ++i) k[g][i] = __builtin_bit_cast(V8, load16(a.kv.k + place + 16 * i + 8 * half));
    }
  }

  // a tile's rows into registers, and from there, in parts, into LDS
  const int my_row = tid >> 3, my_at = (tid & 7) * E;
  typedef std::conditional_t<Q32, f32x4, u32x4> QReg;
  constexpr int QN = Q32 ? E / 4 : E / 8;
  QReg reg[QN];
  float reg_log = 0.0f;
  const auto load = [&](int tile) __attribute__((always_inline)) {
    const int row = min(tile * kTileRows + my_row, rows - 1);
    const int token = seq.row + row / a.group, h = head * a.group + row % a.group;
    const int64_t at = token * a.q_stride + static_cast<int64_t>(h) * D + my_at;
#pragma unroll
    for (int i = 0; i < QN; ++i) {
      if constexpr (Q32)
        reg[i] = *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.q) + at + 4 * i);
      else
        reg[i] = load16(static_cast<const uint16_t*>(a.q) + at + 8 * i);
    }
    reg_log = row_log2(a, static_cast<int64_t>(token) * a.q_heads + h, tile * kTileRows + my_row < rows);
  };
  const auto store = [&](int buffer) __attribute__((always_inline)) {
    float factor = a.scale * kLog2e;
    if constexpr (Q32) {
      int e = 0;
      if constexpr (!BF16) {
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < QN; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) most = fmaxf(most, fabsf(reg[i][j]));
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) most = fmaxf(most, __shfl_xor(most, off));
        e = most > 0.0f && most < __builtin_inff() ? 14 - __builtin_amdgcn_frexp_expf(most) : 0;
        factor = ldexpf(factor, -e);
      }
#pragma unroll
      for (int c = 0; c < E / 8; ++c) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = ldexpf(reg[2 * c + i / 4][i % 4], e);
        V8 parts[NP];
        split8<BF16, NP>(x, parts);
#pragma unroll
        for (int p = 0; p < NP; ++p)
          *reinterpret_cast<V8*>(q_lds[buffer][p] + q_chunk<D>(my_row, my_at / 8 + c)) = parts[p];
      }
    } else {
#pragma unroll
      for (int c = 0; c < E / 8; ++c) *reinterpret_cast<u32x4*>(q_lds[buffer][0] + q_chunk<D>(my_row, my_at / 8 + c)) = reg[c];
    }
    if ((tid & 7) == 0) {
      factors[buffer][my_row] = factor;
      logs[buffer][my_row] = reg_log;
    }
  };

  float sum[2] = {0.0f, 0.0f};
  if (from < to) {
    load(from);
    store(from & 1);
    if (from + 1 < to) load(from + 1);
    for (int tile = from; tile < to; ++tile) {
      const int buffer = tile & 1;
      __syncthreads();  // tile `tile` is there, and all are done with the one before
      if (tile + 1 < to) {
        store(buffer ^ 1);
        if (tile + 2 < to) load(tile + 2);
      }
      f32x16 x[2] = {};
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const V8 q = *reinterpret_cast<const V8*>(q_lds[buffer][p] + q_chunk<D>(col, 2 * i + half));
#pragma unroll
          for (int g = 0; g < 2; ++g) x[g] = N::mfma32(q, k[g][i], x[g]);
        }
      const auto add = [&](auto masked) __attribute__((always_inline)) {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {  // registers 4 r4 .. hold rows 8 r4 + 4 half ..
          const f32x4 factor = *reinterpret_cast<const f32x4*>(&factors[buffer][8 * r4 + 4 * half]);
          const f32x4 log2_sum = *reinterpret_cast<const f32x4*>(&logs[buffer][8 * r4 + 4 * half]);
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float w = weight_of(x[g][4 * r4 + r], factor[r], log2_sum[r]);
              const bool seen = !decltype(masked)::value || tile * kTileRows + 8 * r4 + 4 * half + r >= least_row[g];
              sum[g] += seen ? w : 0.0f;
            }
        }
      };
      // does every row of the tile see every key of the wave?
      if (tile * kTileRows >= (key0 + kKeysAWave - 1 - seq.first) * a.group)
        add(std::false_type{});
      else
        add(std::true_type{});
    }
  }
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    sum[g] = swap32_sum(sum[g]);
    const int key = key0 + 32 * g + col;
    if (half != g || key >= keys) continue;  // a half of the lanes each group
    if (a.row_parts > 1) {
      const int64_t unit_at = static_cast<int64_t>(s) * a.kv.kv_heads + head, width = static_cast<int64_t>(a.key_parts) * a.part_keys;
      a.parts[(static_cast<int64_t>(row_part) * a.kv.sequences * a.kv.kv_heads + unit_at) * width + key] = sum[g];
    } else {
      const int64_t at = weight_of_key(a, s, key, head);
      if (at >= 0) add_weight(a, seq, s, key, at, a.weight[at], sum[g], true);
    }
  }
  if (__any(bad) && lane == 0) kv_fault(a.kv, QK_KV_FAULT_PAGE);
}

// The sums of the rows' parts, a key a thread.
__global__ __launch_bounds__(256) void kv_weigh_join_kernel(const WeighArgs a) {
  const int head = static_cast<int>(blockIdx.x) % a.kv.kv_heads, unit = static_cast<int>(blockIdx.x) / a.kv.kv_heads;
  const int s = unit / a.key_parts, key = unit % a.key_parts * a.part_keys + static_cast<int>(threadIdx.x);
  KvSequence seq;
  int keys;
  if (!weigh_keys(a, s, false, seq, keys) || key >= keys) return;
  const int64_t unit_at = static_cast<int64_t>(s) * a.kv.kv_heads + head, width = static_cast<int64_t>(a.key_parts) * a.part_keys;
  float sum = 0.0f;
  for (int p = 0; p < a.row_parts; ++p)
    sum += a.parts[(static_cast<int64_t>(p) * a.kv.sequences * a.kv.kv_heads + unit_at) * width + key];
  const int64_t at = weight_of_key(a, s, key, head);
  if (at >= 0) add_weight(a, seq, s, key, at, a.weight[at], sum, true);
}

}  // namespace

hipError_t launch_kv_weigh(WeighArgs a, const WeighPlan& plan, int type, int head_dim, int q_type, void* workspace,
                           hipStream_t stream) {
  a.key_parts = plan.key_parts;
  a.part_keys = plan.part_keys;
  a.row_parts = plan.row_parts;
  a.most_keys = plan.key_parts * plan.part_keys;
  a.parts = static_cast<float*>(workspace);
  const uint32_t units = static_cast<uint32_t>(a.kv.sequences) * a.kv.kv_heads * plan.key_parts;
  const bool q32 = q_type == QK_TYPE_F32;
  auto go = [&](auto kernel, uint32_t grid) { kernel<<<grid, 64 * kWaves, 0, stream>>>(a); };
  auto by_type = [&](auto dim, auto kind) {
    constexpr int D = decltype(dim)::value, KIND = decltype(kind)::value;
    if (plan.few)
      q32 ? go(kv_weigh_few_kernel<D, KIND, true>, units) : go(kv_weigh_few_kernel<D, KIND, false>, units);
    else
      q32 ? go(kv_weigh_many_kernel<D, KIND, true>, units * plan.row_parts)
          : go(kv_weigh_many_kernel<D, KIND, false>, units * plan.row_parts);
  };
  auto by_dim = [&](auto dim) {
    if (type == QK_TYPE_BF16)
      by_type(dim, std::integral_constant<int, QK_TYPE_BF16>{});
    else if (type == QK_TYPE_Q4_1)
      by_type(dim, std::integral_constant<int, QK_TYPE_Q4_1>{});
    else
      by_type(dim, std::integral_constant<int, QK_TYPE_F16>{});
  };
  head_dim == 128 ? by_dim(std::integral_constant<int, 128>{}) : by_dim(std::integral_constant<int, 64>{});
  note(plan.few ? "kv_weigh_few_kernel" : "kv_weigh_many_kernel", units, head_dim, type, q32, plan.row_parts > 1);
  const hipError_t error = hipGetLastError();
  if (error != hipSuccess || plan.row_parts == 1) return error;
  kv_weigh_join_kernel<<<units, 256, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace qk
