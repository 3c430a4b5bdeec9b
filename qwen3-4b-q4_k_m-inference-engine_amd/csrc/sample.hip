// The next token of each row by temperature, top-k, top-p and min-p from a
// given uniform, in two launches.
//
// sample_scan_kernel reads every logit once, one workgroup per chunk of a row
// (2048 or 8192 logits, all in registers): the chunk's maximum; how many
// logits lie in each of 128 bands below it, a fifth wide (without top-k a quarter
// of the temperature at most), and, where no top-k bounds the kept set, the sum of
// their weights; and the logits of the top bands themselves, band by band, as many
// as the row's top-k can take from one chunk. sample_draw_kernel, one workgroup per row,
// adds the bands up, which gives the band that a filter's border falls into,
// and then
//   - where the chunks' lists reach down to that band (the usual filters), finds
//     everything among the listed logits: few of them, or those of an even part of
//     them that holds a border, are ranked one against another;
//   - without top-k, reads the row once more for the logits of that band
//     alone (several workgroups if there are few rows), or not at all if there
//     is no border (bare temperature), picks the drawn token's chunk by the
//     chunks' sums and reads that again;
//   - else (thousands of logits around a border: equal ones, high
//     temperatures) searches the row digit by digit.
//
// Values are ranked by a 32-bit key whose unsigned order is the order of the
// logits (NaN and -inf: 0, never drawn). Weights are fixed-point integers,
// rint(exp((z - max) / T) * 2^shift) of a 64-bit exponential with 2^shift *
// vocabulary <= 2^62 and shift <= 44, so their sums are exact and no order of additions can
// change a result; a chunk whose own maximum is not the row's is weighed by
// its own and scaled once per band, in 64-bit floating point. Bands only say
// where to look; no result depends on their width.
// Measured: one row of 151936, top-k 20 and top-p 0.95: 15 us; 200 rows: greedy 24
// (5.0 TB/s), top-k 20 37, filters of their own (a fifth without top-k) 80.
#include "qk_device.hpp"
#include "qk_launch.hpp"
#include "serving.hpp"

namespace qk {
namespace {

constexpr int kThreads = 1024;     // of the draw
constexpr int kBins = 2048;        // of a digit
constexpr int kScanThreads = 256;
constexpr int kBands = 128;
constexpr int kList = 512;         // most listed logits of a chunk
constexpr int kItems = 6144;       // most logits of a band that the draw holds: two workgroups' LDS fits a compute unit
constexpr int kSorted = 2 * kThreads;
constexpr int kMostChunk = 8192;   // logits of a chunk
constexpr int kMostChunks = 2048;  // chunks of a row
constexpr int kHelped = 128;       // most rows that get more than one draw workgroup
constexpr int kShift = 44;         // most fraction bits of a weight
constexpr int kCopies = 16;        // of the scan's bands: a wave's lanes with the same two low bits share one
constexpr int kCountAt = 54;       // a band's count above its sum: 512 logits of 2^44 stay below 2^54
constexpr int kFew = 128;          // listed logits of a chunk without top-k
constexpr int kPairs = 128;        // most items that are ranked pair by pair

// What the scan leaves of a chunk.
struct ChunkHead {
  uint32_t key, index;     // of its largest logit (0: nothing to draw, and nothing else is written)
  int32_t listed, through; // entries of its list: the logits of bands 0 .. through - 1
};
struct SamplePlan {
  int32_t chunk, chunks, list, shift;
  ChunkHead* heads;   // [rows x chunks]
  uint16_t* counts;   // [rows x chunks][kBands]
  uint64_t* weights;  // [rows x chunks][kBands]
  uint64_t* lists;    // [rows x chunks][list]: key << 32 | ~index, by band
  int32_t helpers;    // draw workgroups a row; above 1:
  uint32_t* gathered; // [rows][2]: items and workgroups so far, zero between calls
  uint64_t* items;    // [rows][kItems]
  size_t bytes;
};

__device__ __forceinline__ uint32_t rank_key(float v) {
  if (!(v > -__builtin_inff())) return 0;
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);  // -0 -> +0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __builtin_bit_cast(float, (key & 0x80000000u) ? key & 0x7FFFFFFFu : ~key);
}

// 2^t for t <= 0, to about 2^-50 of itself; nothing below 2^-128: the power
// series of e^(f ln 2) up to f^12 over |f| <= 1/2, a third of the instructions
// of a correctly scaled 64-bit exponential.
__device__ __forceinline__ double exp2_part(double t) {
  t = fmax(t, -128.0);  // NaN too
  const double n = rint(t), f = t - n;
  constexpr double c[13] = {1.0,
                            0.69314718055994531,
                            0.24022650695910072,
                            0.055504108664821580,
                            0.0096181291076284772,
                            0.0013333558146428443,
                            0.00015403530393381610,
                            0.000015252733804059841,
                            0.0000013215486790144310,
                            1.0178086009239699e-7,
                            7.0549116208011234e-9,
                            4.4455382718708114e-10,
                            2.5678435993488206e-11};
  double y = c[12];
#pragma unroll
  for (int i = 11; i >= 0; --i) y = __builtin_fma(y, f, c[i]);
  return ldexp(y, static_cast<int>(n));
}

struct Weigher {
  double max, rate, one;  // rate: log2(e) / T
  __device__ __forceinline__ double ratio_of(float z) const {
    return exp2_part(z == max ? 0.0 : (static_cast<double>(z) - max) * rate);
  }
  __device__ __forceinline__ double ratio(uint32_t key) const { return ratio_of(key_value(key)); }
  // The sum's low 52 bits are the product, at most 2^44, rounded to an integer.
  __device__ __forceinline__ uint64_t fixed_of(float z) const {
    return __builtin_bit_cast(uint64_t, __builtin_fma(ratio_of(z), one, 0x1p52)) & 0xFFFFFFFFFFFFFull;
  }
  __device__ __forceinline__ uint64_t fixed(uint32_t key) const { return key == 0 ? 0 : fixed_of(key_value(key)); }
};
__device__ __forceinline__ Weigher weigher(uint32_t top, float heat, int shift) {
  return Weigher{static_cast<double>(key_value(top)), 1.4426950408889634 / heat, static_cast<double>(uint64_t{1} << shift)};
}

// The band of v below top (v <= top, both above -inf). The same for a chunk's
// maximum against the row's, so that bands of chunks add up: values times
// `scale` that are closer than kBands have exact differences.
__device__ __forceinline__ int band_of(float v, float top, float scale) {
  if (v == top) return 0;
  const float d = floorf(top * scale) - floorf(v * scale);
  return d < static_cast<float>(kBands - 1) ? static_cast<int>(d) : kBands - 1;  // NaN (of infinities): the last
}
// A fifth wide where top-k bounds the kept set and only ranks matter (its border
// then lies in a band for logits up to 25 below the maximum), else a quarter of
// the temperature at most.
__device__ __forceinline__ float band_scale(float heat, bool cut) { return cut ? 5.0f : fmaxf(4.0f / heat, 5.0f); }
__device__ __forceinline__ uint64_t item_of(uint32_t key, int index) {
  return static_cast<uint64_t>(key) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(index));
}
__device__ __forceinline__ uint32_t item_key(uint64_t item) { return static_cast<uint32_t>(item >> 32); }
__device__ __forceinline__ int item_index(uint64_t item) { return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(item)); }
__device__ __forceinline__ void lds_add(uint64_t* p, uint64_t v) {
  atomicAdd(reinterpret_cast<unsigned long long*>(p), static_cast<unsigned long long>(v));
}
// Four logits from x[at]; what lies past n reads as -inf.
template <bool ONCE = false>
__device__ __forceinline__ f32x4 load_logits(const float* x, int at, int n) {
  if (at + 4 <= n) {
    if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const f32x4_a4*>(x + at));
    return *reinterpret_cast<const f32x4_a4*>(x + at);
  }
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = at + e < n ? x[at + e] : -__builtin_inff();
  return v;
}
// Appends the lanes' items where `mine`, a place for each from *count.
__device__ __forceinline__ void append(bool mine, uint64_t item, uint64_t* items, uint32_t* count, uint32_t most) {
  const uint64_t who = __ballot(mine);
  if (!who) return;
  const int lane = static_cast<int>(threadIdx.x & 63), leader = __builtin_ctzll(who);
  uint32_t base = 0;
  if (lane == leader) base = atomicAdd(count, static_cast<uint32_t>(__popcll(who)));
  base = __builtin_amdgcn_readlane(base, leader);
  const uint32_t at = base + static_cast<uint32_t>(__popcll(who & ((uint64_t{1} << lane) - 1)));
  if (mine && at < most) items[at] = item;
}

// The scan. HBM bounds it: 200 rows of 151936 logits, 121 MB. A thread's
// logits are all loaded before any is looked at (16 bytes x E in flight a
// lane). Band counts are spread over copies, as neighbouring logits often
// share a band; with weights, count and sum are one 64-bit addition.
template <int E>
__global__ __launch_bounds__(kScanThreads) void sample_scan_kernel(const SampleArgs a, const SamplePlan p) {
  static_assert(E <= 8 && kScanThreads / 64 * 4 == kCopies && 16 * E * 4 <= 512);
  __shared__ uint64_t bands[kBands * kCopies];
  __shared__ float tops[kScanThreads / 64], groups[kScanThreads];
  __shared__ uint32_t first, places[kBands];  // where a band's next listed logit goes
  __shared__ int32_t depth;
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = tid >> 6;
  const int row = static_cast<int>(blockIdx.y), lo = static_cast<int>(blockIdx.x) * p.chunk;
  const int n = min(a.vocabulary - lo, p.chunk);
  const int64_t unit = static_cast<int64_t>(row) * p.chunks + blockIdx.x;
  const float* x = a.logits + row * a.row_stride + lo;
  const int at0 = tid * 4;  // element e of load i is logit lo + at0 + i * 4 * kScanThreads + e
  const float heat = a.temperature[row];
  const int k = a.top_k ? a.top_k[row] : 0;
  const bool greedy = !(heat > 0.0f);
  const bool cut = k > 0 && k < a.vocabulary;  // the kept set is bounded: no sums of bands are needed
  f32x4 v[E];
  if (E == 8 && (cut || greedy)) {  // large batches: rows that the draw hardly reads again
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = load_logits<true>(x, at0 + i * 4 * kScanThreads, n);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = load_logits(x, at0 + i * 4 * kScanThreads, n);
  }
  const bool bounded = cut && k <= kScanThreads && !greedy;
  uint32_t* const counts = reinterpret_cast<uint32_t*>(bands);  // of a cut row: [band][4]
  if (cut) {
    for (int i = tid; i < kBands * 2; i += kScanThreads) bands[i] = 0;
  } else if (!greedy) {
    for (int i = tid; i < kBands * kCopies; i += kScanThreads) bands[i] = 0;
  }
  if (tid == 0) first = 0xFFFFFFFFu;
  float mine = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < E; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) mine = fmaxf(mine, v[i][e]);  // NaN: the other operand
  if (bounded) {
    float group = mine;
    if (k <= kScanThreads / 4) {
      group = fmaxf(group, __shfl_xor(group, 1));
      group = fmaxf(group, __shfl_xor(group, 2));
    }
    groups[tid] = group;
  }
  float top = mine;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kScanThreads / 64; ++w) top = fmaxf(top, tops[w]);
  if (!(top > -__builtin_inff())) {
    if (tid == 0) p.heads[unit] = ChunkHead{0, 0, 0, 0};
    return;
  }
  const uint32_t top_key = rank_key(top);
  if (mine == top) {
    uint32_t at = 0xFFFFFFFFu;
#pragma unroll
    for (int i = E - 1; i >= 0; --i)
#pragma unroll
      for (int e = 3; e >= 0; --e)
        if (v[i][e] == top) at = static_cast<uint32_t>(lo + at0 + i * 4 * kScanThreads + e);
    atomicMin(&first, at);
  }
  if (greedy) {
    __syncthreads();
    if (tid == 0) p.heads[unit] = ChunkHead{top_key, first, 0, 0};
    return;
  }
  const float scale = band_scale(heat, cut);
  // the lane's logits to count or to list: bit 4 i + e
  uint32_t some = 0;
  const auto each = [&](auto visit) {  // few: read again, not picked from registers
    for (uint32_t left = some; __any(left != 0); left &= left - 1) {
      const int bit = left ? __builtin_ctz(left) : 0, at = at0 + (bit >> 2) * 4 * kScanThreads + (bit & 3);
      visit(left != 0, left ? x[at] : 0.0f, at);
    }
  };
  if (bounded) {
    // The k-th largest of the maxima of k groups or more has k logits of the
    // chunk at or above it: what is below it is in no row's top-k and need not
    // be looked at. Its upper 18 bits, by bisection: groups of four lanes
    // (k <= 64) leave little more than k logits, single lanes a few times k.
    const bool quads = k <= kScanThreads / 4;
    uint32_t key[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) key[j] = quads ? (j ? 0 : rank_key(groups[4 * lane])) : rank_key(groups[64 * j + lane]);
    uint32_t least = 0;
    for (int bit = 31; bit >= 14; --bit) {
      const uint32_t candidate = least | 1u << bit;
      int reach = __popcll(__ballot(key[0] >= candidate));
      if (!quads) {
#pragma unroll
        for (int j = 1; j < 4; ++j) reach += __popcll(__ballot(key[j] >= candidate));
      }
      if (reach >= k) least = candidate;
    }
    const float bound = least >= rank_key(-3.4028234e38f) ? key_value(least) : -3.4028234e38f;
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) some |= v[i][e] >= bound ? 1u << (4 * i + e) : 0u;
    each([&](bool in, float z, int) {
      if (in) atomicAdd(&counts[band_of(z, top, scale) * 4 + (lane & 3)], 1u);
    });
  } else if (cut) {
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (v[i][e] > -__builtin_inff()) atomicAdd(&counts[band_of(v[i][e], top, scale) * 4 + (lane & 3)], 1u);
  } else {
    const Weigher w = weigher(top_key, heat, p.shift);
    const int copy = wave * 4 + (lane & 3);
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float z = v[i][e];
        if (z > -__builtin_inff())
          lds_add(&bands[band_of(z, top, scale) * kCopies + copy], w.fixed_of(z) | uint64_t{1} << kCountAt);
      }
  }
  __syncthreads();
  if (wave == 0) {  // lane: bands 2 lane and 2 lane + 1
    uint32_t c[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int band = 2 * lane + i;
      c[i] = 0;
      if (cut) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c[i] += counts[band * 4 + j];
      } else {
        uint64_t sum = 0;
#pragma unroll
        for (int j = 0; j < kCopies; ++j) {
          const uint64_t both = bands[band * kCopies + ((j + lane) & (kCopies - 1))];  // lanes start at different banks
          c[i] += static_cast<uint32_t>(both >> kCountAt);
          sum += both & ((uint64_t{1} << kCountAt) - 1);
        }
        p.weights[unit * kBands + band] = sum;
      }
    }
    reinterpret_cast<uint32_t*>(p.counts + unit * kBands)[lane] = c[0] | c[1] << 16;
    uint32_t run = c[0] + c[1];
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t other = __shfl_up(run, off);
      if (lane >= off) run += other;
    }
    places[2 * lane] = run - c[1] - c[0];
    places[2 * lane + 1] = run - c[1];
    // as many bands as hold what the row may need of this chunk, and as the list holds
    const uint32_t want = cut ? k : kFew, most = p.list;
    const int enough = __popcll(__ballot(run - c[1] < want)) + __popcll(__ballot(run < want)) + 1;
    const int fit = __popcll(__ballot(run - c[1] <= most)) + __popcll(__ballot(run <= most));
    const int through = min(min(enough, fit), kBands);
    const uint32_t held = through == 0 ? 0 : __shfl(through & 1 ? run - c[1] : run, (through - 1) >> 1);
    if (lane == 0) {
      depth = through;
      p.heads[unit] = ChunkHead{top_key, first, static_cast<int32_t>(held), through};
    }
  }
  __syncthreads();
  const int through = depth;
  if (!bounded) {
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        some |= v[i][e] > -__builtin_inff() && band_of(v[i][e], top, scale) < through ? 1u << (4 * i + e) : 0u;
  }
  uint64_t* list = p.lists + unit * p.list;
  each([&](bool in, float z, int at) {
    const int band = band_of(z, top, scale);
    if (!in || band >= through) return;
    const uint32_t to = atomicAdd(&places[band], 1u);
    if (to < static_cast<uint32_t>(p.list)) list[to] = item_of(rank_key(z), lo + at);
  });
}

struct Shared {
  union {
    uint64_t items[kItems];
    struct {
      uint64_t sorted[2][kSorted];  // listed logits (later by rank), by index
      union {
        uint64_t ranked[kSorted];  // weights by rank
        struct {
          uint64_t key[kPairs], value[kPairs], before[kPairs];  // of rank_pairs
          uint32_t ahead[kPairs], counts[kThreads];             // items of even parts of the keys
        };
      };
    };
    uint64_t bins[kBins];  // of a digit's search
  };
  union {
    struct {
      uint64_t parts[kThreads], part[kThreads];  // sums of even parts, and a band's items of one
    };
    uint64_t sums[kMostChunks];  // of the chunks' kept logits
  };
  uint64_t weight[kBands];
  uint32_t count[kBands];  // later its running sums
  // of each chunk: where its bands lie in the row's (kBands: it has none), and
  // its head's `through` and `listed`
  uint8_t base[kMostChunks], through[kMostChunks];
  uint16_t listed[kMostChunks], active[kMostChunks];
  uint64_t wave[16];
  uint64_t found[3];
  uint64_t above, total;
  uint32_t border, floor_key, n, actives, low, high;
};
static_assert(sizeof(Shared) <= 80 * 1024);

__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}
__device__ uint64_t group_sum(uint64_t v, Shared& sh) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t t = 0;
  for (int i = 0; i < kThreads / 64; ++i) t += sh.wave[i];
  return t;
}

// visit(index, key) for every logit of the row, by all threads; indices past the
// row's end come with key 0.
template <class F>
__device__ __forceinline__ void each_logit(const float* x, int n, F visit) {
  for (int base = 4 * static_cast<int>(threadIdx.x); base < n; base += 8 * kThreads) {
    const f32x4 v = load_logits(x, base, n), w = load_logits(x, base + 4 * kThreads, n);
#pragma unroll
    for (int e = 0; e < 4; ++e) visit(base + e, rank_key(v[e]));
#pragma unroll
    for (int e = 0; e < 4; ++e) visit(base + 4 * kThreads + e, rank_key(w[e]));
  }
}

// The largest key whose measure of {key >= it} reaches target (1 <= target <=
// the measure of all), and in `above` the measure of the larger ones.
template <class F>
__device__ uint32_t descend(const float* x, int n, uint64_t target, F measure, uint64_t& above, Shared& sh) {
  uint32_t prefix = 0;
  above = 0;
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bits = digit == 2 ? 10 : 11;
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
    __syncthreads();
    each_logit(x, n, [&](int, uint32_t key) {
      if (digit == 0 || key >> (shift + bits) == prefix) {
        const uint64_t m = measure(key);
        if (m) lds_add(&sh.bins[(key >> shift) & ((1u << bits) - 1)], m);
      }
    });
    __syncthreads();
    // bins from the top: thread t has bins n-1-2t and n-2-2t
    const int count = 1 << bits, hi = count - 1 - 2 * static_cast<int>(threadIdx.x);
    const uint64_t b0 = hi >= 0 ? sh.bins[hi] : 0, b1 = hi >= 1 ? sh.bins[hi - 1] : 0;
    uint64_t run = b0 + b1;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint64_t other = __shfl_up(run, off);
      if (lane >= off) run += other;
    }
    if (lane == 63) sh.wave[threadIdx.x >> 6] = run;
    __syncthreads();
    uint64_t before = above;
    for (int i = 0; i < static_cast<int>(threadIdx.x >> 6); ++i) before += sh.wave[i];
    before += run - (b0 + b1);
    if (before < target && before + b0 + b1 >= target) {
      const bool upper = before + b0 >= target;
      sh.found[0] = static_cast<uint64_t>(upper ? hi : hi - 1);
      sh.found[1] = upper ? before : before + b0;
    }
    __syncthreads();
    prefix = (prefix << bits) | static_cast<uint32_t>(sh.found[0]);
    above = sh.found[1];
  }
  return prefix;
}

__device__ __forceinline__ uint64_t lane_value(uint64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), lane);
  return static_cast<uint64_t>(hi) << 32 | lo;
}

// Exclusive running sum of v over the workgroup, and the sum of all.
__device__ uint64_t group_prefix(uint64_t v, uint64_t& all, Shared& sh) {
  const int lane = static_cast<int>(threadIdx.x & 63), wave = static_cast<int>(threadIdx.x >> 6);
  uint64_t run = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint64_t other = __shfl_up(run, off);
    if (lane >= off) run += other;
  }
  __syncthreads();
  if (lane == 63) sh.wave[wave] = run;
  __syncthreads();
  uint64_t before = 0;
  all = 0;
  for (int i = 0; i < kThreads / 64; ++i) {
    if (i < wave) before += sh.wave[i];
    all += sh.wave[i];
  }
  return before + run - v;
}

// Index of the first element, in index order, at which the running sum of
// measure (0 of key 0) exceeds beyond_of(total); n if it never does. A run of neighbours a
// thread, then one wave over the run that crosses.
template <class F, class G>
__device__ int walk(const float* x, int n, G beyond_of, F measure, uint64_t& total, Shared& sh) {
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
  const int per = ((n + kThreads - 1) / kThreads + 3) & ~3;
  const int lo = static_cast<int>(min(static_cast<int64_t>(n), static_cast<int64_t>(tid) * per)), hi = min(n, lo + per);
  uint64_t sum = 0;
  for (int i = lo; i < hi; i += 8) {
    const f32x4 v = load_logits(x, i, hi), w = load_logits(x, i + 4, hi);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += measure(rank_key(v[e]), i + e);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += measure(rank_key(w[e]), i + 4 + e);
  }
  __syncthreads();
  if (tid == 0) sh.found[0] = kThreads;
  uint64_t before = group_prefix(sum, total, sh);
  const uint64_t beyond = beyond_of(total);
  if (before <= beyond && before + sum > beyond) {
    sh.found[0] = static_cast<uint64_t>(tid);
    sh.found[1] = before;
  }
  __syncthreads();
  if (sh.found[0] == kThreads) return n;
  if (tid < 64) {
    before = sh.found[1];
    const int first = static_cast<int>(sh.found[0]) * per, end = min(n, first + per);
    for (int base = first; base < end; base += 64) {
      const int i = base + lane;
      uint64_t run = i < end ? measure(rank_key(x[i]), i) : 0;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const uint64_t other = __shfl_up(run, off);
        if (lane >= off) run += other;
      }
      const uint64_t crossed = __ballot(before + run > beyond);
      if (crossed) {
        if (lane == 0) sh.found[2] = static_cast<uint64_t>(base + __builtin_ctzll(crossed));
        break;
      }
      before += __shfl(run, 63);
    }
  }
  __syncthreads();
  return static_cast<int>(sh.found[2]);
}

// For each of sh.key[0 .. n), n <= kPairs: how many others are larger, added to
// sh.ahead, and the sum of their sh.value, added to sh.before. A lane a key and
// 8 or 16 groups of waves that share the others: 1 us, a sort of as many and
// running sums 6. All threads call it after a barrier, a barrier ends it.
__device__ void rank_pairs(int n, Shared& sh) {
  const int tid = static_cast<int>(threadIdx.x);
  const int width = n <= 64 ? 64 : kPairs, groups = kThreads / width, at = tid & (width - 1);
  const uint64_t key = sh.key[at];
  uint64_t before = 0;
  uint32_t ahead = 0;
  for (int j0 = tid / width; j0 < n; j0 += 4 * groups) {
    uint64_t other[4], value[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = min(j0 + u * groups, n - 1);
      other[u] = sh.key[j];
      value[u] = sh.value[j];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool larger = j0 + u * groups < n && other[u] > key;
      before += larger ? value[u] : 0;
      ahead += larger;
    }
  }
  if (at < n && ahead) {
    lds_add(&sh.before[at], before);
    atomicAdd(&sh.ahead[at], ahead);
  }
  __syncthreads();
}

// items[0 .. n) sorted downwards, n <= kSorted, in room for the next power of
// two; all threads call it after a barrier, a barrier ends it. Steps
// over a distance of up to 64 stay within the 128 items of a wave's 64 pairs.
__device__ void sort_down(uint64_t* items, int n) {
  const int tid = static_cast<int>(threadIdx.x);
  int size = 2;
  while (size < n) size <<= 1;
  for (int i = n + tid; i < size; i += kThreads) items[i] = 0;
  __syncthreads();
  for (int run = 2; run <= size; run <<= 1)
    for (int d = run >> 1; d > 0; d >>= 1) {
      if (tid < size / 2) {
        const int i = (tid & ~(d - 1)) << 1 | (tid & (d - 1));
        const uint64_t x = items[i], y = items[i + d];
        if ((x < y) == ((i & run) == 0)) {
          items[i] = y;
          items[i + d] = x;
        }
      }
      const int next = d > 1 ? d >> 1 : run;
      if (d > 64 || next > 64) {
        __syncthreads();
      } else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
    }
  __syncthreads();
}

// One pass over logits [begin, end) of the row (begin a multiple of 4) that puts
// those of `band` into sh.items, sh.n of them (more than fit are counted).
__device__ void gather_band(const float* x, int begin, int end, int band, float top, float scale, Shared& sh) {
  const float origin = floorf(top * scale), want = static_cast<float>(band);
  // band_of decided for one band: one subtraction and a comparison where
  // neither infinities nor NaN can be in it
  const bool plain = band < kBands - 1 && fabsf(origin) < __builtin_inff();
  constexpr int kAhead = 8;  // loads in flight a lane
  const int first = begin + static_cast<int>(threadIdx.x) * 4;
  for (int base = first; __any(base < end); base += 4 * kThreads * kAhead) {
    f32x4 v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) v[i] = load_logits(x, base + i * 4 * kThreads, end);
    uint32_t hits = 0;
    if (plain) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) hits |= origin - floorf(v[i][e] * scale) == want ? 1u << (4 * i + e) : 0u;
    } else {
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          hits |= v[i][e] > -__builtin_inff() && band_of(v[i][e], top, scale) == band ? 1u << (4 * i + e) : 0u;
    }
    uint32_t at = hits ? atomicAdd(&sh.n, static_cast<uint32_t>(__popc(hits))) : 0;
    for (; hits; hits &= hits - 1, ++at) {  // the places; a register cannot be picked by its number
      const int bit = __builtin_ctz(hits);
      if (at < kItems) sh.items[at] = static_cast<uint64_t>(base + (bit >> 2) * 4 * kThreads + (bit & 3));
    }
  }
  __syncthreads();
  const int items = min(static_cast<int>(sh.n), kItems);
  for (int i = static_cast<int>(threadIdx.x); i < items; i += kThreads) {
    const int index = static_cast<int>(sh.items[i]);
    sh.items[i] = item_of(rank_key(x[index]), index);
  }
  __syncthreads();
}

// The helpers' items together in the last of a row's workgroups to get here,
// where this is true.
__device__ bool join_items(const SamplePlan& p, int row, Shared& sh) {
  uint32_t* const counters = p.gathered + 2 * row;
  uint64_t* const all = p.items + static_cast<int64_t>(row) * kItems;
  const int tid = static_cast<int>(threadIdx.x), mine = min(static_cast<int>(sh.n), kItems);
  if (tid == 0) sh.low = __hip_atomic_fetch_add(counters, static_cast<uint32_t>(mine), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  const int at = static_cast<int>(sh.low);
  for (int i = tid; i < mine && at + i < kItems; i += kThreads)
    __hip_atomic_store(all + at + i, sh.items[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the thread's stores have reached memory
  __syncthreads();
  if (tid == 0) {
    const uint32_t n = __hip_atomic_fetch_add(counters + 1, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sh.high = n + 1 == static_cast<uint32_t>(p.helpers);
    if (sh.high) {
      sh.n = __hip_atomic_load(counters, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(counters, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(counters + 1, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __syncthreads();
  if (!sh.high) return false;
  const int items = min(static_cast<int>(sh.n), kItems);
  for (int i = tid; i < items; i += kThreads)
    sh.items[i] = __hip_atomic_load(all + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  return true;
}

// The draw: a few dependent reads of what the scan left, a ranking in LDS and
// running sums; latency bounds it: 8 us a row for top-k 20, 9 for 50, 16 for 300;
// without top-k 23 to 30 where sixteen workgroups read the row again, 30 to 38
// where one does.
__global__ __launch_bounds__(kThreads) void sample_draw_kernel(const SampleArgs a, const SamplePlan p) {
  __shared__ Shared sh;
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = tid >> 6;
  const int row = static_cast<int>(blockIdx.x), helper = static_cast<int>(blockIdx.y), n = a.vocabulary;
  const float* x = a.logits + row * a.row_stride;
  const int64_t unit0 = static_cast<int64_t>(row) * p.chunks;
  const ChunkHead* heads = p.heads + unit0;
  const float heat = a.temperature[row];
  const int k = a.top_k ? a.top_k[row] : 0;
  const bool cut = k > 0 && k < n;
  const double share = a.top_p ? static_cast<double>(a.top_p[row]) : 1.0;
  const double floor_w = a.min_p ? static_cast<double>(a.min_p[row]) : 0.0;
  const float uniform = a.uniform[row];
  // the others only help where a border may lie deep in the row
  if (helper > 0 && (cut || !(heat > 0.0f) || (!(share < 1.0) && floor_w <= 0.0))) return;
  if (tid < kBands) sh.count[tid] = 0, sh.weight[tid] = 0;
  if (tid == 0) sh.n = 0, sh.actives = 0, sh.low = 0xFFFFFFFFu;
  // the first of the chunks' counts are on their way before the row's maximum is known
  const int units = p.chunks * (kBands / 8);
  u16x8 counts{};
  if (tid < units) counts = *reinterpret_cast<const u16x8*>(p.counts + unit0 * kBands + 8 * tid);
  uint64_t best = 0;
  for (int c = tid; c < p.chunks; c += kThreads) {
    const ChunkHead h = heads[c];
    sh.through[c] = static_cast<uint8_t>(h.through);
    sh.listed[c] = static_cast<uint16_t>(h.listed);
    const uint64_t item = h.key ? item_of(h.key, static_cast<int>(h.index)) : 0;
    best = item > best ? item : best;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint64_t other = __shfl_xor(best, off);
    best = other > best ? other : best;
  }
  if (lane == 0) sh.wave[wave] = best;
  __syncthreads();
  for (int i = 0; i < kThreads / 64; ++i) best = sh.wave[i] > best ? sh.wave[i] : best;
  if (!(heat > 0.0f) || best == 0) {
    if (tid == 0 && helper == 0) {
      a.token[row] = best ? static_cast<uint32_t>(item_index(best)) : 0xFFFFFFFFu;
      if (a.probability) a.probability[row] = best ? 1.0f : 0.0f;
    }
    return;
  }
  const uint32_t top = item_key(best);
  const float top_value = key_value(top), scale = band_scale(heat, cut);
  const Weigher w = weigher(top, heat, p.shift);

  for (int c = tid; c < p.chunks; c += kThreads) {
    const uint32_t key = heads[c].key;
    sh.base[c] = static_cast<uint8_t>(key ? band_of(key_value(key), top_value, scale) : kBands);
  }
  __syncthreads();
  // the row's bands: those of chunk c are base[c] further down. A unit is
  // eight bands of a chunk.
  const auto chunk_sums = [&](int c, int64_t at, uint64_t (&out)[8]) {
    const uint64_t* q = p.weights + at;
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = q[j];
    const uint32_t key = heads[c].key;
    if (key != top) {
      const double factor = w.ratio(key);
#pragma unroll
      for (int j = 0; j < 8; ++j) out[j] = static_cast<uint64_t>(rint(static_cast<double>(out[j]) * factor));
    }
  };
  for (int u = tid; u < units; u += kThreads) {
    const int c = u / (kBands / 8), j0 = u % (kBands / 8) * 8;
    if (sh.base[c] == kBands) continue;
    const int base = sh.base[c] + j0;
    const int64_t at = (unit0 + c) * kBands + j0;
    if (u != tid) counts = *reinterpret_cast<const u16x8*>(p.counts + at);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (counts[j]) atomicAdd(&sh.count[min(base + j, kBands - 1)], static_cast<uint32_t>(counts[j]));
    if (!cut) {
      uint64_t sums[8];
      chunk_sums(c, at, sums);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (sums[j]) lds_add(&sh.weight[min(base + j, kBands - 1)], sums[j]);
    }
  }
  __syncthreads();
  const auto target_of = [&](uint64_t total) {  // fewest whose weights reach the share: the sum to reach
    const double goal = ceil(share * static_cast<double>(total));
    return goal < 1.0 ? uint64_t{1} : min(total, static_cast<uint64_t>(goal));
  };
  if (wave == 0) {  // lane: bands 2 lane and 2 lane + 1; the border band of top-k, or else of top-p
    const uint32_t c0 = sh.count[2 * lane], c1 = sh.count[2 * lane + 1];
    const uint64_t w0 = sh.weight[2 * lane], w1 = sh.weight[2 * lane + 1];
    uint32_t counts = c0 + c1;
    uint64_t sums = w0 + w1;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t c = __shfl_up(counts, off);
      const uint64_t s = __shfl_up(sums, off);
      if (lane >= off) counts += c, sums += s;
    }
    sh.count[2 * lane] = counts - c1;
    sh.count[2 * lane + 1] = counts;
    const uint64_t total = __shfl(sums, 63);
    if (cut) {
      const uint32_t want = static_cast<uint32_t>(k);
      const int b = __popcll(__ballot(counts - c1 < want)) + __popcll(__ballot(counts < want));
      if (lane == 0) sh.border = min(b, kBands - 1);
    } else {
      const uint64_t target = target_of(total);
      const int b = __popcll(__ballot(sums - w1 < target)) + __popcll(__ballot(sums < target));
      const uint64_t before = __shfl(b & 1 ? sums - w1 : sums - w1 - w0, min(b >> 1, 63));
      if (lane == 0) {
        sh.border = share < 1.0 ? b : kBands;
        sh.above = before;
        sh.total = total;
      }
    }
  } else if (wave == 1) {  // the smallest key that min-p keeps, 64 candidates at a time
    uint32_t lo = 1, hi = top;
    if (!(floor_w <= 0.0))
      while (lo < hi) {
        const uint32_t step = (hi - lo) / 64 + 1, off = step * static_cast<uint32_t>(lane);
        const uint32_t key = off < hi - lo ? lo + off : hi;
        const uint64_t stays = __ballot(key == top || w.ratio(key) >= floor_w);
        const int at = stays ? __builtin_ctzll(stays) : 64;  // 64: between the last candidate and hi
        if (stays) hi = __shfl(key, at);
        if (at > 0) lo = __shfl(key, at - 1) + 1;
      }
    else
      hi = 1;
    if (lane == 0) sh.floor_key = hi;
  }
  __syncthreads();
  const uint32_t floor_key = sh.floor_key;
  const int share_band = sh.border;  // kBands: top-p takes all
  const int floor_band = floor_key > 1 ? band_of(key_value(floor_key), top_value, scale) : kBands;
  const int border = cut ? share_band : min(share_band, floor_band);
  const auto draw_from = [&](uint64_t total) {
    const double aim = static_cast<double>(uniform) * static_cast<double>(total);
    const uint64_t beyond =
        aim >= 0.0 ? (aim < static_cast<double>(total) ? static_cast<uint64_t>(aim) : total - 1) : 0;
    return min(beyond, total - 1);
  };
  const auto answer = [&](int index, uint64_t weight, uint64_t total) {
    a.token[row] = static_cast<uint32_t>(index);
    if (a.probability) a.probability[row] = static_cast<float>(static_cast<double>(weight) / static_cast<double>(total));
  };

  // do the lists reach through the border band?
  bool reach = border < kBands && sh.count[min(border, kBands - 1)] <= kSorted;
  if (reach)
    for (int c = tid; c < p.chunks; c += kThreads) {
      if (sh.base[c] > border) continue;
      reach = reach && (border == kBands - 1 ? sh.through[c] == kBands : border - sh.base[c] < sh.through[c]);
      sh.active[atomicAdd(&sh.actives, 1u)] = static_cast<uint16_t>(c);
    }
  if (__syncthreads_and(reach)) {
    if (helper > 0) return;
    // 8 to 512 lanes a chunk, each until its items are past the border: one step for most
    const int actives = static_cast<int>(sh.actives);
    int lanes = 512;
    while (lanes > 8 && lanes * actives > kThreads) lanes >>= 1;
    for (int i = tid / lanes; i < actives; i += kThreads / lanes) {
      const int c = sh.active[i], listed = sh.listed[c];
      const uint64_t* list = p.lists + (unit0 + c) * p.list;
      bool more = true;
      for (int at = tid & (lanes - 1); more && at < listed; at += lanes * 8) {
        uint64_t item[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) item[j] = at + lanes * j < listed ? list[at + lanes * j] : 0;
        uint32_t hits = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          hits |= item[j] && band_of(key_value(item_key(item[j])), top_value, scale) <= border ? 1u << j : 0u;
        more = hits >> 7;
        uint32_t to = hits ? atomicAdd(&sh.n, static_cast<uint32_t>(__popc(hits))) : 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (hits >> j & 1) {
            if (to < kSorted) sh.sorted[0][to] = item[j];
            ++to;
          }
      }
    }
    __syncthreads();
    const int listed = min(static_cast<int>(sh.n), kSorted);
    const int held = cut ? min(listed, k) : listed;
    const auto target_in = [&](uint64_t all) { return share < 1.0 ? target_of(cut ? all : sh.total) : ~uint64_t{0}; };
    const auto place = [&](int at, uint64_t key, uint64_t value) {
      sh.key[at] = key;
      sh.value[at] = value;
      sh.before[at] = 0;
      sh.ahead[at] = 0;
    };
    if (listed <= kPairs) {
      // an item a thread
      const bool in = tid < listed;
      const uint64_t item = in ? sh.sorted[0][tid] : 0, f = w.fixed(item_key(item));
      if (in) place(tid, item, f);
      if (tid == 0) sh.found[1] = 0;
      __syncthreads();
      rank_pairs(listed, sh);
      const int rank = in ? static_cast<int>(sh.ahead[tid]) : 0;
      const uint64_t before = in ? sh.before[tid] : 0;
      if (in && rank == held - 1) sh.found[0] = before + f;
      __syncthreads();
      const bool kept = in && rank < held && (rank == 0 || (before < target_in(sh.found[0]) && item_key(item) >= floor_key));
      const uint64_t mine = kept ? f : 0;
      if (in) place(tid, static_cast<uint32_t>(item), mine);  // by index
      if (wave < kPairs / 64) {
        const uint64_t sum = wave_sum(mine);
        if (lane == 0) lds_add(&sh.found[1], sum);
      }
      __syncthreads();
      rank_pairs(listed, sh);
      const uint64_t total = sh.found[1], beyond = draw_from(total), run = in ? sh.before[tid] : 0;
      if (mine && run <= beyond && run + mine > beyond) answer(item_index(item), mine, total);
      return;
    }
    // More: sums over even parts of the keys, then of the indices, say which
    // part holds an end of the kept set or the drawn token, and its items alone
    // are ranked: 600 items in 8 us, sorted by both 14. False where a part
    // holds too many (equal logits).
    const auto draw_by_parts = [&] {
      uint64_t item[2], f[2];
      uint32_t low = 0xFFFFFFFFu;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = tid + i * kThreads;
        item[i] = at < listed ? sh.sorted[0][at] : 0;
        f[i] = w.fixed(item_key(item[i]));
        if (at < listed) low = min(low, item_key(item[i]));
      }
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) low = min(low, static_cast<uint32_t>(__shfl_xor(low, off)));
      if (lane == 0) atomicMin(&sh.low, low);
      sh.parts[tid] = 0;
      sh.counts[tid] = 0;
      if (tid == 0) sh.found[0] = ~uint64_t{0};
      __syncthreads();
      int step = 0;
      while ((top - sh.low) >> step >= static_cast<uint32_t>(kThreads)) ++step;
      const auto part_of = [&](uint64_t of) { return (top - item_key(of)) >> step; };
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (item[i]) {
          lds_add(&sh.parts[part_of(item[i])], f[i]);
          atomicAdd(&sh.counts[part_of(item[i])], 1u);
        }
      __syncthreads();
      // the listed items where `in` for rank_pairs: how many
      const auto collect = [&](auto in, auto key) {
        if (tid == 0) sh.n = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (item[i] && in(item[i])) {
            const uint32_t at = atomicAdd(&sh.n, 1u);
            if (at < kPairs) place(static_cast<int>(at), key(item[i]), f[i]);
          }
        __syncthreads();
        return static_cast<int>(sh.n);
      };
      const auto itself = [](uint64_t of) { return of; };
      const uint64_t sum = sh.parts[tid];
      uint64_t all;
      const uint64_t before = group_prefix(sum, all, sh);
      uint64_t least = 0;  // the last item that is kept
      if (held < listed) {
        const uint64_t count = sh.counts[tid];
        uint64_t counted;
        const uint64_t fore = group_prefix(count, counted, sh), want = static_cast<uint64_t>(held);
        if (fore < want && fore + count >= want) {
          sh.found[0] = static_cast<uint64_t>(tid);
          sh.found[1] = before;
          sh.found[2] = want - fore;
        }
        __syncthreads();
        const uint32_t part = static_cast<uint32_t>(sh.found[0]);
        const uint64_t ahead = sh.found[1], rank = sh.found[2] - 1;
        const int some = collect([&](uint64_t of) { return part_of(of) == part; }, itself);
        if (some > kPairs) return false;
        rank_pairs(some, sh);
        if (tid < some && sh.ahead[tid] == rank) {
          sh.found[0] = ~uint64_t{0};
          sh.found[1] = sh.key[tid];
          sh.found[2] = ahead + sh.before[tid] + sh.value[tid];
        }
        __syncthreads();
        least = sh.found[1];
        all = sh.found[2];
        __syncthreads();
      }
      if (share < 1.0) {
        const uint64_t target = target_in(all);
        if (before < target && before + sum >= target) {
          sh.found[0] = static_cast<uint64_t>(tid);
          sh.found[1] = before;
        }
        __syncthreads();
        if (sh.found[0] != ~uint64_t{0}) {  // else (a rounding short of the row's sum) all are kept
          const uint32_t part = static_cast<uint32_t>(sh.found[0]);
          const uint64_t ahead = sh.found[1];
          const int some = collect([&](uint64_t of) { return part_of(of) == part; }, itself);
          if (some > kPairs) return false;
          rank_pairs(some, sh);
          if (tid < some) {
            const uint64_t run = ahead + sh.before[tid];
            if (run < target && run + sh.value[tid] >= target) sh.found[2] = sh.key[tid];
          }
          __syncthreads();
          least = sh.found[2] > least ? sh.found[2] : least;
        }
      }
      // in the order of the vocabulary
      int wide = 0;
      while ((n - 1) >> wide >= kThreads) ++wide;
      __syncthreads();
      sh.parts[tid] = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (item[i] != best && (item[i] < least || item_key(item[i]) < floor_key)) item[i] = f[i] = 0;
        if (f[i]) lds_add(&sh.parts[item_index(item[i]) >> wide], f[i]);
      }
      __syncthreads();
      const uint64_t here = sh.parts[tid];
      uint64_t total;
      const uint64_t run = group_prefix(here, total, sh);
      uint64_t beyond = draw_from(total);
      if (run <= beyond && run + here > beyond) {
        sh.found[0] = static_cast<uint64_t>(tid);
        sh.found[1] = run;
      }
      __syncthreads();
      const int part = static_cast<int>(sh.found[0]);
      beyond -= sh.found[1];
      const int some = collect([&](uint64_t of) { return item_index(of) >> wide == part; },
                               [](uint64_t of) { return uint64_t{static_cast<uint32_t>(of)}; });
      if (some > kPairs) return false;
      rank_pairs(some, sh);
      if (tid < some && sh.before[tid] <= beyond && sh.before[tid] + sh.value[tid] > beyond)
        answer(item_index(sh.key[tid]), sh.value[tid], total);
      return true;
    };
    if (draw_by_parts()) return;
    sort_down(sh.sorted[0], listed);
    // ranks 2 tid and 2 tid + 1
    uint64_t mine[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) mine[i] = 2 * tid + i < held ? w.fixed(item_key(sh.sorted[0][2 * tid + i])) : 0;
    if (tid == 0) sh.found[0] = sh.found[1] = 0;
    uint64_t all;
    const uint64_t before = group_prefix(mine[0] + mine[1], all, sh);
    const uint64_t target = target_in(all);
    // the kept ones are the first ranks
    const auto stays = [&](int rank, uint64_t ahead) {
      return rank < held && (rank == 0 || (ahead < target && item_key(sh.sorted[0][rank]) >= floor_key));
    };
    const bool stay0 = stays(2 * tid, before), stay1 = stays(2 * tid + 1, before + mine[0]);
    if (!stay0) mine[0] = 0;
    if (!stay1) mine[1] = 0;
    const uint64_t some = __ballot(stay0);
    if (some && lane == 63 - __builtin_clzll(some)) {
      atomicMax(reinterpret_cast<unsigned long long*>(&sh.found[0]), static_cast<unsigned long long>(2 * tid + 1 + stay1));
      atomicMax(reinterpret_cast<unsigned long long*>(&sh.found[1]),
                static_cast<unsigned long long>(before + mine[0] + mine[1]));
    }
    // in the order of the vocabulary
    uint64_t* order = sh.sorted[1];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int rank = 2 * tid + i;
      sh.ranked[rank] = mine[i];
      if (i ? stay1 : stay0) order[rank] = ~(static_cast<uint64_t>(item_index(sh.sorted[0][rank])) << 11 | static_cast<uint64_t>(rank));
    }
    __syncthreads();
    const int kept = static_cast<int>(sh.found[0]);
    const uint64_t total = sh.found[1];
    sort_down(order, kept);
#pragma unroll
    for (int i = 0; i < 2; ++i) mine[i] = 2 * tid + i < kept ? sh.ranked[~order[2 * tid + i] & (kSorted - 1)] : 0;
    const uint64_t run = group_prefix(mine[0] + mine[1], all, sh);
    const uint64_t beyond = draw_from(total);
    if (run <= beyond && run + mine[0] + mine[1] > beyond) {
      const int i = run + mine[0] > beyond ? 0 : 1;
      answer(static_cast<int>(~order[2 * tid + i] >> 11), mine[i], total);
    }
    return;
  }

  bool answers = helper == 0;  // or the last of the helpers to arrive
  uint32_t least = 1;
  int last = n;
  const int in_border = border < kBands ? sh.count[border] - (border > 0 ? sh.count[border - 1] : 0) : 0;
  if (!cut && in_border <= kItems) {
    bool done = true;
    int items = 0;
    if (border == kBands && helper > 0) return;
    if (border < kBands) {
      const int per = (n + 4 * p.helpers - 1) / (4 * p.helpers) * 4;
      gather_band(x, helper * per, min(n, helper * per + per), border, top_value, scale, sh);
      if (p.helpers > 1 && !join_items(p, row, sh)) return;
      answers = true;
      items = min(static_cast<int>(sh.n), kItems);
      __syncthreads();
      if (border == share_band) {
        // top-p's border: which of kThreads even parts of the band's keys, then the rank in it
        uint32_t low = 0xFFFFFFFFu, high = 0;
        for (int i = tid; i < items; i += kThreads) {
          low = min(low, item_key(sh.items[i]));
          high = max(high, item_key(sh.items[i]));
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
          low = min(low, static_cast<uint32_t>(__shfl_xor(low, off)));
          high = max(high, static_cast<uint32_t>(__shfl_xor(high, off)));
        }
        if (tid == 0) sh.low = 0xFFFFFFFFu, sh.high = 0;
        __syncthreads();
        if (lane == 0) {
          atomicMin(&sh.low, low);
          atomicMax(&sh.high, high);
        }
        __syncthreads();
        low = sh.low;
        high = sh.high;
        int step = 0;
        while ((high - low) >> step >= static_cast<uint32_t>(kThreads)) ++step;
        sh.parts[tid] = 0;
        if (tid == 0) sh.n = 0, sh.found[0] = ~uint64_t{0};
        __syncthreads();
        for (int i = tid; i < items; i += kThreads) {
          const uint32_t key = item_key(sh.items[i]);
          const uint64_t f = w.fixed(key);
          if (f) lds_add(&sh.parts[(high - key) >> step], f);
        }
        __syncthreads();
        const uint64_t target = target_of(sh.total) - sh.above;
        const uint64_t mine_part = sh.parts[tid];
        uint64_t all;
        const uint64_t before = group_prefix(mine_part, all, sh);
        if (before < target && before + mine_part >= target) {
          sh.found[0] = static_cast<uint64_t>(tid);
          sh.found[1] = before;
        }
        __syncthreads();
        const bool met = sh.found[0] != ~uint64_t{0};  // else (a rounding short of the band's sum): its last item
        const uint32_t part = met ? static_cast<uint32_t>(sh.found[0]) : (high - low) >> step;
        const uint64_t ahead = met ? sh.found[1] : all;
        for (int base = 0; base < items; base += kThreads) {
          const int i = base + tid;
          const bool in = i < items && (high - item_key(sh.items[i])) >> step == part;
          append(in, i < items ? sh.items[i] : 0, sh.part, &sh.n, kThreads);
        }
        __syncthreads();
        const int listed = static_cast<int>(sh.n);
        done = listed <= kThreads;
        if (listed <= 64) {  // one wave, an item a lane
          if (wave == 0) {
            const uint64_t item = lane < listed ? sh.part[lane] : 0;
            const uint64_t f = lane < listed ? w.fixed(item_key(item)) : 0;
            uint64_t run = ahead + f;  // up to and with the lane's, downwards
            for (int i = 0; i < listed; ++i) run += lane_value(item, i) > item ? lane_value(f, i) : 0;
            // the item where the target is met, else the last
            const uint64_t met_here = __ballot(lane < listed && run >= target && run - f < target);
            int rank = 0;
            for (int i = 0; i < listed; ++i) rank += lane_value(item, i) > item;
            const uint64_t final = __ballot(lane < listed && rank == listed - 1);
            if (lane == 0) sh.found[2] = static_cast<uint64_t>(__builtin_ctzll(met_here ? met_here : final));
          }
          __syncthreads();
        } else if (done) {
          sort_down(sh.part, listed);
          uint64_t mine[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) mine[i] = 2 * tid + i < listed ? w.fixed(item_key(sh.part[2 * tid + i])) : 0;
          const uint64_t run = ahead + group_prefix(mine[0] + mine[1], all, sh);
          if (tid == 0) sh.found[2] = static_cast<uint64_t>(listed - 1);
          __syncthreads();
          if (run < target && run + mine[0] + mine[1] >= target) sh.found[2] = static_cast<uint64_t>(2 * tid + (run + mine[0] < target));
          __syncthreads();
        }
        if (done) {
          const uint64_t item = sh.part[sh.found[2]];
          least = item_key(item);
          last = item_index(item);
          __syncthreads();
        }
      }
    }
    if (done) {
      for (int c = tid; c < p.chunks; c += kThreads) sh.sums[c] = 0;
      __syncthreads();
      const auto kept = [&](uint32_t key, int i) {
        return (key > least || (key == least && i <= last)) && key >= floor_key ? w.fixed(key) : 0;
      };
      // the kept sum of each chunk: its bands above the border, and its part of that
      for (int u = tid; u < units; u += kThreads) {
        const int c = u / (kBands / 8), j0 = u % (kBands / 8) * 8;
        if (sh.base[c] == kBands) continue;
        const int base = sh.base[c] + j0;
        if (min(base, kBands - 1) >= border) continue;
        uint64_t sums[8], sum = 0;
        chunk_sums(c, (unit0 + c) * kBands + j0, sums);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (min(base + j, kBands - 1) < border) sum += sums[j];
        if (sum) lds_add(&sh.sums[c], sum);
      }
      for (int i = tid; i < items; i += kThreads) {
        const uint64_t item = sh.items[i];
        const uint64_t f = kept(item_key(item), item_index(item));
        if (f) lds_add(&sh.sums[item_index(item) / p.chunk], f);
      }
      __syncthreads();
      // the chunk where the running sum passes the draw (two a thread), then the place in it
      const uint64_t s0 = 2 * tid < p.chunks ? sh.sums[2 * tid] : 0, s1 = 2 * tid + 1 < p.chunks ? sh.sums[2 * tid + 1] : 0;
      uint64_t total;
      uint64_t run = group_prefix(s0 + s1, total, sh);
      uint64_t beyond = draw_from(total);
      if (run <= beyond && run + s0 + s1 > beyond) {
        const bool second = run + s0 <= beyond;
        sh.found[0] = static_cast<uint64_t>(2 * tid + second);
        sh.found[1] = second ? run + s0 : run;
      }
      if (tid == 0) sh.found[2] = 0;
      __syncthreads();
      const int per = p.chunk / kThreads, at = static_cast<int>(sh.found[0]) * p.chunk + tid * per;
      beyond -= sh.found[1];
      f32x4 v[kMostChunk / kThreads / 4];
#pragma unroll
      for (int i = 0; i < kMostChunk / kThreads / 4; ++i) v[i] = load_logits(x, at + 4 * i, 4 * i < per ? n : 0);
      uint64_t mine[kMostChunk / kThreads], sum = 0;
#pragma unroll
      for (int i = 0; i < kMostChunk / kThreads; ++i) {
        mine[i] = i < per ? kept(rank_key(v[i / 4][i % 4]), at + i) : 0;
        sum += mine[i];
      }
      uint64_t all;
      run = group_prefix(sum, all, sh);
      // a chunk weighed by its own maximum may add up to a rounding less here:
      // then its last kept token (its largest, if all weights round to nothing)
      if (all == 0) {
        if (tid == 0) answer(static_cast<int>(heads[sh.found[0]].index), 0, total);
        return;
      }
      if (beyond >= all) beyond = all - 1;
      if (run <= beyond && run + sum > beyond) {
        int i = 0;
#pragma unroll
        for (int j = 0; j < kMostChunk / kThreads; ++j)
          if (run <= beyond) {
            run += mine[j];
            i = j;
          }
        answer(at + i, kept(rank_key(x[at + i]), at + i), total);
      }
      return;
    }
  }

  // digit by digit: up to eleven reads of the row, 25 us each (top-k 5000 of 151936: 168 us,
  // with top-p 312)
  if (!answers) return;
  // kept: keys above `least`, and of those equal to it the ones up to index
  // `last`
  uint64_t mine = 0, above, total;
  if (cut) {
    each_logit(x, n, [&](int, uint32_t key) { mine += key != 0; });
    if (group_sum(mine, sh) > static_cast<uint64_t>(k)) {
      least = descend(x, n, k, [](uint32_t key) { return key ? uint64_t{1} : 0; }, above, sh);
      last = walk(x, n, [&](uint64_t) { return k - above - 1; },
                  [=](uint32_t key, int) { return key == least ? uint64_t{1} : 0; }, total, sh);
    }
  }
  if (share < 1.0) {
    mine = 0;
    each_logit(x, n, [&](int i, uint32_t key) { mine += key > least || (key == least && i <= last) ? w.fixed(key) : 0; });
    const uint64_t target = target_of(group_sum(mine, sh));
    // equal keys beyond `last` weigh more than their share here; the search
    // then ends at `least` itself, and the count below is cut to `last`
    const uint32_t key = descend(x, n, target, [&](uint32_t q) { return q >= least ? w.fixed(q) : 0; }, above, sh);
    const uint64_t each = w.fixed(key), keep = (target - above + each - 1) / each;
    const int upto = walk(x, n, [&](uint64_t) { return keep - 1; },
                          [=](uint32_t q, int) { return q == key ? uint64_t{1} : 0; }, total, sh);
    if (key > least) {
      least = key;
      last = upto;
    } else {
      last = min(last, upto);
    }
  }
  const auto kept = [&](uint32_t key, int i) -> uint64_t {
    if (key < least || (key == least && i > last)) return 0;
    return key >= floor_key ? w.fixed(key) : 0;
  };
  const int index = walk(x, n, draw_from, kept, total, sh);
  if (tid == 0) answer(index, kept(rank_key(x[index]), index), total);
}

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Small problems in chunks of 2048 (one row of 151936: 75 workgroups instead
// of 19), large ones of 8192 (fewer bands and lists to write and add).
SamplePlan plan_sample(int64_t rows, int64_t vocabulary, void* workspace) {
  SamplePlan p{};
  const bool fine = rows * up(vocabulary, 8192) < 512 && vocabulary <= 2048 * kMostChunks;
  p.chunk = fine ? 2048 : 8192;
  p.chunks = static_cast<int32_t>(up(vocabulary, p.chunk));
  p.list = static_cast<int32_t>(vocabulary < kList ? vocabulary : kList);
  p.shift = kShift;
  while ((int64_t{1} << (62 - p.shift)) < vocabulary) --p.shift;
  const size_t units = static_cast<size_t>(rows) * p.chunks;
  char* at = static_cast<char*>(workspace);
  size_t bytes = 0;
  const auto take = [&](size_t size) {
    char* part = at ? at + bytes : nullptr;
    bytes += (size + 255) & ~size_t{255};
    return part;
  };
  // the counters first, whatever the batch: no call's lists lie where another's counters are
  p.gathered = reinterpret_cast<uint32_t*>(take(kHelped * 2 * sizeof(uint32_t)));
  // One compute unit reads a row of 151936 in 25 us, sixteen in 3: a row's draw
  // has as many workgroups as leave one a compute unit, 4096 logits each at least
  // (us, top-p 0.95 at temperature 1.3, with and without: one row 44 and 59; at
  // 64 rows 74 and 73; two or four times as many: 200 rows 142 and 146 against 121,
  // though with mixed filters, where most leave at once, 80 and 79 against 83).
  const int64_t share = vocabulary / 4096 < 256 / rows ? vocabulary / 4096 : 256 / rows;
  p.helpers = static_cast<int32_t>(share < 1 ? 1 : share < 16 ? share : 16);
  if (p.helpers > 1) p.items = reinterpret_cast<uint64_t*>(take(static_cast<size_t>(rows) * kItems * sizeof(uint64_t)));
  p.heads = reinterpret_cast<ChunkHead*>(take(units * sizeof(ChunkHead)));
  p.counts = reinterpret_cast<uint16_t*>(take(units * kBands * sizeof(uint16_t)));
  p.weights = reinterpret_cast<uint64_t*>(take(units * kBands * sizeof(uint64_t)));
  p.lists = reinterpret_cast<uint64_t*>(take(units * p.list * sizeof(uint64_t)));
  p.bytes = bytes;
  return p;
}

}  // namespace

size_t sample_workspace(int64_t rows, int64_t vocabulary) { return rows == 0 ? 0 : plan_sample(rows, vocabulary, nullptr).bytes; }

hipError_t launch_sample(const SampleArgs& a, void* workspace, hipStream_t stream) {
  const SamplePlan p = plan_sample(a.rows, a.vocabulary, workspace);
  const dim3 grid(static_cast<uint32_t>(p.chunks), static_cast<uint32_t>(a.rows));
  if (p.chunk == 2048)
    sample_scan_kernel<2><<<grid, kScanThreads, 0, stream>>>(a, p);
  else
    sample_scan_kernel<8><<<grid, kScanThreads, 0, stream>>>(a, p);
  const hipError_t error = hipGetLastError();
  if (error != hipSuccess) return error;
  sample_draw_kernel<<<dim3(static_cast<uint32_t>(a.rows), static_cast<uint32_t>(p.helpers)), kThreads, 0, stream>>>(a, p);
  note("sample_scan_kernel", static_cast<int64_t>(p.chunks) * a.rows, p.chunk);
  return hipGetLastError();
}

}  // namespace qk
