// Sequences cut to a budget, in place: of each key/value head the tokens that stay are
// the latest ones and the ones with the most weight, and those of them that lie past the
// budget move into the places that the others leave before it. Attention does not ask
// for an order of keys that were rotated when they were stored.
//
// Launches: every token's rank as 32 bits; of each (sequence, head) the rank that
// the budget ends at, by a search digit by digit in one workgroup, and the list of
// moves, in the order of the slots; the moves. Sources lie past the budget and
// places before it, so moves do not meet. The search bounds it, which one compute unit
// does for each head: loads of ranks and dependent steps through LDS counters, of which
// there are copies, since the ranks of like weights fall together. 32 sequences of up to 2304
// cut to 2048: ranks 6 us, search 18, moves 8 (8 heads of 128, F16); one of 65536 cut to
// 8192 in Q4_1: 8, 54 and 9.
#include "q4_1.hpp"
#include "qk_device.hpp"
#include "qk_launch.hpp"
#include "serving.hpp"

namespace qk {
namespace {

constexpr int kRankKeys = 1024;  // slots of a workgroup that ranks
constexpr int kThreads = 1024, kWaves = kThreads / 64, kAhead = 4;  // of one that selects; loads of four ranks in flight
constexpr int kBits = 11, kBins = 1 << kBits, kCopies = 4;  // of a digit; copies of the counts, against collisions
constexpr uint32_t kLatest = 0xFFFFFFFFu;

// Ranks of a (sequence, head) begin at 16 bytes each.
__host__ __device__ constexpr int64_t rank_stride(int64_t width) { return (width + 3) & ~int64_t{3}; }

// A sequence's context and budget, or a budget of all where nothing is to be done.
struct Cut {
  int context, keep;
  bool fault, beyond;
};
__device__ __forceinline__ Cut cut_of(const EvictArgs& a, int s) {
  const int context = a.kv.context[s], keep = a.keep[s];
  Cut c;
  c.fault = context < 0 || context > a.width;
  c.beyond = context > static_cast<int64_t>(a.kv.table_pages) * a.kv.page_size;
  c.context = c.fault || c.beyond ? 0 : context;
  c.keep = keep > 0 && keep < c.context ? keep : c.context;
  return c;
}

// Larger is more wanted: the latest tokens, then the weights in their order (both zeros
// alike), NaN last.
__device__ __forceinline__ uint32_t rank_of(float weight, bool latest) {
  if (latest) return kLatest;
  const uint32_t bits = __builtin_bit_cast(uint32_t, weight + 0.0f);
  return weight != weight ? 0u : bits >> 31 ? ~bits : bits | 0x80000000u;
}

__global__ __launch_bounds__(256) void kv_evict_rank_kernel(const EvictArgs a) {
  const int parts = (a.width + kRankKeys - 1) / kRankKeys;
  const int part = static_cast<int>(blockIdx.x) % parts, unit = static_cast<int>(blockIdx.x) / parts;
  const int s = unit / a.kv.kv_heads, head = unit % a.kv.kv_heads;
  const Cut c = cut_of(a, s);
  if (c.keep == c.context) return;
  const int64_t seen = a.seen ? a.seen[s] : c.context, from = seen - (a.recent[s] > 0 ? a.recent[s] : 0);
  uint32_t* ranks = a.ranks + static_cast<int64_t>(unit) * rank_stride(a.width);
  for (int slot = part * kRankKeys + static_cast<int>(threadIdx.x); slot < min(c.context, (part + 1) * kRankKeys); slot += 256) {
    const int entry = slot / a.kv.page_size, page = kv_page(a.kv, s, entry);
    uint32_t rank = 0;
    if (page >= 0) {
      const int64_t at = (static_cast<int64_t>(page) * a.kv.kv_heads + head) * a.kv.page_size + slot - entry * a.kv.page_size;
      rank = rank_of(a.weight[at], a.position[at] >= from);
    }
    ranks[slot] = rank;
  }
}

// Sums over the workgroup's threads before the calling one, and of all.
__device__ __forceinline__ int before_mine(int mine, int (&waves)[kWaves], int& all) {
  const int lane = static_cast<int>(threadIdx.x & 63), wave = static_cast<int>(threadIdx.x >> 6);
  int run = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int other = __shfl_up(run, off);
    if (lane >= off) run += other;
  }
  __syncthreads();  // of the call before
  if (lane == 63) waves[wave] = run;
  __syncthreads();
  int before = 0, total = 0;
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? waves[w] : 0;
    total += waves[w];
  }
  all = total;
  return before + run - mine;
}

// The same of a number a wave, for all of its lanes.
__device__ __forceinline__ int before_wave(int mine, int (&waves)[kWaves], int& all) {
  const int wave = static_cast<int>(threadIdx.x >> 6);
  __syncthreads();  // of the call before
  if ((threadIdx.x & 63) == 0) waves[wave] = mine;
  __syncthreads();
  int before = 0;
  all = 0;
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? waves[w] : 0;
    all += waves[w];
  }
  return before;
}

__global__ __launch_bounds__(kThreads) void kv_evict_select_kernel(const EvictArgs a) {
  __shared__ uint32_t counts[kCopies][kBins];
  __shared__ int waves[kWaves];
  __shared__ uint32_t digit_found, above_found, alike_found;
  const int tid = static_cast<int>(threadIdx.x);
  const int unit = static_cast<int>(blockIdx.x), s = unit / a.kv.kv_heads, head = unit % a.kv.kv_heads;
  const Cut c = cut_of(a, s);
  if (tid == 0 && head == 0) {
    if (c.fault) kv_fault(a.kv, QK_KV_FAULT_LENGTH);
    if (c.beyond) kv_fault(a.kv, QK_KV_FAULT_PAGE);
  }
  // a page that is none: the sequence stays as it is
  int bad = 0;
  if (c.keep < c.context)
    for (int e = tid; e <= (c.context - 1) / a.kv.page_size; e += kThreads) bad |= kv_page(a.kv, s, e) < 0;
  bad = __syncthreads_or(bad);
  if (tid == 0) {
    if (bad) kv_fault(a.kv, QK_KV_FAULT_PAGE);
    if (head == 0) a.context_out[s] = bad || c.fault || c.beyond ? a.kv.context[s] : c.keep;
    a.moves[unit] = 0;
  }
  if (bad || c.keep == c.context) return;
  const uint32_t* ranks = a.ranks + static_cast<int64_t>(unit) * rank_stride(a.width);

  const int last_four = (c.context - 1) & ~3;  // what four loads past the end take instead

  // the rank that the keep-th stands at, digit by digit; `wanted` of those that share the digits so far
  uint32_t prefix = 0;
  int wanted = c.keep, shift = 32;
  while (shift > 0) {
    const int bits = shift > kBits ? kBits : shift;
    shift -= bits;
    for (int i = tid; i < kCopies * kBins; i += kThreads) (&counts[0][0])[i] = 0;
    __syncthreads();
    for (int base = 4 * tid; base < c.context; base += 4 * kAhead * kThreads) {
      u32x4 rank[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) rank[k] = load16(ranks + min(base + 4 * k * kThreads, last_four));
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (base + 4 * k * kThreads + j < c.context && (shift + bits == 32 || rank[k][j] >> (shift + bits) == prefix))
            atomicAdd(&counts[tid >> 6 & (kCopies - 1)][rank[k][j] >> shift & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    // bins from the highest down, two a thread
    const int high = kBins - 1 - 2 * tid;
    uint32_t of[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < kCopies; ++k) {
      of[0] += counts[k][high];
      of[1] += counts[k][high - 1];
    }
    int all;
    const int before = before_mine(static_cast<int>(of[0] + of[1]), waves, all);
    int above = before;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int here = static_cast<int>(of[k]);
      if (above < wanted && above + here >= wanted) {
        digit_found = static_cast<uint32_t>(high - k);
        above_found = static_cast<uint32_t>(above);
        alike_found = static_cast<uint32_t>(here);
      }
      above += here;
    }
    __syncthreads();
    prefix = prefix << bits | digit_found;
    wanted -= static_cast<int>(above_found);
  }

  // Slots in runs, one a wave, four a lane at a time: those that stay and lie past the
  // budget, and the places that others leave before it, numbered in the order of the
  // slots. Of slots with that last rank the first `wanted` stay.
  constexpr int kTurn = 4 * 64;
  const int lane = tid & 63, run = (c.context + kTurn * kWaves - 1) / (kTurn * kWaves) * kTurn;
  const int lo = (tid >> 6) * run, hi = min(lo + run, c.context);
  const auto walk = [&](auto&& at) {
    for (int base = lo + 4 * lane; base - 4 * lane < hi; base += kTurn * kAhead) {
      u32x4 rank[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) rank[k] = load16(ranks + min(base + kTurn * k, last_four));
#pragma unroll
      for (int k = 0; k < kAhead; ++k) at(base + kTurn * k, rank[k]);
    }
  };
  const uint64_t lower = (uint64_t{1} << lane) - 1;
  // of four flags a lane: how many in the lanes before this one, and in all
  const auto count = [&](const bool (&flag)[4], int& in_all) {
    int before = 0;
    in_all = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t lanes = __ballot(flag[j]);
      before += __builtin_popcountll(lanes & lower);
      in_all += __builtin_popcountll(lanes);
    }
    return before;
  };
  int all, ties_before = 0;
  const bool in_order = static_cast<int>(alike_found) > wanted;
  if (in_order) {
    int ties = 0;
    walk([&](int at, const u32x4& rank) {
      bool alike[4];
      int in_all;
#pragma unroll
      for (int j = 0; j < 4; ++j) alike[j] = at + j < hi && rank[j] == prefix;
      count(alike, in_all);
      ties += in_all;
    });
    ties_before = before_wave(ties, waves, all);
  }
  int tie = ties_before;
  const auto staying = [&](int at, const u32x4& rank, bool (&stays)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) stays[j] = at + j < hi && rank[j] >= prefix;
    if (!in_order) return;
    bool alike[4];
    int in_all;
#pragma unroll
    for (int j = 0; j < 4; ++j) alike[j] = at + j < hi && rank[j] == prefix;
    int before = tie + count(alike, in_all);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      stays[j] &= !alike[j] || before < wanted;
      before += alike[j];
    }
    tie += in_all;
  };
  const auto moving = [&](int at, const u32x4& rank, bool (&leaves)[4], bool (&moves)[4]) {
    bool stays[4];
    staying(at, rank, stays);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      leaves[j] = at + j < hi && !stays[j] && at + j < c.keep;
      moves[j] = stays[j] && at + j >= c.keep;
    }
  };
  int free_places = 0, sources = 0;
  walk([&](int at, const u32x4& rank) {
    bool leaves[4], moves[4];
    int in_all;
    moving(at, rank, leaves, moves);
    count(leaves, in_all);
    free_places += in_all;
    count(moves, in_all);
    sources += in_all;
  });
  int place_at = before_wave(free_places, waves, all), source_at = before_wave(sources, waves, all);
  const int most = (a.width + 1) / 2;
  int32_t* const places = a.lists + static_cast<int64_t>(unit) * 2 * most;
  tie = ties_before;
  walk([&](int at, const u32x4& rank) {
    bool leaves[4], moves[4];
    int places_here, sources_here;
    moving(at, rank, leaves, moves);
    int place = place_at + count(leaves, places_here), source = source_at + count(moves, sources_here);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (leaves[j]) places[place++] = at + j;
      if (moves[j]) places[most + source++] = at + j;
    }
    place_at += places_here;
    source_at += sources_here;
  });
  if (tid == 0) a.moves[unit] = static_cast<uint32_t>(all);
}

// Rows of BYTES a lane and LANES lanes, aligned to 4 bytes.
template <int BYTES, int LANES>
__global__ __launch_bounds__(256) void kv_evict_move_kernel(const EvictArgs a) {
  constexpr int kRows = 256 / LANES;
  typedef uint32_t Piece __attribute__((ext_vector_type(BYTES / 4)));
  typedef Piece Piece_a4 __attribute__((aligned(4)));
  const int tid = static_cast<int>(threadIdx.x), lane = tid % LANES, row = tid / LANES;
  const int unit = static_cast<int>(blockIdx.x) % (a.kv.sequences * a.kv.kv_heads);
  const int part = static_cast<int>(blockIdx.x) / (a.kv.sequences * a.kv.kv_heads);
  const int s = unit / a.kv.kv_heads, head = unit % a.kv.kv_heads, moves = static_cast<int>(a.moves[unit]);
  if (row >= kRows) return;
  const int most = (a.width + 1) / 2;
  const int32_t* const places = a.lists + static_cast<int64_t>(unit) * 2 * most;
  const auto find = [&](int slot, int64_t& row_at, int64_t& weight_at) {
    const int entry = slot / a.kv.page_size, in = slot - entry * a.kv.page_size, page = kv_page(a.kv, s, entry);
    row_at = kv_place(a.kv, page, in, head) * a.unit_bytes / a.unit_values;
    weight_at = (static_cast<int64_t>(page) * a.kv.kv_heads + head) * a.kv.page_size + in;
  };
  for (int i = part * kRows + row; i < moves; i += a.move_parts * kRows) {
    int64_t to, from, weight_to, weight_from;
    find(places[i], to, weight_to);
    find(places[most + i], from, weight_from);
    uint8_t* const k = reinterpret_cast<uint8_t*>(a.kv.k) + lane * BYTES;
    uint8_t* const v = reinterpret_cast<uint8_t*>(a.kv.v) + lane * BYTES;
    const Piece k_piece = *reinterpret_cast<const Piece_a4*>(k + from), v_piece = *reinterpret_cast<const Piece_a4*>(v + from);
    *reinterpret_cast<Piece_a4*>(k + to) = k_piece;
    *reinterpret_cast<Piece_a4*>(v + to) = v_piece;
    if (lane == 0) {
      const float weight = a.weight[weight_from];
      const int32_t position = a.position[weight_from];
      a.weight[weight_to] = weight;
      a.position[weight_to] = position;
    }
  }
}

}  // namespace

size_t evict_workspace(int64_t sequences, int64_t kv_heads, int64_t width) {
  const int64_t units = sequences * kv_heads;
  return static_cast<size_t>(((units * 4 + 255) & ~int64_t{255}) + units * rank_stride(width) * 4 + units * 2 * ((width + 1) / 2) * 4);
}

hipError_t launch_kv_evict(EvictArgs a, int type, int head_dim, void* workspace, hipStream_t stream) {
  const int64_t units = static_cast<int64_t>(a.kv.sequences) * a.kv.kv_heads;
  char* ws = static_cast<char*>(workspace);
  a.moves = reinterpret_cast<uint32_t*>(ws);
  a.ranks = reinterpret_cast<uint32_t*>(ws + ((units * 4 + 255) & ~int64_t{255}));
  a.lists = reinterpret_cast<int32_t*>(a.ranks + units * rank_stride(a.width));
  const bool q4 = type == QK_TYPE_Q4_1;
  a.unit_values = q4 ? kQ4Values : 1;
  a.unit_bytes = q4 ? kQ4Bytes : 2;
  const uint32_t ranking = static_cast<uint32_t>(units * ((a.width + kRankKeys - 1) / kRankKeys));
  kv_evict_rank_kernel<<<ranking, 256, 0, stream>>>(a);
  hipError_t error = hipGetLastError();
  if (error != hipSuccess) return error;
  kv_evict_select_kernel<<<static_cast<uint32_t>(units), kThreads, 0, stream>>>(a);
  error = hipGetLastError();
  if (error != hipSuccess) return error;
  const auto move = [&](auto kernel, int rows) {
    // a few workgroups for each compute unit; no more than half of the tokens move
    int64_t parts = (2048 + units - 1) / units;
    const int64_t most = ((a.width + 1) / 2 + rows - 1) / rows;
    a.move_parts = static_cast<int32_t>(parts < most ? parts : most);
    kernel<<<static_cast<uint32_t>(units * a.move_parts), 256, 0, stream>>>(a);
    note("kv_evict_move_kernel", units * a.move_parts, head_dim, type);
  };
  if (q4)
    head_dim == 128 ? move(kv_evict_move_kernel<16, 5>, 256 / 5) : move(kv_evict_move_kernel<8, 5>, 256 / 5);
  else
    head_dim == 128 ? move(kv_evict_move_kernel<16, 16>, 16) : move(kv_evict_move_kernel<16, 8>, 32);
  return hipGetLastError();
}

}  // namespace qk
