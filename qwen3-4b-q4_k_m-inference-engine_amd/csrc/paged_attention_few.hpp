// What the attention kernels for few rows a sequence share: which tile of R rows a
// workgroup takes.
#pragma once

#include "paged_attention.hpp"

namespace qk {

constexpr int kBlock = 32;  // keys of a block

// In LDS beside a kernel's own.
struct FewShared {
  __attribute__((aligned(16))) int32_t keys[kOrdered];
  int32_t chosen;
  uint32_t bad, arrived;
};

// Tiles by the length of their sequences' contexts, where no sequence has more
// than one (false otherwise): the `pairs` longest in the first round of
// workgroups, one a compute unit, the next ones in the second, which the card
// places on the same units in the same order, from the shortest up; then the
// rest. Each unit's two contexts so have about the same length together: 64
// sequences of up to 8192 keys, uneven, 225 us as they come, 175 paired. Every
// workgroup ranks the lengths itself, a thread a sequence.
template <int R>
__device__ __forceinline__ bool find_by_length(const AttentionArgs& a, int tile, bool report, FewShared& sh,
                                               AttentionTile& t) {
  const int s = static_cast<int>(threadIdx.x);
  int mine = -1;
  bool single = true;
  if (s < a.kv.sequences) {
    const KvSequence q = kv_sequence(a.kv, s);
    if (report && q.fault) kv_fault(a.kv, QK_KV_FAULT_LENGTH);
    single = q.count * a.group <= R;
    if (q.count > 0) {
      mine = kv_keys(q);
      mine = a.window > 0 && mine > a.window ? a.window : mine;
    }
  }
  if (s < kOrdered) sh.keys[s] = mine;
  if (s == 0) sh.chosen = -1;
  const int tiles = __syncthreads_count(mine >= 0);
  if (!__syncthreads_and(single)) return false;
  int rank = 0;
  for (int i = 0; i < a.kv.sequences; i += 4) {
    const i32x4 other = *reinterpret_cast<const i32x4*>(&sh.keys[i]);
#pragma unroll
    for (int e = 0; e < 4; ++e) rank += other[e] > mine || (other[e] == mine && i + e < s);
  }
  const int second = 2 * a.pairs < tiles ? 2 * a.pairs : tiles;
  const int wanted = tile < a.pairs || tile >= second ? tile : second - 1 - (tile - a.pairs);
  if (mine >= 0 && rank == wanted) sh.chosen = s;
  __syncthreads();
  t.s = __builtin_amdgcn_readfirstlane(sh.chosen);
  if (t.s < 0) return true;
  const KvSequence q = kv_sequence(a.kv, t.s);
  t.row = q.row;
  t.count = q.count;
  t.first = q.first;
  t.beyond = q.beyond;
  t.begin = 0;
  tile_keys(a.group, a.window, R, t);
  return true;
}

// The tile of this workgroup (uniform); its s is -1 if it has none.
template <int R>
__device__ __forceinline__ AttentionTile few_tile(const AttentionArgs& a, int tile, FewShared& sh) {
  const bool report = blockIdx.x == 0;
  AttentionTile t;
  if (a.pairs == 0 || !find_by_length<R>(a, tile, report, sh, t)) t = find_tile(a, tile, R, report);
  return t;
}

}  // namespace qk
