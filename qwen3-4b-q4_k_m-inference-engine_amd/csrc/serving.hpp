// The operators between the projections: arguments and launchers of the cache
// append (kv_append.hip), the paged attention (paged_attention*.hip) and the
// sampler (sample.hip). Shapes are validated by the C-ABI layer (serving.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "attention_plan.hpp"
#include "kv_index.hpp"
#include "qk_abi.h"
#include "weigh_plan.hpp"

namespace qk {

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ void kv_fault(const KvArgs& a, uint32_t bit) {
  if (a.fault) atomicOr(a.fault, bit);
}

struct AppendArgs {
  KvArgs kv;
  const int32_t* seen;  // tokens of each sequence for the angles' positions; nullptr: the contexts
  const float* q;
  const float* k;
  const float* v;
  int64_t q_stride, k_stride, v_stride;
  int32_t q_heads;
  void* q_out;
  const float* q_norm;
  const float* k_norm;
  float eps;
  double turns_log2;  // log2(base) * -2 / dims
  int32_t dims, interleaved;
};
hipError_t launch_kv_append(const AppendArgs& a, int type, int head_dim, int q_type, hipStream_t stream);

struct RowsArgs {
  KvArgs kv;
  void* k_out;  // either may be nullptr
  void* v_out;
};
hipError_t launch_kv_rows(const RowsArgs& a, int type, int head_dim, int out_type, hipStream_t stream);

struct WeighArgs {
  KvArgs kv;
  const int32_t* seen;  // tokens of each sequence, for the new ones' positions; nullptr: the contexts
  const void* q;
  int64_t q_stride;
  int32_t q_heads, group;
  float scale;
  const float* lse;
  float* weight;      // [pages x kv_heads x page_size], as position
  int32_t* position;
  // the plan's part (launch_kv_weigh)
  int32_t key_parts, part_keys, row_parts, most_keys;
  float* parts;
};
hipError_t launch_kv_weigh(WeighArgs a, const WeighPlan& plan, int type, int head_dim, int q_type, void* workspace,
                           hipStream_t stream);

struct EvictArgs {
  KvArgs kv;  // token_start is not looked at
  const int32_t* seen;
  const int32_t* keep;
  const int32_t* recent;
  float* weight;
  int32_t* position;
  int32_t* context_out;
  int32_t width;  // the longest context that the workspace has room for
  // launch_kv_evict's part
  uint32_t* moves;  // [sequences x kv_heads]
  uint32_t* ranks;  // [sequences x kv_heads x width, up to a multiple of 4]
  int32_t* lists;   // [sequences x kv_heads x 2 x half of width]: places, then sources
  int32_t move_parts, unit_values, unit_bytes;
};
hipError_t launch_kv_evict(EvictArgs a, int type, int head_dim, void* workspace, hipStream_t stream);
size_t evict_workspace(int64_t sequences, int64_t kv_heads, int64_t width);

hipError_t launch_kv_fault_clear(uint32_t* word, uint32_t bits, hipStream_t stream);

struct AttentionArgs {
  KvArgs kv;
  const void* q;
  int64_t q_stride;
  int32_t q_heads, group;
  float scale;
  int32_t window;  // 0: none
  void* out;
  float* lse;
  // the plan's part (launch_paged_attention)
  int32_t tiles, splits, fill;
  PageDivision pages;
  int32_t pairs;      // tiles of a round of workgroups, one a compute unit, if sequences are taken by length; else 0
  uint32_t* arrived;  // [tiles x kv_heads], zero between calls
  float* sums;        // [tiles x kv_heads x splits x rows] (maximum, sum) pairs
  float* parts;       // [tiles x kv_heads x splits x rows x head_dim]
};

hipError_t launch_paged_attention(AttentionArgs a, const AttentionPlan& plan, int type, int head_dim, int q_type,
                                  void* workspace, hipStream_t stream);
hipError_t launch_attention_few(const AttentionArgs& a, int type, int head_dim, int q_type, hipStream_t stream);
hipError_t launch_attention_few_q4(const AttentionArgs& a, int tile_rows, int head_dim, int q_type, hipStream_t stream);
hipError_t launch_attention_many(const AttentionArgs& a, int key_groups, int type, int head_dim, int q_type, hipStream_t stream);

struct SampleArgs {
  const float* logits;
  int64_t row_stride;
  int32_t rows, vocabulary;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniform;
  uint32_t* token;
  float* probability;
};
hipError_t launch_sample(const SampleArgs& a, void* workspace, hipStream_t stream);
size_t sample_workspace(int64_t rows, int64_t vocabulary);

}  // namespace qk
