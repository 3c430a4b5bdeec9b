// The operators between the projections: arguments and launchers of the cache
// append (kv_append.hip), the paged attention (paged_attention*.hip) and the
// sampler (sample.hip). Shapes are validated by the C-ABI layer (serving.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "attention_plan.hpp"
#include "kv_index.hpp"
#include "qk_abi.h"

namespace qk {

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ void kv_fault(const KvArgs& a, uint32_t bit) {
  if (a.fault) atomicOr(a.fault, bit);
}

struct AppendArgs {
  KvArgs kv;
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
  int32_t pairs;      // tiles of a round of workgroups, one a compute unit, if sequences are taken by length; else 0
  uint32_t* arrived;  // [tiles x kv_heads], zero between calls
  float* sums;        // [tiles x kv_heads x splits x rows] (maximum, sum) pairs
  float* parts;       // [tiles x kv_heads x splits x rows x head_dim]
};

hipError_t launch_paged_attention(AttentionArgs a, const AttentionPlan& plan, int type, int head_dim, int q_type,
                                  void* workspace, hipStream_t stream);
hipError_t launch_attention_few(const AttentionArgs& a, int type, int head_dim, int q_type, hipStream_t stream);
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
