// The launch of a paged attention call as its plan says.
#include "paged_attention.hpp"

namespace qk {

hipError_t launch_paged_attention(AttentionArgs a, const AttentionPlan& plan, int type, int head_dim, int q_type,
                                  void* workspace, hipStream_t stream) {
  a.tiles = plan.tiles;
  a.splits = plan.splits;
  a.fill = plan.fill;
  a.pairs = plan.pairs;
  a.pages = page_division(a.kv.page_size);
  char* ws = static_cast<char*>(workspace);
  a.arrived = reinterpret_cast<uint32_t*>(ws);
  a.sums = reinterpret_cast<float*>(ws + plan.sums_at);
  a.parts = reinterpret_cast<float*>(ws + plan.parts_at);
  if (plan.few && type == QK_TYPE_Q4_1) return launch_attention_few_q4(a, plan.rows, head_dim, q_type, stream);
  return plan.few ? launch_attention_few(a, type, head_dim, q_type, stream)
                  : launch_attention_many(a, plan.key_groups, type, head_dim, q_type, stream);
}

}  // namespace qk
