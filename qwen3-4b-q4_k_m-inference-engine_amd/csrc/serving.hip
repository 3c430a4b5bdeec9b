// C-ABI entry points of the cache append, the paged attention and the sampler:
// arguments are checked here, on the host, before any HIP call; what only the
// device can see (page ids, lengths) the kernels check.
#include "serving.hpp"

#include <cmath>

#include "q4_1.hpp"
#include "qk_launch.hpp"

namespace {

using qk::KvArgs;

int refuse(const char* message, int code = QK_ERR_INVALID_ARGUMENT) {
  return qk::set_error(code, message, hipSuccess);
}
int finish(hipError_t error, const char* message) {
  return error == hipSuccess ? QK_OK : qk::set_error(QK_ERR_RUNTIME, message, error);
}
bool misaligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }
hipStream_t as_stream(qk_stream_t s) { return static_cast<hipStream_t>(s); }

// Lengths and strides of a cache and a batch (pointers: check_pointers).
int check_shapes(const qk_kv_cache* c, const qk_kv_batch* b) {
  if (!c || !b) return refuse("cache and batch must be non-null");
  if (c->type != QK_TYPE_F16 && c->type != QK_TYPE_BF16 && c->type != QK_TYPE_Q4_1)
    return refuse("caches are F16, BF16 or Q4_1", QK_ERR_UNSUPPORTED_TYPE);
  if (c->head_dim != 64 && c->head_dim != 128) return refuse("cache head_dim must be 64 or 128");
  if (c->pages < 1 || c->pages > INT32_MAX || c->page_size < 1 || c->page_size > 65536)
    return refuse("cache needs 1 .. 2^31-1 pages of 1 .. 65536 tokens");
  if (c->kv_heads < 1 || c->kv_heads > 4096) return refuse("cache needs 1 .. 4096 heads");
  const int64_t most = int64_t{1} << 30;
  const int64_t unit = c->type == QK_TYPE_Q4_1 ? qk::kQ4Values : 8;
  if (c->token_stride % unit != 0 || c->head_stride % unit != 0 || c->page_stride % unit != 0)
    return refuse("cache strides must be multiples of 8 elements, of a Q4_1 cache of 32");
  if (c->token_stride < c->head_dim || c->head_stride < c->head_dim || c->token_stride > most || c->head_stride > most ||
      c->page_stride < 0 || c->page_stride > (int64_t{1} << 40))
    return refuse("cache strides must hold a head's values and stay below 2^30 elements (pages: 2^40)");
  if (b->sequences < 0 || b->sequences > 65535 || b->tokens < 0 || b->tokens >= (int64_t{1} << 24))
    return refuse("batch needs 0 .. 65535 sequences and 0 .. 2^24 - 1 tokens");
  if (b->table_stride < 1) return refuse("batch table_stride must be positive");
  return QK_OK;
}

int check_pointers(const qk_kv_cache* c, const qk_kv_batch* b) {
  if (!c->k || !c->v || !b->token_start || !b->context || !b->page_table)
    return refuse("cache and batch pointers must be non-null");
  if (misaligned(c->k, 16) || misaligned(c->v, 16)) return refuse("cache arrays must be 16-byte aligned");
  if (misaligned(b->token_start, 4) || misaligned(b->context, 4) || misaligned(b->page_table, 4) || misaligned(c->fault, 4))
    return refuse("batch arrays must be 4-byte aligned");
  return QK_OK;
}

// The 16-bit type that a cache's rows are read as.
int value_type(const qk_kv_cache* c) { return c->type == QK_TYPE_Q4_1 ? QK_TYPE_F16 : c->type; }

// q heads against the cache's, and q's type.
int check_heads(const qk_kv_cache* c, const qk_kv_batch* b, int64_t q_heads, int q_type) {
  if (q_type != QK_TYPE_F32 && q_type != value_type(c))
    return refuse("q must be F32 or of the cache's type (F16 for Q4_1)", QK_ERR_UNSUPPORTED_TYPE);
  if (q_heads < 1 || q_heads > 4096 || q_heads % c->kv_heads != 0)
    return refuse("q_heads must be a multiple of the cache's heads, at most 4096");
  if (b->tokens * q_heads > (int64_t{1} << 28)) return refuse("tokens x q_heads must stay within 2^28");
  return QK_OK;
}

int check_weights(const qk_kv_weights* w) {
  if (!w || !w->weight || !w->position) return refuse("weights must be non-null");
  if (misaligned(w->weight, 4) || misaligned(w->position, 4)) return refuse("weights must be 4-byte aligned");
  return QK_OK;
}

int check_workspace(const void* workspace, size_t bytes, size_t need) {
  if (need != 0 && !workspace) return refuse("workspace must be non-null");
  if (bytes < need) return refuse("workspace too small");
  if (misaligned(workspace, 256)) return refuse("workspace must be 256-byte aligned");
  return QK_OK;
}

// Whether `n` and `m` 32-bit entries from a and b on share any.
bool overlap(const int32_t* a, uint64_t n, const int32_t* b, uint64_t m) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && (x < y ? y - x < 4 * n : x - y < 4 * m);
}

// Slots that a list and a grid hold.
bool evict_fits(const qk_kv_cache* c, const qk_kv_batch* b, int64_t max_context) {
  const int64_t units = b->sequences * c->kv_heads;
  return max_context <= qk::kMostPositions && units <= (int64_t{1} << 21) && units * max_context <= (int64_t{1} << 32);
}

KvArgs kv_args(const qk_kv_cache* c, const qk_kv_batch* b) {
  KvArgs a;
  a.k = static_cast<uint16_t*>(c->k);
  a.v = static_cast<uint16_t*>(c->v);
  a.page_stride = c->page_stride;
  a.token_stride = static_cast<int32_t>(c->token_stride);
  a.head_stride = static_cast<int32_t>(c->head_stride);
  a.pages = static_cast<int32_t>(c->pages);
  a.page_size = static_cast<int32_t>(c->page_size);
  a.kv_heads = static_cast<int32_t>(c->kv_heads);
  a.sequences = static_cast<int32_t>(b->sequences);
  a.tokens = static_cast<int32_t>(b->tokens);
  a.table_pages = static_cast<int32_t>(b->table_stride < INT32_MAX ? b->table_stride : INT32_MAX);
  a.table_stride = b->table_stride;
  a.token_start = b->token_start;
  a.context = b->context;
  a.page_table = b->page_table;
  a.fault = c->fault;
  return a;
}

}  // namespace

extern "C" {

int qk_kv_append(const qk_kv_cache* cache, const qk_kv_batch* batch, const float* q, int64_t q_stride, const float* k,
                 int64_t k_stride, const float* v, int64_t v_stride, int64_t q_heads, const qk_rope* rope, void* q_out,
                 int q_type, qk_stream_t stream) {
  return qk_kv_append_at(cache, batch, nullptr, q, q_stride, k, k_stride, v, v_stride, q_heads, rope, q_out, q_type, stream);
}

int qk_kv_append_at(const qk_kv_cache* cache, const qk_kv_batch* batch, const int32_t* seen, const float* q,
                    int64_t q_stride, const float* k, int64_t k_stride, const float* v, int64_t v_stride,
                    int64_t q_heads, const qk_rope* rope, void* q_out, int q_type, qk_stream_t stream) {
  int status = check_shapes(cache, batch);
  if (status != QK_OK) return status;
  if (q_heads != 0) status = check_heads(cache, batch, q_heads, q_type);
  if (status != QK_OK) return status;
  if (rope) {
    if (rope->dims < 0 || rope->dims > cache->head_dim || rope->dims % 8 != 0)
      return refuse("rope dims must be a multiple of 8, at most head_dim");
    if (rope->dims > 0 && (!(rope->base > 0.0f) || !std::isfinite(rope->base)))
      return refuse("rope base must be positive and finite");
    if ((rope->q_norm || rope->k_norm) && !(rope->eps > 0.0f)) return refuse("head norms need a positive epsilon");
  }
  if (batch->tokens == 0 || batch->sequences == 0) return QK_OK;
  const int64_t kv_width = cache->kv_heads * cache->head_dim, most = int64_t{1} << 40;
  if (k_stride < kv_width || v_stride < kv_width || k_stride > most || v_stride > most ||
      (q_heads != 0 && (q_stride < q_heads * cache->head_dim || q_stride > most)))
    return refuse("q, k and v strides must hold a token's heads");
  status = check_pointers(cache, batch);
  if (status != QK_OK) return status;
  if (misaligned(seen, 4)) return refuse("batch arrays must be 4-byte aligned");
  if (!k || !v || (q_heads != 0 && (!q || !q_out))) return refuse("append pointers must be non-null");
  if (misaligned(q, 4) || misaligned(k, 4) || misaligned(v, 4) || (q_heads != 0 && misaligned(q_out, 16)))
    return refuse("append inputs must be 4-byte, q_out 16-byte aligned");
  if (rope && (misaligned(rope->q_norm, 4) || misaligned(rope->k_norm, 4)))
    return refuse("append inputs must be 4-byte, q_out 16-byte aligned");
  if (q_heads != 0 && q_out == static_cast<const void*>(q) &&
      (q_type != QK_TYPE_F32 || q_stride != q_heads * cache->head_dim))
    return refuse("q_out may be q only for F32 rows without gaps");
  qk::AppendArgs a{};
  a.kv = kv_args(cache, batch);
  a.seen = seen;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.q_heads = static_cast<int32_t>(q_heads);
  a.q_out = q_out;
  if (rope) {
    a.q_norm = rope->q_norm;
    a.k_norm = rope->k_norm;
    a.eps = rope->eps;
    a.dims = static_cast<int32_t>(rope->dims);
    a.interleaved = rope->interleaved != 0;
    if (a.dims > 0) a.turns_log2 = std::log2(static_cast<double>(rope->base)) * -2.0 / a.dims;
  }
  return finish(qk::launch_kv_append(a, cache->type, static_cast<int>(cache->head_dim), q_type, as_stream(stream)),
                "cache append launch failed");
}

size_t qk_paged_attention_workspace_size(const qk_kv_cache* cache, const qk_kv_batch* batch, int q_type,
                                         int64_t q_heads, int64_t window, int64_t max_context) {
  if (check_shapes(cache, batch) != QK_OK || check_heads(cache, batch, q_heads, q_type) != QK_OK || window < 0 ||
      max_context < 0)
    return 0;
  const qk::AttentionPlan plan =
      qk::plan_attention(batch->tokens, batch->sequences, q_heads, cache->kv_heads, static_cast<int>(cache->head_dim),
                         cache->type, q_type, window, max_context);
  return qk::plan_fits(plan, cache->kv_heads, cache->type, q_type) ? plan.bytes : 0;
}

int qk_paged_attention(const qk_kv_cache* cache, const qk_kv_batch* batch, const void* q, int q_type, int64_t q_stride,
                       int64_t q_heads, float scale, int64_t window, int64_t max_context, void* out, float* lse,
                       void* workspace, size_t workspace_bytes, qk_stream_t stream) {
  int status = check_shapes(cache, batch);
  if (status == QK_OK) status = check_heads(cache, batch, q_heads, q_type);
  if (status != QK_OK) return status;
  if (window < 0 || max_context < 0) return refuse("attention window and max_context must not be negative");
  if (!std::isfinite(scale)) return refuse("attention scale must be finite");
  if (batch->tokens == 0 || batch->sequences == 0) return QK_OK;
  if (q_stride < q_heads * cache->head_dim || q_stride > (int64_t{1} << 40))
    return refuse("attention q_stride must hold a token's heads");
  if (q_stride % (q_type == QK_TYPE_F32 ? 4 : 8) != 0) return refuse("attention q rows must be 16-byte aligned");
  status = check_pointers(cache, batch);
  if (status != QK_OK) return status;
  if (!q || !out) return refuse("attention pointers must be non-null");
  if (misaligned(q, 16) || misaligned(out, 16) || misaligned(lse, 4))
    return refuse("attention q and out must be 16-byte, lse 4-byte aligned");
  const qk::AttentionPlan plan =
      qk::plan_attention(batch->tokens, batch->sequences, q_heads, cache->kv_heads, static_cast<int>(cache->head_dim),
                         cache->type, q_type, window, max_context);
  if (!qk::plan_fits(plan, cache->kv_heads, cache->type, q_type))
    return refuse("attention of so many tokens and heads does not fit one launch");
  const size_t need = plan.bytes;
  if (need != 0 && !workspace) return refuse("attention workspace must be non-null");
  if (workspace_bytes < need) return refuse("attention workspace too small");
  if (misaligned(workspace, 256)) return refuse("attention workspace must be 256-byte aligned");
  qk::AttentionArgs a{};
  a.kv = kv_args(cache, batch);
  a.q = q;
  a.q_stride = q_stride;
  a.q_heads = static_cast<int32_t>(q_heads);
  a.group = static_cast<int32_t>(q_heads / cache->kv_heads);
  a.scale = scale;
  a.window = static_cast<int32_t>(qk::bounded_window(window));
  a.out = out;
  a.lse = lse;
  return finish(qk::launch_paged_attention(a, plan, cache->type, static_cast<int>(cache->head_dim), q_type, workspace,
                                           as_stream(stream)),
                "paged attention launch failed");
}

int qk_kv_rows(const qk_kv_cache* cache, const qk_kv_batch* batch, void* k_out, void* v_out, int out_type,
               qk_stream_t stream) {
  int status = check_shapes(cache, batch);
  if (status != QK_OK) return status;
  if (out_type != QK_TYPE_F32 && out_type != value_type(cache))
    return refuse("rows are F32 or of the cache's type (F16 for Q4_1)", QK_ERR_UNSUPPORTED_TYPE);
  if (batch->tokens == 0 || batch->sequences == 0) return QK_OK;
  status = check_pointers(cache, batch);
  if (status != QK_OK) return status;
  if (!k_out && !v_out) return refuse("rows need somewhere to go");
  if (misaligned(k_out, 16) || misaligned(v_out, 16)) return refuse("row outputs must be 16-byte aligned");
  qk::RowsArgs a{kv_args(cache, batch), k_out, v_out};
  return finish(qk::launch_kv_rows(a, cache->type, static_cast<int>(cache->head_dim), out_type, as_stream(stream)),
                "cache rows launch failed");
}

size_t qk_kv_weigh_workspace_size(const qk_kv_cache* cache, const qk_kv_batch* batch, int q_type, int64_t q_heads,
                                  int64_t max_context) {
  if (check_shapes(cache, batch) != QK_OK || check_heads(cache, batch, q_heads, q_type) != QK_OK || max_context < 0) return 0;
  const qk::WeighPlan plan = qk::plan_weigh(batch->tokens, batch->sequences, q_heads, cache->kv_heads, max_context);
  return qk::weigh_fits(plan, batch->sequences, cache->kv_heads) ? plan.bytes : 0;
}

int qk_kv_weigh(const qk_kv_cache* cache, const qk_kv_batch* batch, const int32_t* seen, const void* q, int q_type,
                int64_t q_stride, int64_t q_heads, float scale, const float* lse, int64_t max_context,
                const qk_kv_weights* weights, void* workspace, size_t workspace_bytes, qk_stream_t stream) {
  int status = check_shapes(cache, batch);
  if (status == QK_OK) status = check_heads(cache, batch, q_heads, q_type);
  if (status != QK_OK) return status;
  if (max_context < 0) return refuse("weigh max_context must not be negative");
  if (!std::isfinite(scale)) return refuse("weigh scale must be finite");
  if (batch->tokens == 0 || batch->sequences == 0) return QK_OK;
  if (q_stride < q_heads * cache->head_dim || q_stride > (int64_t{1} << 40)) return refuse("weigh q_stride must hold a token's heads");
  if (q_stride % (q_type == QK_TYPE_F32 ? 4 : 8) != 0) return refuse("weigh q rows must be 16-byte aligned");
  status = check_pointers(cache, batch);
  if (status == QK_OK) status = check_weights(weights);
  if (status != QK_OK) return status;
  if (!q || !lse) return refuse("weigh pointers must be non-null");
  if (misaligned(q, 16) || misaligned(lse, 4) || misaligned(seen, 4)) return refuse("weigh q must be 16-byte, lse and seen 4-byte aligned");
  const qk::WeighPlan plan = qk::plan_weigh(batch->tokens, batch->sequences, q_heads, cache->kv_heads, max_context);
  if (!qk::weigh_fits(plan, batch->sequences, cache->kv_heads))
    return refuse("weights of so many sequences, heads and keys do not fit one launch");
  status = check_workspace(workspace, workspace_bytes, plan.bytes);
  if (status != QK_OK) return status;
  qk::WeighArgs a{};
  a.kv = kv_args(cache, batch);
  a.seen = seen;
  a.q = q;
  a.q_stride = q_stride;
  a.q_heads = static_cast<int32_t>(q_heads);
  a.group = static_cast<int32_t>(q_heads / cache->kv_heads);
  a.scale = scale;
  a.lse = lse;
  a.weight = weights->weight;
  a.position = weights->position;
  return finish(qk::launch_kv_weigh(a, plan, cache->type, static_cast<int>(cache->head_dim), q_type, workspace, as_stream(stream)),
                "weigh launch failed");
}

size_t qk_kv_evict_workspace_size(const qk_kv_cache* cache, const qk_kv_batch* batch, int64_t max_context) {
  if (check_shapes(cache, batch) != QK_OK || batch->sequences == 0 || max_context < 1 || !evict_fits(cache, batch, max_context))
    return 0;
  return qk::evict_workspace(batch->sequences, cache->kv_heads, max_context);
}

int qk_kv_evict(const qk_kv_cache* cache, const qk_kv_batch* batch, const int32_t* seen, const qk_kv_weights* weights,
                const int32_t* keep, const int32_t* recent, int64_t max_context, int32_t* context_out, void* workspace,
                size_t workspace_bytes, qk_stream_t stream) {
  int status = check_shapes(cache, batch);
  if (status != QK_OK) return status;
  if (max_context < 1) return refuse("evict max_context must be positive");
  if (batch->sequences == 0) return QK_OK;
  if (!evict_fits(cache, batch, max_context)) return refuse("eviction of so many sequences, heads and tokens does not fit one launch");
  status = check_pointers(cache, batch);
  if (status == QK_OK) status = check_weights(weights);
  if (status != QK_OK) return status;
  if (!keep || !recent || !context_out) return refuse("evict pointers must be non-null");
  if (misaligned(keep, 4) || misaligned(recent, 4) || misaligned(context_out, 4) || misaligned(seen, 4))
    return refuse("evict arrays must be 4-byte aligned");
  // workgroups of other heads still read those when the first lengths are written
  const uint64_t n = static_cast<uint64_t>(batch->sequences), stride = static_cast<uint64_t>(batch->table_stride);
  const uint64_t table = stride < (uint64_t{1} << 40) ? n * stride : n << 40;  // no address space holds more
  if (overlap(context_out, n, batch->context, n) || overlap(context_out, n, keep, n) || overlap(context_out, n, recent, n) ||
      overlap(context_out, n, seen, n) || overlap(context_out, n, batch->page_table, table))
    return refuse("evict context_out must be an array of its own");
  status = check_workspace(workspace, workspace_bytes, qk::evict_workspace(batch->sequences, cache->kv_heads, max_context));
  if (status != QK_OK) return status;
  qk::EvictArgs a{};
  a.kv = kv_args(cache, batch);
  a.seen = seen;
  a.keep = keep;
  a.recent = recent;
  a.weight = weights->weight;
  a.position = weights->position;
  a.context_out = context_out;
  a.width = static_cast<int32_t>(max_context);
  return finish(qk::launch_kv_evict(a, cache->type, static_cast<int>(cache->head_dim), workspace, as_stream(stream)),
                "evict launch failed");
}

int qk_kv_check(const qk_kv_cache* cache, qk_stream_t stream) {
  if (!cache) return refuse("cache must be non-null");
  if (!cache->fault) return QK_OK;
  if (misaligned(cache->fault, 4)) return refuse("the fault word must be 4-byte aligned");
  uint32_t fault = 0;
  const int status = qk_memcpy_d2h(&fault, cache->fault, sizeof(fault), stream);
  if (status != QK_OK || fault == 0) return status;
  // the bits that were read and no others: a call on another stream may set one meanwhile
  hipError_t error = qk::launch_kv_fault_clear(cache->fault, fault, as_stream(stream));
  if (error == hipSuccess) error = hipStreamSynchronize(as_stream(stream));
  if (error != hipSuccess) return finish(error, "clearing the fault word failed");
  const bool page = fault & QK_KV_FAULT_PAGE, length = fault & QK_KV_FAULT_LENGTH;
  return refuse(page && length ? "a page id or position outside the cache was met, and token_start or context did not fit the batch"
                : page         ? "a page id or position outside the cache was met"
                               : "token_start or context did not fit the batch",
                QK_ERR_RUNTIME);
}

size_t qk_sample_workspace_size(int64_t rows, int64_t vocabulary) {
  if (rows < 0 || rows > 65535 || vocabulary < 1 || vocabulary > (int64_t{1} << 24)) return 0;
  return qk::sample_workspace(rows, vocabulary);
}

int qk_sample(const float* logits, int64_t rows, int64_t vocabulary, int64_t row_stride, const float* temperature,
              const int32_t* top_k, const float* top_p, const float* min_p, const float* uniform, uint32_t* token,
              float* probability, void* workspace, size_t workspace_bytes, qk_stream_t stream) {
  if (rows < 0 || rows > 65535 || vocabulary < 1 || vocabulary > (int64_t{1} << 24))
    return refuse("sample needs 0 .. 65535 rows of 1 .. 2^24 logits");
  if (row_stride < vocabulary || row_stride > (int64_t{1} << 40)) return refuse("sample row_stride must hold a row");
  if (rows == 0) return QK_OK;
  if (!logits || !temperature || !uniform || !token) return refuse("sample pointers must be non-null");
  for (const void* p : {static_cast<const void*>(logits), static_cast<const void*>(temperature),
                        static_cast<const void*>(top_k), static_cast<const void*>(top_p),
                        static_cast<const void*>(min_p), static_cast<const void*>(uniform),
                        static_cast<const void*>(token), static_cast<const void*>(probability)})
    if (misaligned(p, 4)) return refuse("sample arrays must be 4-byte aligned");
  const size_t need = qk::sample_workspace(rows, vocabulary);
  if (need != 0 && !workspace) return refuse("sample workspace must be non-null");
  if (workspace_bytes < need) return refuse("sample workspace too small");
  if (misaligned(workspace, 256)) return refuse("sample workspace must be 256-byte aligned");
  qk::SampleArgs a{logits,
                   row_stride,
                   static_cast<int32_t>(rows),
                   static_cast<int32_t>(vocabulary),
                   temperature,
                   top_k,
                   top_p,
                   min_p,
                   uniform,
                   token,
                   probability};
  return finish(qk::launch_sample(a, workspace, as_stream(stream)), "sample launch failed");
}

}  // extern "C"
