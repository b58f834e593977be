// C ABI of the paged KV cache (include/infer_paged.h): argument checks, then
// the launches of paged_kernels.hip and page_plan.hip.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "infer_paged.h"
#include "paged_kernels.hpp"
#include "status.hpp"

using namespace qlin;

namespace {

constexpr int kMaxSequences = 65535;  // a grid dimension
constexpr int kMaxHeads = 65535;
constexpr int kMaxPositions = 1 << 30;  // of a sequence

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_pool(const infer_hip_kv_pages* p, KvPool* out, const char* what) {
  if (!p) return fail(INFER_HIP_INVALID_ARGUMENT, "%s: null pages", what);
  if (p->format != INFER_HIP_KV_BF16 && p->format != INFER_HIP_KV_INT8 &&
      p->format != INFER_HIP_KV_FP8) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: unknown cache format %d", what, p->format);
  }
  int shift = 4;
  while (shift < 8 && (1 << shift) != p->page_size) ++shift;
  if ((1 << shift) != p->page_size) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: page_size %d (16, 32, 64, 128 or 256)", what,
                p->page_size);
  }
  if (p->head_dim != 64 && p->head_dim != 128) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: head_dim %d (64 or 128)", what, p->head_dim);
  }
  if (p->num_pages < 1 || p->num_kv_heads < 1 || p->num_kv_heads > kMaxHeads) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: bad pool (%d pages, %d kv heads)", what,
                p->num_pages, p->num_kv_heads);
  }
  const bool scaled = p->format != INFER_HIP_KV_BF16;
  if (!p->key_pages || !p->value_pages || (scaled && (!p->key_scales || !p->value_scales))) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: null pages or scales", what);
  }
  if (!aligned16(p->key_pages) || !aligned16(p->value_pages) ||
      (scaled && (!aligned16(p->key_scales) || !aligned16(p->value_scales)))) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: pages and scales must be 16-byte aligned", what);
  }
  *out = KvPool{p->format, p->num_pages, shift, p->num_kv_heads, p->head_dim,
                p->key_pages, p->value_pages, scaled ? p->key_scales : nullptr,
                scaled ? p->value_scales : nullptr};
  return INFER_HIP_OK;
}

int check_table(const infer_hip_kv_table* t, const KvPool& pool, KvTable* out,
                const char* what) {
  if (!t || !t->pages) return fail(INFER_HIP_INVALID_ARGUMENT, "%s: null block table", what);
  if (t->num_sequences < 1 || t->num_sequences > kMaxSequences || t->max_pages < 1 ||
      t->stride < t->max_pages || t->max_pages > (kMaxPositions >> pool.page_shift)) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "%s: bad block table (%d sequences of at most %d, %d pages of at most %d "
                "positions, stride %d)",
                what, t->num_sequences, kMaxSequences, t->max_pages, kMaxPositions, t->stride);
  }
  *out = KvTable{t->pages, t->num_sequences, t->max_pages, t->stride};
  return INFER_HIP_OK;
}

// One of query, key, value, query_out: [tokens][heads][head_dim], `stride`
// elements between tokens.
int check_rows(const uint16_t* p, long long stride, long long row, const char* name,
               const char* what) {
  if (!p) return fail(INFER_HIP_INVALID_ARGUMENT, "%s: null %s", what, name);
  if (!aligned16(p) || stride % 8 != 0) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "%s: %s must be 16-byte aligned with a stride that is a multiple of 8", what,
                name);
  }
  if (stride < row) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: %s stride %lld under its %lld elements a token",
                what, name, stride, row);
  }
  return INFER_HIP_OK;
}

}  // namespace

extern "C" int infer_hip_kv_pages_store(
    const infer_hip_kv_pages* pages, const infer_hip_kv_table* table, const int* sequences,
    const int* positions, int tokens, const uint16_t* query, long long query_stride,
    int num_heads, const uint16_t* key, long long key_stride, const uint16_t* value,
    long long value_stride, const float* rope, int rope_positions, uint16_t* query_out,
    long long query_out_stride, hipStream_t stream) {
  const char* what = "kv_pages_store";
  KvStoreArgs a{};
  int rc = check_pool(pages, &a.pool, what);
  if (rc == INFER_HIP_OK) rc = check_table(table, a.pool, &a.table, what);
  if (rc != INFER_HIP_OK) return rc;
  if (tokens < 1 || !positions || (!sequences && tokens > a.table.sequences)) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "%s: %d tokens of %d sequences, positions%s given, sequences%s", what, tokens,
                a.table.sequences, positions ? "" : " not", sequences ? "" : " not");
  }
  if ((query == nullptr) != (num_heads == 0) || num_heads < 0) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: %d query heads with%s query", what, num_heads,
                query ? "" : "out");
  }
  const long long d = a.pool.head_dim;
  if (query) {
    rc = check_rows(query, query_stride, num_heads * d, "query", what);
    if (rc == INFER_HIP_OK) {
      rc = check_rows(query_out, query_out_stride, num_heads * d, "query_out", what);
    }
  }
  const long long kv_row = a.pool.kv_heads * d;
  if (rc == INFER_HIP_OK) rc = check_rows(key, key_stride, kv_row, "key", what);
  if (rc == INFER_HIP_OK) rc = check_rows(value, value_stride, kv_row, "value", what);
  if (rc != INFER_HIP_OK) return rc;
  if (rope && (rope_positions < 1 || !aligned16(rope))) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "%s: rope needs a position (%d given) and 16-byte alignment", what,
                rope_positions);
  }
  a.sequence_ids = sequences;
  a.positions = positions;
  a.tokens = tokens;
  a.heads = num_heads;
  a.q = query;
  a.k = key;
  a.v = value;
  a.q_out = query_out;
  a.q_stride = query_stride;
  a.k_stride = key_stride;
  a.v_stride = value_stride;
  a.q_out_stride = query_out_stride;
  a.rope = rope;
  a.rope_positions = rope_positions;
  if (!kv_store_supported(a)) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: %d tokens are too many for one call", what,
                tokens);
  }
  launch_kv_store(a, stream);
  return check_launch(what);
}

extern "C" int infer_hip_kv_pages_load(const infer_hip_kv_pages* pages,
                                       const infer_hip_kv_table* table, const int* lengths,
                                       uint16_t* key_cache, uint16_t* value_cache, int capacity,
                                       hipStream_t stream) {
  const char* what = "kv_pages_load";
  KvLoadArgs a{};
  int rc = check_pool(pages, &a.pool, what);
  if (rc == INFER_HIP_OK) rc = check_table(table, a.pool, &a.table, what);
  if (rc != INFER_HIP_OK) return rc;
  if (!lengths || !key_cache || !value_cache) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: null pointer", what);
  }
  if (!aligned16(key_cache) || !aligned16(value_cache) || capacity < 1) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "%s: caches must be 16-byte aligned, with a capacity (%d) of at least 1", what,
                capacity);
  }
  a.lengths = lengths;
  a.key_cache = key_cache;
  a.value_cache = value_cache;
  a.capacity = capacity;
  if (!kv_load_supported(a)) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "%s: %d positions of a sequence are too many for one call", what, capacity);
  }
  launch_kv_load(a, stream);
  return check_launch(what);
}

extern "C" size_t infer_hip_attention_paged_decode_workspace_bytes(int num_sequences,
                                                                   int num_heads,
                                                                   int num_kv_heads,
                                                                   int head_dim) {
  if (num_sequences < 1 || num_sequences > kMaxSequences || num_kv_heads < 1 ||
      num_heads < num_kv_heads || num_heads > kMaxHeads || num_heads % num_kv_heads != 0 ||
      (head_dim != 64 && head_dim != 128)) {
    return 0;
  }
  return paged_attention_workspace_bytes(num_heads, num_kv_heads, head_dim);
}

extern "C" int infer_hip_attention_paged_decode(const infer_hip_kv_pages* pages,
                                                const infer_hip_kv_table* table,
                                                const int* lengths, const uint16_t* query,
                                                long long query_stride, int num_heads,
                                                uint16_t* output, void* workspace,
                                                size_t workspace_bytes, hipStream_t stream) {
  const char* what = "attention_paged_decode";
  PagedAttnArgs a{};
  int rc = check_pool(pages, &a.pool, what);
  if (rc == INFER_HIP_OK) rc = check_table(table, a.pool, &a.table, what);
  if (rc != INFER_HIP_OK) return rc;
  if (num_heads < 1 || num_heads > kMaxHeads || num_heads % a.pool.kv_heads != 0) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: %d query heads on %d kv heads", what, num_heads,
                a.pool.kv_heads);
  }
  const long long row = static_cast<long long>(num_heads) * a.pool.head_dim;
  rc = check_rows(query, query_stride, row, "query", what);
  if (rc == INFER_HIP_OK) rc = check_rows(output, row, row, "output", what);
  if (rc != INFER_HIP_OK) return rc;
  if (!lengths) return fail(INFER_HIP_INVALID_ARGUMENT, "%s: null lengths", what);
  const size_t need = paged_attention_workspace_bytes(num_heads, a.pool.kv_heads, a.pool.head_dim);
  if (!workspace || !aligned16(workspace) || workspace_bytes < need) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "%s: workspace of %zu bytes, 16-byte aligned, needed (%zu given)", what, need,
                workspace_bytes);
  }
  a.lengths = lengths;
  a.q = query;
  a.q_stride = query_stride;
  a.heads = num_heads;
  a.out = output;
  a.records = static_cast<float*>(workspace);
  if (!paged_attention_supported(a)) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "%s: %d sequences of up to %d pages of %d are too many for one call", what,
                a.table.sequences, a.table.max_pages, 1 << a.pool.page_shift);
  }
  launch_paged_attention(a, stream);
  return check_launch(what);
}

namespace {

constexpr int kMaxPoolPages = 1 << 30;
constexpr int kMaxPlanTokens = 1 << 30;

int check_plan(const PagePlan& p, int page_size, const void* workspace, size_t workspace_bytes,
               PagePlan* out, const char* what) {
  int shift = 4;
  while (shift < 8 && (1 << shift) != page_size) ++shift;
  if ((1 << shift) != page_size) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: page_size %d (16, 32, 64, 128 or 256)", what,
                page_size);
  }
  if (p.sequences < 1 || p.sequences > kMaxSequences || p.max_pages < 1 ||
      p.stride < p.max_pages || p.max_pages > (kMaxPositions >> shift)) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "%s: bad block table (%d sequences of at most %d, %d pages of at most %d "
                "positions, stride %d)",
                what, p.sequences, kMaxSequences, p.max_pages, kMaxPositions, p.stride);
  }
  if (p.num_pages < 1 || p.num_pages > kMaxPoolPages) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: %d pages (1 to %d)", what, p.num_pages,
                kMaxPoolPages);
  }
  if (!p.table || !p.free_count || !p.free_count_out || !p.lengths || !p.lengths_out) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: null pointer", what);
  }
  const size_t need = page_plan_workspace_bytes(p.sequences);
  if (!workspace || !aligned16(workspace) || workspace_bytes < need) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "%s: workspace of %zu bytes, 16-byte aligned, needed (%zu given)", what, need,
                workspace_bytes);
  }
  *out = p;
  out->page_shift = shift;
  return INFER_HIP_OK;
}

}  // namespace

extern "C" size_t infer_hip_kv_pages_plan_workspace_bytes(int num_sequences) {
  if (num_sequences < 1 || num_sequences > kMaxSequences) return 0;
  return page_plan_workspace_bytes(num_sequences);
}

extern "C" int infer_hip_kv_pages_assign(int* table, int num_sequences, int max_pages, int stride,
                                         int page_size, const int* free_pages, int num_pages,
                                         const int* free_count, int* free_count_out,
                                         const int* lengths, const int* added, int* lengths_out,
                                         int tokens, int* positions, int* sequences,
                                         long long* slots, int* starts, void* workspace,
                                         size_t workspace_bytes, hipStream_t stream) {
  const char* what = "kv_pages_assign";
  AssignArgs a{};
  const PagePlan p{table, num_sequences, max_pages, stride, 0, num_pages, free_count,
                   free_count_out, lengths, lengths_out};
  const int rc = check_plan(p, page_size, workspace, workspace_bytes, &a.plan, what);
  if (rc != INFER_HIP_OK) return rc;
  if (!free_pages || !added || !positions) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: null pointer", what);
  }
  if (tokens < 1 || tokens > kMaxPlanTokens ||
      (!sequences && (tokens != num_sequences || starts))) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "%s: %d tokens of %d sequences, sequences%s given, starts%s", what, tokens,
                num_sequences, sequences ? "" : " not", starts ? "" : " not");
  }
  a.free_pages = free_pages;
  a.added = added;
  a.tokens = tokens;
  a.positions = positions;
  a.ids = sequences;
  a.slots = slots;
  a.starts = starts;
  launch_pages_assign(a, workspace, stream);
  return check_launch(what);
}

extern "C" int infer_hip_kv_pages_release(const int* table, int num_sequences, int max_pages,
                                          int stride, int page_size, int* free_pages,
                                          int num_pages, const int* free_count,
                                          int* free_count_out, const int* lengths,
                                          const int* finished, int* lengths_out, void* workspace,
                                          size_t workspace_bytes, hipStream_t stream) {
  const char* what = "kv_pages_release";
  ReleaseArgs a{};
  const PagePlan p{const_cast<int*>(table), num_sequences, max_pages, stride, 0, num_pages,
                   free_count, free_count_out, lengths, lengths_out};
  const int rc = check_plan(p, page_size, workspace, workspace_bytes, &a.plan, what);
  if (rc != INFER_HIP_OK) return rc;
  if (!free_pages || !finished) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: null pointer", what);
  }
  a.free_pages = free_pages;
  a.finished = finished;
  launch_pages_release(a, workspace, stream);
  return check_launch(what);
}
