// Internal launch interface of the paged KV cache kernels (paged_kernels.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "infer_paged.h"

namespace qlin {

struct KvPool {
  int format;
  int num_pages;
  int page_shift;  // log2(page_size)
  int kv_heads;
  int head_dim;
  void* key;
  void* value;
  float* key_scales;
  float* value_scales;
};

struct KvTable {
  const int* pages;
  int sequences;
  int max_pages;
  int stride;
};

struct KvStoreArgs {
  KvPool pool;
  KvTable table;
  const int* sequence_ids;  // null: token t is sequence t's
  const int* positions;
  int tokens;
  int heads;  // 0: no query
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* q_out;
  long long q_stride, k_stride, v_stride, q_out_stride;
  const float* rope;  // null: no rotation
  int rope_positions;
};

struct KvLoadArgs {
  KvPool pool;
  KvTable table;
  const int* lengths;
  uint16_t* key_cache;
  uint16_t* value_cache;
  int capacity;
};

struct PagedAttnArgs {
  KvPool pool;
  KvTable table;
  const int* lengths;
  const uint16_t* q;
  long long q_stride;
  int heads;
  uint16_t* out;
  float* records;   // [workgroups][2][heads of a unit][D + 4]: O, maximum, sum
  // set by the launch
  int head_blocks;  // of a KV head: its query heads / 16, rounded up
  int units;        // KV heads x head blocks
  int waves;        // of the grid
  int whole;        // units are not cut
  int join_heads;   // a workgroup of the join per query head
  int piece_waves;  // of a workgroup that the join's parts come from
};

// Whether the launch's threads can be counted in 32 bits.
bool kv_store_supported(const KvStoreArgs& a);
bool kv_load_supported(const KvLoadArgs& a);
void launch_kv_store(const KvStoreArgs& a, hipStream_t stream);
void launch_kv_load(const KvLoadArgs& a, hipStream_t stream);
// Whether the tiles of the largest possible lengths can be counted in 32 bits.
bool paged_attention_supported(const PagedAttnArgs& a);
void launch_paged_attention(PagedAttnArgs a, hipStream_t stream);
size_t paged_attention_workspace_bytes(int heads, int kv_heads, int head_dim);

// Pages of a step (page_plan.hip).
struct PagePlan {
  int* table;
  int sequences, max_pages, stride, page_shift;
  int num_pages;
  const int* free_count;
  int* free_count_out;
  const int* lengths;
  int* lengths_out;
};

struct AssignArgs {
  PagePlan plan;
  const int* free_pages;
  const int* added;
  int tokens;
  int* positions;
  int* ids;  // null: token s is sequence s's
  long long* slots;  // null: not wanted
  int* starts;       // null: not wanted
};

struct ReleaseArgs {
  PagePlan plan;
  int* free_pages;
  const int* finished;
};

size_t page_plan_workspace_bytes(int sequences);
void launch_pages_assign(const AssignArgs& a, void* workspace, hipStream_t stream);
void launch_pages_release(const ReleaseArgs& a, void* workspace, hipStream_t stream);

}  // namespace qlin
