/*
 * C ABI of the paged KV cache: the decode step's cache operators for several
 * sequences at once, whose keys and values live in pages of one pool.
 *
 * No reference counterpart: the reference keeps one sequence's contiguous BF16
 * cache (store_kv_bf16 and attention_decode_bf16, include/infer/cuda_ops.hpp:
 * 78-91, Greedy-cy/qwen2.5-jetson-inference).  These are the same steps of a
 * layer — RoPE, cache store, attention of the new token — over block tables:
 *
 *   infer_hip_kv_pages_store           RoPE of q and k, k and v written into
 *                                      pages as BF16, INT8 or FP8
 *   infer_hip_kv_pages_load            pages read back as the contiguous BF16
 *                                      cache the other operators use
 *   infer_hip_attention_paged_decode   attention of one new token a sequence
 *
 * Conventions are infer_linear.h's: caller-owned device memory, BF16 as 16-bit
 * words, work enqueued on `stream` of the current device and never
 * synchronised, nothing allocated, and a nonzero status with a message in
 * infer_hip_last_error on bad arguments (checked on the host before any
 * launch).  Every operator can be captured into a HIP graph; lengths,
 * positions and tables are read on the device when the work runs.
 */
#ifndef INFER_PAGED_H
#define INFER_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#include "infer_linear.h"

#ifdef __cplusplus
extern "C" {
#endif

/* How a pool holds its elements.  A row is one (token, KV head)'s head_dim
 * keys or values.  The 8-bit formats keep one FP32 scale per row:
 *   INT8  scale = max|v| / 127, element = rint(v / scale)
 *   FP8   scale = max|v| / 448, element = e4m3(v / scale) (OCP E4M3, round to
 *         nearest even)
 * both from the FP32 row, so nothing is rounded twice.  A row of zeros has
 * scale 0; a row with a NaN or an infinity has scale NaN and reads as NaN. */
enum infer_hip_kv_format {
  INFER_HIP_KV_BF16 = 0,
  INFER_HIP_KV_INT8 = 1,
  INFER_HIP_KV_FP8 = 2
};

/* A pool of pages (device memory).  key_pages and value_pages are
 * [num_pages][num_kv_heads][page_size][head_dim] elements, 16-byte aligned;
 * key_scales and value_scales [num_pages][num_kv_heads][page_size] FP32,
 * 16-byte aligned (ignored for BF16).  page_size 16, 32, 64, 128 or 256,
 * head_dim 64 or 128. */
typedef struct infer_hip_kv_pages {
  int format; /* infer_hip_kv_format */
  int num_pages;
  int page_size;
  int num_kv_heads;
  int head_dim;
  void* key_pages;
  void* value_pages;
  float* key_scales;
  float* value_scales;
} infer_hip_kv_pages;

/* Block table (device memory): position p of sequence s is slot p % page_size
 * of page pages[s * stride + p / page_size].  max_pages entries of a row may be
 * used; entries behind a sequence's last page are never read.  max_pages bounds
 * the lengths, and the launches go by that bound, as they cannot see the
 * lengths: where a table is wider than any sequence of the batch, pass the
 * columns that are in use (max_pages smaller than stride). */
typedef struct infer_hip_kv_table {
  const int* pages;
  int num_sequences; /* at most 65535 */
  int max_pages;     /* at most 2^30 positions */
  int stride;        /* entries between rows, >= max_pages */
} infer_hip_kv_table;

/* For each of `tokens` tokens t at positions[t] of sequence sequences[t]
 * (sequences NULL: token t belongs to sequence t, the decode step's form):
 *   query_out[t] <- rope(query[t]) in BF16 (one rounding),
 *   the pages' row of (t, KV head) <- rope(key[t]), value[t].
 * rope is [rope_positions][head_dim / 2] (cos, sin) pairs as
 * infer_hip_rope_row gives them, applied as infer_hip_rms_norm_qkv_rope_w8a16
 * does; NULL: no rotation.  query, key and value are BF16 [tokens][heads]
 * [head_dim] with their own distance between tokens in elements (a multiple of
 * 8, so that column blocks of one projection's output can be passed), 16-byte
 * aligned.  query NULL (then num_heads 0): only the cache is written.
 * query_out may be query itself with the same stride; no other overlap.
 *
 * A token with a negative position (padding), or with rope one at or past
 * rope_positions, writes nothing.  One whose sequence is not in the table,
 * whose position is past the table's pages or whose page is not in the pool
 * stores nothing (its query is still rotated).  Two tokens of a call must not
 * share a slot: that slot then holds an unspecified row.  A call takes at most
 * 2^36 - 4096 elements: tokens x (num_heads + 2 num_kv_heads) x head_dim. */
int infer_hip_kv_pages_store(const infer_hip_kv_pages* pages, const infer_hip_kv_table* table,
                             const int* sequences, const int* positions, int tokens,
                             const uint16_t* query, long long query_stride, int num_heads,
                             const uint16_t* key, long long key_stride, const uint16_t* value,
                             long long value_stride, const float* rope, int rope_positions,
                             uint16_t* query_out, long long query_out_stride,
                             hipStream_t stream);

/* Positions [0, min(lengths[s], capacity)) of every sequence of the table,
 * dequantised to BF16 (bf16(element * scale)), into contiguous caches
 * [num_sequences][num_kv_heads][capacity][head_dim] — per sequence the layout
 * of infer_hip_attention_prefill_bf16.  Rows at or past a sequence's length
 * keep what they hold.  Lengths past the table's pages end there; rows on a
 * page that is not in the pool read as NaN.  The smaller of capacity and the
 * table's positions times head_dim is at most 2^35 - 2048. */
int infer_hip_kv_pages_load(const infer_hip_kv_pages* pages, const infer_hip_kv_table* table,
                            const int* lengths, uint16_t* key_cache, uint16_t* value_cache,
                            int capacity, hipStream_t stream);

/* Attention of one new token a sequence: for sequence s of lengths[s] cached
 * positions (the token's own among them), query head h and its KV head
 * h / (num_heads / num_kv_heads)
 *   output[s][h] = bf16(softmax(query[s][h] K^T / sqrt(head_dim)) V).
 * query is BF16 [num_sequences][num_heads][head_dim] with query_stride elements
 * between sequences (a multiple of 8), already rotated; output is contiguous
 * and overlaps nothing; both 16-byte aligned.  FP32 softmax statistics and
 * sums; the sum of weights (up to 2^6 each) times values is divided at the
 * end, so values near FP32's largest overflow, and values under some 2^-110
 * lose bits to its smallest normal number.  An infinite value of BF16 pages
 * gives that infinity, or NaN where the other one meets it or its weight is 0
 * in FP32.  A length of zero or less (an empty slot of the batch) gives zeros;
 * a length past the table's pages ends there.  Scores that are all -infinity give NaN, as the
 * quotient does.  A sequence whose pages within its length are not all in the
 * pool gives NaN.  Rows behind a sequence's length never count, whatever they
 * hold.
 *
 * The work of all sequences is cut into equal parts over the chip on the
 * device, from the lengths, and the parts of a head joined in a fixed order:
 * results do not change from run to run.  lengths must not change while the
 * call runs.  workspace: device memory of
 * infer_hip_attention_paged_decode_workspace_bytes, 16-byte aligned, holding
 * nothing between calls; calls that share one must not overlap.  Its size goes
 * by the heads and head_dim alone, and is 0 for shapes that a call refuses.
 * num_sequences x the table's positions x the KV heads (each counted once for
 * 16 of its query heads) are at most 6.8e10. */
size_t infer_hip_attention_paged_decode_workspace_bytes(int num_sequences, int num_heads,
                                                        int num_kv_heads, int head_dim);
int infer_hip_attention_paged_decode(const infer_hip_kv_pages* pages,
                                     const infer_hip_kv_table* table, const int* lengths,
                                     const uint16_t* query, long long query_stride,
                                     int num_heads, uint16_t* output, void* workspace,
                                     size_t workspace_bytes, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* INFER_PAGED_H */
