/*
 * C ABI of operators beside a served batch's Linears and LM head: low-rank
 * adapters of many requests at once, and the choice of each sequence's next
 * token.
 *
 * No reference counterpart: the reference runs one sequence of one model and
 * takes the argmax of its logits (src/qwen2.cpp:597-674, lm_head_bf16 in
 * include/infer/cuda_ops.hpp:42-45, Greedy-cy/qwen2.5-jetson-inference).
 *
 * Conventions are infer_linear.h's: caller-owned device memory, BF16 as 16-bit
 * words, work enqueued on `stream` of the current device and never
 * synchronised, nothing allocated, and a nonzero status with a message in
 * infer_hip_last_error on bad arguments (checked on the host before any
 * launch).  Both operators can be captured into a HIP graph; identifiers,
 * ranks and settings are read on the device when the work runs.  A workspace
 * holds nothing between calls; calls that share one must not overlap.
 */
#ifndef INFER_BATCH_H
#define INFER_BATCH_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#include "infer_linear.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- Low-rank adapters -----------------------------------------------------
 * For every token t with adapter i = ids[t] and every target, a projection of
 * the same input x:
 *   output[t] = bf16(base[t] + scales[i] * B[i] (A[i] x[t])),
 * FP32 sums.  A token whose id is not in [0, adapters) (-1, say) has no
 * adapter: its base is copied.
 *
 * x is BF16 [tokens][in_features], x_stride elements between tokens (a multiple
 * of 8).  Per target: a BF16 [adapters][max_rank][in_features] and b BF16
 * [adapters][out_features][max_rank], contiguous; base and output BF16
 * [tokens][out_features] with strides of their own (any from out_features up).
 * output may be base itself with the same stride (the projection's output is
 * then updated); base NULL: zeros.  No other overlap.  ranks[i] (NULL: max_rank
 * for all; clamped to [0, max_rank]): rows of A[i] and columns of B[i] from
 * there on are not used, whatever they hold.  scales NULL: 1.
 *
 * x, a, b and the workspace are 16-byte aligned; in_features a multiple of 8
 * up to 2^22, max_rank a multiple of 8 up to 128, out_features up to 2^22, at
 * most 2^20 tokens and adapters, 1 to INFER_HIP_LORA_TARGETS targets.  Outputs and
 * bases that are 16-byte aligned with strides that are a multiple of 8 are
 * faster.
 *
 * A[i] x[t] times the scale is kept as the sum of two BF16 numbers (a relative
 * 2^-16, up to FP32's largest number) between the products.  An infinite element of
 * B gives an infinity or NaN in its row of the tokens with that adapter, and no
 * other.  Results do not change from run to run. */
#define INFER_HIP_LORA_TARGETS 3

typedef struct infer_hip_lora_target {
  const uint16_t* a;
  const uint16_t* b;
  const uint16_t* base;
  uint16_t* output;
  int out_features;
  long long base_stride;
  long long output_stride;
} infer_hip_lora_target;

/* Bytes for calls of up to `tokens` tokens (0: refused shapes). */
size_t infer_hip_lora_workspace_bytes(int tokens, int max_rank, int targets);
int infer_hip_lora_bf16(const uint16_t* x, long long x_stride, const int* ids, int tokens,
                        int in_features, const infer_hip_lora_target* targets, int num_targets,
                        int adapters, int max_rank, const int* ranks, const float* scales,
                        void* workspace, size_t workspace_bytes, hipStream_t stream);

/* ---- Sampling -----------------------------------------------------------------
 * The next token of every row of logits, BF16 [rows][vocab] with `stride`
 * elements between rows (any from vocab up), from a given random number.  In 64
 * bits, a row's tokens stand in descending order of logit, ties in ascending
 * order of index, each with the weight
 *   w = exp((logit - largest logit) / temperature);
 * kept are
 *   the first top_k of them (top_k <= 0: all),
 *   of those the shortest run that holds at least top_p of their weight
 *   (top_p >= 1: all), but one at least,
 *   of those the ones with w >= min_p (min_p <= 0: all), but one at least;
 * the token is the first kept one whose running sum of w exceeds uniform times
 * the sum of all kept.  So a smaller random number never gives a token of a
 * smaller logit.  probabilities[row] (may be NULL) is its w over that sum.
 *
 * Settings are arrays [rows] in device memory, NULL for temperature 1, top_k 0,
 * top_p 1 and min_p 0 in every row.  A temperature of 0 or less takes the first
 * token, whatever the other settings (its probability is 1).  uniform[row] in
 * [0, 1) (values outside: the nearer end).  Logits of -infinity (masked tokens)
 * have weight 0 and are never taken; +infinity leaves the tokens that have it,
 * equally.  A row with nothing but -infinity gives token -1 and probability 0,
 * a row with a NaN among its logits or settings, or for its random number, token
 * -1 and probability NaN.
 *
 * logits at least 2-byte aligned (rows that are 16-byte aligned are faster),
 * vocab up to 2^20, rows up to 2^20, the workspace 16-byte aligned.  A row takes some 50
 * times as long where 32768 tokens or more have one magnitude (both signs counted
 * together), other than those of one value, a mask's: the lowest, or a low one that more
 * tokens have than any below it. */
/* Bytes for calls of up to `rows` rows of `vocab` (0: refused shapes).  16 now,
 * which nothing is written to: a row's state lies in its workgroup. */
size_t infer_hip_sample_workspace_bytes(int rows, int vocab);
int infer_hip_sample_bf16(const uint16_t* logits, long long stride, int rows, int vocab,
                          const float* temperature, const int* top_k, const float* top_p,
                          const float* min_p, const float* uniform, int* tokens,
                          float* probabilities, void* workspace, size_t workspace_bytes,
                          hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* INFER_BATCH_H */
