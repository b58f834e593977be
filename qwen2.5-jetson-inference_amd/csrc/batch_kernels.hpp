// Internal launch interface of the operators of infer_batch.h (lora.hip,
// sample.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "infer_batch.h"

namespace qlin {

struct LoraTarget {
  const uint16_t* a;
  const uint16_t* b;
  const uint16_t* base;
  uint16_t* out;
  int n;
  long long base_stride, out_stride;
};

struct LoraArgs {
  const uint16_t* x;
  long long x_stride;
  const int* ids;
  int tokens, k;
  LoraTarget target[INFER_HIP_LORA_TARGETS];
  int targets, adapters, max_rank;
  const int* ranks;     // null: max_rank
  const float* scales;  // null: 1
  uint16_t* h;          // [targets][tokens][2][rank_pitch(max_rank)]
  // set by the launch
  int* groups;   // of more tokens than a workgroup gathers by itself
  int units;     // of the call, or of a chunk
  int by_token;  // a unit is a token that is the first with its adapter, not an adapter
  int blocks;    // of columns, where a launch counts units and blocks together
  int parts;     // of K, each with sums in 32 bits: float [parts][targets][tokens][rank_pitch]
};

struct SampleArgs {
  const uint16_t* logits;
  long long stride;
  int rows, vocab;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniform;
  int* tokens;
  float* probabilities;
};

size_t lora_workspace_bytes(int tokens, int max_rank, int targets);
void launch_lora(LoraArgs a, hipStream_t stream);
size_t sample_workspace_bytes(int rows, int vocab);
void launch_sample(const SampleArgs& a, hipStream_t stream);

}  // namespace qlin
