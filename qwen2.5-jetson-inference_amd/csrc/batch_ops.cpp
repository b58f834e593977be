// C ABI of the adapters and of sampling (include/infer_batch.h): argument
// checks, then the launches of lora.hip and sample.hip.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "batch_kernels.hpp"
#include "infer_batch.h"
#include "status.hpp"

using namespace qlin;

namespace {

constexpr int kMaxTokens = 1 << 20;
constexpr int kMaxAdapters = 1 << 20;
constexpr int kMaxFeatures = 1 << 22;
constexpr int kMaxRank = 128;
constexpr int kMaxRows = 1 << 20;
constexpr int kMaxVocab = 1 << 20;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool lora_shape(int tokens, int max_rank, int targets) {
  return tokens >= 1 && tokens <= kMaxTokens && max_rank >= 8 && max_rank <= kMaxRank &&
         max_rank % 8 == 0 && targets >= 1 && targets <= INFER_HIP_LORA_TARGETS;
}

bool sample_shape(int rows, int vocab) {
  return rows >= 1 && rows <= kMaxRows && vocab >= 1 && vocab <= kMaxVocab;
}

int check_workspace(const void* workspace, size_t bytes, size_t need, const char* what) {
  if (!workspace || !aligned16(workspace) || bytes < need) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "%s: workspace of %zu bytes, 16-byte aligned, needed (%zu given)", what, need,
                bytes);
  }
  return INFER_HIP_OK;
}

}  // namespace

extern "C" size_t infer_hip_lora_workspace_bytes(int tokens, int max_rank, int targets) {
  return lora_shape(tokens, max_rank, targets) ? lora_workspace_bytes(tokens, max_rank, targets)
                                               : 0;
}

extern "C" int infer_hip_lora_bf16(const uint16_t* x, long long x_stride, const int* ids,
                                   int tokens, int in_features,
                                   const infer_hip_lora_target* targets, int num_targets,
                                   int adapters, int max_rank, const int* ranks,
                                   const float* scales, void* workspace, size_t workspace_bytes,
                                   hipStream_t stream) {
  const char* what = "lora";
  if (!lora_shape(tokens, max_rank, num_targets) || adapters < 1 || adapters > kMaxAdapters) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "%s: %d tokens, %d adapters (1 to %d), rank %d (a multiple of 8 up to %d), %d "
                "targets (1 to %d)",
                what, tokens, adapters, kMaxTokens, max_rank, kMaxRank, num_targets,
                INFER_HIP_LORA_TARGETS);
  }
  if (in_features < 8 || in_features % 8 != 0 || in_features > kMaxFeatures) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: in_features %d (a multiple of 8 up to %d)", what,
                in_features, kMaxFeatures);
  }
  if (!x || !ids || !targets) return fail(INFER_HIP_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!aligned16(x) || x_stride % 8 != 0 || x_stride < in_features) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "%s: x must be 16-byte aligned with a stride (%lld) that is a multiple of 8, from "
                "%d up",
                what, x_stride, in_features);
  }
  LoraArgs a{};
  for (int i = 0; i < num_targets; ++i) {
    const infer_hip_lora_target& t = targets[i];
    if (!t.a || !t.b || !t.output) {
      return fail(INFER_HIP_INVALID_ARGUMENT, "%s: null pointer in target %d", what, i);
    }
    if (!aligned16(t.a) || !aligned16(t.b)) {
      return fail(INFER_HIP_INVALID_ARGUMENT, "%s: a and b must be 16-byte aligned (target %d)",
                  what, i);
    }
    if (t.out_features < 1 || t.out_features > kMaxFeatures ||
        t.output_stride < t.out_features || (t.base && t.base_stride < t.out_features)) {
      return fail(INFER_HIP_INVALID_ARGUMENT,
                  "%s: out_features %d (1 to %d), stride %lld of the output and %lld of the base "
                  "(target %d)",
                  what, t.out_features, kMaxFeatures, t.output_stride, t.base_stride, i);
    }
    if (t.base == t.output && t.base_stride != t.output_stride) {
      return fail(INFER_HIP_INVALID_ARGUMENT,
                  "%s: an output that is its base has the base's stride (target %d)", what, i);
    }
    a.target[i] = LoraTarget{t.a, t.b, t.base, t.output, t.out_features, t.base_stride,
                             t.output_stride};
  }
  const int rc = check_workspace(workspace, workspace_bytes,
                                 lora_workspace_bytes(tokens, max_rank, num_targets), what);
  if (rc != INFER_HIP_OK) return rc;
  a.x = x;
  a.x_stride = x_stride;
  a.ids = ids;
  a.tokens = tokens;
  a.k = in_features;
  a.targets = num_targets;
  a.adapters = adapters;
  a.max_rank = max_rank;
  a.ranks = ranks;
  a.scales = scales;
  a.h = static_cast<uint16_t*>(workspace);
  launch_lora(a, stream);
  return check_launch(what);
}

extern "C" size_t infer_hip_sample_workspace_bytes(int rows, int vocab) {
  return sample_shape(rows, vocab) ? sample_workspace_bytes(rows, vocab) : 0;
}

extern "C" int infer_hip_sample_bf16(const uint16_t* logits, long long stride, int rows,
                                     int vocab, const float* temperature, const int* top_k,
                                     const float* top_p, const float* min_p, const float* uniform,
                                     int* tokens, float* probabilities, void* workspace,
                                     size_t workspace_bytes, hipStream_t stream) {
  const char* what = "sample";
  if (!sample_shape(rows, vocab)) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: %d rows (1 to %d) of %d tokens (1 to %d)", what,
                rows, kMaxRows, vocab, kMaxVocab);
  }
  if (!logits || !uniform || !tokens) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "%s: null pointer", what);
  }
  if ((reinterpret_cast<uintptr_t>(logits) & 1u) != 0 || stride < vocab) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "%s: logits must be 2-byte aligned, with a stride (%lld) from %d up", what, stride,
                vocab);
  }
  const int rc = check_workspace(workspace, workspace_bytes, sample_workspace_bytes(rows, vocab),
                                 what);
  if (rc != INFER_HIP_OK) return rc;
  launch_sample(SampleArgs{logits, stride, rows, vocab, temperature, top_k, top_p, min_p, uniform,
                           tokens, probabilities},
                stream);
  return check_launch(what);
}
