// 4-bit weight-only products of a few tokens (W4A16) for gfx950, with the
// host packer of their weights (include/infer_linear.h).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cmath>

#include "device_common.hpp"
#include "infer_linear.h"
#include "status.hpp"

using namespace qlin;

namespace {

constexpr int kThreads = 256;
constexpr int kTileRows = 16, kTileCols = 128;
constexpr int kTileBytes = kTileRows * kTileCols / 2;
constexpr int kMaxTokens = 16;

struct W4Args {
  const uint8_t* w;
  const uint16_t* s;
  const uint16_t* bias;
  const uint16_t* x;
  uint16_t* y;
  int tokens, n, k, group;
};

// A wave per output row: lane (tile t of four, dword d) holds 8 columns.
__global__ __launch_bounds__(kThreads) void w4a16_gemv_kernel(W4Args a) {
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x * (kThreads / kWave) + (threadIdx.x >> 6);
  if (row >= a.n) return;
  const int tiles = (a.k + kTileCols - 1) / kTileCols;
  const int b = (lane & 15) >> 2, step = lane & 3, r = row % kTileRows;
  const uint8_t* w = a.w + static_cast<size_t>(row / kTileRows) * tiles * kTileBytes;
  const uint16_t* s = a.s + static_cast<size_t>(row / kTileRows) * (a.k / a.group) * kTileRows + r;
  float acc[kMaxTokens] = {};
  for (int t = lane >> 4; t < tiles; t += 4) {
    const int col = t * kTileCols + 32 * step + 8 * b;
    if (col >= a.k) continue;
    const uint32_t q = *reinterpret_cast<const uint32_t*>(w + static_cast<size_t>(t) * kTileBytes +
                                                          16 * (b * kTileRows + r) + 4 * step);
    const float scale = bf16_to_f32(s[col / a.group * kTileRows]);
    for (int m = 0; m < kMaxTokens; ++m) {
      if (m >= a.tokens) break;
      const uint16_t* x = a.x + static_cast<size_t>(m) * a.k + col;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int nibble = (i >> 1) + 4 * (i & 1);
        const int value = static_cast<int>((q >> (4 * nibble)) & 15u) - 8;
        acc[m] = fmaf(scale * value, bf16_to_f32(x[i]), acc[m]);
      }
    }
  }
  for (int m = 0; m < kMaxTokens; ++m) {
    if (m >= a.tokens) break;
    const float v = wave_sum(acc[m]);
    if (lane == 0) {
      a.y[static_cast<size_t>(m) * a.n + row] =
          f32_to_bf16(a.bias ? v + bf16_to_f32(a.bias[row]) : v);
    }
  }
}

bool group_ok(int group, int k) {
  return (group == 32 || group == 64 || group == 128) && k > 0 && k % group == 0;
}

}  // namespace

extern "C" size_t infer_hip_w4a16_weight_bytes(int out_features, int in_features) {
  if (out_features < 1 || in_features < 1) return 0;
  return static_cast<size_t>((static_cast<long long>(out_features) + kTileRows - 1) / kTileRows) *
         ((static_cast<long long>(in_features) + kTileCols - 1) / kTileCols) * kTileBytes;
}

extern "C" size_t infer_hip_w4a16_scale_count(int out_features, int in_features, int group_size) {
  if (out_features < 1 || !group_ok(group_size, in_features)) return 0;
  return static_cast<size_t>((static_cast<long long>(out_features) + kTileRows - 1) / kTileRows) *
         (in_features / group_size) * kTileRows;
}

extern "C" int infer_hip_w4a16_pack(const int8_t* values, const uint16_t* scales, int group_size,
                                    int out_features, int in_features, uint8_t* packed_weight,
                                    uint16_t* packed_scales) {
  if (!values || !scales || !packed_weight || !packed_scales) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "w4a16_pack: null pointer");
  }
  if (out_features < 1 || !group_ok(group_size, in_features)) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "w4a16_pack: N=%d K=%d group %d (32, 64 or 128, dividing K)", out_features,
                in_features, group_size);
  }
  const size_t n = out_features, k = in_features, groups = k / group_size;
  const size_t tiles = (k + kTileCols - 1) / kTileCols;
  for (size_t i = 0; i < n * k; ++i) {
    if (values[i] < -8 || values[i] > 7) {
      return fail(INFER_HIP_INVALID_ARGUMENT, "w4a16_pack: value %d at %zu is outside [-8, 7]",
                  values[i], i);
    }
  }
  uint8_t* out = packed_weight;
  for (size_t row0 = 0; row0 < n; row0 += kTileRows) {
    for (size_t t = 0; t < tiles; ++t) {
      for (int b = 0; b < 4; ++b) {
        for (int r = 0; r < kTileRows; ++r) {
          for (int step = 0; step < 4; ++step) {
            uint32_t word = 0;
            for (int i = 0; i < 8; ++i) {
              const size_t row = row0 + r, col = t * kTileCols + 32 * step + 8 * b + i;
              const uint32_t u = row < n && col < k ? values[row * k + col] + 8 : 8;
              word |= u << (4 * ((i >> 1) + 4 * (i & 1)));
            }
            for (int byte = 0; byte < 4; ++byte) *out++ = static_cast<uint8_t>(word >> (8 * byte));
          }
        }
      }
    }
    for (size_t g = 0; g < groups; ++g) {
      for (int r = 0; r < kTileRows; ++r) {
        packed_scales[(row0 / kTileRows * groups + g) * kTileRows + r] =
            row0 + r < n ? scales[(row0 + r) * groups + g] : 0;
      }
    }
  }
  return ok();
}

extern "C" int infer_hip_gemv_w4a16(const uint8_t* weight, const uint16_t* scales, int group_size,
                                    const uint16_t* bias, const uint16_t* input, uint16_t* output,
                                    int tokens, int out_features, int in_features,
                                    hipStream_t stream) {
  if (out_features < 1 || !group_ok(group_size, in_features)) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "gemv_w4a16: N=%d K=%d group %d (32, 64 or 128, dividing K)", out_features,
                in_features, group_size);
  }
  if (tokens < 1 || tokens > kMaxTokens) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "gemv_w4a16: %d tokens (1 to %d)", tokens, kMaxTokens);
  }
  if (!weight || !scales || !input || !output) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "gemv_w4a16: null required pointer");
  }
  if (((reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(scales) |
        reinterpret_cast<uintptr_t>(input)) & 15u) != 0) {
    return fail(INFER_HIP_INVALID_ARGUMENT,
                "gemv_w4a16: weight, scales and input must be 16-byte aligned");
  }
  const W4Args a{weight, scales, bias, input, output, tokens, out_features, in_features, group_size};
  const int per = kThreads / kWave;
  hipLaunchKernelGGL(w4a16_gemv_kernel, dim3((out_features + per - 1) / per), dim3(kThreads), 0,
                     stream, a);
  return check_launch("gemv_w4a16");
}
