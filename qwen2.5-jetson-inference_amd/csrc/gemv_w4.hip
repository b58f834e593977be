// 4-bit weight-only products of a few tokens (W4A16) for gfx950, with the
// host packer of their weights (include/infer_linear.h).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "device_common.hpp"
#include "infer_linear.h"
#include "status.hpp"

using namespace qlin;

namespace {

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

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// Y^T = W X^T on v_mfma_f32_16x16x32_bf16, 16 rows of W by up to 16 tokens.
//
// A nibble u goes into the mantissa of a BF16 number, 1 + u / 16 exactly, with a
// shift and an and-or per pair.  With q = u - 8 that is (q + 24) / 16, so a
// group's accumulator starts from -1.5 sum x (one more MFMA, of the constant,
// shared by the wave's row tiles) and holds sum q x / 16 in FP32; the group's
// scale multiplies it into the FP32 total.  Terms are at most 31/16 |x| where
// q x / 16 reaches 1/2 |x|, which costs two bits of FP32's 24.
//
// A workgroup has R row tiles (16 rows each); its waves split the 128-column
// tiles, each a contiguous KiB of weights in one load, and meet in LDS in the
// order of the waves.  Memory bounds it: per KiB of weights a SIMD issues about
// 40 vector instructions and five MFMAs.
//
// Activations beyond FP32's reach (a sum that is not finite) are summed again
// element by element, q s x in FP32.
template <int G, int R>
struct W4Piece {
  uint4 w[R];
  uint4 x[4];
  uint2 s[R][kTileCols / G];  // four rows' scales
};

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// Eight nibbles as 1 + u / 16 in BF16.
__device__ __forceinline__ bf16x8_t widen_nibbles(uint32_t w) {
  constexpr uint32_t kMantissa = 0x00780078u, kOne = 0x3F803F80u;
  const uint4 v = make_uint4(((w << 3) & kMantissa) | kOne, ((w >> 1) & kMantissa) | kOne,
                             ((w >> 5) & kMantissa) | kOne, ((w >> 9) & kMantissa) | kOne);
  return __builtin_bit_cast(bf16x8_t, v);
}

// Row `row` times token `t`, each product in FP32 as it is.
__device__ float exact_dot(const W4Args& a, int row, int t) {
  const int tiles = (a.k + kTileCols - 1) / kTileCols, r = row % kTileRows;
  const uint8_t* w = a.w + static_cast<size_t>(row / kTileRows) * tiles * kTileBytes;
  const uint16_t* s = a.s + static_cast<size_t>(row / kTileRows) * (a.k / a.group) * kTileRows + r;
  const uint16_t* x = a.x + static_cast<size_t>(t) * a.k;
  float sum = 0.0f;
  for (int col = 0; col < a.k; col += 8) {
    const int at = col % kTileCols;
    const uint32_t q = *reinterpret_cast<const uint32_t*>(
        w + static_cast<size_t>(col / kTileCols) * kTileBytes +
        16 * (at % 32 / 8 * kTileRows + r) + 4 * (at / 32));
    const float scale = bf16_to_f32(s[col / a.group * kTileRows]);
    for (int i = 0; i < 8; ++i) {
      const int value = static_cast<int>((q >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15u) - 8;
      sum = fmaf(scale * value, bf16_to_f32(x[col + i]), sum);
    }
  }
  return sum;
}

template <int G, int R>
__global__ __launch_bounds__(R == 1 ? 1024 : 512) void w4a16_gemv_kernel(W4Args a) {
  constexpr int kGroups = kTileCols / G, kSteps = G / 32;  // of a tile, of a group
  constexpr int kRows = R * kTileRows, kPitch = kRows + 4;
  extern __shared__ __align__(16) float partial[];  // [wave][token][kPitch]
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x / kWave;
  const int tiles = (a.k + kTileCols - 1) / kTileCols;
  const int row_tiles = (a.n + kTileRows - 1) / kTileRows;
  const int first = blockIdx.x * R;
  const int groups = a.k / G;

  auto load = [&](W4Piece<G, R>& p, int t) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int rt = min(first + i, row_tiles - 1);  // past the last: read again, not stored
      p.w[i] = load_stream16(a.w + (static_cast<size_t>(rt) * tiles + t) * kTileBytes + 16 * lane);
#pragma unroll
      for (int j = 0; j < kGroups; ++j) {
        const int group = min(t * kGroups + j, groups - 1);  // past the last: of columns x = 0
        const uint16_t* s = a.s + (static_cast<size_t>(rt) * groups + group) * kTileRows + 4 * g;
        p.s[i][j] = make_uint2(gload(reinterpret_cast<const uint32_t*>(s)),
                               gload(reinterpret_cast<const uint32_t*>(s) + 1));
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = t * kTileCols + 32 * i;
      p.x[i] = make_uint4(0, 0, 0, 0);
      if (col < a.k && r < a.tokens) {
        p.x[i] = load_global16(a.x + static_cast<size_t>(r) * a.k + col + 8 * g);
      }
    }
  };
  const bf16x8_t minus_1_5 =
      __builtin_bit_cast(bf16x8_t, make_uint4(0xBFC0BFC0u, 0xBFC0BFC0u, 0xBFC0BFC0u, 0xBFC0BFC0u));
  f32x4_t total[R];
#pragma unroll
  for (int i = 0; i < R; ++i) total[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  auto add = [&](const W4Piece<G, R>& p) {
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
      f32x4_t base{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        base = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            minus_1_5, __builtin_bit_cast(bf16x8_t, p.x[j * kSteps + i]), base, 0, 0, 0);
      }
#pragma unroll
      for (int t = 0; t < R; ++t) {
        f32x4_t d = base;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              widen_nibbles(word_of(p.w[t], j * kSteps + i)),
              __builtin_bit_cast(bf16x8_t, p.x[j * kSteps + i]), d, 0, 0, 0);
        }
        const uint2 s = p.s[t][j];
        total[t][0] = fmaf(bf16_lo(s.x), d[0], total[t][0]);
        total[t][1] = fmaf(bf16_hi(s.x), d[1], total[t][1]);
        total[t][2] = fmaf(bf16_lo(s.y), d[2], total[t][2]);
        total[t][3] = fmaf(bf16_hi(s.y), d[3], total[t][3]);
      }
    }
  };
  for (int t = wave; t < tiles; t += 2 * waves) {  // two tiles' loads in flight
    W4Piece<G, R> p0, p1;
    load(p0, t);
    const bool two = t + waves < tiles;
    if (two) load(p1, t + waves);
    add(p0);
    if (two) add(p1);
  }

  if (r < a.tokens) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      *reinterpret_cast<f32x4_t*>(partial + (wave * a.tokens + r) * kPitch + i * kTileRows + 4 * g) =
          total[i];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < kRows * a.tokens; e += blockDim.x) {
    const int t = e / kRows, i = e % kRows, row = first * kTileRows + i;
    if (row >= a.n) continue;
    float v = 0.0f;
    for (int w = 0; w < waves; ++w) v += partial[(w * a.tokens + t) * kPitch + i];
    v *= 16.0f;
    if (!__builtin_isfinite(v)) v = exact_dot(a, row, t);
    a.y[static_cast<size_t>(t) * a.n + row] =
        f32_to_bf16(a.bias ? v + bf16_to_f32(a.bias[row]) : v);
  }
}

// Waves of a workgroup: as few tiles each as `most` waves allow, and no wave
// without one.
int waves_for(int tiles, int most) {
  const int per = (tiles + most - 1) / most;
  return (tiles + per - 1) / per;
}

template <int G>
void launch_w4(const W4Args& a, hipStream_t stream) {
  const int row_tiles = (a.n + kTileRows - 1) / kTileRows;
  const int tiles = (a.k + kTileCols - 1) / kTileCols;
  auto launch = [&](auto rows, int most) {
    constexpr int R = decltype(rows)::value;
    const int waves = waves_for(tiles, most);
    const size_t lds = static_cast<size_t>(waves) * a.tokens * (R * kTileRows + 4) * sizeof(float);
    hipLaunchKernelGGL((w4a16_gemv_kernel<G, R>), dim3((row_tiles + R - 1) / R),
                       dim3(waves * kWave), lds, stream, a);
  };
  if (row_tiles >= 2048) {
    launch(std::integral_constant<int, 4>{}, 8);
  } else if (row_tiles >= 1024) {
    launch(std::integral_constant<int, 2>{}, 8);
  } else {
    launch(std::integral_constant<int, 1>{}, 16);
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
  if (group_size == 32) {
    launch_w4<32>(a, stream);
  } else if (group_size == 64) {
    launch_w4<64>(a, stream);
  } else {
    launch_w4<128>(a, stream);
  }
  return check_launch("gemv_w4a16");
}
