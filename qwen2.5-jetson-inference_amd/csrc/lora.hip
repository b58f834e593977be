// Low-rank adapters of many requests beside a shared projection, for gfx950
// (include/infer_batch.h).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "batch_kernels.hpp"
#include "device_common.hpp"

namespace qlin {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// output = base + s B (A x), token by token's adapter.
//
// Units.  The tokens are cut into chunks, and a unit is the tokens of a chunk that
// have one adapter, wherever they stand: they are gathered into tiles of 16, so that
// an adapter's A and B are read once for all of them and the products run on
// v_mfma_f32_16x16x32_bf16.  A unit is named by an adapter's number or by a token that
// is the first of its chunk with its adapter, whichever gives fewer; those without
// tokens end at once.  No sorting, nothing but the ids is read first, and a
// captured graph follows ids that change.
//
// h = s A x: 16 rows of A by 16 tokens a tile, K split over a workgroup's waves and
// joined in LDS in the order of the waves.  h is kept as high + low BF16 (2^-16 of it;
// one BF16 number alone would add as much error as the output's rounding) between
// the launches, and B h takes two products.
constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kTile = 16;         // tokens, and rows of A
constexpr int kMaxChunk = 1024;   // tokens
constexpr int kCols = 128;        // of B h a wave

// Words of a token's high (and low) part in the workspace: whole steps of the MFMA's K.
__host__ __device__ constexpr int rank_pitch(int max_rank) { return (max_rank + 31) / 32 * 32; }

struct Unit {
  int adapter;  // -1: none
  int count;    // of tokens; 0: no such unit
};

__device__ __forceinline__ int adapter_of(const LoraArgs& a, int id) {
  return static_cast<unsigned>(id) < static_cast<unsigned>(a.adapters) ? id : -1;
}

// The unit's tokens, as offsets from the chunk's first, in order.
__device__ Unit gather_tokens(const LoraArgs& a, int first, int unit, uint16_t* list) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int size = min(a.chunk, a.tokens - first);
  if (a.by_token && unit >= size) return {-1, 0};
  const int mine = a.by_token ? adapter_of(a, a.ids[first + unit]) : unit - 1;
  int count = 0;
  for (int base = 0; base < size; base += kWave) {
    const int t = base + lane;
    const bool has = t < size && adapter_of(a, a.ids[first + t]) == mine;
    const unsigned long long mask = __ballot(has);
    if (a.by_token && count == 0 && mask && base + __builtin_ctzll(mask) != unit) return {-1, 0};
    if (has && (base / kWave) % kWaves == wave) {
      list[count + __popcll(mask & ((1ull << lane) - 1))] = t;
    }
    count += __popcll(mask);
  }
  __syncthreads();
  return {mine, count};
}

__device__ __forceinline__ int rank_of(const LoraArgs& a, int adapter) {
  return a.ranks ? min(max(a.ranks[adapter], 0), a.max_rank) : a.max_rank;
}

__device__ __forceinline__ bf16x8_t as_bf16(const uint4& v) {
  return __builtin_bit_cast(bf16x8_t, v);
}

// Eight words from column k on, zero from `rank` on, whatever is there.
__device__ __forceinline__ uint4 cut_words(uint4 v, int k, int rank) {
  if (k + 8 <= rank) return v;
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (k + 2 * i >= rank) {
      w[i] = 0;
    } else if (k + 2 * i + 1 >= rank) {
      w[i] &= 0xFFFFu;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__global__ __launch_bounds__(kThreads) void lora_shrink_kernel(LoraArgs a) {
  __shared__ uint16_t list[kMaxChunk];
  __shared__ f32x4_t part[kWaves][kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int m = lane & 15, g = lane >> 4;
  const int first = blockIdx.x / a.units * a.chunk;
  const Unit u = gather_tokens(a, first, blockIdx.x % a.units, list);
  if (u.count == 0 || u.adapter < 0) return;
  const int rank_tiles = (a.max_rank + kTile - 1) / kTile;
  const int c = blockIdx.y / rank_tiles, rows = blockIdx.y % rank_tiles * kTile;
  const int rank = rank_of(a, u.adapter), pitch = rank_pitch(a.max_rank);
  const float scale = a.scales ? a.scales[u.adapter] : 1.0f;
  const uint16_t* w = a.target[c].a + (static_cast<size_t>(u.adapter) * a.max_rank +
                                       min(rows + m, a.max_rank - 1)) * a.k;
  const int steps = (a.k + 31) / 32;
  for (int tile = blockIdx.z; tile * kTile < u.count; tile += gridDim.z) {
    const int token = first + list[min(tile * kTile + m, u.count - 1)];
    const uint16_t* x = a.x + token * a.x_stride;
    f32x4_t sum{0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = wave; i < steps; i += kWaves) {
      const int k = 32 * i + 8 * g;
      uint4 p = make_uint4(0, 0, 0, 0), q = p;
      if (k < a.k) {
        p = load_global16(w + k);
        q = load_global16(x + k);
      }
      sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16(p), as_bf16(q), sum, 0, 0, 0);
    }
    __syncthreads();
    part[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && tile * kTile + m < u.count) {
      for (int i = 1; i < kWaves; ++i) sum += part[i][lane];
      uint32_t high[4], low[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float h = rows + 4 * g + i < rank ? sum[i] * scale : 0.0f;
        high[i] = f32_to_bf16(h);
        // an infinity has no remainder
        const float rest = h - bf16_to_f32(high[i]);
        low[i] = (high[i] & 0x7F80u) == 0x7F80u ? 0u : f32_to_bf16(rest);
      }
      uint16_t* h = a.h + (static_cast<size_t>(c) * a.tokens + token) * 2 * pitch + rows + 4 * g;
      store_global8(h, make_uint2(high[0] | high[1] << 16, high[2] | high[3] << 16));
      store_global8(h + pitch, make_uint2(low[0] | low[1] << 16, low[2] | low[3] << 16));
    }
  }
}

// KS: steps of 32 of the rank.  A wave takes 128 columns, lane m of each 16 the eight from
// 8 m on, one of each of eight products, so that a token's 128 outputs are stored 16 bytes a
// lane in a row.
template <int KS>
__global__ __launch_bounds__(kThreads) void lora_expand_kernel(LoraArgs a) {
  __shared__ uint16_t list[kMaxChunk];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int m = lane & 15, g = lane >> 4;
  const int first = blockIdx.x / a.units * a.chunk;
  const Unit u = gather_tokens(a, first, blockIdx.x % a.units, list);
  if (u.count == 0) return;
  int block = blockIdx.y * kWaves + wave, c = 0;
  while (c < a.targets && block * kCols >= a.target[c].n) {
    block -= (a.target[c].n + kCols - 1) / kCols;
    ++c;
  }
  if (c == a.targets) return;
  const LoraTarget& t = a.target[c];
  const int n0 = block * kCols + 8 * m;
  const int rank = u.adapter < 0 ? 0 : rank_of(a, u.adapter), pitch = rank_pitch(a.max_rank);
  if (rank == 0 && t.base == t.out) return;
  const bool wide = n0 + 8 <= t.n && (t.out_stride & 7) == 0 &&
                    (reinterpret_cast<uintptr_t>(t.out) & 15) == 0 &&
                    (!t.base || ((t.base_stride & 7) == 0 &&
                                 (reinterpret_cast<uintptr_t>(t.base) & 15) == 0));
  bf16x8_t w[KS][8];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int k = 32 * s + 8 * g;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (k < rank) {
        const size_t row = static_cast<size_t>(u.adapter) * t.n + min(n0 + j, t.n - 1);
        v = cut_words(load_global16(t.b + row * a.max_rank + k), k, rank);
      }
      w[s][j] = as_bf16(v);
    }
  }
  for (int tile = blockIdx.z; tile * kTile < u.count; tile += gridDim.z) {
    const int token = first + list[min(tile * kTile + m, u.count - 1)];
    f32x4_t sum[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const uint16_t* h = a.h + (static_cast<size_t>(c) * a.tokens + token) * 2 * pitch;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int k = 32 * s + 8 * g;
      uint4 high = make_uint4(0, 0, 0, 0), low = high;
      if (k < rank) {
        high = load_global16(h + k);
        low = load_global16(h + pitch + k);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sum[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16(low), w[s][j], sum[j], 0, 0, 0);
        sum[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16(high), w[s][j], sum[j], 0, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = tile * kTile + 4 * g + i;
      if (at >= u.count) break;
      const size_t to = first + list[at];
      uint16_t* out = t.out + to * t.out_stride + n0;
      const uint16_t* base = t.base ? t.base + to * t.base_stride + n0 : nullptr;
      if (wide) {
        uint4 b = base ? load_global16(base) : make_uint4(0, 0, 0, 0);
        if (rank) {
          b = make_uint4(pack2_bf16(bf16_lo(b.x) + sum[0][i], bf16_hi(b.x) + sum[1][i]),
                         pack2_bf16(bf16_lo(b.y) + sum[2][i], bf16_hi(b.y) + sum[3][i]),
                         pack2_bf16(bf16_lo(b.z) + sum[4][i], bf16_hi(b.z) + sum[5][i]),
                         pack2_bf16(bf16_lo(b.w) + sum[6][i], bf16_hi(b.w) + sum[7][i]));
        }
        store_global16(out, b);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (n0 + j >= t.n) continue;
          const uint16_t b = base ? base[j] : 0;
          out[j] = rank ? f32_to_bf16(bf16_to_f32(b) + sum[j][i]) : b;
        }
      }
    }
  }
}

}  // namespace

size_t lora_workspace_bytes(int tokens, int max_rank, int targets) {
  return static_cast<size_t>(targets) * tokens * 4 * rank_pitch(max_rank);
}

void launch_lora(LoraArgs a, hipStream_t stream) {
  a.chunk = min(a.tokens, kMaxChunk);
  const int chunks = (a.tokens + a.chunk - 1) / a.chunk;
  a.by_token = a.adapters + 1 > a.chunk;
  a.units = a.by_token ? a.chunk : a.adapters + 1;
  const int slots = a.tokens <= 256 ? 1 : 16;
  const int rank_tiles = (a.max_rank + kTile - 1) / kTile;
  hipLaunchKernelGGL(lora_shrink_kernel, dim3(chunks * a.units, a.targets * rank_tiles, slots),
                     dim3(kThreads), 0, stream, a);
  int blocks = 0;
  for (int i = 0; i < a.targets; ++i) blocks += (a.target[i].n + kCols - 1) / kCols;
  const dim3 grid(chunks * a.units, (blocks + kWaves - 1) / kWaves, slots);
  const int steps = rank_pitch(a.max_rank) / 32;
  auto run = [&](auto* kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, a);
  };
  steps == 1 ? run(lora_expand_kernel<1>)
  : steps == 2 ? run(lora_expand_kernel<2>)
  : steps == 3 ? run(lora_expand_kernel<3>)
               : run(lora_expand_kernel<4>);
}

}  // namespace qlin
