// Low-rank adapters of many requests beside a shared projection, for gfx950
// (include/infer_batch.h).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "batch_kernels.hpp"
#include "device_common.hpp"

namespace qlin {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// output = base + s B (A x), token by token's adapter.
//
// Units.  The tokens that have one adapter, wherever they stand, are gathered into tiles of
// 16, so that an adapter's A and B are read once for all of them and the products run on
// v_mfma_f32_16x16x32_bf16.  Of up to kGather tokens each workgroup finds its own by
// itself, with a ballot per 64 ids: a unit is an adapter's number, or a token that is the first
// with its adapter, whichever are fewer, and those without tokens end at once.  Of more a
// launch ahead groups each chunk of 1024 by a table in LDS.  Nothing is sorted, and a
// captured graph follows ids that change.
//
// h = s A x: 16 rows of A by 16 tokens a tile, K split over a workgroup's waves and
// joined in LDS in the order of the waves.  h is kept as high + low BF16 (2^-16 of it;
// one BF16 number alone would add as much error as the output's rounding), and B h takes
// two products.
constexpr int kTile = 16;       // tokens, and rows of A
constexpr int kGather = 256;    // tokens
constexpr int kChunk = 1024;    // tokens grouped together beyond
constexpr int kSet = 64;        // tokens of a unit then, at most
constexpr int kCols = 128;      // of B h a wave
constexpr int kExpandWaves = 4;

// Words of a token's high (and low) part in the workspace: whole steps of the MFMA's K.
__host__ __device__ constexpr int rank_pitch(int max_rank) { return (max_rank + 31) / 32 * 32; }

// A unit's tokens; `adapter` -1: none has one.
struct Unit {
  int adapter, count;
};

__device__ __forceinline__ int adapter_of(const LoraArgs& a, int id) {
  return static_cast<unsigned>(id) < static_cast<unsigned>(a.adapters) ? id : -1;
}

// Unit `unit`'s tokens in order, by all of the workgroup's waves; count 0: no such unit.
__device__ __forceinline__ Unit gather_tokens(const LoraArgs& a, int unit, int* list) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  int id[kGather / kWave];
#pragma unroll
  for (int i = 0; i < kGather / kWave; ++i) {
    const int t = i * kWave + lane;
    id[i] = t < a.tokens ? adapter_of(a, a.ids[t]) : -2;
  }
  const int mine = a.by_token ? adapter_of(a, a.ids[unit]) : unit - 1;
  int count = 0, first = -1;
#pragma unroll
  for (int i = 0; i < kGather / kWave; ++i) {
    const unsigned long long mask = __ballot(id[i] == mine);
    if (first < 0 && mask) first = i * kWave + __builtin_ctzll(mask);
    if (id[i] == mine && wave == 0) {
      list[count + __popcll(mask & ((1ull << lane) - 1))] = i * kWave + lane;
    }
    count += __popcll(mask);
  }
  if (a.by_token && first != unit) return {-1, 0};
  __syncthreads();
  return {mine, count};
}

// The groups that a launch ahead has made: of each chunk `sets[chunk]` units, each an
// adapter, the place of its first token in `order`, and the number of them.
struct Groups {
  int* sets;    // [chunks]
  int* order;   // [tokens]
  int4* units;  // [chunks][units of a chunk]
};

__host__ __device__ inline Groups groups_of(const LoraArgs& a) {
  const int chunks = (a.tokens + kChunk - 1) / kChunk;
  return {a.groups, a.groups + (chunks + 3) / 4 * 4,
          reinterpret_cast<int4*>(a.groups + (chunks + 3) / 4 * 4 + (a.tokens + 3) / 4 * 4)};
}

__device__ __forceinline__ Unit grouped_tokens(const LoraArgs& a, int unit, int* list) {
  const Groups g = groups_of(a);
  const int chunk = unit / a.units;
  if (unit % a.units >= g.sets[chunk]) return {-1, 0};
  const int4 u = g.units[unit];
  if (static_cast<int>(threadIdx.x) < u.z) list[threadIdx.x] = g.order[u.y + threadIdx.x];
  __syncthreads();
  return {u.x, u.z};
}

template <bool GROUPED>
__device__ __forceinline__ Unit tokens_of(const LoraArgs& a, int unit, int* list) {
  return GROUPED ? grouped_tokens(a, unit, list) : gather_tokens(a, unit, list);
}

// A chunk's tokens by adapter: a table of the chunk's adapters in LDS (twice as many
// places as tokens, searched on from the adapter's own), how many tokens have each and
// which of them a token is, in whatever order they come: it says only in which column
// of a product a token stands.
__global__ __launch_bounds__(kChunk) void lora_group_kernel(LoraArgs a) {
  constexpr int kPlaces = 2 * kChunk, kWaves = kChunk / kWave;
  __shared__ int key[kPlaces], size[kPlaces];
  __shared__ int start[kPlaces], unit[kPlaces];
  __shared__ int wave_tokens[kWaves], wave_units[kWaves];
  const Groups out = groups_of(a);
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int first = blockIdx.x * kChunk, t = first + threadIdx.x;
  for (int i = threadIdx.x; i < kPlaces; i += kChunk) {
    key[i] = -2;
    size[i] = 0;
  }
  __syncthreads();
  int place = 0, nth = 0;
  if (t < a.tokens) {
    const int id = adapter_of(a, a.ids[t]);
    place = (static_cast<unsigned>(id) * 2654435761u >> 16) % kPlaces;
    for (;;) {  // at most kChunk adapters in kPlaces places
      const int was = atomicCAS(&key[place], -2, id);
      if (was == -2 || was == id) break;
      place = (place + 1) % kPlaces;
    }
    nth = atomicAdd(&size[place], 1);
  }
  __syncthreads();
  const int n0 = size[2 * threadIdx.x], n1 = size[2 * threadIdx.x + 1];
  const int u0 = (n0 + kSet - 1) / kSet, u1 = (n1 + kSet - 1) / kSet;
  int tokens = n0 + n1, units = u0 + u1;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int x = __shfl_up(tokens, d), y = __shfl_up(units, d);
    if (lane >= d) {
      tokens += x;
      units += y;
    }
  }
  if (lane == kWave - 1) {
    wave_tokens[wave] = tokens;
    wave_units[wave] = units;
  }
  __syncthreads();
  int all = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) {
      tokens += wave_tokens[w];
      units += wave_units[w];
    }
    all += wave_units[w];
  }
  start[2 * threadIdx.x] = tokens - n0 - n1;
  start[2 * threadIdx.x + 1] = tokens - n1;
  unit[2 * threadIdx.x] = units - u0 - u1;
  unit[2 * threadIdx.x + 1] = units - u1;
  if (threadIdx.x == 0) out.sets[blockIdx.x] = all;
  __syncthreads();
  if (t < a.tokens) {
    const int at = first + start[place] + nth;
    out.order[at] = t;
    if (nth % kSet == 0) {  // a unit's first
      out.units[blockIdx.x * a.units + unit[place] + nth / kSet] =
          make_int4(key[place], at, min(kSet, size[place] - nth), 0);
    }
  }
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

// A wave's share of RT tiles of rows of A by the tile's tokens: steps of 32 columns,
// each wave neighbouring ones, whose loads are on their way together.
template <int RT>
__device__ __forceinline__ void shrink_steps(f32x4_t (&sum)[RT], const LoraArgs& a,
                                             const uint16_t* const (&w)[RT], const uint16_t* x,
                                             int wave, int waves, int g) {
  constexpr int kDepth = RT >= 4 ? 2 : RT == 2 ? 4 : 8;
  const int steps = (a.k + 31) / 32, each = (steps + waves - 1) / waves;
  const int end = min(steps, (wave + 1) * each);
#pragma unroll
  for (int r = 0; r < RT; ++r) sum[r] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  for (int base = wave * each; base < end; base += kDepth) {
    uint4 p[kDepth][RT], q[kDepth];
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      const int k = 32 * (base + i) + 8 * g;
      const bool in = base + i < end && k < a.k;
      q[i] = make_uint4(0, 0, 0, 0);
      if (in) q[i] = load_global16(x + k);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        p[i][r] = make_uint4(0, 0, 0, 0);
        if (in) p[i][r] = load_global16(w[r] + k);
      }
    }
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        sum[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16(p[i][r]), as_bf16(q[i]), sum[r],
                                                         0, 0, 0);
      }
    }
  }
}

// h as high + low BF16; an infinity has no remainder.
__device__ __forceinline__ void split_word(float h, uint16_t& high, uint16_t& low) {
  high = f32_to_bf16(h);
  low = (high & 0x7F80u) == 0x7F80u ? 0 : f32_to_bf16(h - bf16_to_f32(high));
}

template <int RT, int WAVES, bool GROUPED>
__global__ __launch_bounds__(WAVES * kWave) void lora_shrink_kernel(LoraArgs a) {
  __shared__ int list[GROUPED ? kSet : kGather];
  __shared__ f32x4_t part[WAVES][RT][kWave];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int m = lane & 15, g = lane >> 4;
  const Unit u = tokens_of<GROUPED>(a, blockIdx.x, list);
  if (u.count == 0 || u.adapter < 0) return;
  const int blocks = (a.max_rank + RT * kTile - 1) / (RT * kTile);
  const int c = blockIdx.y / blocks, rows = blockIdx.y % blocks * RT * kTile;
  const int rank = rank_of(a, u.adapter), pitch = rank_pitch(a.max_rank);
  const float scale = a.scales ? a.scales[u.adapter] : 1.0f;
  const uint16_t* w[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    w[r] = a.target[c].a + (static_cast<size_t>(u.adapter) * a.max_rank +
                            min(rows + r * kTile + m, a.max_rank - 1)) * a.k;
  }
  for (int tile = blockIdx.z; tile * kTile < u.count; tile += gridDim.z) {
    f32x4_t sum[RT];
    shrink_steps<RT>(sum, a, w, a.x + list[min(tile * kTile + m, u.count - 1)] * a.x_stride, wave,
                     WAVES, g);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RT; ++r) part[wave][r][lane] = sum[r];
    __syncthreads();
    // element e of a tile: row 4 (e / 64) + e % 4 of token e / 4 % 16
    for (int e = threadIdx.x; e < RT * kTile * kTile; e += WAVES * kWave) {
      const float* p = reinterpret_cast<const float*>(part) + e;
      float h = p[0];
#pragma unroll
      for (int i = 1; i < WAVES; ++i) h += p[i * RT * kWave * 4];
      const int in = e % (kTile * kTile);
      const int row = rows + e / (kTile * kTile) * kTile + in / 64 * 4 + in % 4;
      const int at = tile * kTile + in / 4 % 16;
      if (at < u.count && row < pitch) {
        uint16_t high, low;
        split_word(row < rank ? h * scale : 0.0f, high, low);
        uint16_t* to =
            a.h + (static_cast<size_t>(c) * a.tokens + list[at]) * 2 * pitch + row;
        to[0] = high;
        to[pitch] = low;
      }
    }
  }
}

// KS: steps of 32 of the rank.  A wave takes 128 columns, lane m of each 16 the eight from
// 8 m on, one of each of eight products, so that a token's 128 outputs are loaded and
// stored 16 bytes a lane in a row.
template <int KS>
struct Columns {
  const LoraTarget& t;
  int n0, rank;
  bool wide;  // whole, and aligned
  bf16x8_t w[KS][8];

  __device__ __forceinline__ Columns(const LoraArgs& a, const LoraTarget& target, int block,
                                     int adapter, int lane)
      : t(target), n0(block * kCols + 8 * (lane & 15)), rank(0) {
    if (adapter >= 0) rank = rank_of(a, adapter);
    wide = n0 + 8 <= t.n && (t.out_stride & 7) == 0 &&
           (reinterpret_cast<uintptr_t>(t.out) & 15) == 0 &&
           (!t.base ||
            ((t.base_stride & 7) == 0 && (reinterpret_cast<uintptr_t>(t.base) & 15) == 0));
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int k = 32 * s + 8 * (lane >> 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (k < rank) {
          const size_t row = static_cast<size_t>(adapter) * t.n + min(n0 + j, t.n - 1);
          v = load_global16(t.b + row * a.max_rank + k);
        }
        w[s][j] = as_bf16(v);
      }
    }
  }
  __device__ __forceinline__ void cut(int lane) {
    if (rank % 8 == 0) return;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int k = 32 * s + 8 * (lane >> 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[s][j] = as_bf16(cut_words(__builtin_bit_cast(uint4, w[s][j]), k, rank));
      }
    }
  }
  __device__ __forceinline__ uint4 base_of(int token) const {
    return wide && t.base ? load_global16(t.base + token * t.base_stride + n0)
                          : make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void multiply(f32x4_t (&sum)[8], const uint4 (&high)[KS],
                                           const uint4 (&low)[KS]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sum[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16(low[s]), w[s][j], sum[j], 0, 0, 0);
        sum[j] =
            __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16(high[s]), w[s][j], sum[j], 0, 0, 0);
      }
    }
  }
  // Row i of the sums is the token's.
  __device__ __forceinline__ void store(int token, const f32x4_t (&sum)[8], int i, uint4 b) const {
    uint16_t* out = t.out + token * t.out_stride + n0;
    if (wide) {
      if (rank) {
        b = make_uint4(pack2_bf16(bf16_lo(b.x) + sum[0][i], bf16_hi(b.x) + sum[1][i]),
                       pack2_bf16(bf16_lo(b.y) + sum[2][i], bf16_hi(b.y) + sum[3][i]),
                       pack2_bf16(bf16_lo(b.z) + sum[4][i], bf16_hi(b.z) + sum[5][i]),
                       pack2_bf16(bf16_lo(b.w) + sum[6][i], bf16_hi(b.w) + sum[7][i]));
      }
      store_global16(out, b);
      return;
    }
    const uint16_t* base = t.base ? t.base + token * t.base_stride + n0 : nullptr;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (n0 + j >= t.n) continue;
      const uint16_t v = base ? base[j] : 0;
      out[j] = rank ? f32_to_bf16(bf16_to_f32(v) + sum[j][i]) : v;
    }
  }
};

// Block `block` of 128 columns over all targets: the target and the block within it;
// -1 past the last.
__device__ __forceinline__ int target_of(const LoraArgs& a, int& block) {
  for (int c = 0; c < a.targets; ++c) {
    const int blocks = (a.target[c].n + kCols - 1) / kCols;
    if (block < blocks) return c;
    block -= blocks;
  }
  return -1;
}

template <int KS, bool GROUPED>
__global__ __launch_bounds__(kExpandWaves * kWave) void lora_expand_kernel(LoraArgs a) {
  __shared__ int list[GROUPED ? kSet : kGather];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int m = lane & 15, g = lane >> 4;
  const Unit u = tokens_of<GROUPED>(a, blockIdx.x, list);
  if (u.count == 0) return;
  int block = blockIdx.y * kExpandWaves + wave;
  const int c = target_of(a, block);
  if (c < 0) return;
  const LoraTarget& t = a.target[c];
  if (u.adapter < 0 && t.base == t.out) return;
  Columns<KS> columns(a, t, block, u.adapter, lane);
  const int rank = columns.rank, pitch = rank_pitch(a.max_rank);
  // A tile's h and bases are loaded while the one before it is computed.
  struct Tile {
    uint4 high[KS], low[KS], base[4];
  };
  auto load = [&](Tile& v, int tile) {
    const int token = list[min(tile * kTile + m, u.count - 1)];
    const uint16_t* h = a.h + (static_cast<size_t>(c) * a.tokens + token) * 2 * pitch;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int k = 32 * s + 8 * g;
      v.high[s] = v.low[s] = make_uint4(0, 0, 0, 0);
      if (k < rank) {
        v.high[s] = load_global16(h + k);
        v.low[s] = load_global16(h + pitch + k);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v.base[i] = columns.base_of(list[min(tile * kTile + 4 * g + i, u.count - 1)]);
    }
  };
  const int step = gridDim.z;
  int tile = blockIdx.z;
  if (tile * kTile >= u.count) return;
  Tile now, next;
  load(next, tile);
  columns.cut(lane);
  for (; tile * kTile < u.count; tile += step) {
    now = next;
    if ((tile + step) * kTile < u.count) load(next, tile + step);
    f32x4_t sum[8];
    columns.multiply(sum, now.high, now.low);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = tile * kTile + 4 * g + i;
      if (at < u.count) columns.store(list[at], sum, i, now.base[i]);
    }
  }
}

int chunks_of(int tokens) { return (tokens + kChunk - 1) / kChunk; }
int units_of(int tokens, int adapters) {  // of a chunk
  return (kChunk + kSet - 1) / kSet + std::min(std::min(tokens, kChunk), adapters + 1);
}

size_t h_bytes(int tokens, int max_rank, int targets) {
  return static_cast<size_t>(targets) * tokens * 4 * rank_pitch(max_rank);
}

}  // namespace

size_t lora_workspace_bytes(int tokens, int max_rank, int targets) {
  size_t bytes = h_bytes(tokens, max_rank, targets);
  if (tokens > kGather) {
    const size_t chunks = chunks_of(tokens);
    bytes += 4 * ((chunks + 3) / 4 * 4 + (static_cast<size_t>(tokens) + 3) / 4 * 4) +
             16 * chunks * units_of(tokens, kChunk);
  }
  return bytes;
}

void launch_lora(LoraArgs a, hipStream_t stream) {
  const int rank_tiles = (a.max_rank + kTile - 1) / kTile;
  const int steps = rank_pitch(a.max_rank) / 32;
  int blocks = 0;
  for (int i = 0; i < a.targets; ++i) blocks += (a.target[i].n + kCols - 1) / kCols;
  blocks = (blocks + kExpandWaves - 1) / kExpandWaves;
  if (a.tokens > kGather) {
    a.groups = reinterpret_cast<int*>(reinterpret_cast<char*>(a.h) +
                                      h_bytes(a.tokens, a.max_rank, a.targets));
    a.units = units_of(a.tokens, a.adapters);
    const int chunks = chunks_of(a.tokens), units = chunks * a.units;
    hipLaunchKernelGGL(lora_group_kernel, dim3(chunks), dim3(kChunk), 0, stream, a);
    auto shrink = [&](auto* kernel, int tiles) {
      hipLaunchKernelGGL(kernel, dim3(units, a.targets * ((rank_tiles + tiles - 1) / tiles),
                                      kSet / kTile),
                         dim3(8 * kWave), 0, stream, a);
    };
    rank_tiles == 1   ? shrink(lora_shrink_kernel<1, 8, true>, 1)
    : rank_tiles == 2 ? shrink(lora_shrink_kernel<2, 8, true>, 2)
                      : shrink(lora_shrink_kernel<4, 8, true>, 4);
    auto expand = [&](auto* kernel) {
      hipLaunchKernelGGL(kernel, dim3(units, blocks), dim3(kExpandWaves * kWave), 0, stream, a);
    };
    steps == 1   ? expand(lora_expand_kernel<1, true>)
    : steps == 2 ? expand(lora_expand_kernel<2, true>)
    : steps == 3 ? expand(lora_expand_kernel<3, true>)
                 : expand(lora_expand_kernel<4, true>);
    return;
  }
  a.by_token = a.adapters + 1 > a.tokens;
  a.units = a.by_token ? a.tokens : a.adapters + 1;
  // workgroups side by side for a unit's tiles, as many as it has if units are alike
  const int tiles = (a.tokens + kTile - 1) / kTile;
  const int slots = std::min(tiles, 1 + a.tokens / (kTile * a.units));
  hipLaunchKernelGGL((lora_shrink_kernel<1, 16, false>),
                     dim3(a.units, a.targets * rank_tiles, slots), dim3(16 * kWave), 0, stream, a);
  auto expand = [&](auto* kernel) {
    hipLaunchKernelGGL(kernel, dim3(a.units, blocks, slots), dim3(kExpandWaves * kWave), 0, stream,
                       a);
  };
  steps == 1   ? expand(lora_expand_kernel<1, false>)
  : steps == 2 ? expand(lora_expand_kernel<2, false>)
  : steps == 3 ? expand(lora_expand_kernel<3, false>)
               : expand(lora_expand_kernel<4, false>);
}

}  // namespace qlin
