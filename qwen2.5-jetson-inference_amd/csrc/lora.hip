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
// h = s A x: 16 rows of A by 16 tokens a tile, K split over a workgroup's 16 waves and
// joined in LDS in the order of the waves, and over up to kMostParts workgroups where there
// are few.  h is kept as high + low BF16 (2^-16 of it; one BF16 number alone would add as
// much error as the output's rounding), and B h takes two products.
//
// Small calls take one launch, up to kGather tokens two, more three.  What bounds them, in
// us: one launch its reads one behind the other (ids, rows, then the join; 1 x 896 x 896 at
// rank 8 6.7 of which 1.7 an empty launch, 33 tokens' q, k and v of 1536 at rank 16 7.8);
// A x the same and a CU's loads (128 x 3584 by 2 x 64 rows 7.6; 6001 x 1536 by 32 8.6); B h
// its bytes (128 x 2 x 18944 at rank 64 18.0 for 75 MB, 4.2 TB/s; 6001 x 8960 at rank 32
// 45 for 216 MB, 4.8, a copy 5.07); grouping 3.2-4.7, a launch and LDS atomics.
constexpr int kTile = 16;       // tokens, and rows of A
constexpr int kGather = 256;    // tokens
constexpr int kChunk = 1024;    // tokens grouped together beyond
constexpr int kSet = 64;        // tokens of a unit then, at most
constexpr int kPartWaves = 4;
constexpr int kCus = 256;
// A part's columns, at least: a workgroup's chunk is 1024, and 64 x 896 at rank 64 took 9.7
// us in two parts, 8.9 in one.
constexpr int kMostParts = 4, kPartColumns = 768;

// Words of a token's high (and low) part in the workspace: whole steps of the MFMA's K.
__host__ __device__ constexpr int rank_pitch(int max_rank) { return (max_rank + 31) / 32 * 32; }

// A unit's tokens; `adapter` -1: none has one (and its rank is 0).
struct Unit {
  int adapter, count, rank;
  float scale;
};

__device__ __forceinline__ int adapter_of(const LoraArgs& a, int id) {
  return static_cast<unsigned>(id) < static_cast<unsigned>(a.adapters) ? id : -1;
}

__device__ __forceinline__ Unit unit_of(const LoraArgs& a, int adapter, int count) {
  Unit u{adapter, count, 0, 1.0f};
  if (adapter >= 0) {
    u.rank = a.ranks ? min(max(a.ranks[adapter], 0), a.max_rank) : a.max_rank;
    if (a.scales) u.scale = a.scales[adapter];
  }
  return u;
}

// Unit `unit`'s tokens in order, by all of the workgroup's waves; count 0: no such unit.
__device__ __forceinline__ Unit gather_tokens(const LoraArgs& a, int unit, int* list) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  int id[kGather / kWave];
#pragma unroll
  for (int i = 0; i < kGather / kWave; ++i) {
    const int t = i * kWave + lane;
    id[i] = -2;
    if (i * kWave < a.tokens && t < a.tokens) id[i] = adapter_of(a, a.ids[t]);
  }
  const int mine = a.by_token ? adapter_of(a, a.ids[unit]) : unit - 1;
  Unit u = unit_of(a, mine, 0);  // on its way while the ids are compared
  int first = -1;
#pragma unroll
  for (int i = 0; i < kGather / kWave; ++i) {
    if (i * kWave >= a.tokens) break;
    const unsigned long long mask = __ballot(id[i] == mine);
    if (first < 0 && mask) first = i * kWave + __builtin_ctzll(mask);
    if (id[i] == mine && wave == 0) {
      list[u.count + __popcll(mask & ((1ull << lane) - 1))] = i * kWave + lane;
    }
    u.count += __popcll(mask);
  }
  if (a.by_token && first != unit) return Unit{-1, 0, 0, 1.0f};
  __syncthreads();
  return u;
}

// The groups that a launch ahead has made: units, each an adapter, the place of its first
// token in `order`, and the number of them (0: none).
struct Groups {
  int* order;   // [tokens]
  int4* units;  // [chunks][units of a chunk]
};

__host__ __device__ inline Groups groups_of(const LoraArgs& a) {
  return {a.groups, reinterpret_cast<int4*>(a.groups + (a.tokens + 3) / 4 * 4)};
}

__device__ __forceinline__ Unit grouped_tokens(const LoraArgs& a, int unit, int* list) {
  const Groups g = groups_of(a);
  const int4 v = g.units[unit];
  const int t = threadIdx.x;
  int token = 0;
  if (t < v.z) token = g.order[v.y + t];
  const Unit u = unit_of(a, v.x, v.z);
  if (t < v.z) list[t] = token;
  __syncthreads();
  return u;
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
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
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
    // a wave of one adapter, as in a prompt, asks once: 64 lanes at one address would wait
    // for each other
    const bool alike = !__ballot(id != __builtin_amdgcn_readfirstlane(id));
    const int lanes = __popcll(__ballot(true));
    if (!alike || lane == 0) {
      for (;;) {  // at most kChunk adapters in kPlaces places
        const int was = atomicCAS(&key[place], -2, id);
        if (was == -2 || was == id) break;
        place = (place + 1) % kPlaces;
      }
      nth = atomicAdd(&size[place], alike ? lanes : 1);
    }
    if (alike) {
      place = __builtin_amdgcn_readfirstlane(place);
      nth = __builtin_amdgcn_readfirstlane(nth) + lane;
    }
  }
  __syncthreads();
  const int n0 = size[2 * threadIdx.x], n1 = size[2 * threadIdx.x + 1];
  const int u0 = (n0 + kSet - 1) / kSet, u1 = (n1 + kSet - 1) / kSet;
  int tokens = wave_scan(static_cast<unsigned>(n0 + n1));
  int units = wave_scan(static_cast<unsigned>(u0 + u1));
  if (lane == kWave - 1) {
    wave_tokens[wave] = tokens;
    wave_units[wave] = units;
  }
  __syncthreads();
  const unsigned tokens_in = wave_scan(lane < kWaves ? unsigned(wave_tokens[lane]) : 0u);
  const unsigned units_in = wave_scan(lane < kWaves ? unsigned(wave_units[lane]) : 0u);
  const int all = __builtin_amdgcn_readlane(static_cast<int>(units_in), kWave - 1);
  if (wave) {
    tokens += __builtin_amdgcn_readlane(static_cast<int>(tokens_in), wave - 1);
    units += __builtin_amdgcn_readlane(static_cast<int>(units_in), wave - 1);
  }
  start[2 * threadIdx.x] = tokens - n0 - n1;
  start[2 * threadIdx.x + 1] = tokens - n1;
  unit[2 * threadIdx.x] = units - u0 - u1;
  unit[2 * threadIdx.x + 1] = units - u1;
  for (int i = all + threadIdx.x; i < a.units; i += kChunk) {
    out.units[blockIdx.x * a.units + i] = make_int4(-1, 0, 0, 0);
  }
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

// h of RT (1 or 2) tiles of rows of A by a tile's tokens, by 16 waves.  Each wave loads whole
// rows, a KB in a row (as operands, 16 rows side by side, they would cost the CU's address
// unit four times as much), into LDS, a chunk of columns at a time with kDepth of them on
// their way; there it takes its steps of the chunk for all rows.  Two workgroups share a
// CU, by LDS and by registers (12000 x 1536 at rank 32: one 49.3 us with all of the call,
// two 42.8; four tiles at a time, one to a CU, 2000 x 3584 at rank 128 51.1 us, 43.8).
constexpr int kShrinkWaves = 16;

template <int RT>
struct Stage {
  static constexpr int kLoads = RT == 1 ? 2 : 1;  // of a row's chunk
  static constexpr int kColumns = 512 * kLoads;
  static constexpr int kDepth = 2;
  static constexpr int kSteps = kColumns / 32 / kShrinkWaves;  // of a wave
  static constexpr int kPitch = kColumns + 8;
  union {
    __align__(16) uint16_t rows[(RT + 1) * kTile][kPitch];
    f32x4_t part[kShrinkWaves][RT][kWave];
  };
};

// rows: those of A that the wave loads, row `wave` of each tile, and its token's x, from
// the first of `columns` on.
template <int RT>
__device__ __forceinline__ void shrink_tile(f32x4_t (&sum)[RT], int columns,
                                            const uint16_t* const (&rows)[RT + 1],
                                            Stage<RT>& stage, int wave, int lane) {
  typedef Stage<RT> S;
  const int chunks = (columns + S::kColumns - 1) / S::kColumns;
  uint4 v[S::kDepth][RT + 1][S::kLoads];
  auto load = [&](uint4 (&to)[RT + 1][S::kLoads], int chunk) {
#pragma unroll
    for (int i = 0; i <= RT; ++i) {
#pragma unroll
      for (int j = 0; j < S::kLoads; ++j) {
        const int k = chunk * S::kColumns + 512 * j + 8 * lane;
        to[i][j] = make_uint4(0, 0, 0, 0);
        if (k < columns) to[i][j] = load_global16(rows[i] + k);
      }
    }
  };
#pragma unroll
  for (int d = 0; d < S::kDepth; ++d) {
    if (d < chunks) load(v[d], d);
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) sum[r] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  for (int base = 0; base < chunks; base += S::kDepth) {
#pragma unroll
    for (int d = 0; d < S::kDepth; ++d) {
      if (base + d >= chunks) break;
      lds_barrier();
#pragma unroll
      for (int i = 0; i <= RT; ++i) {
#pragma unroll
        for (int j = 0; j < S::kLoads; ++j) {
          *reinterpret_cast<uint4*>(&stage.rows[i * kTile + wave][512 * j + 8 * lane]) = v[d][i][j];
        }
      }
      lds_barrier();
      if (base + d + S::kDepth < chunks) load(v[d], base + d + S::kDepth);
#pragma unroll
      for (int s = 0; s < S::kSteps; ++s) {
        const int k = 32 * (wave * S::kSteps + s) + 8 * (lane >> 4);
        auto piece = [&](int i) {
          return as_bf16(
              *reinterpret_cast<const uint4*>(&stage.rows[i * kTile + (lane & 15)][k]));
        };
        const bf16x8_t x = piece(RT);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          sum[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(piece(r), x, sum[r], 0, 0, 0);
        }
      }
    }
  }
  lds_barrier();
#pragma unroll
  for (int r = 0; r < RT; ++r) stage.part[wave][r][lane] = sum[r];
  lds_barrier();
}

// Element e of the tile's h, row 16 (e / 256) + 4 (e / 64 % 4) + e % 4 of token e / 4 % 16:
// the waves' sums in order.
template <int RT>
__device__ __forceinline__ float joined(const Stage<RT>& stage, int e) {
  const float* p = reinterpret_cast<const float*>(stage.part) + e;
  float h = p[0];
#pragma unroll
  for (int i = 1; i < kShrinkWaves; ++i) h += p[i * RT * kWave * 4];
  return h;
}
__device__ __forceinline__ int row_of(int e) { return e / 256 * kTile + e / 64 % 4 * 4 + e % 4; }
__device__ __forceinline__ int token_of(int e) { return e / 4 % 16; }

// h as high + low BF16; an infinity has no remainder, and where h rounds to one the largest
// number is high.
__device__ __forceinline__ void split_word(float h, uint16_t& high, uint16_t& low) {
  high = f32_to_bf16(h);
  if ((high & 0x7FFFu) == 0x7F80u && fabsf(h) < INFINITY) --high;
  low = (high & 0x7F80u) == 0x7F80u ? 0 : f32_to_bf16(h - bf16_to_f32(high));
}

// The rows of A that a wave loads of RT tiles from tile `first` on, of all targets' one
// after the other (past the last: that one again).
template <int RT>
__device__ __forceinline__ void stage_rows(const uint16_t* (&rows)[RT + 1], const LoraArgs& a,
                                           int adapter, int first, int wave) {
  const int tiles = (a.max_rank + kTile - 1) / kTile;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int q = min(first + r, a.targets * tiles - 1);
    rows[r] = a.target[q / tiles].a +
              (static_cast<size_t>(max(adapter, 0)) * a.max_rank +
               min(q % tiles * kTile + wave, a.max_rank - 1)) * a.k;
  }
}

template <int RT, bool GROUPED>
__global__ __launch_bounds__(kShrinkWaves * kWave, 8) void lora_shrink_kernel(LoraArgs a) {
  extern __shared__ __align__(16) char shared[];
  Stage<RT>& stage = *reinterpret_cast<Stage<RT>*>(shared);
  int* const list = reinterpret_cast<int*>(shared + sizeof(Stage<RT>));
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const Unit u = tokens_of<GROUPED>(a, blockIdx.x, list);
  if (u.count == 0 || u.rank == 0) return;
  const int tiles = (a.max_rank + kTile - 1) / kTile, first = blockIdx.y * RT;
  const int pitch = rank_pitch(a.max_rank);
  const uint16_t* rows[RT + 1];
  stage_rows<RT>(rows, a, u.adapter, first, wave);
  for (int tile = blockIdx.z; tile * kTile < u.count; tile += gridDim.z) {
    const int token = list[min(tile * kTile + wave, u.count - 1)];
    rows[RT] = a.x + token * a.x_stride;
    f32x4_t sum[RT];
    shrink_tile<RT>(sum, a.k, rows, stage, wave, lane);
    for (int e = threadIdx.x; e < RT * kTile * kTile; e += kShrinkWaves * kWave) {
      const float h = joined<RT>(stage, e);
      const int q = first + row_of(e) / kTile, c = q / tiles;
      const int row = q % tiles * kTile + row_of(e) % kTile, at = tile * kTile + token_of(e);
      if (at < u.count && c < a.targets) {
        uint16_t high, low;
        split_word(row < u.rank ? h * u.scale : 0.0f, high, low);
        uint16_t* to = a.h + (static_cast<size_t>(c) * a.tokens + list[at]) * 2 * pitch + row;
        to[0] = high;
        to[pitch] = low;
      }
    }
  }
}

// Of up to kGather tokens, where units are few: A x in a.parts of K, one to a workgroup, each
// written in 32 bits; B h adds them up.
__host__ __device__ inline int part_columns(const LoraArgs& a) {
  return ((a.k + a.parts - 1) / a.parts + 63) / 64 * 64;
}

__global__ __launch_bounds__(kShrinkWaves * kWave) void lora_shrink_part_kernel(LoraArgs a) {
  extern __shared__ __align__(16) char shared[];
  Stage<1>& stage = *reinterpret_cast<Stage<1>*>(shared);
  int* const list = reinterpret_cast<int*>(shared + sizeof(Stage<1>));
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const Unit u = gather_tokens(a, blockIdx.x, list);
  if (u.count == 0 || u.rank == 0) return;
  const int tiles = (a.max_rank + kTile - 1) / kTile;
  const int part = blockIdx.y % a.parts, q = blockIdx.y / a.parts;
  const int from = part * part_columns(a), columns = min(part_columns(a), a.k - from);
  const int pitch = rank_pitch(a.max_rank);
  const uint16_t* rows[2];
  stage_rows<1>(rows, a, u.adapter, q, wave);
  rows[0] += from;
  float* const h = reinterpret_cast<float*>(a.h) +
                   (static_cast<size_t>(part) * a.targets + q / tiles) * a.tokens * pitch;
  for (int tile = blockIdx.z; tile * kTile < u.count; tile += gridDim.z) {
    rows[1] = a.x + list[min(tile * kTile + wave, u.count - 1)] * a.x_stride + from;
    f32x4_t sum[1];
    shrink_tile<1>(sum, columns, rows, stage, wave, lane);
    const int e = threadIdx.x, at = tile * kTile + token_of(e);
    if (e < kTile * kTile && at < u.count) {
      h[static_cast<size_t>(list[at]) * pitch + q % tiles * kTile + row_of(e)] =
          joined<1>(stage, e);
    }
  }
}

// KS: steps of 32 of the rank.  A wave takes 16 J columns, lane m of each 16 the J from
// J m on, one of each of J products, so that a token's outputs are loaded and stored 2 J
// bytes a lane in a row.
template <int J>
struct Words;
template <>
struct Words<8> {
  typedef u32x4 type;
  typedef uint32_t memory __attribute__((ext_vector_type(4), aligned(2)));
};
template <>
struct Words<4> {
  typedef uint32_t type __attribute__((ext_vector_type(2)));
  typedef uint32_t memory __attribute__((ext_vector_type(2), aligned(2)));
};

template <int KS, int J, bool ONCE>
struct Columns {
  typedef typename Words<J>::type words;
  typedef typename Words<J>::memory memory;
  const LoraTarget& t;
  int n0, rank;
  bool whole;
  bf16x8_t w[KS][J];

  __device__ __forceinline__ Columns(const LoraArgs& a, const LoraTarget& target, int block,
                                     const Unit& u, int lane)
      : t(target), n0(block * J * 16 + J * (lane & 15)), rank(u.rank) {
    whole = n0 + J <= t.n;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int k = 32 * s + 8 * (lane >> 4);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (k < rank) {
          const size_t row = static_cast<size_t>(u.adapter) * t.n + min(n0 + j, t.n - 1);
          v = load_global16(t.b + row * a.max_rank + k);
        }
        w[s][j] = as_bf16(v);
      }
    }
  }
  // Columns of B from the adapter's rank on as zeros.
  __device__ __forceinline__ void cut(int lane) {
    if (rank % 8 == 0) return;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int k = 32 * s + 8 * (lane >> 4);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        w[s][j] = as_bf16(cut_words(__builtin_bit_cast(uint4, w[s][j]), k, rank));
      }
    }
  }
  __device__ __forceinline__ words base_of(int token) const {
    if (!whole || !t.base) return words(0u);
    const QLIN_GLOBAL memory* p =
        (const QLIN_GLOBAL memory*)(t.base + token * t.base_stride + n0);
    return ONCE ? __builtin_nontemporal_load(p) : *p;
  }
  __device__ __forceinline__ void multiply(f32x4_t (&sum)[J], const uint4 (&high)[KS],
                                           const uint4 (&low)[KS]) const {
#pragma unroll
    for (int j = 0; j < J; ++j) sum[j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        sum[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16(low[s]), w[s][j], sum[j], 0, 0, 0);
        sum[j] =
            __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16(high[s]), w[s][j], sum[j], 0, 0, 0);
      }
    }
  }
  // Row i of the sums is the token's.
  __device__ __forceinline__ void store(int token, const f32x4_t (&sum)[J], int i, words b) const {
    uint16_t* out = t.out + token * t.out_stride + n0;
    if (whole) {
      if (rank) {
#pragma unroll
        for (int j = 0; j < J; j += 2) {
          b[j / 2] = pack2_bf16(bf16_lo(b[j / 2]) + sum[j][i], bf16_hi(b[j / 2]) + sum[j + 1][i]);
        }
      }
      QLIN_GLOBAL memory* p = (QLIN_GLOBAL memory*)out;
      if (ONCE) {
        __builtin_nontemporal_store(memory(b), p);
      } else {
        *p = b;
      }
      return;
    }
    const uint16_t* base = t.base ? t.base + token * t.base_stride + n0 : nullptr;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (n0 + j >= t.n) continue;
      const uint16_t v = base ? base[j] : 0;
      out[j] = rank ? f32_to_bf16(bf16_to_f32(v) + sum[j][i]) : v;
    }
  }
};

// Block `block` of `columns` over all targets: the target and the block within it; -1 past
// the last.
__device__ __forceinline__ int target_of(const LoraArgs& a, int columns, int& block) {
  for (int c = 0; c < a.targets; ++c) {
    const int blocks = (a.target[c].n + columns - 1) / columns;
    if (block < blocks) return c;
    block -= blocks;
  }
  return -1;
}

// Workgroups of several waves hold their unit's h in LDS, read once for all (6001 x 1536 x 8960
// at rank 32 58.6 -> 57.2 us, at 128, where registers leave room for one more wave, 112 -> 90).
template <int KS, int J, int WAVES, bool GROUPED, bool ONCE>
__global__ __launch_bounds__(WAVES * kWave) void lora_expand_kernel(LoraArgs a) {
  constexpr bool kShared = WAVES > 1;
  constexpr int kWords = 64 * KS;  // of a token's h
  __shared__ int list[GROUPED ? kSet : kGather];
  __shared__ __align__(16) uint16_t shared[kShared ? kSet : 1][kShared ? kWords + 8 : 8];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int m = lane & 15, g = lane >> 4;
  // neighbouring workgroups have neighbouring columns, where they can be counted so
  const Unit u = tokens_of<GROUPED>(a, a.blocks ? blockIdx.x / a.blocks : blockIdx.x, list);
  if (u.count == 0) return;
  int block = a.blocks ? blockIdx.x % a.blocks : blockIdx.y;
  const int c = target_of(a, WAVES * J * 16, block);
  const LoraTarget& t = a.target[c];
  if (u.adapter < 0 && t.base == t.out) return;
  const int rank = u.rank;
  const uint16_t* const all_h = a.h + static_cast<size_t>(c) * a.tokens * kWords;
  uint4 mine[kShared ? kSet * kWords / 8 / (WAVES * kWave) : 1];
  if constexpr (kShared) {
#pragma unroll
    for (int i = 0; i < kSet * kWords / 8 / (WAVES * kWave); ++i) {
      const int e = i * WAVES * kWave + threadIdx.x;
      const int at = e / (kWords / 8), w = e % (kWords / 8) * 8;
      mine[i] = make_uint4(0, 0, 0, 0);
      if (at < u.count && w % (kWords / 2) < rank) {
        mine[i] = load_global16(all_h + static_cast<size_t>(list[at]) * kWords + w);
      }
    }
  }
  block = block * WAVES + wave;
  Columns<KS, J, ONCE> columns(a, t, block * J * 16 < t.n ? block : 0, u, lane);
  // A tile's bases, and h, are loaded while the one before it is computed.
  struct Tile {
    uint4 high[KS], low[KS];
    typename Words<J>::type base[4];
  };
  auto load = [&](Tile& v, int tile) {
    if constexpr (!kShared) {
      const uint16_t* h =
          all_h + static_cast<size_t>(list[min(tile * kTile + m, u.count - 1)]) * kWords;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int k = 32 * s + 8 * g;
        v.high[s] = v.low[s] = make_uint4(0, 0, 0, 0);
        if (k < rank) {
          v.high[s] = load_global16(h + k);
          v.low[s] = load_global16(h + kWords / 2 + k);
        }
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
  if constexpr (kShared) {
#pragma unroll
    for (int i = 0; i < kSet * kWords / 8 / (WAVES * kWave); ++i) {
      const int e = i * WAVES * kWave + threadIdx.x;
      *reinterpret_cast<uint4*>(&shared[e / (kWords / 8)][e % (kWords / 8) * 8]) = mine[i];
    }
    lds_barrier();
    if (block * J * 16 >= t.n) return;
  }
  columns.cut(lane);
  for (; tile * kTile < u.count; tile += step) {
    now = next;
    if ((tile + step) * kTile < u.count) load(next, tile + step);
    if constexpr (kShared) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const uint16_t* h = &shared[tile * kTile + m][32 * s + 8 * g];
        now.high[s] = *reinterpret_cast<const uint4*>(h);
        now.low[s] = *reinterpret_cast<const uint4*>(h + kWords / 2);
      }
    }
    f32x4_t sum[J];
    columns.multiply(sum, now.high, now.low);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = tile * kTile + 4 * g + i;
      if (at < u.count) columns.store(list[at], sum, i, now.base[i]);
    }
  }
}

// B h from the parts of h: a workgroup's waves add them up in the order of the parts, once
// for all, into LDS.
template <int KS, int J>
__global__ __launch_bounds__(kPartWaves * kWave) void lora_expand_parts_kernel(LoraArgs a) {
  constexpr int kPitch = 32 * KS, kThreads = kPartWaves * kWave;
  constexpr int kFours = kTile * kPitch / 4, kMine = (kFours + kThreads - 1) / kThreads;
  __shared__ int list[kGather];
  __shared__ __align__(16) uint16_t h[2][2][kTile][kPitch + 8];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int m = lane & 15, g = lane >> 4;
  const Unit u = gather_tokens(a, blockIdx.x / a.blocks, list);
  if (u.count == 0) return;
  int block = blockIdx.x % a.blocks;
  const int c = target_of(a, kPartWaves * J * 16, block);
  const LoraTarget& t = a.target[c];
  if (u.adapter < 0 && t.base == t.out) return;
  block = block * kPartWaves + wave;
  const bool has = block * J * 16 < t.n;
  // A tile's parts and bases are loaded while the one before it is computed.
  struct Tile {
    f32x4_t part[kMine][kMostParts];
    typename Words<J>::type base[4];
  };
  auto load_parts = [&](Tile& v, int tile) {
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int e = i * kThreads + threadIdx.x, row = e % (kPitch / 4) * 4;
      const int token = list[min(tile * kTile + e / (kPitch / 4) % kTile, u.count - 1)];
      const float* from = reinterpret_cast<const float*>(a.h) +
                          (static_cast<size_t>(c) * a.tokens + token) * kPitch + row;
#pragma unroll
      for (int p = 0; p < kMostParts; ++p) {
        v.part[i][p] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        if (p < a.parts && row < u.rank) {
          v.part[i][p] = *(const QLIN_GLOBAL f32x4_t*)(
              from + static_cast<size_t>(p) * a.targets * a.tokens * kPitch);
        }
      }
    }
  };
  auto load_base = [&](Tile& v, const auto& columns, int tile) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v.base[i] = columns.base_of(list[min(tile * kTile + 4 * g + i, u.count - 1)]);
    }
  };
  const int step = gridDim.z;
  int tile = blockIdx.z;
  if (tile * kTile >= u.count) return;
  Tile now, next;
  load_parts(next, tile);
  Columns<KS, J, false> columns(a, t, has ? block : 0, u, lane);
  load_base(next, columns, tile);
  columns.cut(lane);
  for (int turn = 0; tile * kTile < u.count; tile += step, turn ^= 1) {
    now = next;
    if ((tile + step) * kTile < u.count) {
      load_parts(next, tile + step);
      load_base(next, columns, tile + step);
    }
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int e = i * kThreads + threadIdx.x, row = e % (kPitch / 4) * 4;
      uint16_t high[4], low[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float sum = now.part[i][0][k];
#pragma unroll
        for (int p = 1; p < kMostParts; ++p) {
          if (p < a.parts) sum += now.part[i][p][k];
        }
        split_word(row + k < u.rank ? sum * u.scale : 0.0f, high[k], low[k]);
      }
      if (kFours % kThreads == 0 || e < kFours) {
        uint16_t* to = &h[turn][0][e / (kPitch / 4)][row];
        *reinterpret_cast<uint2*>(to) =
            make_uint2(high[0] | high[1] << 16, high[2] | high[3] << 16);
        *reinterpret_cast<uint2*>(to + kTile * (kPitch + 8)) =
            make_uint2(low[0] | low[1] << 16, low[2] | low[3] << 16);
      }
    }
    lds_barrier();
    uint4 high[KS], low[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      high[s] = *reinterpret_cast<const uint4*>(&h[turn][0][m][32 * s + 8 * g]);
      low[s] = *reinterpret_cast<const uint4*>(&h[turn][1][m][32 * s + 8 * g]);
    }
    f32x4_t sum[J];
    columns.multiply(sum, high, low);
    if (has) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = tile * kTile + 4 * g + i;
        if (at < u.count) columns.store(list[at], sum, i, now.base[i]);
      }
    }
  }
}

// Both products in one launch, for calls so small that it is launches and round trips
// they wait for: a workgroup takes 16 waves' columns of a unit's target and computes
// the unit's h for itself, in LDS.  A is read once for each such workgroup, from L2 as
// a rule.
template <int RT, int J>
__global__ __launch_bounds__(kShrinkWaves * kWave) void lora_fused_kernel(LoraArgs a) {
  constexpr int KS = (RT + 1) / 2, kPitch = RT * kTile + 8;  // words of a row of h
  extern __shared__ __align__(16) char shared[];
  Stage<RT>& stage = *reinterpret_cast<Stage<RT>*>(shared);
  int* const list = reinterpret_cast<int*>(shared + sizeof(Stage<RT>));
  __shared__ __align__(16) uint16_t h[2][kTile][kPitch];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int m = lane & 15, g = lane >> 4;
  const Unit u = gather_tokens(a, blockIdx.x, list);
  if (u.count == 0) return;
  int block = blockIdx.y;
  const int c = target_of(a, kShrinkWaves * J * 16, block);
  const LoraTarget& t = a.target[c];
  if (u.adapter < 0 && t.base == t.out) return;
  block = block * kShrinkWaves + wave;
  const bool has = block * J * 16 < t.n;
  Columns<KS, J, false> columns(a, t, has ? block : 0, u, lane);
  const uint16_t* rows[RT + 1];
  stage_rows<RT>(rows, a, u.adapter, c * ((a.max_rank + kTile - 1) / kTile), wave);
  for (int tile = blockIdx.z; tile * kTile < u.count; tile += gridDim.z) {
    typename Words<J>::type base[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      base[i] = columns.base_of(list[min(tile * kTile + 4 * g + i, u.count - 1)]);
    }
    uint4 high[KS], low[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) high[s] = low[s] = make_uint4(0, 0, 0, 0);
    if (u.rank) {
      f32x4_t sum[RT];
      rows[RT] = a.x + list[min(tile * kTile + wave, u.count - 1)] * a.x_stride;
      shrink_tile<RT>(sum, a.k, rows, stage, wave, lane);
      for (int e = threadIdx.x; e < RT * kTile * kTile; e += kShrinkWaves * kWave) {
        const int row = row_of(e);
        uint16_t* to = &h[0][token_of(e)][row];
        split_word(row < u.rank ? joined<RT>(stage, e) * u.scale : 0.0f, to[0],
                   to[kTile * kPitch]);
      }
      lds_barrier();
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int k = 32 * s + 8 * g;
        if (k < RT * kTile) {
          high[s] = *reinterpret_cast<const uint4*>(&h[0][m][k]);
          low[s] = *reinterpret_cast<const uint4*>(&h[1][m][k]);
        }
      }
    }
    if (tile == static_cast<int>(blockIdx.z)) columns.cut(lane);
    f32x4_t sum[J];
    columns.multiply(sum, high, low);
    if (has) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = tile * kTile + 4 * g + i;
        if (at < u.count) columns.store(list[at], sum, i, base[i]);
      }
    }
  }
}

int chunks_of(int tokens) { return (tokens + kChunk - 1) / kChunk; }
int units_of(int tokens, int adapters) {  // of a chunk
  return (kChunk + kSet - 1) / kSet + std::min(std::min(tokens, kChunk), adapters + 1);
}

// Of h as two BF16 numbers, or as one part in 32 bits.
size_t h_bytes(int tokens, int max_rank, int targets) {
  return static_cast<size_t>(targets) * tokens * 4 * rank_pitch(max_rank);
}

}  // namespace

size_t lora_workspace_bytes(int tokens, int max_rank, int targets) {
  const size_t parts = kMostParts * h_bytes(std::min(tokens, kGather), max_rank, targets);
  if (tokens <= kGather) return parts;
  const size_t chunks = chunks_of(tokens);
  return std::max(parts, h_bytes(tokens, max_rank, targets) +
                             4 * ((static_cast<size_t>(tokens) + 3) / 4 * 4) +
                             16 * chunks * units_of(tokens, kChunk));
}

// Bytes of bases and outputs beyond which four waves take 512 columns side by side, and beyond
// which they are not left in the caches (6001 tokens by 8960, 215 MB, 67.1 -> 64.1 us; 3000 by
// 2 x 4864, 117 MB, whose bases still are there, 31.6 -> 36.7; 6001 by 8959, whose lines are
// written in parts, 89 -> 102).  Below, a wave is a workgroup, of 64 columns beyond rank 32,
// that starts as soon as it finds room (2000 x 3584 x 3584 at rank 128 43.6 us in fours, 37.3;
// 250 x 3584 x 3584 of 200 adapters 66.9, 64.6; but 3000 x 896 x 2 x 4864 at rank 64 56.6 for
// 47.8, at rank 8 40.3 for 38.6).
constexpr long long kManyBytes = 70ll << 20;
constexpr long long kStreamBytes = 192ll << 20;
constexpr long long kMostThreads = (1ll << 32) - 1;  // of a launch, along x

template <bool GROUPED>
static void launch_expand(LoraArgs a, int units, int slots, hipStream_t stream) {
  const int steps = rank_pitch(a.max_rank) / 32;
  const int sets = (a.tokens + kSet - 1) / kSet;
  long long bytes = 0;
  bool aligned = true;
  for (int i = 0; i < a.targets; ++i) {
    const LoraTarget& t = a.target[i];
    bytes += 4ll * a.tokens * t.n;
    const uintptr_t at = reinterpret_cast<uintptr_t>(t.out) | reinterpret_cast<uintptr_t>(t.base);
    aligned = aligned && (t.out_stride | t.base_stride) % 8 == 0 && at % 16 == 0;
  }
  auto run = [&](auto* kernel, int columns, int waves) {
    int blocks = 0;
    for (int i = 0; i < a.targets; ++i) {
      blocks += (a.target[i].n + columns * waves - 1) / (columns * waves);
    }
    // a unit's four tiles side by side where there would be few workgroups
    const long long few = static_cast<long long>(sets) * blocks;
    const int z = !GROUPED ? slots : waves > 1 || few >= 1024 ? 1 : few >= 512 ? 2 : kSet / kTile;
    const bool flat = static_cast<long long>(units) * blocks * waves * kWave <= kMostThreads;
    a.blocks = flat ? blocks : 0;
    hipLaunchKernelGGL(kernel, flat ? dim3(units * blocks, 1, z) : dim3(units, blocks, z),
                       dim3(waves * kWave), 0, stream, a);
  };
  if constexpr (GROUPED) {
    if (bytes > kStreamBytes && aligned) {
      steps == 1   ? run(lora_expand_kernel<1, 8, 4, true, true>, 128, 4)
      : steps == 2 ? run(lora_expand_kernel<2, 8, 4, true, true>, 128, 4)
      : steps == 3 ? run(lora_expand_kernel<3, 8, 4, true, true>, 128, 4)
                   : run(lora_expand_kernel<4, 8, 4, true, true>, 128, 4);
      return;
    }
    if (bytes > kManyBytes) {
      steps == 1   ? run(lora_expand_kernel<1, 8, 4, true, false>, 128, 4)
      : steps == 2 ? run(lora_expand_kernel<2, 8, 4, true, false>, 128, 4)
      : steps == 3 ? run(lora_expand_kernel<3, 8, 4, true, false>, 128, 4)
                   : run(lora_expand_kernel<4, 8, 4, true, false>, 128, 4);
      return;
    }
  }
  steps == 1   ? run(lora_expand_kernel<1, 8, 1, GROUPED, false>, 128, 1)
  : steps == 2 ? run(lora_expand_kernel<2, 4, 1, GROUPED, false>, 64, 1)
  : steps == 3 ? run(lora_expand_kernel<3, 4, 1, GROUPED, false>, 64, 1)
               : run(lora_expand_kernel<4, 4, 1, GROUPED, false>, 64, 1);
}

static void launch_two(LoraArgs a, int slots, hipStream_t stream) {
  const int rows = a.targets * ((a.max_rank + kTile - 1) / kTile);
  // as long as a part has kPartColumns and the workgroups run at once, one to a CU (128 x
  // 3584 x 2 x 18944 at rank 64 26.4 us in one part, 23.6 in two, 24.2 in four on 416)
  const long long units = std::min(a.units, a.tokens);
  a.parts = 1;
  while (a.parts < kMostParts && a.k >= 2 * a.parts * kPartColumns &&
         2 * a.parts * units * rows * slots <= kCus) {
    a.parts *= 2;
  }
  if (a.parts == 1) {
    auto shrink = [&](auto* kernel, int tiles, size_t lds) {
      hipLaunchKernelGGL(kernel, dim3(a.units, (rows + tiles - 1) / tiles, slots),
                         dim3(kShrinkWaves * kWave), lds + kGather * sizeof(int), stream, a);
    };
    // x for two tiles of rows where there are many (33 tokens' q, k and v of 1536 at rank 64
    // 15.1 us, 12.2)
    units * rows * slots <= kCus ? shrink(lora_shrink_kernel<1, false>, 1, sizeof(Stage<1>))
                                 : shrink(lora_shrink_kernel<2, false>, 2, sizeof(Stage<2>));
    launch_expand<false>(a, a.units, slots, stream);
    return;
  }
  hipLaunchKernelGGL(lora_shrink_part_kernel, dim3(a.units, rows * a.parts, slots),
                     dim3(kShrinkWaves * kWave), sizeof(Stage<1>) + kGather * sizeof(int), stream,
                     a);
  auto run = [&](auto* kernel, int columns) {
    a.blocks = 0;
    for (int i = 0; i < a.targets; ++i) a.blocks += (a.target[i].n + columns - 1) / columns;
    hipLaunchKernelGGL(kernel, dim3(a.units * a.blocks, 1, slots), dim3(kPartWaves * kWave), 0,
                       stream, a);
  };
  const int steps = rank_pitch(a.max_rank) / 32;
  steps == 1   ? run(lora_expand_parts_kernel<1, 8>, 128 * kPartWaves)
  : steps == 2 ? run(lora_expand_parts_kernel<2, 4>, 64 * kPartWaves)
  : steps == 3 ? run(lora_expand_parts_kernel<3, 4>, 64 * kPartWaves)
               : run(lora_expand_parts_kernel<4, 4>, 64 * kPartWaves);
}

// The one launch's largest rank (64 spills registers: 64 x 896 x 896 16.3 us, in two launches
// 8.8; 32 33 tokens' q, k and v of 1536 9.1, in two 10.1), rows of A by columns that each of
// its workgroups takes (5 x 8960 x 1536 at rank 32 19.0 us, in two launches 11.0; 40 x 2048
// x 2048 9.4, 9.7), and A's bytes that all of them may read (100 tokens' 60 adapters by
// 2048 x 2048 at rank 32, 16 MB, 10.6 us, 11.1; 200's 200 by 1536 x 1536 at rank 16, 20 MB, 15.1,
// 13.7; 128's 120 by 896 x 2 x 4864, 34 MB, 24.7, 17.3).
constexpr int kFusedRank = 32, kFusedRows = 1 << 16;
constexpr long long kFusedBytes = 16ll << 20;

static bool launch_fused(const LoraArgs& a, int slots, hipStream_t stream) {
  constexpr int kColumns = kShrinkWaves * 64;
  int blocks = 0;
  for (int i = 0; i < a.targets; ++i) blocks += (a.target[i].n + kColumns - 1) / kColumns;
  const long long units = std::min(a.units, a.tokens);
  if (a.max_rank > kFusedRank || (a.max_rank + kTile - 1) / kTile * kTile * a.k > kFusedRows ||
      2ll * units * blocks * a.max_rank * a.k > kFusedBytes) {
    return false;
  }
  auto run = [&](auto* kernel, size_t lds) {
    hipLaunchKernelGGL(kernel, dim3(a.units, blocks, slots), dim3(kShrinkWaves * kWave),
                       lds + kGather * sizeof(int), stream, a);
  };
  a.max_rank <= 16 ? run(lora_fused_kernel<1, 4>, sizeof(Stage<1>))
                   : run(lora_fused_kernel<2, 4>, sizeof(Stage<2>));
  return true;
}

void launch_lora(LoraArgs a, hipStream_t stream) {
  const int rank_tiles = (a.max_rank + kTile - 1) / kTile;
  if (a.tokens > kGather) {
    a.groups = reinterpret_cast<int*>(reinterpret_cast<char*>(a.h) +
                                      h_bytes(a.tokens, a.max_rank, a.targets));
    a.units = units_of(a.tokens, a.adapters);
    const int chunks = chunks_of(a.tokens), units = chunks * a.units;
    hipLaunchKernelGGL(lora_group_kernel, dim3(chunks), dim3(kChunk), 0, stream, a);
    const int all = a.targets * rank_tiles;
    auto shrink = [&](auto* kernel, int tiles, size_t lds) {
      hipLaunchKernelGGL(kernel, dim3(units, (all + tiles - 1) / tiles, kSet / kTile),
                         dim3(kShrinkWaves * kWave), lds + kSet * sizeof(int), stream, a);
    };
    all == 1 ? shrink(lora_shrink_kernel<1, true>, 1, sizeof(Stage<1>))
             : shrink(lora_shrink_kernel<2, true>, 2, sizeof(Stage<2>));
    launch_expand<true>(a, units, 0, stream);
    return;
  }
  a.by_token = a.adapters + 1 > a.tokens;
  a.units = a.by_token ? a.tokens : a.adapters + 1;
  // workgroups side by side for a unit's tiles, as many as it has if units are alike
  const int tiles = (a.tokens + kTile - 1) / kTile;
  const int slots = std::min(tiles, 1 + a.tokens / (kTile * a.units));
  if (launch_fused(a, slots, stream)) return;
  launch_two(a, slots, stream);
}

}  // namespace qlin
