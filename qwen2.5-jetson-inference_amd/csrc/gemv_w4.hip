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
// q x / 16 reaches 1/2 |x|, which costs two bits of FP32's 24, and a large activation
// leaves its rounding in rows whose q is 0 too.  With q itself (the nibbles as E4M3
// bytes with a sign, converted to BF16 two at a time: 17 instructions a dword for 8, no
// starts) neither is so, but 16 x 151936 x 896 takes 23.0 us for 20.4, 1 x 152064 x 3584
// 65 for 53, 16 x 1536 x 8960 10.7 for 9.7 (1 x 896 x 896 without a bias 3.0 for 3.2).
//
// Two forms.  With many rows (w4a16_rows_kernel) a wave takes whole row tiles
// over all of K, by itself, with the activations and the groups' starts in LDS.
// With fewer (w4a16_split_kernel) the waves of a workgroup split one or two row
// tiles' K and meet in LDS, in the order of the waves; the activations come from
// L2 for every row tile, 128 bytes a token and KiB of weights.  Either keeps DP
// tiles of 128 columns, a contiguous KiB of weights each, in flight per wave.
//
// Bound.  The weights' bytes and the waits at a call's start and end: 16 tokens by
// 151936 x 896 in groups of 32 takes 20 us for 81 MB (4.1 TB/s; a read alone runs at
// 7.0), 1 by 152064 x 3584 in groups of 128 50 us (5.6 TB/s), 1 by 40000 x 4096 18.4
// us (4.7 TB/s), 1 by 896 x 896 3.1 us, of which 1.7 are an empty launch.  The vector
// instructions (60 to 80 a tile, by the group) would allow a KiB in 65 to 85 cycles of
// a CU, whose share of HBM is a KiB in 90.  Where K is long and row tiles are few (16 x
// 1536 x 8960, 9.7 us) it is the activations, all of them read by each CU.
//
// Activations beyond FP32's reach (a sum that is not finite) are summed again
// element by element, q s x in FP32.
struct W4Piece {
  uint4 w;
  uint2 s;  // four rows' scales, of the lane's group
};

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// The constants of widen_nibbles in registers: as literals they cost an instruction
// more a pair (and, or) than the one that takes three operands.
struct NibbleBits {
  uint32_t mantissa = 0x00780078u, one = 0x3F803F80u;
  __device__ __forceinline__ NibbleBits() { asm("" : "+s"(mantissa), "+v"(one)); }
};

// Eight nibbles as 1 + u / 16 in BF16.
__device__ __forceinline__ bf16x8_t widen_nibbles(uint32_t w, const NibbleBits& c) {
  const uint4 v = make_uint4(((w << 3) & c.mantissa) | c.one, ((w >> 1) & c.mantissa) | c.one,
                             ((w >> 5) & c.mantissa) | c.one, ((w >> 9) & c.mantissa) | c.one);
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

// Column tile t of row tile rt.  Lane 16 g + r holds the scales of rows 4 g ..
// + 3 for group r modulo the tile's groups: one load for all of them, and each
// quad of lanes has every group.
template <int G>
__device__ __forceinline__ void load_piece(W4Piece& p, const W4Args& a, int rt, int t, int tiles,
                                           int groups, int lane) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  constexpr int kGroups = kTileCols / G;
  p.w = load_stream16(a.w + (static_cast<size_t>(rt) * tiles + t) * kTileBytes + 16 * lane);
  // past the last group: that one again
  const int group = kGroups == 1 ? t : min(t * kGroups + (lane & (kGroups - 1)), groups - 1);
  const u32x2 v = gload(reinterpret_cast<const u32x2*>(
      a.s + (static_cast<size_t>(rt) * groups + group) * kTileRows + 4 * (lane >> 4)));
  p.s = make_uint2(v.x, v.y);
}

// v of lane J of the quad.
template <int J>
__device__ __forceinline__ float quad_lane(float v) {
  return __int_as_float(
      __builtin_amdgcn_mov_dpp(__float_as_int(v), J * 0x55, 0xF, 0xF, true));
}

// -1.5 sum x over each group of a tile (four steps of 32 columns), for every row.
template <int G>
__device__ __forceinline__ void base_of(f32x4_t (&base)[kTileCols / G], const bf16x8_t (&x)[4]) {
  constexpr int kSteps = G / 32;
  const bf16x8_t minus_1_5 =
      __builtin_bit_cast(bf16x8_t, make_uint4(0xBFC0BFC0u, 0xBFC0BFC0u, 0xBFC0BFC0u, 0xBFC0BFC0u));
#pragma unroll
  for (int j = 0; j < kTileCols / G; ++j) {
    base[j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = j * kSteps; i < (j + 1) * kSteps; ++i) {
      base[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(minus_1_5, x[i], base[j], 0, 0, 0);
    }
  }
}

// total += the tile's products with x, over 16.
template <int G>
__device__ __forceinline__ void add_piece(f32x4_t& total, const W4Piece& p, const bf16x8_t (&x)[4],
                                          const f32x4_t (&base)[kTileCols / G],
                                          const NibbleBits& bits) {
  constexpr int kGroups = kTileCols / G, kSteps = G / 32;
  const float s[4] = {bf16_lo(p.s.x), bf16_hi(p.s.x), bf16_lo(p.s.y), bf16_hi(p.s.y)};
#pragma unroll
  for (int j = 0; j < kGroups; ++j) {
    f32x4_t d = base[j];
#pragma unroll
    for (int i = j * kSteps; i < (j + 1) * kSteps; ++i) {
      d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen_nibbles(word_of(p.w, i), bits), x[i], d, 0,
                                                  0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = kGroups == 1 ? s[i]
                      : j == 0     ? quad_lane<0>(s[i])
                      : j == 1     ? quad_lane<1>(s[i])
                      : j == 2     ? quad_lane<2>(s[i])
                                   : quad_lane<3>(s[i]);
      total[i] = fmaf(f, d[i], total[i]);
    }
  }
}

// The output from a sum over 16.
__device__ __forceinline__ uint16_t finish(const W4Args& a, float v, int row) {
  v *= 16.0f;
  return f32_to_bf16(a.bias ? v + bf16_to_f32(a.bias[row]) : v);
}

// Whether a stored output may be that of a sum that overflowed.
__device__ __forceinline__ bool not_finite(uint16_t y) { return (y & 0x7F80u) == 0x7F80u; }

__device__ void finish_exactly(const W4Args& a, int row, int token) {
  uint16_t* y = a.y + static_cast<size_t>(token) * a.n + row;
  const float v = exact_dot(a, row, token);
  *y = f32_to_bf16(a.bias ? v + bf16_to_f32(a.bias[row]) : v);
}

// Tiles in flight per wave of the rows kernel: 16 x 151936 x 896 20.1 us, 21.0 with 4
// (whose first loads delay the activations), 19.8 with 2, which loses 4-8 % on long K.
constexpr int kRowsDepth = 3, kRowsMaxWaves = 16;
// Workgroups of the rows kernel a CU holds, and their waves, by their LDS: as many as
// the registers allow (two of 8 waves: 16 x 151936 x 896 24.6 us, three: 21.4).
struct RowsShape {
  int per_cu, waves;
  size_t lds;  // at most
};
constexpr RowsShape kRowsShapes[] = {
    {3, 8, 52 * 1024}, {2, 12, 78 * 1024}, {1, kRowsMaxWaves, 156 * 1024}};

// LDS of the rows kernel: the activations [K / 8][pitch][8] for TP tokens, zero past K
// and past the tokens, then the groups' bases [K / G][TP][4].  With 16 tokens a piece
// of 16 bytes more for each 8 columns: a token's neighbouring pieces, which neighbouring
// lanes load, then go to different banks.
constexpr int x_pitch(int tp) { return tp == 16 ? 17 : tp; }
constexpr size_t rows_x_bytes(int tiles, int tp) {
  return static_cast<size_t>(tiles) * kTileCols * 2 * x_pitch(tp);
}
constexpr size_t rows_lds_bytes(int tiles, int tp, int group) {
  return rows_x_bytes(tiles, tp) + static_cast<size_t>(tiles) * (kTileCols / group) * tp * 16;
}

// Workgroup i takes the i-th of equal shares of the row tiles, its waves equal
// shares of that.  TP: room for that many tokens; lanes past it repeat others,
// whose columns of Y^T are dropped.
template <int G, int TP>
__global__ __launch_bounds__(kRowsMaxWaves * kWave, 6) void w4a16_rows_kernel(W4Args a) {
  constexpr int DP = kRowsDepth, kGroups = kTileCols / G;
  constexpr int kHead = TP == 16 ? 4 : TP == 4 ? 2 : 1;
  constexpr int kPieces = kTileCols / 8, kPitch = x_pitch(TP);  // of a tile; in LDS
  extern __shared__ __align__(16) uint4 lds[];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x / kWave;
  const int tiles = (a.k + kTileCols - 1) / kTileCols, groups = a.k / G;
  const int row_tiles = (a.n + kTileRows - 1) / kTileRows;
  const long long share = static_cast<long long>(row_tiles) * blockIdx.x;
  const int begin = share / gridDim.x, end = (share + row_tiles) / gridDim.x;
  const int per_wave = (end - begin + waves - 1) / waves;
  const int first = min(end, begin + wave * per_wave), last = min(end, first + per_wave);
  const int count = (last - first) * tiles;

  // The wave's weights, and scales, follow each other in memory.  Loads run DP
  // tiles ahead, always: past the wave's last tile they read that one again, so
  // that the compiler knows how many are in flight; the addresses are kept from it,
  // as it would copy such a tile instead of loading it, and then wait for all.
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  const int in_last = groups - (tiles - 1) * kGroups;  // groups of a row's last tile
  const uint32_t s_off = ((lane & (kGroups - 1)) * kTileRows + 4 * g) * 2;
  const uint32_t s_off_last = (min(lane & (kGroups - 1), in_last - 1) * kTileRows + 4 * g) * 2;
  const int from = min(first, row_tiles - 1);  // also of a wave with no tiles
  const uint8_t* w_next = a.w + static_cast<size_t>(from) * tiles * kTileBytes;
  const char* s_next =
      reinterpret_cast<const char*>(a.s + static_cast<size_t>(from) * groups * kTileRows);
  const int s_step = kGroups * kTileRows * 2, s_step_last = in_last * kTileRows * 2;
  int t_ahead = 0, ahead = 0;
  auto load_next = [&](W4Piece& p) {
    const bool ends = t_ahead + 1 == tiles;
    p.w = load_stream16(w_next + 16 * lane);
    const u32x2 v = gload(reinterpret_cast<const u32x2*>(s_next + (ends ? s_off_last : s_off)));
    p.s = make_uint2(v.x, v.y);
    const int more = ahead + 1 < count ? -1 : 0;  // a mask: as branches the
    ahead -= more;                                // advance would part the block
    w_next += kTileBytes & more;
    s_next += (ends ? s_step_last : s_step) & more;
    t_ahead -= more;
    t_ahead = t_ahead == tiles ? 0 : t_ahead;
    asm("" : "+s"(w_next), "+s"(s_next));
  };
  // The activations' first loads go ahead of the weights', whose return they would
  // wait for, and reach LDS while those are on their way.
  const int chunks = a.k / 8, pieces = tiles * kPieces * TP;
  auto chunk_of = [&](int i) { return i / (kPieces * TP) * kPieces + i % kPieces; };
  auto token_of = [&](int i) { return i / kPieces % TP; };
  auto inside = [&](int i) { return chunk_of(i) < chunks && token_of(i) < a.tokens; };
  auto load_x = [&](int i) {
    return load_global16(i < pieces && inside(i)
                             ? a.x + static_cast<size_t>(token_of(i)) * a.k + 8 * chunk_of(i)
                             : a.x);
  };
  auto keep_x = [&](int i, const uint4& v) {
    if (i < pieces) {
      lds[chunk_of(i) * kPitch + token_of(i)] = inside(i) ? v : make_uint4(0, 0, 0, 0);
    }
  };
  uint4 head[kHead];
#pragma unroll
  for (int b = 0; b < kHead; ++b) head[b] = load_x(threadIdx.x + b * blockDim.x);
  asm volatile("" ::: "memory");
  W4Piece p[DP];
#pragma unroll
  for (int i = 0; i < DP; ++i) load_next(p[i]);
  asm volatile("" ::: "memory");
#pragma unroll
  for (int b = 0; b < kHead; ++b) keep_x(threadIdx.x + b * blockDim.x, head[b]);
  for (int i = threadIdx.x + kHead * blockDim.x; i < pieces; i += blockDim.x) keep_x(i, load_x(i));
  __syncthreads();
  const int lds_lane = g * kPitch + r % TP;  // of a step's 4 x kPitch pieces
  f32x4_t* const bases = reinterpret_cast<f32x4_t*>(lds + tiles * kPieces * kPitch);
  for (int t = wave; t < tiles; t += waves) {
    bf16x8_t x[4];
    f32x4_t base[kGroups];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = __builtin_bit_cast(bf16x8_t, lds[(t * 4 + j) * 4 * kPitch + lds_lane]);
    }
    base_of<G>(base, x);
    if (lane < TP) {
#pragma unroll
      for (int j = 0; j < kGroups; ++j) bases[(t * kGroups + j) * TP + lane] = base[j];
    }
  }
  __syncthreads();
  if (count <= 0) return;
  const bool wide = (a.n & 3) == 0 && (reinterpret_cast<uintptr_t>(a.y) & 7u) == 0;

  const NibbleBits bits;
  f32x4_t total{0.0f, 0.0f, 0.0f, 0.0f};
  bool again = false;
  int rt = first, t = 0;
  auto piece = [&](int i, auto more) {
    bf16x8_t x[4];
    f32x4_t base[kGroups];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = __builtin_bit_cast(bf16x8_t, lds[(t * 4 + j) * 4 * kPitch + lds_lane]);
    }
#pragma unroll
    for (int j = 0; j < kGroups; ++j) base[j] = bases[(t * kGroups + j) * TP + r % TP];
    add_piece<G>(total, p[i], x, base, bits);
    if (decltype(more)::value) load_next(p[i]);
    if (++t == tiles) {
      const int row = rt * kTileRows + 4 * g;
      if (r < a.tokens) {
        uint16_t* y = a.y + static_cast<size_t>(r) * a.n + row;
        uint16_t v[4];
        f32x4_t b{0.0f, 0.0f, 0.0f, 0.0f};
        if (a.bias) {
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] = bf16_to_f32(a.bias[min(row + j, a.n - 1)]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = f32_to_bf16(fmaf(total[j], 16.0f, b[j]));
          again = again || (row + j < a.n && not_finite(v[j]));
        }
        if (wide) {  // then the four rows are in the matrix or none is
          if (row < a.n) {
            store_global8(y, make_uint2(v[0] | static_cast<uint32_t>(v[1]) << 16,
                                        v[2] | static_cast<uint32_t>(v[3]) << 16));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (row + j < a.n) y[j] = v[j];
          }
        }
      }
      total = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
      t = 0;
      ++rt;
    }
  };
  // DP tiles a pass, left from a single place: with a way out behind each, the wait
  // for the first piece's loads would be for the way from all of them.  The last pass
  // loads nothing.
  int item = 0;
  for (; item + DP < count; item += DP) {
#pragma unroll
    for (int i = 0; i < DP; ++i) piece(i, std::true_type{});
  }
#pragma unroll
  for (int i = 0; i < DP; ++i) {
    if (item + i < count) piece(i, std::false_type{});
  }
  if (again) {  // the lane's own outputs
    for (int row = first * kTileRows; row < min(last * kTileRows, a.n); ++row) {
      if ((row >> 2 & 3) == g && r < a.tokens &&
          not_finite(a.y[static_cast<size_t>(r) * a.n + row])) {
        finish_exactly(a, row, r);
      }
    }
  }
}

constexpr int kSplitWaves = 16;

// v of lane `from` (0 .. S - 1) of the S lanes next to each other that v's lane is of.
template <int S, int FROM>
__device__ __forceinline__ uint4 share_lane(const uint4& v) {
  if (S == 1) return v;
  auto one = [](uint32_t w) {
    constexpr int kPerm = S == 4 ? FROM * 0x55 : FROM ? 0xF5 : 0xA0;  // quad lanes
    return static_cast<uint32_t>(
        __builtin_amdgcn_update_dpp(0, static_cast<int>(w), kPerm, 0xF, 0xF, true));
  };
  return make_uint4(one(v.x), one(v.y), one(v.z), one(v.w));
}

// Workgroup i: row tiles [i R, (i + 1) R); wave w takes their column tiles w, w +
// waves, ..., DP of them in flight.  With R > 1 the activations, four KiB a tile
// at 16 tokens, are read for R KiB of weights.  With at most 16 / S tokens S columns
// of Y^T are one token's, and each of their lanes reads one of S parts of the tile's
// activations and hands it to the others: 4 / S KiB a tile.
template <int G, int S, int DP, int R>
__global__ __launch_bounds__(kSplitWaves * kWave) void w4a16_split_kernel(W4Args a) {
  constexpr int kPitch = R * kTileRows + 4, kLoads = 4 / S, kGroups = kTileCols / G;
  extern __shared__ __align__(16) float partial[];  // [wave][token][kPitch]
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x / kWave;
  const int tiles = (a.k + kTileCols - 1) / kTileCols, groups = a.k / G;
  const int row_tiles = (a.n + kTileRows - 1) / kTileRows;
  const int first = blockIdx.x * R;
  // Lane 16 g + r multiplies token r / S's columns 8 g .. of each step of 32, but loads
  // what the lane with g and r's low bits exchanged does: four lanes in a row then read
  // 64 bytes in a row, not 16 of four tokens (16 x 8960 x 1536 7.4 -> 5.7 us, 16 x 1536 x
  // 8960 12.5 -> 9.7, 5 x 17920 x 1536 in groups of 128 6.8 -> 6.2).
  const int gl = lane & 3, rl = (lane & 12) | g, from = 4 * ((r & 3) << 4 | (r & 12) | g);
  const int x_part = rl % S * kLoads * 32;
  const uint16_t* x_row = a.x + static_cast<size_t>(min(rl / S, a.tokens - 1)) * a.k + 8 * gl;
  const NibbleBits bits;
  f32x4_t total[R];
#pragma unroll
  for (int i = 0; i < R; ++i) total[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  for (int t0 = wave; t0 < tiles; t0 += DP * waves) {
    W4Piece p[DP][R];
    uint4 x[DP][kLoads];
#pragma unroll
    for (int i = 0; i < DP; ++i) {  // past the last tile, or row tile: that one again
      const int t = min(t0 + i * waves, tiles - 1);
#pragma unroll
      for (int j = 0; j < R; ++j) {
        load_piece<G>(p[i][j], a, min(first + j, row_tiles - 1), t, tiles, groups, lane);
      }
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        // columns past K have no scale, from wherever they are read
        const int col = t * kTileCols + x_part + 32 * j;
        x[i][j] = load_global16(x_row + (col < a.k ? col : 0));
      }
    }
    // The loads stay ahead of the products' branch, which else each would move
    // behind (1 x 1536 x 8960 7.9 us so, 6.7 here).
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < DP; ++i) {
      if (t0 + i * waves >= tiles) break;
      bf16x8_t xb[4];
#pragma unroll
      for (int j = 0; j < kLoads; ++j) x[i][j] = lane_of(x[i][j], from);
      auto put = [&](auto from) {
        constexpr int kFrom = decltype(from)::value;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          xb[kFrom * kLoads + j] = __builtin_bit_cast(bf16x8_t, share_lane<S, kFrom>(x[i][j]));
        }
      };
      put(std::integral_constant<int, 0>{});
      if constexpr (S > 1) put(std::integral_constant<int, 1>{});
      if constexpr (S > 2) {
        put(std::integral_constant<int, 2>{});
        put(std::integral_constant<int, 3>{});
      }
      f32x4_t base[kTileCols / G];
      base_of<G>(base, xb);
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (kGroups > 1 && (t0 + i * waves) * kGroups + (lane & (kGroups - 1)) >= groups) {
          p[i][j].s = make_uint2(0, 0);
        }
        add_piece<G>(total[j], p[i][j], xb, base, bits);
      }
    }
  }
  if (r % S == 0 && r / S < a.tokens) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      float* const at = partial + (wave * a.tokens + r / S) * kPitch + j * kTileRows + 4 * g;
      *reinterpret_cast<f32x4_t*>(at) = total[j];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < R * kTileRows * a.tokens; e += blockDim.x) {
    const int token = e / (R * kTileRows), i = e % (R * kTileRows);
    const int row = first * kTileRows + i;
    if (row >= a.n) continue;
    float v = 0.0f;
    for (int w = 0; w < waves; ++w) v += partial[(w * a.tokens + token) * kPitch + i];
    const uint16_t y = finish(a, v, row);
    a.y[static_cast<size_t>(token) * a.n + row] = y;
    if (not_finite(y)) finish_exactly(a, row, token);
  }
}

constexpr int kCus = 256;
// Row tiles from which a wave takes whole ones (1 x 65536 x 1024 10.6 us split, 10.1 in
// rows; 8 x 80000 x 2048 22.7 and 19.9; 1 x 40000 x 4096 18.4 and 20.7).  More than 8
// tokens, whose activations the split kernel reads at the weights' own rate or faster:
// fewer, if K is long (16 x 40000 x 4096 23.9 and 22.2; 16 x 32768 x 1024 6.9 and 9.3).
constexpr int kRowsTiles = 4096, kRowsTilesMany = 2048, kRowsLongTiles = 12;
// Row tiles from which the split kernel takes two a workgroup: half the activations'
// reads, half the workgroups (16 x 17920 x 1536 8.1 -> 7.8 us, 16 x 30000 x 1024 8.9 -> 7.2, 1 x
// 40000 x 4096 21.6 -> 18.1, 1 x 30000 x 1024 6.7 -> 6.5, but 1 x 17920 x 1536 5.8 -> 6.4).
constexpr int kPairTiles = 1536, kPairTilesMany = 1024;
constexpr int kManyTokens = 9;         // tokens from which the above say "many"
constexpr int kSplitRoom = 16 * kCus;  // waves that the split kernel fills the chip with

template <int G>
void launch_w4(const W4Args& a, hipStream_t stream) {
  const int row_tiles = (a.n + kTileRows - 1) / kTileRows;
  const int tiles = (a.k + kTileCols - 1) / kTileCols;
  const int room_for = a.tokens == 1 ? 1 : a.tokens <= 4 ? 4 : 16;
  const bool many = a.tokens >= kManyTokens;
  for (const RowsShape& shape : kRowsShapes) {
    const size_t lds = rows_lds_bytes(tiles, room_for, G);
    if (row_tiles < (many && tiles > kRowsLongTiles ? kRowsTilesMany : kRowsTiles) ||
        lds > shape.lds) {
      continue;
    }
    auto launch = [&](auto tp) {
      hipLaunchKernelGGL((w4a16_rows_kernel<G, decltype(tp)::value>), dim3(shape.per_cu * kCus),
                         dim3(shape.waves * kWave), lds, stream, a);
    };
    if (room_for == 1) {
      launch(std::integral_constant<int, 1>{});
    } else if (room_for == 4) {
      launch(std::integral_constant<int, 4>{});
    } else {
      launch(std::integral_constant<int, 16>{});
    }
    return;
  }
  // Waves for the chip's room, at least eight, of equal shares of the tiles (12 or 16:
  // 1 x 17920 x 1536 7.7 us for 6.3; 4 or 6: 9 x 30000 x 1024 7.0 for 6.5, though 1 x
  // 30000 x 1024 6.2).  A wave's loads in flight are all of its tiles up to five with up
  // to four tokens, two with more (16 x 3584 x 18944 20.0 us with one, 17.0 with two, 18.3
  // with three; 9 x 1536 x 8960 7.8, 8.4, 8.4).
  const int room = kSplitRoom / row_tiles;
  const int most = room < 8 ? 8 : room > kSplitWaves ? kSplitWaves : room;
  const int per = (tiles + most - 1) / most;
  const int waves = (tiles + per - 1) / per;
  auto launch = [&](auto share, auto depth, auto rows) {
    constexpr int R = decltype(rows)::value;
    const size_t lds = static_cast<size_t>(waves) * a.tokens * (R * kTileRows + 4) * sizeof(float);
    hipLaunchKernelGGL((w4a16_split_kernel<G, decltype(share)::value, decltype(depth)::value, R>),
                       dim3((row_tiles + R - 1) / R), dim3(waves * kWave), lds, stream, a);
  };
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  using Four = std::integral_constant<int, 4>;
  using Five = std::integral_constant<int, 5>;
  auto by_share = [&](auto depth, auto rows) {
    if (many) {
      launch(One{}, depth, rows);
    } else {
      a.tokens > 4 ? launch(Two{}, depth, rows) : launch(Four{}, depth, rows);
    }
  };
  if (row_tiles >= (many ? kPairTilesMany : kPairTiles)) {
    per == 1 ? by_share(One{}, Two{}) : by_share(Two{}, Two{});
  } else if (per == 1) {
    by_share(One{}, One{});
  } else if (per == 2 || a.tokens > 4) {
    by_share(Two{}, One{});
  } else {
    per <= 4 ? launch(Four{}, Four{}, One{}) : launch(Four{}, Five{}, One{});
  }
}

// Sizes whose padded forms can be counted in 32 bits.
constexpr int kMaxRows = 1 << 28, kMaxCols = 1 << 24;

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
  if (out_features > kMaxRows || in_features > kMaxCols) {
    return fail(INFER_HIP_INVALID_ARGUMENT, "gemv_w4a16: N=%d K=%d are over %d x %d", out_features,
                in_features, kMaxRows, kMaxCols);
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
  const W4Args a{weight, scales,       bias,        input,     output,
                 tokens, out_features, in_features, group_size};
  if (group_size == 32) {
    launch_w4<32>(a, stream);
  } else if (group_size == 64) {
    launch_w4<64>(a, stream);
  } else {
    launch_w4<128>(a, stream);
  }
  return check_launch("gemv_w4a16");
}
