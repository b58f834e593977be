// Paged KV cache kernels for gfx950: store with RoPE and quantisation, load
// back, and the attention of one new token a sequence.
#include <float.h>
#include <stdint.h>

#include <type_traits>

#include "device_common.hpp"
#include "paged_kernels.hpp"

namespace qlin {

namespace {

constexpr int kThreads = 256;
constexpr int kBf16 = INFER_HIP_KV_BF16, kInt8 = INFER_HIP_KV_INT8, kFp8 = INFER_HIP_KV_FP8;

template <int F>
constexpr float kLimit = F == kInt8 ? 127.0f : 448.0f;

// Index of the pool's row (page, head, slot); page in range.
__device__ __forceinline__ size_t pool_row(const KvPool& p, int page, int head, int slot) {
  return ((static_cast<size_t>(page) * p.kv_heads + head) << p.page_shift) + slot;
}

__device__ __forceinline__ void unpack8(uint4 w, float (&x)[8]) {
  x[0] = bf16_lo(w.x); x[1] = bf16_hi(w.x); x[2] = bf16_lo(w.y); x[3] = bf16_hi(w.y);
  x[4] = bf16_lo(w.z); x[5] = bf16_hi(w.z); x[6] = bf16_lo(w.w); x[7] = bf16_hi(w.w);
}

__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3]), pack2_bf16(x[4], x[5]),
                    pack2_bf16(x[6], x[7]));
}

// Eight elements of a format, v / scale rounded and clamped to its range (scale
// 0 or NaN: v itself; what a row with either holds does not show).
template <int F>
__device__ __forceinline__ uint2 quantise8(const float (&v)[8], float scale) {
  const float by = scale > 0.0f ? scale : 1.0f;
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = fminf(fmaxf(v[i] / by, -kLimit<F>), kLimit<F>);
  uint2 w;
  if (F == kInt8) {
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = static_cast<uint32_t>(static_cast<int>(rintf(q[i]))) & 255u;
    w.x = b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
    w.y = b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24;
  } else {
    int x = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    w.x = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], x, true);
    x = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
    w.y = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], x, true);
  }
  return w;
}

template <int F>
__device__ __forceinline__ void dequantise8(uint2 w, float scale, float (&x)[8]) {
  if (F == kInt8) {
    x[0] = sbyte0(w.x); x[1] = sbyte1(w.x); x[2] = sbyte2(w.x); x[3] = sbyte3(w.x);
    x[4] = sbyte0(w.y); x[5] = sbyte1(w.y); x[6] = sbyte2(w.y); x[7] = sbyte3(w.y);
  } else {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w.x, false);
    const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(w.x, true);
    const auto c = __builtin_amdgcn_cvt_pk_f32_fp8(w.y, false);
    const auto d = __builtin_amdgcn_cvt_pk_f32_fp8(w.y, true);
    x[0] = a[0]; x[1] = a[1]; x[2] = b[0]; x[3] = b[1];
    x[4] = c[0]; x[5] = c[1]; x[6] = d[0]; x[7] = d[1];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= scale;
}

// RoPE of eight pairs (lo[i], hi[i]) by the (cos, sin) at cs.  Each operation
// is rounded by itself (no FMA), so that a quantised element does not depend
// on how the compiler contracts them.
__device__ __forceinline__ void rotate8(float (&lo)[8], float (&hi)[8], const float* cs) {
#pragma clang fp contract(off)
  float c[16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 w = load_global16(cs + 4 * i);
    c[4 * i] = __uint_as_float(w.x);
    c[4 * i + 1] = __uint_as_float(w.y);
    c[4 * i + 2] = __uint_as_float(w.z);
    c[4 * i + 3] = __uint_as_float(w.w);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = lo[i], y = hi[i];
    const float xc = x * c[2 * i], ys = y * c[2 * i + 1];
    const float yc = y * c[2 * i], xs = x * c[2 * i + 1];
    lo[i] = xc - ys;
    hi[i] = yc + xs;
  }
}

// ------------------------------------------------------------------ store --

// q' = q R(pos), k' = k R(pos), v' = v; q' to BF16; a row x of k' or v' to x / s in
// the pool's format, s = max|x| / limit.  A row (token, query head | key head | value
// head) takes D / 16 lanes; lane c holds elements 8 c .. + 8 of both halves, i.e.
// whole RoPE pairs, so a row's maximum is three exchanges at most and nothing waits
// for another row: any number of tokens, of any sequences, is one grid.
//
// Bound: bytes.  6 prompts of up to 5000 tokens of 32 + 2 x 8 heads of 128 in FP8 (396
// MB) 76 us, 5.2 TB/s, a copy 5.0.  A decode step (24 tokens of 14 + 2 x 2 heads of
// 64) is 2.9 us, 1.7 of them the launch, the rest two reads one behind the other:
// position, sequence and row, then page and rotation.  Non-temporal loads or stores
// gained 2-3 % on some sizes and lost as much on others.
template <int F, int D>
__global__ __launch_bounds__(kThreads) void kv_store_kernel(KvStoreArgs a) {
  constexpr int L = D / 16;
  const unsigned rows = a.heads + 2 * a.pool.kv_heads;
  const unsigned item = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const int c = threadIdx.x % L;
  const unsigned t = item / rows;
  if (t >= static_cast<unsigned>(a.tokens)) return;  // whole groups of L lanes
  const int row = item % rows;
  // Position, sequence and row are read together, then the page and the rotation.
  const int pos = a.positions[t];
  const int seq = a.sequence_ids ? a.sequence_ids[t] : static_cast<int>(t);
  const bool is_q = row < a.heads;
  const bool is_v = row >= a.heads + a.pool.kv_heads;
  const int head = is_q ? row : is_v ? row - a.heads - a.pool.kv_heads : row - a.heads;
  const uint16_t* src = (is_q ? a.q + t * a.q_stride : is_v ? a.v + t * a.v_stride
                                                            : a.k + t * a.k_stride) +
                        static_cast<size_t>(head) * D + 8 * c;
  const uint4 row_lo = load_global16(src), row_hi = load_global16(src + D / 2);
  asm volatile("" ::: "memory");  // not behind the ways out
  if (pos < 0 || (a.rope && pos >= a.rope_positions)) return;
  const int index = pos >> a.pool.page_shift;
  const bool placed = !is_q &&
                      static_cast<unsigned>(seq) < static_cast<unsigned>(a.table.sequences) &&
                      index < a.table.max_pages;
  const int page =
      placed ? a.table.pages[static_cast<size_t>(seq) * a.table.stride + index] : -1;
  float lo[8], hi[8];
  unpack8(row_lo, lo);
  unpack8(row_hi, hi);
  if (a.rope && !is_v) {
    rotate8(lo, hi, a.rope + static_cast<size_t>(pos) * D + 16 * c);
  }
  if (is_q) {
    uint16_t* dst = a.q_out + t * a.q_out_stride + static_cast<size_t>(head) * D + 8 * c;
    store_global16(dst, pack8(lo));
    store_global16(dst + D / 2, pack8(hi));
    return;
  }
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.pool.num_pages)) return;
  const size_t at = pool_row(a.pool, page, head, pos & ((1 << a.pool.page_shift) - 1));
  void* pages = is_v ? a.pool.value : a.pool.key;
  if (F == kBf16) {
    uint16_t* dst = static_cast<uint16_t*>(pages) + at * D + 8 * c;
    store_global16(dst, pack8(lo));
    store_global16(dst + D / 2, pack8(hi));
    return;
  }
  // max|v| over the row on the bits of |v|: a NaN is larger than an infinity
  // and both larger than any finite value.
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m = max(m, max(__float_as_uint(fabsf(lo[i])), __float_as_uint(fabsf(hi[i]))));
  }
#pragma unroll
  for (int o = 1; o < L; o <<= 1) {
    m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), o)));
  }
  const float scale = m >= 0x7F800000u ? __uint_as_float(0x7FC00000u)
                                       : __uint_as_float(m) / kLimit<F>;
  uint8_t* dst = static_cast<uint8_t*>(pages) + at * D + 8 * c;
  store_global8(dst, quantise8<F>(lo, scale));
  store_global8(dst + D / 2, quantise8<F>(hi, scale));
  if (c == 0) (is_v ? a.pool.value_scales : a.pool.key_scales)[at] = scale;
}

// ------------------------------------------------------------------- load --

// NT: what is written is not to be kept in the caches.
template <bool NT>
__device__ __forceinline__ void store_as(void* p, uint4 v) {
  const u32x4 w = {v.x, v.y, v.z, v.w};
  if (NT) {
    __builtin_nontemporal_store(w, (QLIN_GLOBAL u32x4*)(p));
  } else {
    *(QLIN_GLOBAL u32x4*)(p) = w;
  }
}

// bf16(element * scale), one rounding.  One lane per 8 elements of a row; blockIdx.x
// over rows, y the KV head, z the sequence; the grid covers the capacity, and rows
// behind a length end after one load.  Bound: bytes (launch_kv_load has the figures).
template <int F, int D, bool NT>
__global__ __launch_bounds__(kThreads) void kv_load_kernel(KvLoadArgs a) {
  constexpr int L = D / 8;
  const int seq = blockIdx.z, head = blockIdx.y, c = threadIdx.x % L;
  const long long r = static_cast<long long>(blockIdx.x) * (kThreads / L) + threadIdx.x / L;
  const int n = min(min(a.lengths[seq], a.capacity), a.table.max_pages << a.pool.page_shift);
  if (r >= n) return;
  const int pos = static_cast<int>(r);
  const int page =
      a.table.pages[static_cast<size_t>(seq) * a.table.stride + (pos >> a.pool.page_shift)];
  const size_t to =
      ((static_cast<size_t>(seq) * a.pool.kv_heads + head) * a.capacity + pos) * D + 8 * c;
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.pool.num_pages)) {
    const uint4 nan = make_uint4(0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u);
    store_as<NT>(a.key_cache + to, nan);
    store_as<NT>(a.value_cache + to, nan);
    return;
  }
  const size_t at = pool_row(a.pool, page, head, pos & ((1 << a.pool.page_shift) - 1));
  if (F == kBf16) {
    const uint4 k = load_global16(static_cast<const uint16_t*>(a.pool.key) + at * D + 8 * c);
    const uint4 v = load_global16(static_cast<const uint16_t*>(a.pool.value) + at * D + 8 * c);
    store_as<NT>(a.key_cache + to, k);
    store_as<NT>(a.value_cache + to, v);
    return;
  }
  const uint2 k = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.pool.key) +
                                                  at * D + 8 * c);
  const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.pool.value) +
                                                  at * D + 8 * c);
  float x[8];
  dequantise8<F>(k, a.pool.key_scales[at], x);
  store_as<NT>(a.key_cache + to, pack8(x));
  dequantise8<F>(v, a.pool.value_scales[at], x);
  store_as<NT>(a.value_cache + to, pack8(x));
}

// -------------------------------------------------------------- attention --
//
// out[s][h] = sum_j p_j v_j / sum_j p_j, p_j = 2^((q.k_j - m) log2(e) / sqrt(d)).
//
// Work.  A unit is a (sequence, KV head, block of at most 16 query heads) and
// has ceil(length / 32) tiles of 32 keys.  All tiles of a call, in the order
// (sequence, unit, tile), are cut into equal pieces, one a workgroup, from the
// lengths on the device: the load is even whatever the lengths, and a graph
// captured once follows them.  A workgroup's waves cut its piece again; each
// walks its tiles alone, without barriers.  A unit that ends inside one wave is
// written by it, one inside a workgroup is joined there through LDS, and one
// over several by a second launch, in the order of its tiles.  (Joined inside
// the launch by the last workgroup to arrive, in two levels of 16, 131001 keys
// of two KV heads took 42 us against 35 with a second launch, before other
// changes: coherent stores, an atomic and the loads of what other XCDs wrote
// cost 4 us a level under load.)  Where the tables leave room for short
// sequences only, the cuts move to the units' ends instead and the second
// launch is left out.
//
// Tile.  S = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_bf16.  With lane =
// 16 g + r: S's lanes hold head r's scores of keys 4 g .. + 3 of the tile's two
// halves of 16, which is the layout P^T is read in if the contraction over keys
// runs in that order, so P never moves between lanes; V^T's lanes read their
// eight keys' dimensions r D / 16 .. and pair them up in registers.  Keys and
// values go from memory to registers once, the next tile's while this one is
// multiplied.  8-bit elements become BF16 exactly; their scales go onto the
// scores and the weights.  A weight is the sum of three BF16 numbers of eight bits
// each, exactly, none of them negative, so that an infinite value gives that infinity
// (rounded to one, the error was 1.35 times the output rounding's own; to two, a
// remainder of 0 or below made NaN of infinities; the third costs 0-4 %).  Maxima,
// sums and O are FP32.  The maximum m is a sum q.k itself and comes off before the
// factor: the difference of two close scores is exact, so the largest one's weight is 1
// however large it is.  (Taken off as a rounded product, it leaves half of the product's
// last bit in the exponent, 2^7 from 2^31 up.)
//
// Bound.  Large calls: the cache's bytes, 1 x 131001 keys of 2 x 128 in BF16 (134 MB)
// 30.5 us, 64 sequences of up to 4000 of 8 x 128 in FP8 (270 MB) 53 us, 5.1 TB/s;
// a read alone runs at 7.0.  A tile in flight a wave and eight waves a CU are what
// the registers hold (two tiles in flight, or more waves, gained nothing).  Small
// calls: the launches and their chains of dependent reads, lengths, table, keys: 1 x
// 101 keys 4.8 us, 16 x 2000 in INT8 9.6 us, 3.1 of them the second launch.

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kTileKeys = 32;
constexpr int kHeadBlock = 16;       // query heads of a unit at most
constexpr float kRescaleSlack = 6.0f;  // p <= 2^6 before the maximum is moved

// log2(e) / sqrt(D): a weight's exponent per unit of q.k.
template <int D>
constexpr float kExponent = D == 64 ? 0.18033688011112042f : 0.12751743082459868f;

// A uniform 32-bit word that nothing writes while the kernel runs, through the
// scalar cache.
__device__ __forceinline__ int scalar_word(const int* p) {
  return *(const __attribute__((address_space(4))) int*)(reinterpret_cast<uintptr_t>(p));
}

// N bytes of a lane; NT: marked as not to be kept in the caches.
template <bool NT, typename T>
__device__ __forceinline__ T load_as(const void* p) {
  const QLIN_GLOBAL T* const at = (const QLIN_GLOBAL T*)(p);
  return NT ? __builtin_nontemporal_load(at) : *at;
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <int N>
struct Words;
template <>
struct Words<4> {
  uint32_t w[1];
  template <bool NT>
  __device__ __forceinline__ void load(const uint8_t* p) {
    w[0] = load_as<NT, uint32_t>(p);
  }
};
template <>
struct Words<8> {
  uint32_t w[2];
  template <bool NT>
  __device__ __forceinline__ void load(const uint8_t* p) {
    const u32x2 v = load_as<NT, u32x2>(p);
    w[0] = v.x;
    w[1] = v.y;
  }
};
template <>
struct Words<16> {
  uint32_t w[4];
  template <bool NT>
  __device__ __forceinline__ void load(const uint8_t* p) {
    const u32x4 v = load_as<NT, u32x4>(p);
    w[0] = v.x;
    w[1] = v.y;
    w[2] = v.z;
    w[3] = v.w;
  }
};

// Low (high) halves of two dwords: a's in bits 0-15.
__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x05040100u);
}
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}

// Byte b of w, an int8, as the FP32 whose high half is its BF16.
template <int B>
__device__ __forceinline__ uint32_t int8_f32(uint32_t w) {
  return __float_as_uint(B == 0 ? sbyte0(w) : B == 1 ? sbyte1(w) : B == 2 ? sbyte2(w) : sbyte3(w));
}

// Two FP8 of a dword (its low or high half) as a BF16 pair.
template <bool HIGH>
__device__ __forceinline__ uint32_t fp8_pair(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH));
}

// Eight 8-bit elements in order as BF16.
template <int F>
__device__ __forceinline__ bf16x8_t widen8(uint32_t lo, uint32_t hi) {
  uint4 r;
  if (F == kInt8) {
    r.x = high_halves(int8_f32<0>(lo), int8_f32<1>(lo));
    r.y = high_halves(int8_f32<2>(lo), int8_f32<3>(lo));
    r.z = high_halves(int8_f32<0>(hi), int8_f32<1>(hi));
    r.w = high_halves(int8_f32<2>(hi), int8_f32<3>(hi));
  } else {
    r.x = fp8_pair<false>(lo);
    r.y = fp8_pair<true>(lo);
    r.z = fp8_pair<false>(hi);
    r.w = fp8_pair<true>(hi);
  }
  return __builtin_bit_cast(bf16x8_t, r);
}

// V^T fragments of a lane: frag[j] = dimension j of eight keys, key e in
// element e, from the keys' words.
template <int F, int D, int N>
__device__ __forceinline__ void turn_values(const Words<N> (&v)[8], bf16x8_t (&frag)[D / 16]) {
#pragma unroll
  for (int w = 0; w < N / 4; ++w) {
    uint32_t out[F == kBf16 ? 2 : 4][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t a = v[2 * e].w[w], b = v[2 * e + 1].w[w];
      if (F == kBf16) {
        out[0][e] = low_halves(a, b);
        out[1][e] = high_halves(a, b);
      } else if (F == kInt8) {
        out[0][e] = high_halves(int8_f32<0>(a), int8_f32<0>(b));
        out[1][e] = high_halves(int8_f32<1>(a), int8_f32<1>(b));
        out[2][e] = high_halves(int8_f32<2>(a), int8_f32<2>(b));
        out[3][e] = high_halves(int8_f32<3>(a), int8_f32<3>(b));
      } else {
        const uint32_t al = fp8_pair<false>(a), bl = fp8_pair<false>(b);
        const uint32_t ah = fp8_pair<true>(a), bh = fp8_pair<true>(b);
        out[0][e] = low_halves(al, bl);
        out[1][e] = high_halves(al, bl);
        out[2][e] = low_halves(ah, bh);
        out[3][e] = high_halves(ah, bh);
      }
    }
    constexpr int per = F == kBf16 ? 2 : 4;
#pragma unroll
    for (int j = 0; j < per; ++j) {
      frag[w * per + j] = __builtin_bit_cast(
          bf16x8_t, make_uint4(out[j][0], out[j][1], out[j][2], out[j][3]));
    }
  }
}

// The top eight bits of eight numbers of one sign, as BF16, and the rest left of them:
// taken three times, all 24.
__device__ __forceinline__ bf16x8_t take_top8(float (&p)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = high_halves(__float_as_uint(p[2 * i]), __float_as_uint(p[2 * i + 1]));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) p[i] -= __uint_as_float(__float_as_uint(p[i]) & 0xFFFF0000u);
  return __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
}

// A lower part that is 0 as 2^-126: an infinite value times every part of a weight is
// that infinity then, where 0 would make it NaN.  8-bit pages hold no infinities.
template <int F>
__device__ __forceinline__ bf16x8_t part_above_zero(bf16x8_t p) {
  typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
  if (F != kBf16) return p;
  const u16x8 least = 0x0080, bits = __builtin_bit_cast(u16x8, p);
  return __builtin_bit_cast(bf16x8_t, __builtin_elementwise_max(bits, least));
}

// Over the four lanes r, 16 + r, 32 + r, 48 + r.
__device__ __forceinline__ float groups_max(float v) {
  int w = __float_as_int(v);
  const auto a = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  v = fmaxf(__int_as_float(a[0]), __int_as_float(a[1]));
  w = __float_as_int(v);
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return fmaxf(__int_as_float(b[0]), __int_as_float(b[1]));
}
__device__ __forceinline__ float groups_sum(float v) {
  v = swap16_sum(v, v);
  return swap32_sum(v, v);
}

// Inclusive prefix sums over the wave.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr:1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15, 31
  return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
}

// Tiles of the walk a wave takes, of all in `waves` equal parts.
__device__ __forceinline__ int piece_of(int total, int waves) {
  return max(1, (total + waves - 1) / waves);
}

// What O is divided by, inverted: without any weight NaN (the 2^-126s of
// part_above_zero leave O a little off 0).
__device__ __forceinline__ float inverse(float sum) {
  return sum == 0.0f ? __uint_as_float(0x7FC00000u) : 1.0f / sum;
}

// Four dimensions of the output from O and the sum of the weights.
__device__ __forceinline__ void store_out(uint16_t* out, f32x4_t o, float sum) {
  const float inv = inverse(sum);
  store_global8(out, make_uint2(pack2_bf16(o[0] * inv, o[1] * inv),
                                pack2_bf16(o[2] * inv, o[3] * inv)));
}

__device__ __forceinline__ int tiles_of(int n) { return (n + kTileKeys - 1) / kTileKeys; }

// One tile of the walk (wave-uniform).
struct TileAt {
  int seq, unit;    // unit: KV head * head blocks + head block
  int kvh, block;
  int tile, tiles;  // of the unit
  int n;            // length of the sequence
};

// A part of a unit that is not whole: which tiles, and where the unit lies in
// the walk.
struct PartTag {
  int first;  // the unit's first tile in the walk
  int tiles;
  int seq, unit;
  int begin, end;  // the part's tiles; end 0: no part
};

// W waves a workgroup; HB: room for that many query heads of a unit in LDS; NT:
// keys and values are not to be kept in the caches.
template <int F, int D, int W, int HB, bool NT>
__global__ __launch_bounds__(W * kWave, 2) void paged_attention_kernel(PagedAttnArgs a) {
  constexpr int ES = F == kBf16 ? 2 : 1;
  constexpr int RB = D * ES;       // bytes of a row
  constexpr int KC = RB / 64;      // 16-byte pieces of a key per lane
  constexpr int VB = RB / 16;      // bytes of a value row per lane
  constexpr int NQ = D / 32;       // MFMA steps of q.k
  constexpr int NO = D / 16;       // dimensions of O per lane and register row
  // the states of parts of units: O [2 W][HB][D], then (maximum, sum)
  __shared__ __align__(16) float smem[2 * W * HB * (D + 2)];
  __shared__ PartTag tags[2 * W];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int units = a.units, cap = a.table.max_pages << a.pool.page_shift;
  const int heads_per_kv = a.heads / a.pool.kv_heads;
  const int hb = min(heads_per_kv, kHeadBlock);  // query heads of a full unit
  const int mask = (1 << a.pool.page_shift) - 1;

  // ---- the wave's part of the walk.  Lane i: sequence i's tiles, and those of
  // all up to it (of the first 64 sequences).
  auto length = [&](int i) {
    return i < a.table.sequences ? max(0, min(a.lengths[i], cap)) : 0;
  };
  const int n_first = length(lane), upto_first = wave_scan(tiles_of(n_first));
  int total = __builtin_amdgcn_readlane(upto_first, kWave - 1);
  if (a.table.sequences > kWave) {
    int more = 0;
    for (int i = kWave + lane; i < a.table.sequences; i += kWave) more += tiles_of(length(i));
    total += __builtin_amdgcn_readlane(wave_scan(more), kWave - 1);
  }
  total *= units;
  // Where tile x < total of the walk lies.
  auto locate = [&](int x) {
    TileAt at{};
    int n = n_first, upto = upto_first;
    for (int base = 0, run = 0; base < a.table.sequences; base += kWave) {
      if (base > 0) {
        n = length(base + lane);
        upto = wave_scan(tiles_of(n));
      }
      const unsigned long long hit = __ballot((run + upto) * units > x);
      if (hit) {
        const int i = __builtin_ctzll(hit);
        at.seq = base + i;
        at.n = __builtin_amdgcn_readlane(n, i);
        at.tiles = tiles_of(at.n);
        const unsigned rest = x - (run + __builtin_amdgcn_readlane(upto, i) - at.tiles) * units;
        at.unit = rest / static_cast<unsigned>(at.tiles);
        at.tile = rest - at.unit * at.tiles;
        at.kvh = HB == 8 ? at.unit : at.unit / a.head_blocks;
        at.block = HB == 8 ? 0 : at.unit - at.kvh * a.head_blocks;
        break;
      }
      run += __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    return at;
  };
  const int piece = piece_of(total, a.waves) * W;
  int group_start = min(total, static_cast<int>(blockIdx.x) * piece);
  int group_end = min(total, group_start + piece);
  if (a.whole) {  // to the nearer end of the unit that a cut is in
    auto moved = [&](int x) {
      if (x >= total) return total;
      const TileAt at = locate(x);
      return 2 * at.tile <= at.tiles ? x - at.tile : x - at.tile + at.tiles;
    };
    group_start = moved(group_start);
    group_end = moved(group_end);
  }
  const int chunk = (group_end - group_start + W - 1) / W;
  const int start = min(group_end, group_start + wave * chunk);
  const int end = min(group_end, start + chunk);

  if (lane < 2) tags[2 * wave + lane].end = 0;

  if (start < end) {
    const TileAt at = locate(start);

    auto advance = [&](TileAt& t) {
      if (++t.tile < t.tiles) return;
      t.tile = 0;
      if (HB == 8 || ++t.block == a.head_blocks) {
        t.block = 0;
        ++t.kvh;
      }
      if (++t.unit < units) return;
      t.unit = 0;
      t.kvh = 0;
      do {  // a later tile exists, so a later sequence with keys does
        ++t.seq;
        t.n = max(0, min(scalar_word(a.lengths + t.seq), cap));
        t.tiles = tiles_of(t.n);
      } while (t.tiles == 0 && t.seq + 1 < a.table.sequences);
    };

    bf16x8_t q[NQ], q_next[NQ];
    auto load_q = [&](const TileAt& t, bf16x8_t (&to)[NQ]) {
      const int h = t.kvh * heads_per_kv + min(t.block * kHeadBlock + r, heads_per_kv - 1);
      const uint16_t* p = a.q + t.seq * a.q_stride + static_cast<size_t>(h) * D;
#pragma unroll
      for (int m = 0; m < NQ; ++m) {
        const int dim = F == kBf16 ? 32 * m + 8 * g : 64 * (m >> 1) + 16 * g + 8 * (m & 1);
        to[m] = __builtin_bit_cast(bf16x8_t, load_global16(p + dim));
      }
    };

    // A tile's two halves of 16 keys each lie in one page.  Rows of a half past
    // the sequence's end are read with it (the page is there) and dropped; a
    // second half wholly past the end reads the first again.
    const bool small_pages = a.pool.page_shift == 4;
    const uint32_t page_rows = static_cast<uint32_t>(a.pool.kv_heads) << a.pool.page_shift;
    int e0 = 0, e1 = 0;  // page entries of the tile to be loaded next
    auto look_up = [&](const TileAt& t) {
      const int* row = a.table.pages + static_cast<size_t>(t.seq) * a.table.stride;
      e0 = scalar_word(row + (t.tile * kTileKeys >> a.pool.page_shift));
      if (small_pages) {
        e1 = scalar_word(row + (t.tile * 2 + (t.tile * kTileKeys + 16 < t.n ? 1 : 0)));
      }
    };
    size_t row[2];  // of the pool, the halves' first keys
    bool bad;       // a page is not in the pool
    auto find_rows = [&](const TileAt& t) {
      const uint32_t pages = a.pool.num_pages;
      const bool two = t.tile * kTileKeys + 16 < t.n;
      const uint32_t head_row = static_cast<uint32_t>(t.kvh) << a.pool.page_shift;
      bad = static_cast<uint32_t>(e0) >= pages;
      row[0] = static_cast<size_t>(bad ? 0 : e0) * page_rows + head_row +
               (t.tile * kTileKeys & mask);
      row[1] = row[0] + (two ? 16 : 0);
      if (small_pages) {
        const bool bad1 = static_cast<uint32_t>(e1) >= pages;
        row[1] = static_cast<size_t>(bad1 ? 0 : e1) * page_rows + head_row;
        bad = bad || bad1;
      }
    };

    u32x4 k[2][KC];
    Words<VB> v[8];
    f32x4_t ks[2], vs[2];
    // In BF16 a lane loads of the keys what the lane with g and r's low bits exchanged
    // multiplies: four lanes in a row then read 64 bytes in a row, not 16 of four keys (28
    // / 4 / 128 heads: 1 x 500 keys 9.0 -> 8.1 us, 16 x 500 9.4 -> 8.5, 1 x 131001 30.7 ->
    // 30.4).  8-bit keys, half the loads, lose by the exchange (in INT8 8.4 -> 9.1, 8.6 ->
    // 9.2).
    constexpr bool kTurned = F == kBf16;
    const uint32_t k_off = kTurned ? ((lane & 12) | g) * RB + 16 * (lane & 3) : r * RB + 16 * g;
    const uint32_t v_off = 4 * g * RB + r * VB;
    const int from = 4 * ((r & 3) << 4 | (r & 12) | g);
    auto load_keys = [&] {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* base = static_cast<const uint8_t*>(a.pool.key) + row[h] * RB;
#pragma unroll
        for (int c = 0; c < KC; ++c) k[h][c] = load_as<NT, u32x4>(base + k_off + 64 * c);
        if (F != kBf16) {
          ks[h] = gload(reinterpret_cast<const f32x4_t*>(a.pool.key_scales + row[h]) + g);
        }
      }
    };
    auto load_values = [&] {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* base = static_cast<const uint8_t*>(a.pool.value) + row[h] * RB;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * h + i].template load<NT>(base + v_off + i * RB);
        if (F != kBf16) {
          vs[h] = gload(reinterpret_cast<const f32x4_t*>(a.pool.value_scales + row[h]) + g);
        }
      }
    };

    f32x4_t acc[NO];
    float m = -FLT_MAX, l = 0.0f;
#pragma unroll
    for (int j = 0; j < NO; ++j) acc[j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

    TileAt next = at;
    look_up(next);
    load_q(next, q);
    find_rows(next);
    load_keys();
    load_values();
    int begin = at.tile;  // of the part of the current unit
    bool first_part = true, part_bad = bad;
    TileAt t = at;
    if (start + 1 < end) {
      advance(next);
      look_up(next);
    }

    // One tile; MORE (a constant): another follows, whose loads are issued on the
    // way.  The last tile is apart from the loop, so that every pass of the loop
    // has the same loads in flight and waits for those it needs alone.
    auto step = [&](int idx, auto more_tiles) {
      constexpr bool more = decltype(more_tiles)::value;
      // S of both halves, times the keys' scales
      float s[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f32x4_t d{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          if (F == kBf16) {
            const uint4 mine = lane_of(__builtin_bit_cast(uint4, k[h][c]), from);
            d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, mine), q[c], d,
                                                        0, 0, 0);
          } else {
            d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8<F>(k[h][c].x, k[h][c].y), q[2 * c],
                                                        d, 0, 0, 0);
            d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8<F>(k[h][c].z, k[h][c].w),
                                                        q[2 * c + 1], d, 0, 0, 0);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * h + i] = F == kBf16 ? d[i] : d[i] * ks[h][i];
      }
      const bool unit_ends = more && next.tile == 0;
      if (more) {
        find_rows(next);
        load_keys();
        if (unit_ends) load_q(next, q_next);
      }
      const int keys = t.n - t.tile * kTileKeys;  // that the sequence holds
      if (keys < kTileKeys) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (16 * (e >> 2) + 4 * g + (e & 3) >= keys) s[e] = -INFINITY;
        }
      }
      float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])),
                        fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
      top = groups_max(top);
      if (__any(top - m > kRescaleSlack / kExponent<D>)) {
        const float up = fmaxf(m, top);
        const float old = __builtin_amdgcn_exp2f((m - up) * kExponent<D>);
        m = up;
        l *= old;
#pragma unroll
        for (int j = 0; j < NO; ++j) acc[j] *= old;
      }
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f((s[e] - m) * kExponent<D>);
        l += p[e];
        if (F != kBf16) p[e] *= vs[e >> 2][e & 3];
      }
      if (keys < kTileKeys) {  // what is read past the end counts for nothing
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (16 * (e >> 2) + 4 * g + (e & 3) >= keys) {
            p[e] = 0.0f;
#pragma unroll
            for (int w = 0; w < VB / 4; ++w) v[e].w[w] = 0;
          }
        }
      }
      const bf16x8_t p_hi = take_top8(p);
      const bf16x8_t p_mid = part_above_zero<F>(take_top8(p));
      const bf16x8_t p_lo = part_above_zero<F>(take_top8(p));
      bf16x8_t vf[NO];
      turn_values<F, D, VB>(v, vf);
#pragma unroll
      for (int j = 0; j < NO; ++j) {
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[j], p_hi, acc[j], 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < NO; ++j) {
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[j], p_mid, acc[j], 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < NO; ++j) {
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[j], p_lo, acc[j], 0, 0, 0);
      }
      if (more) load_values();
      if (!more || unit_ends) {
        float sum_l = groups_sum(l);
        if (part_bad) sum_l = __uint_as_float(0x7FC00000u);
        const int h = t.block * kHeadBlock + r;
        if (begin == 0 && t.tile + 1 == t.tiles) {
          if (h < heads_per_kv) {
            const float inv = inverse(sum_l);
            const int head = t.kvh * heads_per_kv + h;
            uint16_t* out =
                a.out + (static_cast<size_t>(t.seq) * a.heads + head) * D + 4 * g * NO;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t w[NO / 2];
#pragma unroll
              for (int j = 0; j < NO / 2; ++j) {
                w[j] = pack2_bf16(acc[2 * j][i] * inv, acc[2 * j + 1][i] * inv);
              }
              if constexpr (NO == 8) {
                store_global16(out + i * NO, make_uint4(w[0], w[1], w[2], w[3]));
              } else {
                store_global8(out + i * NO, make_uint2(w[0], w[1]));
              }
            }
          }
        } else {
          const int slot = 2 * wave + (first_part ? 0 : 1);
          if (r < hb) {
            float* rec = smem + (slot * HB + r) * D + 4 * g * NO;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
              for (int j = 0; j < NO; ++j) rec[i * NO + j] = acc[j][i];
            }
            if (g == 0) {
              float* ml = smem + 2 * W * HB * D + (slot * HB + r) * 2;
              ml[0] = m;
              ml[1] = sum_l;
            }
          }
          if (lane == 0) {
            tags[slot] = PartTag{idx - t.tile, t.tiles, t.seq, t.unit, begin, t.tile + 1};
          }
        }
        first_part = false;
        begin = 0;
        part_bad = false;
        m = -FLT_MAX;
        l = 0.0f;
#pragma unroll
        for (int j = 0; j < NO; ++j) acc[j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NQ; ++i) q[i] = q_next[i];
      }
      if (more) {
        part_bad = part_bad || bad;
        t = next;
        if (idx + 2 < end) {
          advance(next);
          look_up(next);
        }
      }
    };
    for (int idx = start; idx < end - 1; ++idx) step(idx, std::true_type{});
    step(end - 1, std::false_type{});
  }

  // ---- empty sequences
  if (a.table.sequences > kWave || __ballot(lane < a.table.sequences && n_first == 0)) {
    for (int s = blockIdx.x; s < a.table.sequences; s += gridDim.x) {
      if (scalar_word(a.lengths + s) > 0) continue;
      uint16_t* out = a.out + static_cast<size_t>(s) * a.heads * D;
      for (int e = threadIdx.x; e < a.heads * (D / 8); e += W * kWave) {
        store_global16(out + 8 * e, make_uint4(0, 0, 0, 0));
      }
    }
  }
  if (group_start >= group_end) return;  // the whole workgroup
  __syncthreads();

  // ---- the workgroup's parts: neighbours of one unit together
  const float* ml_at = smem + 2 * W * HB * D;
  {
    const PartTag mine = tags[lane & (2 * W - 1)];
    const uint32_t there = static_cast<uint32_t>(__ballot(lane < 2 * W && mine.end != 0));
    const uint32_t before = there & ((1u << (lane & 31)) - 1u);
    const int previous = __shfl(mine.first, before ? 31 - __builtin_clz(before) : 0);
    const uint32_t starts = static_cast<uint32_t>(__ballot(
        lane < 2 * W && mine.end != 0 && (before == 0 || previous != mine.first)));
    const int runs = __builtin_popcount(starts), per_run = hb * (D / 4);
    for (int x = threadIdx.x; x < runs * per_run; x += W * kWave) {
      const int run = x / per_run, e = x - run * per_run;
      uint32_t left = starts;
      for (int i = 0; i < run; ++i) left &= left - 1;
      const int i = __builtin_ctz(left);
      left &= left - 1;
      const uint32_t in = there & ~((1u << i) - 1u) & (left ? (left & -left) - 1u : ~0u);
      const int last = 31 - __builtin_clz(in);
      const PartTag tag = tags[i];
      const bool whole = tag.begin == 0 && tags[last].end == tag.tiles;
      const int kvh = HB == 8 ? tag.unit : tag.unit / a.head_blocks;
      const int block = HB == 8 ? 0 : tag.unit - kvh * a.head_blocks;
      const int h = e / (D / 4), d = 4 * (e % (D / 4));
      const int head = block * kHeadBlock + h;
      if (head >= heads_per_kv) continue;
      float top = -FLT_MAX, sum_l = 0.0f;
      for (uint32_t w = in; w; w &= w - 1) {
        top = fmaxf(top, ml_at[(__builtin_ctz(w) * HB + h) * 2]);
      }
      f32x4_t o{0.0f, 0.0f, 0.0f, 0.0f};
      for (uint32_t w = in; w; w &= w - 1) {
        const int at = __builtin_ctz(w) * HB + h;
        const float f = __builtin_amdgcn_exp2f((ml_at[at * 2] - top) * kExponent<D>);
        sum_l += f * ml_at[at * 2 + 1];
        o += f * *reinterpret_cast<const f32x4_t*>(smem + at * D + d);
      }
      if (whole) {
        const size_t out_head = static_cast<size_t>(tag.seq) * a.heads + kvh * heads_per_kv + head;
        store_out(a.out + out_head * D + d, o, sum_l);
      } else {
        const int side = tag.begin == 0 ? 1 : 0;  // 1: the unit's first workgroup
        float* rec = a.records + (static_cast<size_t>(blockIdx.x * 2 + side) * hb + h) * (D + 4);
        *reinterpret_cast<f32x4_t*>(rec + d) = o;
        if (d == 0) *reinterpret_cast<f32x4_t*>(rec + D) = f32x4_t{top, sum_l, 0.0f, 0.0f};
      }
    }
  }
}

// Joins the units that lie over several workgroups of the launch before: a
// workgroup of T threads per (unit, sequence), or (a.join_heads 1) per query head
// of one.
template <int D, int T>
__global__ __launch_bounds__(T) void paged_attention_join_kernel(PagedAttnArgs a) {
  constexpr int kJoinBatch = T == 512 ? 8 : 4;  // parts that a thread has in flight
  __shared__ f32x4_t part_o[T + 1];  // the last: no part
  __shared__ float2 part_ml[T + 1];
  const int lane = threadIdx.x & 63;
  const int seq = blockIdx.y;
  const int cap = a.table.max_pages << a.pool.page_shift;
  const int heads_per_kv = a.heads / a.pool.kv_heads;
  const int hb = min(heads_per_kv, kHeadBlock);
  int before = 0, all = 0, tiles = 0;
  for (int i = lane; i < a.table.sequences; i += kWave) {
    const int t = tiles_of(max(0, min(a.lengths[i], cap)));
    all += t;
    if (i < seq) before += t;
    if (i == seq) tiles = t;
  }
  before = __builtin_amdgcn_readlane(wave_scan(before), kWave - 1);
  all = __builtin_amdgcn_readlane(wave_scan(all), kWave - 1);
  tiles = __builtin_amdgcn_readlane(wave_scan(tiles), kWave - 1);
  const int piece = piece_of(all * a.units, a.waves) * a.piece_waves;
  const int unit = a.join_heads ? blockIdx.x / hb : blockIdx.x;
  const int first = before * a.units + unit * tiles;
  const int from = first / piece, to = (first + tiles - 1) / piece;
  if (tiles == 0 || from == to) return;
  const int kvh = unit / a.head_blocks, block = unit - kvh * a.head_blocks;
  const int h0 = a.join_heads ? blockIdx.x - unit * hb : 0;
  const int live = min(hb, heads_per_kv - block * kHeadBlock);  // heads of the unit
  if (h0 >= live) return;
  const int items = (a.join_heads ? 1 : live) * (D / 4);

  // The threads are as many rows of `items` as fit, row i taking parts i, i +
  // rows, ...; what the rows found is joined through LDS.
  const int rows = max(1, T / items), row = rows > 1 ? threadIdx.x / items : 0;
  for (int e0 = 0; e0 < items; e0 += T) {
    const int e = rows > 1 ? static_cast<int>(threadIdx.x) - row * items
                           : e0 + static_cast<int>(threadIdx.x);
    const bool busy = e < items && row < rows;
    const int h = h0 + e / (D / 4), d = 4 * (e % (D / 4));
    float top = -FLT_MAX, sum_l = 0.0f;
    f32x4_t o{0.0f, 0.0f, 0.0f, 0.0f};
    for (int part = busy ? from + row : to + 1; part <= to; part += kJoinBatch * rows) {
      f32x4_t x[kJoinBatch], ml[kJoinBatch];
#pragma unroll
      for (int b = 0; b < kJoinBatch; ++b) {
        const int wg = part + b * rows;
        x[b] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        ml[b] = f32x4_t{-FLT_MAX, 0.0f, 0.0f, 0.0f};
        if (wg > to) continue;
        const float* rec =
            a.records + (static_cast<size_t>(wg * 2 + (wg == from ? 1 : 0)) * hb + h) * (D + 4);
        x[b] = gload(reinterpret_cast<const f32x4_t*>(rec + d));
        ml[b] = gload(reinterpret_cast<const f32x4_t*>(rec + D));
      }
      float next = top;
#pragma unroll
      for (int b = 0; b < kJoinBatch; ++b) next = fmaxf(next, ml[b][0]);
      const float old = __builtin_amdgcn_exp2f((top - next) * kExponent<D>);
      top = next;
      sum_l *= old;
      o *= old;
#pragma unroll
      for (int b = 0; b < kJoinBatch; ++b) {
        const float w = __builtin_amdgcn_exp2f((ml[b][0] - next) * kExponent<D>);
        sum_l += w * ml[b][1];
        o += w * x[b];
      }
    }
    if (rows > 1) {
      if (busy) {
        part_o[row * items + e] = o;
        part_ml[row * items + e] = make_float2(top, sum_l);
      }
      if (threadIdx.x == 0) {
        part_o[T] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        part_ml[T] = make_float2(-FLT_MAX, 0.0f);
      }
      __syncthreads();
      for (int i = 1; i < rows && row == 0; i += kJoinBatch) {
        f32x4_t x[kJoinBatch];
        float2 ml[kJoinBatch];
        float next = top;
#pragma unroll
        for (int b = 0; b < kJoinBatch; ++b) {
          const int at = i + b < rows ? (i + b) * items + e : T;
          x[b] = part_o[at];
          ml[b] = part_ml[at];
          next = fmaxf(next, ml[b].x);
        }
        const float old = __builtin_amdgcn_exp2f((top - next) * kExponent<D>);
        top = next;
        sum_l *= old;
        o *= old;
#pragma unroll
        for (int b = 0; b < kJoinBatch; ++b) {
          const float w = __builtin_amdgcn_exp2f((ml[b].x - next) * kExponent<D>);
          sum_l += w * ml[b].y;
          o += w * x[b];
        }
      }
    }
    if (busy && row == 0) {
      const int head = kvh * heads_per_kv + block * kHeadBlock + h;
      store_out(a.out + (static_cast<size_t>(seq) * a.heads + head) * D + d, o, sum_l);
    }
  }
}

}  // namespace

// Runs f.template operator()<format, head_dim>() for the pool's.
template <typename Fn>
static void by_format(const KvPool& p, Fn&& f) {
  auto by_dim = [&](auto format) {
    if (p.head_dim == 64) {
      f(format, std::integral_constant<int, 64>{});
    } else {
      f(format, std::integral_constant<int, 128>{});
    }
  };
  if (p.format == kBf16) {
    by_dim(std::integral_constant<int, kBf16>{});
  } else if (p.format == kInt8) {
    by_dim(std::integral_constant<int, kInt8>{});
  } else {
    by_dim(std::integral_constant<int, kFp8>{});
  }
}

static long long store_rows(const KvStoreArgs& a) {
  return a.tokens * (a.heads + 2ll * a.pool.kv_heads);
}

// Threads of a grid's x, whole workgroups of them, are under 2^32.
static bool countable(long long rows, int lanes) {
  return rows <= ((1ll << 32) - kThreads) / lanes;
}

bool kv_store_supported(const KvStoreArgs& a) {
  return countable(store_rows(a), a.pool.head_dim / 16);
}

void launch_kv_store(const KvStoreArgs& a, hipStream_t stream) {
  const long long items = store_rows(a);
  by_format(a.pool, [&](auto f, auto d) {
    constexpr int per = kThreads / (decltype(d)::value / 16);
    const unsigned blocks = static_cast<unsigned>((items + per - 1) / per);
    hipLaunchKernelGGL((kv_store_kernel<decltype(f)::value, decltype(d)::value>), dim3(blocks),
                       dim3(kThreads), 0, stream, a);
  });
}

// Bytes that little is left of in the 256 MB memory-side cache when they are read
// again, next to what else a model's layers read.
constexpr long long kStreamBytes = 96ll << 20;

// Positions of a sequence that a load's grid covers.
static long long load_rows(const KvLoadArgs& a) {
  const long long most = static_cast<long long>(a.table.max_pages) << a.pool.page_shift;
  return a.capacity < most ? a.capacity : most;
}

bool kv_load_supported(const KvLoadArgs& a) {
  return countable(load_rows(a), a.pool.head_dim / 8);
}

// A load into caches of more than kStreamBytes does not leave them there: 12 x
// 9000 rows of 4 x 128 INT8 36 -> 25.5 us, 64 x 1000 of 8 x 64 FP8 32 -> 18.  A
// kernel that reads all of it next, and does nothing else, is slower by as much
// (both together 111 us either way; after a store of the same rows 287 -> 284); a
// smaller load's reader finds it in the cache (8 x 8000 of 2 x 64: 18.9 us for both,
// 20.8 without).  So the gain is the load's own, and that of what runs between; the next
// reader pays it back.
void launch_kv_load(const KvLoadArgs& a, hipStream_t stream) {
  const long long rows = load_rows(a);
  by_format(a.pool, [&](auto f, auto d) {
    constexpr int per = kThreads / (decltype(d)::value / 8);
    const dim3 grid(static_cast<unsigned>((rows + per - 1) / per), a.pool.kv_heads,
                    a.table.sequences);
    constexpr int F = decltype(f)::value, D = decltype(d)::value;
    const long long bytes = 4ll * a.table.sequences * a.pool.kv_heads * rows * D;
    if (bytes > kStreamBytes) {
      hipLaunchKernelGGL((kv_load_kernel<F, D, true>), grid, dim3(kThreads), 0, stream, a);
    } else {
      hipLaunchKernelGGL((kv_load_kernel<F, D, false>), grid, dim3(kThreads), 0, stream, a);
    }
  });
}

// Workgroups of the attention: 8 waves a CU, the registers' limit at head_dim
// 128, in workgroups of 8 (of 4 where a unit has more than 8 query heads, whose
// states fill the LDS).
constexpr int kCus = 256;
// Units of more tiles, by the tables' room, are cut.  The join's launch takes 3.1 to
// 5.9 us; a unit left whole is read by one CU, 1.2 us a tile of each wave (one sequence
// of 14 / 2 / 64 heads in BF16: 500 keys 7.4 whole against 9.9 cut, 1000 keys 9.9 against
// 9.8; 28 / 4 / 128 in INT8: 500 keys 9.2 against 10.3, 1000 keys 12.3 against 10.4).
// With more than two units a workgroup the pieces' sizes differ by up to a unit,
// 0.3 us a tile (100 sequences of 500 keys, 28 / 4 / 128 in BF16: 15.7 against
// 17.6; beyond, only small ones stay whole).
constexpr int kWholeTiles = 24, kWholeTilesMany = 8;
// Parts of a unit from which a workgroup of the join has 512 threads (8 heads of 64 on
// one KV head, 131001 keys, 256 parts: 19.1 us, 24.2 with 256; 14 / 2 / 64, 20000 keys,
// 128 parts: 12.3 and 12.9; 12 / 2 / 128, 131001 keys, 128 parts: 30.5 and 31.1; 28 / 4 /
// 128, 30000 keys, 128 parts: 19.7 and 19.8; 16 x 2000 keys, 16 parts: 10.3 and 9.4).
constexpr int kJoinParts = 96;
// Units up to which the join has a workgroup for each of their query heads (1 x
// 131001 keys 30.6 us, 46.0 with one a unit; 8 x 20000 keys of 14 / 2 / 64, 16 units,
// 14.0 and 18.6; 64 x 4000 keys, 512 units, 55.0 and 52.7).
constexpr int kJoinHeadUnits = 64;

// Workgroups of 4 waves instead of 8 start and meet sooner, and spread cut units
// over more CUs: where all units are whole and small or few (1 x 101 keys 5.5 ->
// 4.8 us, 100 x 250 of 14 / 2 / 64 heads 7.4 -> 6.5, but 100 x 500 8.7 -> 9.9), and
// for cut ones of calls with at most kSmallTiles tiles (16 x 2000 keys 10.7 -> 10.0;
// 1 x 100000, as many waves and twice the parts, 16.0 -> 19.1).
constexpr int kSmallWholeTiles = 8, kSmallWholeUnits = 64, kSmallTiles = 4096;

struct PagedAttnShape {
  int head_blocks, units;
  int block_heads;  // query heads of a full unit
  int max_groups;   // workgroups at most
  int record_floats;
};

static PagedAttnShape paged_attention_shape(int heads, int kv_heads, int head_dim) {
  PagedAttnShape s{};
  const int per_kv = heads / kv_heads;
  s.head_blocks = (per_kv + kHeadBlock - 1) / kHeadBlock;
  s.units = kv_heads * s.head_blocks;
  s.block_heads = per_kv < kHeadBlock ? per_kv : kHeadBlock;
  s.max_groups = 2 * kCus;
  s.record_floats = s.block_heads * (head_dim + 4);
  return s;
}

size_t paged_attention_workspace_bytes(int heads, int kv_heads, int head_dim) {
  const PagedAttnShape s = paged_attention_shape(heads, kv_heads, head_dim);
  return static_cast<size_t>(s.max_groups) * 2 * s.record_floats * sizeof(float);
}

// Tiles of a sequence that fills its table.
static long long most_tiles(const PagedAttnArgs& a) {
  return ((static_cast<long long>(a.table.max_pages) << a.pool.page_shift) + kTileKeys - 1) /
         kTileKeys;
}

bool paged_attention_supported(const PagedAttnArgs& a) {
  const PagedAttnShape s = paged_attention_shape(a.heads, a.pool.kv_heads, a.pool.head_dim);
  return most_tiles(a) * a.table.sequences * s.units < 2147000000LL;
}

// A call whose tables have room for more keys and values than kStreamBytes reads
// them past the caches, unless several head blocks read the same keys.  134 MB: 34.5
// -> 30.6 us, 350 MB: 67 -> 60.6; of 256 short sequences, 268 MB of room and half of it
// live, 32.5 -> 29.3.  Where the lengths fall far short of the tables'
// room it costs nothing with cold caches (39 MB 13.9 -> 14.0 us, 123 MB 29.4 ->
// 27.2), and up to a fifth where earlier calls left all of it in the cache (200
// sequences, 131 MB of room and half of it live: 18.2 -> 19.9).
void launch_paged_attention(PagedAttnArgs a, hipStream_t stream) {
  const PagedAttnShape s = paged_attention_shape(a.heads, a.pool.kv_heads, a.pool.head_dim);
  a.head_blocks = s.head_blocks;
  a.units = s.units;
  const long long tiles = most_tiles(a);
  const long long units = static_cast<long long>(a.table.sequences) * s.units;
  a.whole = tiles <= (units <= 2 * kCus ? kWholeTiles : kWholeTilesMany);
  const bool small =
      s.block_heads > 8 || (a.whole ? tiles <= kSmallWholeTiles || units <= kSmallWholeUnits
                                    : tiles * units <= kSmallTiles);
  const long long bytes = tiles * a.table.sequences * kTileKeys * 2 * a.pool.kv_heads *
                          a.pool.head_dim * (a.pool.format == kBf16 ? 2 : 1);
  const bool streams = bytes > kStreamBytes && s.head_blocks == 1;
  // no more workgroups than the tables have tiles for, one a wave
  const int waves = small ? 4 : 8, room = small ? 2 * kCus : kCus;
  const long long wanted = (tiles * units + waves - 1) / waves;
  const int groups = static_cast<int>(wanted < room ? wanted : room);
  a.waves = groups * waves;
  by_format(a.pool, [&](auto f, auto d) {
    constexpr int F = decltype(f)::value, D = decltype(d)::value;
    auto launch = [&](auto w, auto hb, auto nt) {
      constexpr int W = decltype(w)::value, HB = decltype(hb)::value;
      hipLaunchKernelGGL((paged_attention_kernel<F, D, W, HB, decltype(nt)::value>), dim3(groups),
                         dim3(W * kWave), 0, stream, a);
    };
    using Four = std::integral_constant<int, 4>;
    using Eight = std::integral_constant<int, 8>;
    using Sixteen = std::integral_constant<int, 16>;
    auto by_caches = [&](auto w, auto hb) {
      streams ? launch(w, hb, std::true_type{}) : launch(w, hb, std::false_type{});
    };
    if (s.block_heads > 8) {
      by_caches(Four{}, Sixteen{});
    } else if (small) {
      by_caches(Four{}, Eight{});
    } else {
      by_caches(Eight{}, Eight{});
    }
  });
  if (a.whole) return;
  a.join_heads = units <= kJoinHeadUnits;
  a.piece_waves = waves;
  const dim3 grid(a.join_heads ? s.units * s.block_heads : s.units, a.table.sequences);
  auto join = [&](auto d, auto threads) {
    constexpr int D = decltype(d)::value, T = decltype(threads)::value;
    hipLaunchKernelGGL((paged_attention_join_kernel<D, T>), grid, dim3(T), 0, stream, a);
  };
  auto by_dim = [&](auto threads) {
    if (a.pool.head_dim == 64) {
      join(std::integral_constant<int, 64>{}, threads);
    } else {
      join(std::integral_constant<int, 128>{}, threads);
    }
  };
  if (groups / units >= kJoinParts) {
    by_dim(std::integral_constant<int, 512>{});
  } else {
    by_dim(std::integral_constant<int, 256>{});
  }
}

}  // namespace qlin
