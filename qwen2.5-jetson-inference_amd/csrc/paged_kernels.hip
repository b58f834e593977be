// Paged KV cache kernels for gfx950: store with RoPE and quantisation, load
// back, and the attention of one new token a sequence.
#include <float.h>
#include <stdint.h>

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

// A row (token, query head | key head | value head) takes D / 16 lanes; lane c
// holds elements 8 c .. + 8 of both halves, i.e. whole RoPE pairs.
template <int F, int D>
__global__ __launch_bounds__(kThreads) void kv_store_kernel(KvStoreArgs a) {
  constexpr int L = D / 16;
  const unsigned rows = a.heads + 2 * a.pool.kv_heads;
  const unsigned item = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const int c = threadIdx.x % L;
  const unsigned t = item / rows;
  if (t >= static_cast<unsigned>(a.tokens)) return;  // whole groups of L lanes
  const int row = item % rows;
  const int pos = a.positions[t];
  if (pos < 0 || (a.rope && pos >= a.rope_positions)) return;

  const bool is_q = row < a.heads;
  const bool is_v = row >= a.heads + a.pool.kv_heads;
  const int head = is_q ? row : is_v ? row - a.heads - a.pool.kv_heads : row - a.heads;
  const uint16_t* src = (is_q ? a.q + t * a.q_stride : is_v ? a.v + t * a.v_stride
                                                            : a.k + t * a.k_stride) +
                        static_cast<size_t>(head) * D + 8 * c;
  float lo[8], hi[8];
  unpack8(load_global16(src), lo);
  unpack8(load_global16(src + D / 2), hi);
  if (a.rope && !is_v) {
    rotate8(lo, hi, a.rope + static_cast<size_t>(pos) * D + 16 * c);
  }
  if (is_q) {
    uint16_t* dst = a.q_out + t * a.q_out_stride + static_cast<size_t>(head) * D + 8 * c;
    store_global16(dst, pack8(lo));
    store_global16(dst + D / 2, pack8(hi));
    return;
  }
  const int seq = a.sequence_ids ? a.sequence_ids[t] : static_cast<int>(t);
  const int index = pos >> a.pool.page_shift;
  if (static_cast<unsigned>(seq) >= static_cast<unsigned>(a.table.sequences) ||
      index >= a.table.max_pages) {
    return;
  }
  const int page = a.table.pages[static_cast<size_t>(seq) * a.table.stride + index];
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
  for (int o = 1; o < L; o <<= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), o)));
  const float scale = m >= 0x7F800000u ? __uint_as_float(0x7FC00000u)
                                       : __uint_as_float(m) / kLimit<F>;
  uint8_t* dst = static_cast<uint8_t*>(pages) + at * D + 8 * c;
  store_global8(dst, quantise8<F>(lo, scale));
  store_global8(dst + D / 2, quantise8<F>(hi, scale));
  if (c == 0) (is_v ? a.pool.value_scales : a.pool.key_scales)[at] = scale;
}

// ------------------------------------------------------------------- load --

// One lane per 8 elements of a row; blockIdx.x over rows, y the KV head, z the
// sequence.
template <int F, int D>
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
    store_global16(a.key_cache + to, nan);
    store_global16(a.value_cache + to, nan);
    return;
  }
  const size_t at = pool_row(a.pool, page, head, pos & ((1 << a.pool.page_shift) - 1));
  if (F == kBf16) {
    const uint4 k = load_global16(static_cast<const uint16_t*>(a.pool.key) + at * D + 8 * c);
    const uint4 v = load_global16(static_cast<const uint16_t*>(a.pool.value) + at * D + 8 * c);
    store_global16(a.key_cache + to, k);
    store_global16(a.value_cache + to, v);
    return;
  }
  const uint2 k = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.pool.key) + at * D + 8 * c);
  const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.pool.value) + at * D + 8 * c);
  float x[8];
  dequantise8<F>(k, a.pool.key_scales[at], x);
  store_global16(a.key_cache + to, pack8(x));
  dequantise8<F>(v, a.pool.value_scales[at], x);
  store_global16(a.value_cache + to, pack8(x));
}

// -------------------------------------------------------------- attention --

// The plain form of the kernel: a workgroup per (query head, sequence), each
// wave every fourth key with its own running maximum and sum (a lane holds
// D / 64 dimensions), the four states joined through LDS.
template <int F, int D>
__global__ __launch_bounds__(kThreads) void paged_attention_kernel(PagedAttnArgs a) {
  constexpr int N = D / 64;
  const int head = blockIdx.x, seq = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = head / (a.heads / a.pool.kv_heads);
  const int n = min(a.lengths[seq], a.table.max_pages << a.pool.page_shift);
  const uint16_t* qp = a.q + seq * a.q_stride + static_cast<size_t>(head) * D + N * lane;
  float q[N], acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    q[i] = bf16_to_f32(qp[i]) * (1.0f / sqrtf(static_cast<float>(D)));
    acc[i] = 0.0f;
  }
  float m = -FLT_MAX, l = 0.0f;
  for (int p = wave; p < n; p += kThreads / kWave) {
    const int page =
        a.table.pages[static_cast<size_t>(seq) * a.table.stride + (p >> a.pool.page_shift)];
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.pool.num_pages)) {
      l = __uint_as_float(0x7FC00000u);
      break;
    }
    const size_t at = pool_row(a.pool, page, g, p & ((1 << a.pool.page_shift) - 1));
    float k[N], v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const size_t e = at * D + N * lane + i;
      if (F == kBf16) {
        k[i] = bf16_to_f32(static_cast<const uint16_t*>(a.pool.key)[e]);
        v[i] = bf16_to_f32(static_cast<const uint16_t*>(a.pool.value)[e]);
      } else {
        float x[8];
        dequantise8<F>(make_uint2(static_cast<const uint8_t*>(a.pool.key)[e], 0), a.pool.key_scales[at], x);
        k[i] = x[0];
        dequantise8<F>(make_uint2(static_cast<const uint8_t*>(a.pool.value)[e], 0), a.pool.value_scales[at], x);
        v[i] = x[0];
      }
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(q[i], k[i], s);
    s = wave_sum(s);
    const float top = fmaxf(m, s), old = expf(m - top), w = expf(s - top);
    m = top;
    l = l * old + w;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = acc[i] * old + w * v[i];
  }
  __shared__ float sm[4], sl[4], sa[4][D];
  if (lane == 0) {
    sm[wave] = m;
    sl[wave] = l;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) sa[wave][N * lane + i] = acc[i];
  __syncthreads();
  if (threadIdx.x >= D) return;
  float top = sm[0];
  for (int w = 1; w < 4; ++w) top = fmaxf(top, sm[w]);
  float sum = 0.0f, total = 0.0f;
  for (int w = 0; w < 4; ++w) {
    const float e = expf(sm[w] - top);
    sum += e * sa[w][threadIdx.x];
    total += e * sl[w];
  }
  a.out[(static_cast<size_t>(seq) * a.heads + head) * D + threadIdx.x] =
      f32_to_bf16(total == 0.0f ? 0.0f : sum / total);
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

void launch_kv_store(const KvStoreArgs& a, hipStream_t stream) {
  const long long items = static_cast<long long>(a.tokens) * (a.heads + 2 * a.pool.kv_heads);
  by_format(a.pool, [&](auto f, auto d) {
    constexpr int per = kThreads / (decltype(d)::value / 16);
    const unsigned blocks = static_cast<unsigned>((items + per - 1) / per);
    hipLaunchKernelGGL((kv_store_kernel<decltype(f)::value, decltype(d)::value>), dim3(blocks),
                       dim3(kThreads), 0, stream, a);
  });
}

void launch_kv_load(const KvLoadArgs& a, hipStream_t stream) {
  const long long most = static_cast<long long>(a.table.max_pages) << a.pool.page_shift;
  const long long rows = a.capacity < most ? a.capacity : most;
  by_format(a.pool, [&](auto f, auto d) {
    constexpr int per = kThreads / (decltype(d)::value / 8);
    const dim3 grid(static_cast<unsigned>((rows + per - 1) / per), a.pool.kv_heads,
                    a.table.sequences);
    hipLaunchKernelGGL((kv_load_kernel<decltype(f)::value, decltype(d)::value>), grid,
                       dim3(kThreads), 0, stream, a);
  });
}

size_t paged_attention_workspace_bytes(int, int, int, int) { return 256; }

void launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream) {
  by_format(a.pool, [&](auto f, auto d) {
    hipLaunchKernelGGL((paged_attention_kernel<decltype(f)::value, decltype(d)::value>),
                       dim3(a.heads, a.table.sequences), dim3(kThreads), 0, stream, a);
  });
}

}  // namespace qlin
