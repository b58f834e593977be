// The next token of every row of logits from a given random number, for gfx950
// (include/infer_batch.h).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "batch_kernels.hpp"
#include "device_common.hpp"

namespace qlin {

namespace {

// BF16 logits have at most 65536 values, so a row is a count per value: a kept set is
// a run of values from the largest down, of whose last one only the first few tokens
// may stay.  All sums of weights are counts times one exponential per value in 64
// bits, in a fixed order, and a token is told from its neighbour in the running sum
// down to some 1e-15 of the total, where 32 bits would err by some 1e-7, once in a
// thousand rows of a flat distribution over 151936 tokens.
//
// Keys order the values: a BF16 word's bits, all turned over for negative ones, the
// sign for the others; -0 counts as 0.
constexpr int kThreads = 1024, kWaves = kThreads / kWave;
constexpr int kKeyMinusInf = 0x007F, kKeyInf = 0xFF80;  // NaNs lie outside
constexpr int kKeyLowest = kKeyMinusInf + 1;            // of a token that counts

__device__ __forceinline__ int key_of(uint32_t word) {
  if (word == 0x8000u) word = 0;
  return static_cast<int>((word & 0x8000u) ? word ^ 0xFFFFu : word | 0x8000u);
}

__device__ __forceinline__ double value_of(int key) {
  const uint32_t word = (key & 0x8000) ? key ^ 0x8000 : key ^ 0xFFFF;
  return static_cast<double>(__uint_as_float(word << 16));
}

// exp((value - largest) / temperature), 1 for the largest also if that is infinite.
struct Weight {
  int top_key;
  double top, temperature;
  __device__ __forceinline__ double operator()(int key) const {
    if (key >= top_key) return 1.0;
    if (key <= kKeyMinusInf || top_key == kKeyInf) return 0.0;
    return exp((value_of(key) - top) / temperature);
  }
};

// A value, how many tokens have a larger one and their weight, and how many have it.
struct Border {
  int key;
  unsigned above;
  double above_mass;
  unsigned count;
};

struct Setting {
  double temperature, top_p, min_p, uniform;
  unsigned top_k;  // 0: all
  bool bad;        // a NaN
};

__device__ __forceinline__ Setting setting_of(const SampleArgs& a, int row) {
  const float t = a.temperature ? a.temperature[row] : 1.0f;
  const float p = a.top_p ? a.top_p[row] : 1.0f;
  const float m = a.min_p ? a.min_p[row] : 0.0f;
  const float u = a.uniform[row];
  const int k = a.top_k ? a.top_k[row] : 0;
  Setting s{t, p, m, 0.0, k > 0 ? static_cast<unsigned>(k) : 0u, t != t || p != p || m != m || u != u};
  // 1 - 2^-24, the last number under 1: a target under the sum of all
  s.uniform = fminf(fmaxf(u, 0.0f), 0x1.fffffep-1f);
  if (!(t > 0.0f)) s = Setting{1.0, 1.0, 0.0, 0.0, 1u, s.bad};
  return s;
}

struct Pick {
  int key;
  unsigned nth;  // of the tokens with that value, in order of index
  double probability;
};

// The kept run's end after each setting, then the token.  Row finds values by the counts
// and sums of those from the largest down: by_count(k) the first with k tokens or
// more (the lowest of all if there are none), by_mass(m, strict, floor) the first
// with a sum of m or more (more than m), floor if none is before it, at(key) any.
template <class Row>
__device__ __forceinline__ Pick choose(Row& row, const Setting& s, const Weight& w) {
  Border b = s.top_k ? row.by_count(s.top_k) : row.at(kKeyLowest);
  unsigned kept = b.count;  // of the tokens at the border
  if (s.top_k && s.top_k - b.above < kept) kept = s.top_k - b.above;
  if (s.top_p < 1.0) {
    const double mass = s.top_p * (b.above_mass + kept * w(b.key));
    const int last = b.key;
    b = row.by_mass(mass, false, last);
    const unsigned most = b.key == last ? kept : b.count;
    const double need = ceil((mass - b.above_mass) / w(b.key));
    // NaN and infinity where the border's weight is 0
    kept = need < most ? static_cast<unsigned>(fmax(need, 0.0)) : most;
    if (b.above + kept == 0) kept = 1;
  }
  if (s.min_p > 0.0 && w(b.key) < s.min_p) {
    int lo = b.key, hi = w.top_key;  // w(lo) < min_p, hi stays
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (w(mid) < s.min_p) {
        lo = mid;
      } else {
        hi = mid;
      }
    }
    b = row.at(hi);
    kept = b.count;
    // more than the largest weight: one token
    if (hi == w.top_key && s.min_p > 1.0) kept = 1;
  }
  const double total = b.above_mass + kept * w(b.key);
  const double target = s.uniform * total;
  const Border at = row.by_mass(target, true, b.key);
  const double each = w(at.key);
  const unsigned most = at.key == b.key ? kept : at.count;
  const double nth = floor((target - at.above_mass) / each);
  Pick pick{at.key, 0u, each / total};
  if (nth > 0.0) pick.nth = nth < most ? static_cast<unsigned>(nth) : most - 1;
  return pick;
}

// ------------------------------------------------------- bisecting kernel --

struct Lds {
  unsigned count[kWaves];
  double mass[kWaves];
  int low, high;
};

__device__ __forceinline__ unsigned wave_total(unsigned v) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) v += __shfl_xor(v, d);
  return v;
}

__device__ __forceinline__ double wave_total(double v) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) v += __shfl_xor(v, d);
  return v;
}

// A row that is read again for every question: 16 passes a border.
struct ReadRow {
  const uint16_t* logits;
  int vocab;
  Weight w;
  Lds& lds;

  __device__ void sum_from(int key, unsigned& count, double& mass) {
    unsigned c = 0;
    double m = 0.0;
    for (int i = threadIdx.x; i < vocab; i += kThreads) {
      const int k = key_of(logits[i]);
      if (k >= key) {
        ++c;
        m += w(k);
      }
    }
    c = wave_total(c);
    m = wave_total(m);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) {
      lds.count[threadIdx.x / kWave] = c;
      lds.mass[threadIdx.x / kWave] = m;
    }
    __syncthreads();
    count = 0;
    mass = 0.0;
    for (int i = 0; i < kWaves; ++i) {
      count += lds.count[i];
      mass += lds.mass[i];
    }
  }

  __device__ Border at(int key) {
    Border b{key, 0u, 0.0, 0u};
    unsigned c;
    double m;
    sum_from(key, c, m);
    sum_from(key + 1, b.above, b.above_mass);
    b.count = c - b.above;
    return b;
  }

  // The largest key from floor up for which ok of the sums from it holds, else floor.
  template <class F>
  __device__ Border largest(int floor, F ok) {
    int lo = floor, hi = w.top_key + 1;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      unsigned c;
      double m;
      sum_from(mid, c, m);
      if (ok(c, m)) {
        lo = mid;
      } else {
        hi = mid;
      }
    }
    return at(lo);
  }

  __device__ Border by_count(unsigned k) {
    return largest(kKeyLowest, [&](unsigned c, double) { return c >= k; });
  }
  __device__ Border by_mass(double target, bool strict, int floor) {
    return largest(floor, [&](unsigned, double m) { return strict ? m > target : m >= target; });
  }
};

__device__ void finish(const SampleArgs& a, int row, int token, double probability) {
  a.tokens[row] = token;
  if (a.probabilities) a.probabilities[row] = static_cast<float>(probability);
}

__global__ __launch_bounds__(kThreads) void sample_bisect_kernel(SampleArgs a) {
  __shared__ Lds lds;
  const int row = blockIdx.x, wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const uint16_t* logits = a.logits + row * a.stride;
  const Setting s = setting_of(a, row);
  if (threadIdx.x == 0) {
    lds.low = 0xFFFF;
    lds.high = 0;
  }
  __syncthreads();
  int low = 0xFFFF, high = 0;
  for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
    const int k = key_of(logits[i]);
    low = min(low, k);
    high = max(high, k);
  }
  atomicMin(&lds.low, low);
  atomicMax(&lds.high, high);
  __syncthreads();
  low = lds.low;
  high = lds.high;
  if (s.bad || low < kKeyMinusInf || high > kKeyInf || high == kKeyMinusInf) {
    if (threadIdx.x == 0) {
      const bool masked = !s.bad && low == kKeyMinusInf && high == kKeyMinusInf;
      finish(a, row, -1, masked ? 0.0 : __builtin_nan(""));
    }
    return;
  }
  const Weight w{high, value_of(high), s.temperature};
  ReadRow r{logits, a.vocab, w, lds};
  const Pick pick = choose(r, s, w);

  // The nth token with the value, 1024 at a time.
  unsigned before = 0;
  for (int base = 0; base < a.vocab; base += kThreads) {
    const int i = base + threadIdx.x;
    const bool has = i < a.vocab && key_of(logits[i]) == pick.key;
    const unsigned long long mask = __ballot(has);
    __syncthreads();
    if (lane == 0) lds.count[wave] = __popcll(mask);
    __syncthreads();
    unsigned mine = before;
    for (int v = 0; v < kWaves; ++v) {
      if (v < wave) mine += lds.count[v];
      before += lds.count[v];
    }
    mine += __popcll(mask & ((1ull << lane) - 1));
    if (has && mine == pick.nth) finish(a, row, i, pick.probability);
    if (before > pick.nth) break;
  }
}

}  // namespace

size_t sample_workspace_bytes(int rows, int vocab) {
  (void)rows;
  (void)vocab;
  return 16;
}

void launch_sample(const SampleArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(sample_bisect_kernel, dim3(a.rows), dim3(kThreads), 0, stream, a);
}

}  // namespace qlin
