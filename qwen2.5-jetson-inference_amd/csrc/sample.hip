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
constexpr int kThreads = 512, kWaves = kThreads / kWave;
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

// e^x in 64 bits for x <= 0: 2^n e^r with |r| <= ln(2) / 2 and e^r's series up to r^13
// (the next term is 4e-18).  Some 20 instructions, expf's double counterpart takes twice
// that for ranges that do not occur here.
__device__ __forceinline__ double exp_nonpos(double x) {
  x = fmax(x, -800.0);  // 0 as the result is
  const double n = rint(x * 1.4426950408889634);
  double r = fma(n, -0x1.62e42fefa39efp-1, x);  // ln(2), and what it lacks
  r = fma(n, -0x1.abc9e3b39803fp-56, r);
  double p = 1.0 / 6227020800.0;
  p = fma(p, r, 1.0 / 479001600.0);
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return ldexp(p, static_cast<int>(n));
}

// exp((value - largest) / temperature), 1 for the largest also if that is infinite.
struct Weight {
  int top_key;
  double top, temperature, inverse;
  __device__ Weight(int key, double t)
      : top_key(key), top(value_of(key)), temperature(t), inverse(1.0 / t) {}
  __device__ __forceinline__ double operator()(int key) const {
    const double w = exp_nonpos((value_of(key) - top) * inverse);
    return key >= top_key ? 1.0 : key <= kKeyMinusInf || top_key == kKeyInf ? 0.0 : w;
  }
};

// A value and its weight, how many tokens have a larger one and their weight, and how
// many have it.
struct Border {
  int key;
  unsigned above;
  double above_mass;
  unsigned count;
  double weight;
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
  Setting s{t, p, m, 0.0, k > 0 ? static_cast<unsigned>(k) : 0u,
            t != t || p != p || m != m || u != u};
  // 1 - 2^-24, the last number under 1: a target under the sum of all
  s.uniform = fminf(fmaxf(u, 0.0f), 0x1.fffffep-1f);
  if (!(t > 0.0f)) s = Setting{1.0, 1.0, 0.0, 0.0, 1u, s.bad};
  return s;
}

struct Pick {
  int key;
  unsigned nth;    // of the tokens with that value, in order of index
  unsigned count;  // of them
  double probability;
};

// The smallest key from lo + 1 to the largest one whose weight is at least min_p, where
// lo's is not.  64 keys around the one that the logarithm gives are tried at
// once; the interval is halved where those do not hold the border (values near 0, whose keys
// lie closer than the logarithm is exact).
__device__ __forceinline__ int lowest_with(double min_p, int lo, const Weight& w) {
  int hi = w.top_key;
  const float value = static_cast<float>(w.top + w.temperature * log(min_p));
  const int guess = key_of(__float_as_uint(value) >> 16) - kWave / 2;
  const int key = min(max(guess + static_cast<int>(threadIdx.x & (kWave - 1)), lo), hi);
  const unsigned long long heavy = __ballot(w(key) >= min_p), light = ~heavy;
  if (heavy && light) {
    hi = __builtin_amdgcn_readlane(key, __builtin_ctzll(heavy));
    lo = __builtin_amdgcn_readlane(key, kWave - 1 - __builtin_clzll(light));
  }
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (w(mid) < min_p) {
      lo = mid;
    } else {
      hi = mid;
    }
  }
  return hi;
}

// What is asked of a row: the first value, from the largest down, where the count up to it
// has `count` tokens; where the sum of weights up to it reaches `mass` (is more than it, if
// strict), no lower than key; or key itself, whether any token has it or not.
struct Query {
  enum { kCount, kMass, kKey } by;
  unsigned count;
  double mass;
  bool strict;
  int key;
};

// The kept run's end after each setting, then the token: one question after the other, in
// a loop, as code that runs once is fetched at some 500 cycles per KB.
template <class Row>
__device__ __forceinline__ Pick choose(Row& row, const Setting& s, const Weight& w) {
  Border b{kKeyLowest, 0u, 0.0, 0u, 0.0};
  unsigned kept = 0;  // of the tokens at the border
  double total = 0.0, target = 0.0;
#pragma unroll 1
  for (int stage = 0; stage < 4; ++stage) {
    Query q{Query::kKey, 0u, 0.0, false, kKeyLowest};
    if (stage == 0) {
      if (s.top_k) {
        q.by = Query::kCount;
        q.count = s.top_k;
      } else if (row.all(b)) {
        continue;
      }
    } else if (stage == 2) {
      if (!(s.min_p > 0.0 && b.weight < s.min_p)) continue;
      q.key = lowest_with(s.min_p, b.key, w);
    } else {
      if (stage == 1 && !(s.top_p < 1.0)) continue;
      total = b.above_mass + kept * b.weight;
      target = (stage == 1 ? s.top_p : s.uniform) * total;
      q = Query{Query::kMass, 0u, target, stage == 3, b.key};
    }
    const int last = b.key;
    b = row.find(q);
    const unsigned most = stage & 1 && b.key == last ? kept : b.count;
    kept = most;
    if (stage == 0 && s.top_k && s.top_k - b.above < kept) kept = s.top_k - b.above;
    if (stage == 1) {
      const double need = ceil((target - b.above_mass) / b.weight);
      // NaN and infinity where the border's weight is 0
      kept = need < most ? static_cast<unsigned>(fmax(need, 0.0)) : most;
      if (b.above + kept == 0) kept = 1;
    }
    // a min_p over the largest weight: one token
    if (stage == 2 && b.key == w.top_key && s.min_p > 1.0) kept = 1;
  }
  const double nth = floor((target - b.above_mass) / b.weight);
  Pick pick{b.key, 0u, b.count, b.weight / total};
  if (nth > 0.0) pick.nth = nth < kept ? static_cast<unsigned>(nth) : kept - 1;
  return pick;
}

// ------------------------------------------------- sums over a wave's lanes --

__device__ __forceinline__ unsigned at_lane(unsigned v, int lane) {
  return __builtin_amdgcn_readlane(static_cast<int>(v), lane);
}
__device__ __forceinline__ double at_lane(double v, int lane) {
  const unsigned long long w = __builtin_bit_cast(unsigned long long, v);
  return __builtin_bit_cast(
      double, static_cast<unsigned long long>(at_lane(static_cast<unsigned>(w >> 32), lane)) << 32 |
                  at_lane(static_cast<unsigned>(w), lane));
}

template <class T>
__device__ __forceinline__ T wave_total(T v) {
  return at_lane(wave_scan(v), kWave - 1);
}

// ------------------------------------------------------- bisecting kernel --

struct Lds {
  unsigned count[kWaves];
  double mass[kWaves];
  int low, high;
};

// A row that is read again for every question, 16 passes a border: 16 rows of 151936 that
// have two values with half of the tokens each 1880 us, where the count takes 21 to 111.
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

  __device__ __forceinline__ bool all(Border&) { return false; }
  __device__ __forceinline__ Border find(const Query& q) {
    // the largest key from lo up for which the sums from it pass, else lo
    int lo = q.by == Query::kCount ? kKeyLowest : q.key;
    int hi = q.by == Query::kKey ? lo + 1 : w.top_key + 1;
    unsigned count = 0;
    double mass = 0.0;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      sum_from(mid, count, mass);
      const bool ok = q.by == Query::kCount ? count >= q.count
                      : q.strict            ? mass > q.mass
                                            : mass >= q.mass;
      if (ok) {
        lo = mid;
      } else {
        hi = mid;
      }
    }
    Border b{lo, 0u, 0.0, 0u, w(lo)};
    for (int i = 0; i < 2; ++i) {
      sum_from(lo + i, count, mass);
      if (i == 0) b.count = count;
    }
    b.above = count;
    b.above_mass = mass;
    b.count -= count;
    return b;
  }
};

__device__ __forceinline__ void finish(const SampleArgs& a, int row, int token,
                                       double probability) {
  a.tokens[row] = token;
  if (a.probabilities) a.probabilities[row] = static_cast<float>(probability);
}

// The row's answer by bisection, for a row whose counts do not fit the other
// kernel's.
__device__ __forceinline__ void sample_by_bisection(const SampleArgs& a, int row,
                                                    const Setting& s, Lds& lds) {
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const uint16_t* logits = a.logits + row * a.stride;
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
  if (low < kKeyMinusInf || high > kKeyInf || high == kKeyMinusInf) {
    if (threadIdx.x == 0) {
      const bool masked = low == kKeyMinusInf && high == kKeyMinusInf;
      finish(a, row, -1, masked ? 0.0 : __builtin_nan(""));
    }
    return;
  }
  const Weight w(high, s.temperature);
  ReadRow r{logits, a.vocab, w, lds};
  const Pick pick = choose(r, s, w);

  // The nth token with the value, 512 at a time.
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

// --------------------------------------------------------- counting kernel --

// A workgroup counts a row's values in LDS.  Dword v & 0x7FFF counts the words of both
// signs in 17 bits and those with the sign in the 15 above: its address and what is added
// to it are two instructions from a shifted word.  Where 32768 tokens or more have one
// magnitude, which a dword's total shows, the row is taken by bisection; but for those of
// one value, a mask's: a low one, the row's lowest or one of more tokens than those below it,
// as far as a wave has seen.  A wave counts them in a register, as they would also meet at one
// address.
//
// Groups of 64 values are ordered from the largest down: 0 to 511 the positive ones,
// 512 to 1023 the negative ones.  A group's values are equally far apart, so that its
// weights are a geometric series, w q^l, and its sum a polynomial in q of the
// counts: two exponentials a group, and 8 lanes for the polynomial.  One wave then asks
// its questions of the sums of the groups with tokens, some 50 to 90 of a model's row.
//
// Bound: chains within one workgroup, as a row's counts meet in one CU's LDS.  Of the 46000
// cycles of a row of 151936 (19.9 us with a launch) the count takes 22000, 8 LDS additions a
// 16-byte piece at some 8 cycles a wave; the groups' sums 7000; the questions, one wave's
// dependent 64-bit steps, 6000; the token's place 5000-7000 over the row in registers.  256
// such rows take 26.2 us (78 MB, 3.0 TB/s), 17 of 32003 12.7, of which the counts are 5000
// cycles.  Parts of a row counted by several workgroups need a launch to add them up: 1 x
// 151936 24.7 us, 1 x 40000 22 for 12.4.  512 threads, so that the row stays in registers
// beside the work.
constexpr int kBins = 32768, kGroups = 1024;
constexpr int kInfBin = 0x7F80;
constexpr int kLastGroup = (0xFFFF - kKeyLowest) / kWave;  // with tokens that count
constexpr unsigned kBinTotal = 0x1FFFFu;
constexpr int kBinShift = 17;

struct Heavy {
  unsigned word, count;
};

struct CountLds {
  unsigned bins[kBins];
  // of the groups with tokens, in order; then up to and with each
  unsigned list_count[kGroups];
  double list_mass[kGroups];
  uint16_t list_group[kGroups];
  // which of a wave's groups have tokens: positive ones from the last down, negative ones
  unsigned long long positive[kWaves], negative[kWaves];
  Heavy heavy[kWaves];
  unsigned wave_count[kWaves], found[kWave];
  unsigned total, many, nan;
  Pick pick;
  Lds bisect;
};

typedef __attribute__((address_space(3))) unsigned LdsWord;
typedef __attribute__((address_space(3))) char LdsByte;

// The bins lie in static LDS: the compiler knows their address, so that a shifted word needs
// no addition (of dynamic LDS it takes one a word).
struct Bins {
  LdsByte* first;

  __device__ explicit Bins(unsigned* bins) : first((LdsByte*)bins) {}
  // `shifted` has the word's 16 bits from bit 2 on.
  __device__ __forceinline__ void add_shifted(uint32_t shifted, unsigned times) const {
    const unsigned one = (shifted & (1u << kBinShift)) | 1u;
    __hip_atomic_fetch_add((LdsWord*)(first + (shifted & (4u * (kBins - 1)))), one * times,
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  }
  __device__ __forceinline__ void add_word(uint32_t word, unsigned times) const {
    add_shifted(word << 2, times);
  }
};

__device__ __forceinline__ int key_of_lane(int group, int lane) {
  return 0xFFFF - (group * kWave + lane);
}

__device__ __forceinline__ unsigned lanes_max(unsigned v) {
  v = max(v, from_lane<kDppQuadSwap1>(v));
  v = max(v, from_lane<kDppQuadSwap2>(v));
  v = max(v, from_lane<kDppRowHalfMirror>(v));
  v = max(v, from_lane<kDppRowMirror>(v));
  return max(max(at_lane(v, 0), at_lane(v, 16)), max(at_lane(v, 32), at_lane(v, 48)));
}

struct Counted {
  CountLds& lds;
  int heavy_key;
  unsigned heavy;

  // Tokens of a group's value.
  __device__ __forceinline__ unsigned count(int group, int lane) const {
    const int key = key_of_lane(group, lane);
    const unsigned word = lds.bins[key & 0x8000 ? key ^ 0x8000 : 0x7FFF - key];
    const unsigned total = word & kBinTotal, negative = word >> kBinShift;
    unsigned c = key > 0x8000    ? total - negative
                 : key == 0x8000 ? total  // -0 is 0
                 : key == 0x7FFF ? 0u
                                 : negative;
    if (key == heavy_key) c += heavy;
    return key <= kKeyMinusInf ? 0u : c;
  }
};

// Questions of the list, by one wave; every lane gets the answer.
struct CountedRow {
  const Counted& c;
  const Weight& w;
  int entries, lane;

  // All tokens that count, as those above the lowest value; false if that has some.
  __device__ __forceinline__ bool all(Border& b) {
    const int lowest = (0xFFFF - kKeyLowest) % kWave;
    if (at_lane(c.count(kLastGroup, lane), lowest)) return false;
    b.above = at_lane(c.lds.list_count[entries - 1], 0);
    b.above_mass = at_lane(c.lds.list_mass[entries - 1], 0);
    return true;
  }

  __device__ __forceinline__ Border find(Query q) {
    for (;;) {
      const int q_group = (0xFFFF - q.key) / kWave, q_lane = (0xFFFF - q.key) % kWave;
      auto passed = [&](unsigned count, double mass) {
        return q.by == Query::kCount ? count >= q.count
               : q.strict            ? mass > q.mass
                                     : mass >= q.mass;
      };
      // the groups before the one with the answer, and their sums
      int e = 0;
      for (int base = 0; base < entries; base += kWave) {
        const int i = min(base + lane, entries - 1);
        const bool before = q.by == Query::kKey
                                ? c.lds.list_group[i] < q_group
                                : !passed(c.lds.list_count[i], c.lds.list_mass[i]);
        const int here = __popcll(__ballot(base + lane < entries && before));
        e += here;
        if (here < kWave) break;
      }
      if (q.by != Query::kKey && e == entries) {  // none
        q = Query{Query::kKey, 0u, 0.0, false, q.by == Query::kCount ? kKeyLowest : q.key};
        continue;
      }
      const unsigned count = e ? at_lane(c.lds.list_count[e - 1], 0) : 0u;
      const double mass = e ? at_lane(c.lds.list_mass[e - 1], 0) : 0.0;
      const int group = q.by == Query::kKey
                            ? q_group
                            : static_cast<int>(at_lane(unsigned{c.lds.list_group[e]}, 0));
      const int key = key_of_lane(group, lane);
      const unsigned n = c.count(group, lane);
      const double each = w(key);
      const unsigned n_in = wave_scan(n);
      const double m_in = wave_scan(n * each);
      const unsigned long long hit = __ballot(
          q.by == Query::kKey ? lane >= q_lane : n && passed(count + n_in, mass + m_in));
      // the last value with tokens if the group's sums, added in another order, said that
      // one would do
      const int at = hit ? __builtin_ctzll(hit) : kWave - 1 - __builtin_clzll(__ballot(n != 0) | 1);
      const Border b{static_cast<int>(at_lane(static_cast<unsigned>(key), at)),
                     count + at_lane(n_in, at) - at_lane(n, at),
                     at ? mass + at_lane(m_in, at - 1) : mass, at_lane(n, at), at_lane(each, at)};
      if (q.by != Query::kMass || b.key >= q.key) return b;
      q.by = Query::kKey;
    }
  }
};

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t larger_words(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                 __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ uint32_t add_words(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_bit_cast(u16x2, a) + __builtin_bit_cast(u16x2, b));
}
__device__ __forceinline__ uint32_t smaller_words(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2, a),
                                                                 __builtin_bit_cast(u16x2, b)));
}

// A row as 16-byte pieces between two edges of up to 7 words each.
struct RowSpan {
  const uint16_t* body;
  int head, pieces, tail;

  __device__ RowSpan(const uint16_t* row, int vocab) {
    head = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / 2, vocab);
    body = row + head;
    pieces = (vocab - head) / 8;
    tail = vocab - head - 8 * pieces;
  }
  // Lanes 0-7 the head's words, 8-15 the tail's.
  __device__ __forceinline__ bool edge(int lane, uint32_t& word, int& index) const {
    const bool in_head = lane < head, in_tail = lane >= 8 && lane - 8 < tail;
    index = in_head ? lane : head + 8 * pieces + lane - 8;
    word = in_head || in_tail ? body[index - head] : 0u;
    return in_head || in_tail;
  }
};

// NR pieces of a thread, 512 apart, of those in [first, last).  Past them they are 0, by the
// loads' own bounds check: a piece's place goes into their vector offset, which is sure to
// be in it, also beyond the row.
template <int NR>
struct Pieces {
  u32x4 x[NR];

  // Pieces [from, to) of them.
  template <int from, int to>
  __device__ __forceinline__ void load(const RowSpan& span, int first, int last) {
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(span.body), 0, 16 * last, 0x00020000);
#pragma unroll
    for (int i = from; i < to && i < NR; ++i) {
      x[i] = __builtin_amdgcn_raw_buffer_load_b128(
          rsrc, 16 * (first + i * kThreads + static_cast<int>(threadIdx.x)), 0, 0);
    }
  }
  // Piece i as a copy of its own, made here: what is computed of it is not computed
  // ahead for all pieces, nor kept for the next time.
  __device__ __forceinline__ u32x4 get(int i) const {
    u32x4 y = x[i];
    asm volatile("" : "+v"(y)::"memory");
    return y;
  }
  // Piece i, a number that the wave shares: by halves, as a jump over each piece's copy
  // would fetch the code of all.
  template <int from = 0, int to = NR>
  __device__ __forceinline__ u32x4 pick(int i) const {
    if constexpr (to - from == 1) {
      return get(from);
    } else {
      constexpr int middle = (from + to) / 2;
      return i < middle ? pick<from, middle>(i) : pick<middle, to>(i);
    }
  }
};

// The words of the pieces into the bins.  The first kAhead pieces are loaded before;
// the others in the loop, so that counting begins while they are on their way (all of a
// thread's loads at once wait for room: 256 rows of 151936 36 -> 30 us).  A piece in which
// kHeavyLanes lanes of a wave or more have a word as low as the heavy one, a low one of
// those kAhead, is left for later: it is read again, and its heavy words, a mask's, are
// counted in a register.  A value of fewer lanes has at most 1 / 16 of the tokens.
constexpr int kAhead = 6, kHeavyLanes = 5, kManyLanes = 16;
struct Counting {
  const RowSpan& span;
  const Bins bins;
  Heavy heavy{0u, 0u};  // of the wave
  unsigned lead = 0;    // tokens that have it beyond those that were counted against it

  __device__ __forceinline__ static unsigned largest(const u32x4& x) {
    const uint32_t pair =
        larger_words(larger_words(x[0], x[1]), larger_words(x[2], x[3]));
    return max(pair & 0xFFFFu, pair >> 16);
  }

  __device__ __forceinline__ static uint32_t word_of(const u32x4& x, int j) {
    return j & 1 ? x[j / 2] >> 16 : x[j / 2] & 0xFFFFu;
  }

  template <int NR, int I = 0>
  __device__ __forceinline__ void add_pieces(Pieces<NR>& p, int first, int last,
                                             unsigned long long& later) {
    if constexpr (I < NR) {
      p.template load<I + kAhead, I + kAhead + 1>(span, first, last);
      if (first + I * kThreads < last) {
        const u32x4 x = p.get(I);
        if (__popcll(__ballot(largest(x) >= heavy.word)) >= kHeavyLanes) {
          later |= 1ull << I;
        } else if (first + I * kThreads + static_cast<int>(threadIdx.x) < last) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            bins.add_shifted(x[j] << 2, 1);
            bins.add_shifted(x[j] >> 14, 1);
          }
        }
      }
      add_pieces<NR, I + 1>(p, first, last, later);
    }
  }

  template <int NR>
  __device__ __forceinline__ void add(Pieces<NR>& p, int first, int last) {
    if (heavy.word == 0 && heavy.count == 0) {  // zeros that were counted stay zeros
      unsigned most = 0;
#pragma unroll
      for (int i = 0; i < kAhead && i < NR; ++i) most = max(most, largest(p.x[i]));
      // the lowest, or where that is far below what many more lanes have, as -infinity in few
      // places is below a mask, theirs
      heavy.word = lanes_max(most);
      const unsigned some = min(min(at_lane(most, 0), at_lane(most, 21)), at_lane(most, 42));
      if (heavy.word - some >= 256) {  // twice the exponent's step: ordinary rows end here
        const int lanes = __popcll(__ballot(most == some));
        if (lanes >= kManyLanes && lanes > __popcll(__ballot(most == heavy.word))) {
          heavy.word = some;
        }
      }
    }
    unsigned long long later = 0;
    add_pieces(p, first, last, later);
#pragma unroll 1
    for (; later; later &= later - 1) {
      const int piece =
          first + __builtin_ctzll(later) * kThreads + static_cast<int>(threadIdx.x);
      const bool live = piece < last;
      const u32x4 x = live ? *(const QLIN_GLOBAL u32x4*)(span.body + 8ll * piece)
                           : u32x4{0, 0, 0, 0};
      // The piece's lowest value, or the next if more lanes have that, takes the heavy one's
      // place when more tokens have it than the heavy one leads by (a lower value alone did:
      // 16 rows of 151936 at -10^4 but for 300 -infinities each took 1260 us, now 38).
      const unsigned low = largest(x);
      unsigned word = lanes_max(low);
      const int lanes = __popcll(__ballot(low == word));
      if (word != heavy.word || lanes < kWave / 2) {
        const unsigned other = lanes_max(low == word ? 0u : low);
        if (other && __popcll(__ballot(low == other)) > lanes) word = other;
        if (word != heavy.word) {
          unsigned n = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) n += __popcll(__ballot(live && word_of(x, j) == word));
          if (n > lead) {
            if (heavy.count && (threadIdx.x & (kWave - 1)) == 0) {
              bins.add_word(heavy.word, heavy.count);
            }
            heavy = Heavy{word, 0u};
            lead = 0;
          } else {
            lead -= n;
          }
        }
      }
      unsigned count = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool is_heavy = word_of(x, j) == heavy.word;
        count += __popcll(__ballot(live && is_heavy));
        if (live && !is_heavy) bins.add_word(word_of(x, j), 1);
      }
      heavy.count += count;
      lead += count;
    }
  }
};

__device__ __forceinline__ void clear_bins(CountLds& lds) {
  uint4* const zero = reinterpret_cast<uint4*>(lds.bins);
#pragma unroll
  for (int i = 0; i < kBins / 4 / kThreads; ++i) {
    zero[i * kThreads + threadIdx.x] = make_uint4(0, 0, 0, 0);
  }
  if (threadIdx.x < kWave) lds.found[threadIdx.x] = 0;
  if (threadIdx.x == 0) lds.total = lds.many = lds.nan = 0;
}

// One heavy value of the waves', from the lane that holds each: the lowest of those of
// which a wave has kManyHeavy tokens, or else of all.  The others go into the bins.
constexpr unsigned kManyHeavy = 1024;
__device__ __forceinline__ Heavy join_heavy(CountLds& lds, Heavy h, bool has, bool adds) {
  has = has && h.count;
  const unsigned many = h.count >= kManyHeavy ? 0x10000u : 0u;
  const unsigned word = lanes_max(has ? h.word | many : 0u) & 0xFFFFu;
  const bool same = has && h.word == word;
  if (adds && has && !same) Bins(lds.bins).add_word(h.word, h.count);
  return Heavy{word, wave_total(same ? h.count : 0u)};
}

// The sum of weights of a group other than the largest value's, in lane 0 of each 8
// lanes, which hold eight of its values each.
__device__ __forceinline__ double group_mass(const Counted& c, const Weight& w, int group,
                                             int lane) {
  const int j = lane & 7;
  const bool positive = group < kGroups / 2;
  const int first = positive ? kBins - 8 - kWave * group - 8 * j
                             : kWave * (group - kGroups / 2) + 8 * j;  // of the dwords
  const uint4* const bins = reinterpret_cast<const uint4*>(c.lds.bins + first);
  const uint4 u = bins[positive ? 1 : 0], v = bins[positive ? 0 : 1];
  unsigned n[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 8; i += 4) {  // the larger values first
    const unsigned a = n[i], b = n[i + 1];
    n[i] = positive ? n[i + 3] : a;
    n[i + 1] = positive ? n[i + 2] : b;
    n[i + 2] = positive ? b : n[i + 2];
    n[i + 3] = positive ? a : n[i + 3];
  }
  const int key = key_of_lane(group, 8 * j);
  // values of one exponent are 2^(exponent - 134) apart, also those of exponent 0
  const int exponent = max(first >> 7, 1);
  const double apart = __uint_as_float(static_cast<unsigned>(exponent) << 23) * 0x1p-7;
  // one exponential: the first value's weight in even lanes, q in odd ones
  const double weight = exp_nonpos((lane & 1 ? -apart : value_of(key) - w.top) * w.inverse);
  const double q = from_lane<0xF5>(weight);  // quad_perm [1, 1, 3, 3]
  double sum = 0.0;
#pragma unroll
  for (int i = 7; i >= 0; --i) {
    unsigned count = n[i] >> kBinShift;
    if (positive) count = (n[i] & kBinTotal) - (key - i == 0x8000 ? 0u : count);  // -0 is 0
    if (key - i == 0x7FFF) count = 0;
    if (key - i == c.heavy_key) count += c.heavy;
    sum = fma(sum, q, double(count));
  }
  const double q2 = q * q, q4 = q2 * q2, q8 = q4 * q4, q16 = q8 * q8;
  sum = fma(from_lane<0x101>(sum), q8, sum);  // row_shl 1, 2, 4
  sum = fma(from_lane<0x102>(sum), q16, sum);
  sum = fma(from_lane<0x104>(sum), q16 * q16, sum);
  return w.top_key == kKeyInf ? 0.0 : weight * sum;
}

// Everything after the bins: the token's value, and its place among those that have it,
// in lds.pick.  False where the row has been answered.
__device__ __forceinline__ bool choose_value(const SampleArgs& a, int row, const Setting& s,
                                             const Heavy& heavy, CountLds& lds) {
  const int t = threadIdx.x, lane = t & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(t / kWave);
  // Thread t's 64 dwords are groups 511 - t and 512 + t; 16 bytes at a time in an order
  // that spreads the lanes over the banks.  Eight dwords are added as they are while none
  // has 4096.
  unsigned total = 0, negative = 0, seen = 0;
#pragma unroll
  for (int j = 0; j < 16; j += 2) {
    const uint4* bins = reinterpret_cast<const uint4*>(lds.bins) + 16 * t;
    const uint4 v = bins[(j + t) & 15], u = bins[(j + 1 + t) & 15];
    const unsigned sum = ((v.x + v.y) + (v.z + v.w)) + ((u.x + u.y) + (u.z + u.w));
    seen |= (v.x | v.y | v.z) | (v.w | u.x | u.y) | (u.z | u.w);
    total += sum & kBinTotal;
    negative += sum >> kBinShift;
  }
  if (seen & 0x1F000u) {
    total = negative = 0;
    for (int j = 0; j < kWave; ++j) {
      const unsigned w = lds.bins[kWave * t + j];
      total += w & kBinTotal;
      negative += w >> kBinShift;
    }
    if (seen & 0x18000u) lds.many = 1;
  }
  if (t == 0) negative -= lds.bins[0] >> kBinShift;  // -0 is 0
  const unsigned all = wave_total(total);
  if (lane == 0) atomicAdd(&lds.total, all);
  unsigned positive = total - negative;
  if (t >= kInfBin / kWave) {  // infinities and NaN: +infinity alone counts
    const unsigned inf = t == kInfBin / kWave ? lds.bins[kInfBin] : 0u;
    if (total != (inf & kBinTotal)) lds.nan = 1;
    positive = (inf & kBinTotal) - (inf >> kBinShift);
    negative = 0;
  }
  const int heavy_key = key_of(heavy.word);
  const Counted counted{lds, heavy_key, heavy_key <= kKeyMinusInf ? 0u : heavy.count};
  const int heavy_group = (0xFFFF - heavy_key) / kWave;
  if (heavy_group == 511 - t) positive += counted.heavy;
  if (heavy_group == 512 + t) negative += counted.heavy;
  const unsigned long long has_positive = __ballot(positive != 0);
  const unsigned long long has_negative = __ballot(negative != 0);
  if (lane == 0) {
    lds.positive[wave] = has_positive;
    lds.negative[wave] = has_negative;
  }
  lds_barrier();

  if (lds.total + heavy.count != static_cast<unsigned>(a.vocab) || lds.many) {
    if (s.bad) {
      if (t == 0) finish(a, row, -1, __builtin_nan(""));
    } else {
      sample_by_bisection(a, row, s, lds.bisect);
    }
    return false;
  }
  if (s.bad || lds.nan || (heavy.count && (heavy.word & 0x7FFFu) > kInfBin)) {
    if (t == 0) finish(a, row, -1, __builtin_nan(""));
    return false;
  }
  // Places in the list: lane i the waves' masks in the order of the groups.
  const unsigned in_mask =
      lane < kWaves       ? __popcll(lds.positive[kWaves - 1 - lane])
      : lane < 2 * kWaves ? __popcll(lds.negative[lane - kWaves])
                          : 0u;
  const unsigned up_to = wave_scan(in_mask);
  int entries = at_lane(up_to, kWave - 1);
  if (entries == 0) {  // all masked
    if (t == 0) finish(a, row, -1, 0.0);
    return false;
  }
  if (positive) {
    const int e = at_lane(up_to, kWaves - 1 - wave) - __popcll(has_positive) +
                  __popcll(has_positive >> lane >> 1);
    lds.list_group[e] = 511 - t;
    lds.list_count[e] = positive;
  }
  if (negative) {
    const int e = at_lane(up_to, kWaves + wave) - __popcll(has_negative) +
                  __popcll(has_negative & ((1ull << lane) - 1));
    lds.list_group[e] = 512 + t;
    lds.list_count[e] = negative;
  }
  lds_barrier();
  const int top_group = lds.list_group[0];
  const unsigned in_top = counted.count(top_group, lane);
  const int top_key = key_of_lane(top_group, __builtin_ctzll(__ballot(in_top != 0)));
  const Weight weight(top_key, s.temperature);
  if (s.top_k) {  // no further than the first top_k
    unsigned count = 0;
    for (int base = 0; base < entries; base += kWave) {
      const int e = base + lane;
      const unsigned sum = count + wave_scan(e < entries ? lds.list_count[e] : 0u);
      const unsigned long long enough = __ballot(sum >= s.top_k);
      if (enough) {
        entries = min(entries, base + __builtin_ctzll(enough) + 1);
        break;
      }
      count = at_lane(sum, kWave - 1);
    }
  }
  // The groups of the list, one to 8 lanes; the largest value's from its weights.
#pragma unroll 1
  for (int base = 8 * wave; base < entries; base += 8 * kWaves) {
    const int e = base + (lane >> 3);
    const double m = group_mass(counted, weight, lds.list_group[min(e, entries - 1)], lane);
    if ((lane & 7) == 0 && e && e < entries) lds.list_mass[e] = m;
  }
  if (wave == kWaves - 1) {
    const double m = wave_total(in_top * weight(key_of_lane(top_group, lane)));
    if (lane == 0) lds.list_mass[0] = m;
  }
  lds_barrier();
  if (wave == 0) {
    double mass = 0.0;
    unsigned count = 0;
    for (int base = 0; base < entries; base += kWave) {
      const int e = base + lane;
      const double m = mass + wave_scan(e < entries ? lds.list_mass[e] : 0.0);
      const unsigned n = count + wave_scan(e < entries ? lds.list_count[e] : 0u);
      if (e < entries) {
        lds.list_mass[e] = m;
        lds.list_count[e] = n;
      }
      mass = at_lane(m, kWave - 1);
      count = at_lane(n, kWave - 1);
    }
    CountedRow r{counted, weight, entries, lane};
    const Pick pick = choose(r, s, weight);
    if (lane == 0) lds.pick = pick;
  }
  lds_barrier();
  return true;
}

// A value as the words that have it: zeros are both.
struct Wanted {
  uint32_t word, mask;
  __device__ explicit Wanted(int key)
      : word(key & 0x8000 ? key ^ 0x8000 : key ^ 0xFFFF), mask(word ? 0xFFFFu : 0x7FFFu) {}
  __device__ __forceinline__ bool is(uint32_t w) const { return (w & mask) == word; }
  // Halves that are 0 have it.
  __device__ __forceinline__ uint32_t differs(uint32_t pair) const {
    return (pair & (mask | mask << 16)) ^ (word | word << 16);
  }
};

// The nth token with the value among the pieces, in order of index: true if it is there
// (written by its thread), else nth less their number; of a value that one token has, false
// in any case.  The counts of each 512 pieces first, then of the waves of those that
// have it.
template <int NR>
__device__ __forceinline__ bool locate(const SampleArgs& a, int row, const RowSpan& span,
                                       const Pieces<NR>& p, int first, int last, const Wanted& v,
                                       const Pick& pick, unsigned& nth, CountLds& lds) {
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  auto live = [&](int i) {
    return first + i * kThreads + static_cast<int>(threadIdx.x) < last;
  };
  // Which of the eight words of piece i, any number that the wave shares, have it.
  auto words = [&](int i) {
    unsigned m = 0;
    const u32x4 x = p.pick(i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t d = v.differs(x[j]);
      m |= (d & 0xFFFFu ? 0u : 1u << 2 * j) | (d >> 16 ? 0u : 2u << 2 * j);
    }
    return live(i) ? m : 0u;
  };
  auto take = [&](int i, unsigned m, unsigned skip) {
    for (; skip; --skip) m &= m - 1;
    finish(a, row, span.head + 8 * (first + i * kThreads + static_cast<int>(threadIdx.x)) +
                       __builtin_ctz(m),
           pick.probability);
  };
  constexpr int kPart = 4;  // pieces looked at together
  int hit = -1;
#pragma unroll
  for (int k = 0; k < NR; k += kPart) {
    uint32_t least = 0xFFFFFFFFu;
#pragma unroll
    for (int i = k; i < NR && i < k + kPart; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) least = smaller_words(least, v.differs(p.x[i][j]));
    }
    if (!__ballot(min(least & 0xFFFFu, least >> 16) == 0)) continue;
#pragma unroll
    for (int i = k; i < NR && i < k + kPart; ++i) {
      const u32x4 x = p.get(i);
      uint32_t others = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        others = add_words(others, smaller_words(v.differs(x[j]), 0x10001u));
      }
      const unsigned n = 8 - (others & 0xFFFFu) - (others >> 16);
      if (n && live(i)) {
        atomicAdd(&lds.found[i], n);
        hit = i;
      }
    }
  }
  if (pick.count == 1) {  // no other
    const unsigned long long has = __ballot(hit >= 0);
    if (has) {
      const int at = __builtin_amdgcn_readlane(hit, __builtin_ctzll(has));
      const unsigned m = words(at);
      if (m) take(at, m, 0);
    }
    return false;
  }
  lds_barrier();
  const unsigned n = lane < NR ? lds.found[lane] : 0u, in = wave_scan(n);
  const unsigned long long past = __ballot(in > nth);
  if (!past) {
    nth -= at_lane(in, kWave - 1);
    return false;
  }
  const int at = __builtin_ctzll(past);
  nth -= at_lane(in, at) - at_lane(n, at);
  const unsigned m = words(at);
  const unsigned mine_in = wave_scan(static_cast<unsigned>(__popc(m)));
  if (lane == kWave - 1) lds.wave_count[wave] = mine_in;
  lds_barrier();
  unsigned before = lane < wave ? lds.wave_count[lane & (kWaves - 1)] : 0u;
  before = wave_total(before) + mine_in - __popc(m);
  if (nth >= before && nth < before + __popc(m)) take(at, m, nth - before);
  return true;
}

// NR: pieces a thread takes at a time; HELD: that is the row, kept in registers.
template <int NR, bool HELD>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  __shared__ __align__(16) CountLds lds;
  const int row = blockIdx.x, lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const RowSpan span(a.logits + row * a.stride, a.vocab);
  constexpr int kStep = NR * kThreads;
  clear_bins(lds);
  Pieces<NR> p;
  p.template load<0, kAhead>(span, 0, span.pieces);
  const Setting s = setting_of(a, row);
  uint32_t edge_word;
  int edge_index;
  const bool has_edge = span.edge(lane, edge_word, edge_index);
  lds_barrier();

  const Bins bins(lds.bins);
  Counting counting{span, bins};
  for (int base = 0; base < span.pieces; base += kStep) {
    if (!HELD && base) p.template load<0, kAhead>(span, base, span.pieces);
    counting.add(p, base, span.pieces);
  }
  if (wave == 0 && has_edge) bins.add_word(edge_word, 1);
  if (lane == 0) lds.heavy[wave] = counting.heavy;
  lds_barrier();
  const Heavy heavy = join_heavy(lds, lds.heavy[lane & (kWaves - 1)], lane < kWaves, wave == 0);
  lds_barrier();
  if (!choose_value(a, row, s, heavy, lds)) return;

  const Pick pick = lds.pick;
  const Wanted wanted(__builtin_amdgcn_readfirstlane(pick.key));
  unsigned nth = __builtin_amdgcn_readfirstlane(pick.nth);
  const unsigned long long edges = __ballot(has_edge && wanted.is(edge_word));
  const unsigned in_head = __popcll(edges & 0xFFull);
  // The nth of the edge's words with the value.
  auto take_edge = [&](unsigned long long which) {
    if (wave == 0 && (which >> lane & 1) && __popcll(which & ((1ull << lane) - 1)) == nth) {
      finish(a, row, edge_index, pick.probability);
    }
  };
  if (nth < in_head) {
    take_edge(edges & 0xFFull);
    return;
  }
  nth -= in_head;
  for (int base = 0; base < span.pieces; base += kStep) {
    if (!HELD) {
      p.template load<0, NR>(span, base, span.pieces);
      if (base) {
        lds_barrier();
        if (threadIdx.x < kWave) lds.found[threadIdx.x] = 0;
        lds_barrier();
      }
    }
    if (locate(a, row, span, p, base, span.pieces, wanted, pick, nth, lds)) return;
  }
  take_edge(edges & ~0xFFull);
}

}  // namespace

size_t sample_workspace_bytes(int rows, int vocab) {
  (void)rows;
  (void)vocab;
  return 16;
}

void launch_sample(const SampleArgs& a, hipStream_t stream) {
  const int pieces = (a.vocab + 7) / 8, each = (pieces + kThreads - 1) / kThreads;
  auto run = [&](auto* kernel) {
    hipLaunchKernelGGL(kernel, dim3(a.rows), dim3(kThreads), 0, stream, a);
  };
  each <= 2    ? run(sample_kernel<2, true>)
  : each <= 4  ? run(sample_kernel<4, true>)
  : each <= 8  ? run(sample_kernel<8, true>)
  : each <= 16 ? run(sample_kernel<16, true>)
  : each <= 26 ? run(sample_kernel<26, true>)
  : each <= 38 ? run(sample_kernel<38, true>)
               : run(sample_kernel<16, false>);
}

}  // namespace qlin
