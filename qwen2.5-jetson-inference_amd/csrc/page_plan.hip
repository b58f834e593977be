// Pages of a step for gfx950: block tables, positions and slots of new tokens
// from the sequences' lengths, and the pages of ended sequences back.
#include <stdint.h>

#include "device_common.hpp"
#include "paged_kernels.hpp"

namespace qlin {

namespace {

constexpr int kWide = 1024;  // threads of a scan

// Sums of the plan saturate at 2^31 - 1: a sum of two such fits in 32 bits, and
// taking the minimum after each addition gives the same whatever the order.
__device__ __forceinline__ unsigned add_sat(unsigned a, unsigned b) {
  return min(a + b, 0x7FFFFFFFu);
}

__device__ __forceinline__ unsigned scan_sat(unsigned v) { return wave_scan(v, add_sat); }

// What a token needs of its sequence: the first free entry of its new pages
// (the j-th is entry first - j), and the positions it held, -1 if not served.
struct Share {
  int* starts;  // [sequences + 1]
  int* held;    // [sequences]
  int* first;   // [sequences]
};

struct ScanLds {
  unsigned add[kWide / kWave], need[kWide / kWave];
  unsigned used;
};

// Of the sums that each of `waves` waves left in LDS, and what came before them: those
// before the wave, and all.
struct SumPair {
  unsigned before, all;
};

__device__ __forceinline__ SumPair sums_before(const unsigned* of_wave, int wave, int waves,
                                               unsigned before) {
  const int lane = threadIdx.x & (kWave - 1);
  const unsigned in = add_sat(before, scan_sat(lane < waves ? of_wave[lane] : 0u));
  const unsigned mine = __builtin_amdgcn_readlane(static_cast<int>(in), max(wave - 1, 0));
  return {wave ? mine : before,
          static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(in), kWave - 1))};
}

__device__ __forceinline__ int unused_pages(const PagePlan& p) {
  return min(max(*p.free_count, 0), p.num_pages);
}

// The plan of all sequences by one workgroup of blockDim.x threads; returns the
// pages taken in every thread.  Written here: share, and where `out` lengths_out and
// starts (all of lengths is read before; the caller writes free_count_out).
__device__ int scan_sequences(const AssignArgs& a, const Share& share, ScanLds& lds, bool out) {
  const PagePlan& p = a.plan;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int waves = blockDim.x / kWave;
  const unsigned positions = static_cast<unsigned>(p.max_pages) << p.page_shift;
  const unsigned round = (1u << p.page_shift) - 1;
  const int count = unused_pages(p);
  unsigned add_before = 0, need_before = 0;
  if (threadIdx.x == 0) lds.used = 0;
  // a thread's next sequence is read while this one is added up
  int next_kept = 0, next_added = 0;
  auto read = [&](int s) {
    if (s < p.sequences) {
      next_kept = p.lengths[s];
      next_added = a.added[s];
    }
  };
  read(threadIdx.x);
  for (int base = 0; base < p.sequences; base += blockDim.x) {
    const int s = base + threadIdx.x, kept = next_kept, added = next_added;
    unsigned length = 0, add = 0, need = 0;
    bool fits = false;
    read(s + blockDim.x);
    if (s < p.sequences) {
      length = max(kept, 0);
      add = max(added, 0);
      fits = length + add <= positions && (a.ids || add <= 1);
      if (fits) {
        need = ((length + add + round) >> p.page_shift) - ((length + round) >> p.page_shift);
      }
    }
    const unsigned add_in = scan_sat(add), need_in = scan_sat(need);
    if (lane == kWave - 1) {
      lds.add[wave] = add_in;
      lds.need[wave] = need_in;
    }
    __syncthreads();
    const SumPair adds = sums_before(lds.add, wave, waves, add_before);
    const SumPair needs = sums_before(lds.need, wave, waves, need_before);
    const unsigned add_wave = adds.before, need_wave = needs.before;
    const unsigned add_end = add_sat(add_wave, add_in), need_end = add_sat(need_wave, need_in);
    // An exclusive sum as the inclusive one of the lane before: a saturated sum
    // cannot be taken back.
    unsigned start = __shfl_up(add_in, 1), before = __shfl_up(need_in, 1);
    start = lane ? add_sat(add_wave, start) : add_wave;
    before = lane ? add_sat(need_wave, before) : need_wave;
    if (s < p.sequences) {
      const bool served = fits && (need == 0 || need_end <= static_cast<unsigned>(count)) &&
                          (!a.ids || add == 0 || add_end <= static_cast<unsigned>(a.tokens));
      if (served && need) atomicMax(&lds.used, need_end);
      share.starts[s] = start;
      share.held[s] = served ? static_cast<int>(length) : -1;
      share.first[s] = count - 1 - static_cast<int>(before);
      if (s == p.sequences - 1) share.starts[p.sequences] = add_end;
      if (out) {
        p.lengths_out[s] = served ? static_cast<int>(length + add) : kept;
        if (a.starts) {
          a.starts[s] = start;
          if (s == p.sequences - 1) a.starts[p.sequences] = add_end;
        }
      }
    }
    add_before = adds.all;
    need_before = needs.all;
    __syncthreads();
  }
  return lds.used;
}

// Position, sequence and slot of N tokens, `apart` from t on, and the table's entry where a
// token is the first of a new page, which every new page has.  Step by step for all of
// them, without branches, so that their reads are on their way together.
template <int N>
__device__ __forceinline__ void place_tokens(const AssignArgs& a, const Share& share, int t,
                                             int apart) {
  const PagePlan& p = a.plan;
  const int page_mask = (1 << p.page_shift) - 1, last = p.sequences - 1;
  int s[N], at[N], held[N], first[N], page[N];
  bool live[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int token = t + i * apart;
    live[i] = token < a.tokens;
    s[i] = live[i] ? token : 0;
    at[i] = 0;  // of the sequence's new tokens
  }
  if (a.ids) {  // how many sequences end at or before each: the first that does not
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = 0;
    for (int step = 1 << (31 - __builtin_clz(p.sequences)); step > 0; step >>= 1) {
      int start[N];
#pragma unroll
      for (int i = 0; i < N; ++i) start[i] = share.starts[min(s[i] + step, p.sequences)];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int next = s[i] + step;
        s[i] = next <= p.sequences && start[i] <= t + i * apart ? next : s[i];
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      live[i] = live[i] && s[i] <= last;
      s[i] = min(s[i], last);
      at[i] = t + i * apart - share.starts[s[i]];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) live[i] = live[i] && a.added[s[i]] > 0;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    held[i] = share.held[s[i]];
    first[i] = share.first[s[i]];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    live[i] = live[i] && held[i] >= 0;
    const int pos = held[i] + at[i], index = pos >> p.page_shift;
    const int old_pages = (held[i] + page_mask) >> p.page_shift;
    const int* from = index < old_pages
                          ? p.table + static_cast<size_t>(s[i]) * p.stride + index
                          : a.free_pages + (first[i] - (index - old_pages));
    page[i] = live[i] ? *from : -1;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int token = t + i * apart, pos = held[i] + at[i];
    if (live[i] && (pos & page_mask) == 0) {  // of no page that was there
      p.table[static_cast<size_t>(s[i]) * p.stride + (pos >> p.page_shift)] = page[i];
    }
    const bool placed = static_cast<unsigned>(page[i]) < static_cast<unsigned>(p.num_pages);
    if (token < a.tokens) {
      a.positions[token] = live[i] ? pos : -1;
      if (a.ids) a.ids[token] = live[i] ? s[i] : -1;
      if (a.slots) {
        a.slots[token] = live[i] && placed ? (static_cast<long long>(page[i]) << p.page_shift) +
                                                 (pos & page_mask)
                                           : -1;
      }
    }
  }
}

__device__ __forceinline__ Share share_of(int* workspace, int sequences) {
  return {workspace, workspace + sequences + 1, workspace + 2 * sequences + 1};
}

// Up to kHere sequences and one workgroup's tokens, or where nothing is written in place:
// every workgroup plans all sequences for itself, in LDS, and the first writes the plan's
// outputs.  Otherwise a launch of one workgroup writes the plan into the workspace and a
// second one places the tokens.
//
// Bound: a step's launch and its chain of reads: lengths, then free entries or pages.  24
// sequences 3.0 us (1.7 an empty launch), 25 000 tokens of 8 prompts 3.5, 620 000 of 2000
// sequences 10.8 for 10 MB, mostly written.
constexpr int kHere = 2048;
// Tokens from which a thread takes four.
constexpr int kManyTokens = 1 << 16;

template <int NT, int N>
__global__ __launch_bounds__(NT) void assign_kernel(AssignArgs a) {
  __shared__ ScanLds lds;
  __shared__ int starts[kHere + 1], held[kHere], first[kHere];
  const Share share{starts, held, first};
  const int used = scan_sequences(a, share, lds, blockIdx.x == 0);
  // every thread of the workgroup has read the count by now
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.plan.free_count_out = unused_pages(a.plan) - used;
  const int t = blockIdx.x * NT * N + threadIdx.x;
  if (t < a.tokens) place_tokens<N>(a, share, t, NT);
}

__global__ __launch_bounds__(kWide) void assign_scan_kernel(AssignArgs a, int* workspace) {
  __shared__ ScanLds lds;
  const int used = scan_sequences(a, share_of(workspace, a.plan.sequences), lds, true);
  if (threadIdx.x == 0) *a.plan.free_count_out = unused_pages(a.plan) - used;
}

// The starts are searched in LDS while they fit.
constexpr int kStarts = 8192, kFillTokens = 1024;

template <bool FITS>
__global__ __launch_bounds__(256) void assign_fill_kernel(AssignArgs a, int* workspace) {
  __shared__ int starts[FITS ? kStarts : 1];
  Share share = share_of(workspace, a.plan.sequences);
  if (FITS && a.ids) {
#pragma unroll 8
    for (int i = threadIdx.x; i <= a.plan.sequences; i += 256) starts[i] = share.starts[i];
    __syncthreads();
  }
  if (FITS) share.starts = starts;
  const int t = blockIdx.x * kFillTokens + threadIdx.x;
  if (t < a.tokens) place_tokens<kFillTokens / 256>(a, share, t, 256);
}

}  // namespace

size_t page_plan_workspace_bytes(int sequences) {
  return (static_cast<size_t>(sequences) * 3 + 1 + 3) / 4 * 16;
}

void launch_pages_assign(const AssignArgs& a, void* workspace, hipStream_t stream) {
  int* ws = static_cast<int*>(workspace);
  const PagePlan& p = a.plan;
  auto blocks = [&](int each) { return static_cast<unsigned>((a.tokens - 1) / each + 1); };
  const int threads = p.sequences <= 256 && a.tokens <= kManyTokens ? 256 : kWide;
  const bool in_place = p.lengths_out == p.lengths || p.free_count_out == p.free_count;
  if (p.sequences <= (in_place ? threads : kHere) && (a.tokens <= threads || !in_place)) {
    if (threads == 256) {
      hipLaunchKernelGGL((assign_kernel<256, 1>), dim3(blocks(256)), dim3(256), 0, stream, a);
    } else if (a.tokens <= kManyTokens) {
      hipLaunchKernelGGL((assign_kernel<kWide, 1>), dim3(blocks(kWide)), dim3(kWide), 0, stream,
                         a);
    } else {
      hipLaunchKernelGGL((assign_kernel<kWide, 4>), dim3(blocks(4 * kWide)), dim3(kWide), 0,
                         stream, a);
    }
    return;
  }
  hipLaunchKernelGGL(assign_scan_kernel, dim3(1), dim3(kWide), 0, stream, a, ws);
  if (p.sequences < kStarts) {
    hipLaunchKernelGGL(assign_fill_kernel<true>, dim3(blocks(kFillTokens)), dim3(256), 0, stream,
                       a, ws);
  } else {
    hipLaunchKernelGGL(assign_fill_kernel<false>, dim3(blocks(kFillTokens)), dim3(256), 0, stream,
                       a, ws);
  }
}

namespace {

// Pages that go back, of sequence s.
__device__ __forceinline__ unsigned ended_pages(const ReleaseArgs& a, int s, int length) {
  const PagePlan& p = a.plan;
  if (a.finished[s] == 0) return 0;
  const unsigned round = (1u << p.page_shift) - 1;
  return min((static_cast<unsigned>(max(length, 0)) + round) >> p.page_shift,
             static_cast<unsigned>(p.max_pages));
}

// Sequence s's pages to the entries above `above`, the unused ones and the pages that go
// back after its own, its last page first.  Such a sum is right, or so large that its
// entries lie past the list.
__device__ __forceinline__ void give_back(const ReleaseArgs& a, int s, int pages,
                                          unsigned above) {
  const PagePlan& p = a.plan;
  const int top = static_cast<int>(add_sat(above, pages)) - 1;
  const int* row = p.table + static_cast<size_t>(s) * p.stride;
  for (int i = threadIdx.x; i < pages; i += blockDim.x) {
    const int place = top - i;
    if (place < p.num_pages) a.free_pages[place] = row[i];
  }
}

// Up to kReleaseHere sequences, nothing in place: a workgroup of each adds up the pages
// that go back after its own; the first sequence's has the whole count so.  Otherwise one
// workgroup writes each sequence's place into the workspace, and a second launch copies.
//
// Bound: as above; 64 sequences 2.4 us, 860 000 pages of 1350 sequences 3.9 for 6.9 MB.
constexpr int kReleaseHere = 4096;

__global__ __launch_bounds__(256) void release_kernel(ReleaseArgs a) {
  constexpr int kWaves = 256 / kWave;
  __shared__ unsigned after_wave[kWaves];
  const PagePlan& p = a.plan;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, s = blockIdx.x;
  const int length = p.lengths[s];
  const unsigned mine = ended_pages(a, s, length);
  if (threadIdx.x == 0) p.lengths_out[s] = a.finished[s] ? 0 : length;
  if (!mine && s) return;  // the same in all threads
  unsigned after = 0;
  for (int i = s + 1 + threadIdx.x; i < p.sequences; i += 256) {
    after = add_sat(after, ended_pages(a, i, p.lengths[i]));
  }
  after = scan_sat(after);
  if (lane == kWave - 1) after_wave[wave] = after;
  __syncthreads();
  unsigned above = unused_pages(p);
  for (int i = 0; i < kWaves; ++i) above = add_sat(above, after_wave[i]);
  if (s == 0 && threadIdx.x == 0) {
    *p.free_count_out = min(add_sat(above, mine), static_cast<unsigned>(p.num_pages));
  }
  give_back(a, s, mine, above);
}

// Where the pages of each ended sequence go: share.first[s] entries lie below its last one,
// share.held[s] how many there are.  From the last sequence down.
__global__ __launch_bounds__(kWide) void release_scan_kernel(ReleaseArgs a, int* workspace) {
  __shared__ ScanLds lds;
  const PagePlan& p = a.plan;
  const Share share = share_of(workspace, p.sequences);
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  unsigned below = unused_pages(p);
  for (int base = 0; base < p.sequences; base += kWide) {
    const int s = p.sequences - 1 - base - static_cast<int>(threadIdx.x);
    unsigned pages = 0;
    if (s >= 0) {
      const int length = p.lengths[s];
      pages = ended_pages(a, s, length);
      p.lengths_out[s] = a.finished[s] ? 0 : length;
    }
    const unsigned in = scan_sat(pages);
    if (lane == kWave - 1) lds.need[wave] = in;
    __syncthreads();
    const SumPair sums = sums_before(lds.need, wave, kWide / kWave, below);
    const unsigned mine = sums.before;
    unsigned first = __shfl_up(in, 1);
    first = lane ? add_sat(mine, first) : mine;
    if (s >= 0) {
      share.held[s] = pages;
      share.first[s] = first;
    }
    below = sums.all;
    __syncthreads();
  }
  if (threadIdx.x == 0) *p.free_count_out = min(below, static_cast<unsigned>(p.num_pages));
}

__global__ __launch_bounds__(256) void release_copy_kernel(ReleaseArgs a, int* workspace) {
  const Share share = share_of(workspace, a.plan.sequences);
  const int s = blockIdx.x;
  give_back(a, s, share.held[s], share.first[s]);
}

}  // namespace

void launch_pages_release(const ReleaseArgs& a, void* workspace, hipStream_t stream) {
  int* ws = static_cast<int*>(workspace);
  const PagePlan& p = a.plan;
  const bool in_place = p.lengths_out == p.lengths || p.free_count_out == p.free_count;
  if (p.sequences <= kReleaseHere && !in_place) {
    hipLaunchKernelGGL(release_kernel, dim3(p.sequences), dim3(256), 0, stream, a);
    return;
  }
  hipLaunchKernelGGL(release_scan_kernel, dim3(1), dim3(kWide), 0, stream, a, ws);
  hipLaunchKernelGGL(release_copy_kernel, dim3(p.sequences), dim3(256), 0, stream, a, ws);
}

}  // namespace qlin
