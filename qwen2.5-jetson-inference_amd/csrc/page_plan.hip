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

__device__ __forceinline__ unsigned wave_scan(unsigned v, int lane) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const unsigned o = __shfl_up(v, d);
    if (lane >= d) v = add_sat(v, o);
  }
  return v;
}

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

__device__ __forceinline__ int unused_pages(const PagePlan& p) {
  return min(max(*p.free_count, 0), p.num_pages);
}

// The plan of all sequences by one workgroup of blockDim.x threads; returns the
// pages taken in every thread.  Written here: share, and where `out` lengths_out and
// starts (all of lengths is read before; the caller writes free_count_out).
__device__ int scan_sequences(const AssignArgs& a, const Share& share, ScanLds& lds, bool out) {
  const PagePlan& p = a.plan;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int waves = blockDim.x / kWave;
  const unsigned positions = static_cast<unsigned>(p.max_pages) << p.page_shift;
  const unsigned round = (1u << p.page_shift) - 1;
  const int count = unused_pages(p);
  unsigned add_before = 0, need_before = 0;
  if (threadIdx.x == 0) lds.used = 0;
  for (int base = 0; base < p.sequences; base += blockDim.x) {
    const int s = base + threadIdx.x;
    unsigned length = 0, add = 0, need = 0;
    int kept = 0;
    bool fits = false;
    if (s < p.sequences) {
      kept = p.lengths[s];
      length = max(kept, 0);
      add = max(a.added[s], 0);
      fits = length + add <= positions && (a.ids || add <= 1);
      if (fits) {
        need = ((length + add + round) >> p.page_shift) - ((length + round) >> p.page_shift);
      }
    }
    const unsigned add_in = wave_scan(add, lane), need_in = wave_scan(need, lane);
    if (lane == kWave - 1) {
      lds.add[wave] = add_in;
      lds.need[wave] = need_in;
    }
    __syncthreads();
    unsigned add_sum = add_before, need_sum = need_before, add_wave = 0, need_wave = 0;
    for (int w = 0; w < waves; ++w) {
      if (w == wave) {
        add_wave = add_sum;
        need_wave = need_sum;
      }
      add_sum = add_sat(add_sum, lds.add[w]);
      need_sum = add_sat(need_sum, lds.need[w]);
    }
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
    add_before = add_sum;
    need_before = need_sum;
    __syncthreads();
  }
  return lds.used;
}

// Position, sequence and slot of tokens [t, t + 4), and the table's entry where a
// token is the first of a new page, which every new page has.
__device__ __forceinline__ void place_tokens(const AssignArgs& a, const Share& share, int t) {
  const PagePlan& p = a.plan;
  const int page_mask = (1 << p.page_shift) - 1;
  // The first sequence from `from` whose tokens end past `token`.
  auto sequence_of = [&](int from, int token) {
    int hi = p.sequences;
    while (from < hi) {
      const int mid = (from + hi) / 2;
      if (share.starts[mid + 1] > token) {
        hi = mid;
      } else {
        from = mid + 1;
      }
    }
    return from;
  };
  int s = a.ids ? sequence_of(0, t) : t;
  int position[4], id[4];
  long long slot[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    position[i] = id[i] = -1;
    slot[i] = -1;
    int at = 0;  // of the sequence's new tokens
    bool live = t + i < a.tokens;
    if (a.ids) {
      if (s < p.sequences && share.starts[s + 1] <= t + i) s = sequence_of(s + 1, t + i);
      live = live && s < p.sequences;
      if (live) at = t + i - share.starts[s];
    } else {
      s = t + i;
      live = live && a.added[s] > 0;
    }
    if (!live) continue;
    const int held = share.held[s];
    if (held < 0) continue;
    const int pos = held + at, index = pos >> p.page_shift;
    const int old_pages = (held + page_mask) >> p.page_shift;
    int* entry = p.table + static_cast<size_t>(s) * p.stride + index;
    int page;
    if (index < old_pages) {
      page = *entry;
    } else {
      page = a.free_pages[share.first[s] - (index - old_pages)];
      if ((pos & page_mask) == 0) *entry = page;
    }
    position[i] = pos;
    id[i] = s;
    if (static_cast<unsigned>(page) < static_cast<unsigned>(p.num_pages)) {
      slot[i] = (static_cast<long long>(page) << p.page_shift) + (pos & page_mask);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (t + i < a.tokens) {
      a.positions[t + i] = position[i];
      if (a.ids) a.ids[t + i] = id[i];
      if (a.slots) a.slots[t + i] = slot[i];
    }
  }
}

__device__ __forceinline__ Share share_of(int* workspace, int sequences) {
  return {workspace, workspace + sequences + 1, workspace + 2 * sequences + 1};
}

__global__ __launch_bounds__(kWide) void assign_scan_kernel(AssignArgs a, int* workspace) {
  __shared__ ScanLds lds;
  const int used = scan_sequences(a, share_of(workspace, a.plan.sequences), lds, true);
  // every thread has read the count by now
  if (threadIdx.x == 0) *a.plan.free_count_out = unused_pages(a.plan) - used;
}

__global__ __launch_bounds__(256) void assign_fill_kernel(AssignArgs a, int* workspace) {
  const int t = 4 * (blockIdx.x * blockDim.x + threadIdx.x);
  if (t < a.tokens) place_tokens(a, share_of(workspace, a.plan.sequences), t);
}

}  // namespace

size_t page_plan_workspace_bytes(int sequences) {
  return (static_cast<size_t>(sequences) * 3 + 1 + 3) / 4 * 16;
}

void launch_pages_assign(const AssignArgs& a, void* workspace, hipStream_t stream) {
  int* ws = static_cast<int*>(workspace);
  hipLaunchKernelGGL(assign_scan_kernel, dim3(1), dim3(kWide), 0, stream, a, ws);
  const unsigned blocks = static_cast<unsigned>((a.tokens + 1023ll) / 1024);
  hipLaunchKernelGGL(assign_fill_kernel, dim3(blocks), dim3(256), 0, stream, a, ws);
}

namespace {

// Where the pages of each ended sequence go: share.first[s] is its first page's entry,
// share.held[s] how many there are.
__global__ __launch_bounds__(kWide) void release_scan_kernel(ReleaseArgs a, int* workspace) {
  __shared__ ScanLds lds;
  const PagePlan& p = a.plan;
  const Share share = share_of(workspace, p.sequences);
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const unsigned round = (1u << p.page_shift) - 1;
  const int count = unused_pages(p);
  unsigned before = 0;
  for (int base = 0; base < p.sequences; base += kWide) {
    const int s = base + threadIdx.x;
    unsigned pages = 0;
    if (s < p.sequences) {
      const int length = p.lengths[s];
      const bool ended = a.finished[s] != 0;
      if (ended) {
        pages = min((static_cast<unsigned>(max(length, 0)) + round) >> p.page_shift,
                    static_cast<unsigned>(p.max_pages));
      }
      p.lengths_out[s] = ended ? 0 : length;
    }
    const unsigned in = wave_scan(pages, lane);
    if (lane == kWave - 1) lds.need[wave] = in;
    __syncthreads();
    unsigned sum = before, mine = 0;
    for (int w = 0; w < kWide / kWave; ++w) {
      if (w == wave) mine = sum;
      sum = add_sat(sum, lds.need[w]);
    }
    unsigned first = __shfl_up(in, 1);
    first = lane ? add_sat(mine, first) : mine;
    if (s < p.sequences) {
      share.held[s] = pages;
      share.first[s] = first;
    }
    before = sum;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    share.starts[0] = add_sat(count, before);  // where the last released page's place ends
    *p.free_count_out = min(add_sat(count, before), static_cast<unsigned>(p.num_pages));
  }
}

__global__ __launch_bounds__(256) void release_copy_kernel(ReleaseArgs a, int* workspace) {
  const PagePlan& p = a.plan;
  const Share share = share_of(workspace, p.sequences);
  for (int s = blockIdx.x; s < p.sequences; s += gridDim.x) {
    const int pages = share.held[s];
    const int top = share.starts[0] - 1 - share.first[s];
    for (int i = threadIdx.x; i < pages; i += blockDim.x) {
      const int place = top - i;
      if (place >= 0 && place < p.num_pages) {
        a.free_pages[place] = p.table[static_cast<size_t>(s) * p.stride + i];
      }
    }
  }
}

}  // namespace

void launch_pages_release(const ReleaseArgs& a, void* workspace, hipStream_t stream) {
  int* ws = static_cast<int*>(workspace);
  hipLaunchKernelGGL(release_scan_kernel, dim3(1), dim3(kWide), 0, stream, a, ws);
  hipLaunchKernelGGL(release_copy_kernel, dim3(a.plan.sequences), dim3(256), 0, stream, a, ws);
}

}  // namespace qlin
