// plan.hip — what a step's new tokens make of a paged batch, on the device: starts, lengths and the page table, the pages taken
// from a stack, and for each token its sequence, position and slot; and pages given back to the stack.
//
// Two sums in a row: of the new tokens (a sequence's start), then of the pages that the tokens which fit need (where in the stack
// its pages are).  One block takes the sequences 1024 at a time, and its threads the pages one each: a page's sequence is found in
// the sums in LDS (a thread a sequence waits for a long prompt's pages one after another).  Rows find their sequence in the starts
// alike, by the same block where all sequences are in LDS and the rows are a few a thread, else by a launch of its own.
// Dependent loads and barriers bound it, not bytes.  32 single tokens: 5.5 us in one launch (4.2 + 1.9 and a launch more in two); 1024
// ragged requests: 11.4 us and 4.2 for their rows (17.9 and 5.5 where a thread wrote a sequence's pages and searched in memory).
#include "paged.hpp"

namespace hq {

namespace {

constexpr int kThreads = 1024;
constexpr int kFew = 4 * kThreads;  // rows that the planning block maps itself

// the sum of v over the threads before this one, and over all in `total` (every thread calls it; `part`: 16 words of LDS)
HQ_DEV int64_t sum_before(int64_t v, int64_t *part, int64_t &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t sum = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t other = __shfl_up(sum, o, 64);
    if (lane >= o) sum += other;
  }
  __syncthreads();  // (what the call before read)
  if (lane == 63) part[wave] = sum;
  __syncthreads();
  // (a lane a wave: the sums up to each)
  int64_t waves = part[lane & 15];
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    const int64_t other = __shfl_up(waves, o, 16);
    if ((lane & 15) >= o) waves += other;
  }
  total = __shfl(waves, 15, 16);
  const int64_t before = wave ? __shfl(waves, wave - 1, 16) : 0;
  return before + sum - v;
}

// what is written for row t: its sequence's number and its place there (s < 0: no sequence has it)
HQ_DEV void map_row(const Plan &a, const Pool &p, int32_t t, int32_t s, int32_t position) {
  if (a.sequence) a.sequence[t] = s;
  if (a.position) a.position[t] = s < 0 ? -1 : position;
  if (!a.slot) return;
  const int32_t entry = position >> p.shift;
  const int32_t page = s >= 0 && entry < a.width ? a.table[(int64_t)s * a.width + entry] : -1;
  a.slot[t] = (uint32_t)page < (uint32_t)p.pages ? ((int64_t)page << p.shift) + (position & ((1 << p.shift) - 1)) : -1;
}

// the last of 1024 rising numbers that is not more than t (the first is not)
HQ_DEV int32_t last_up_to(const int32_t *numbers, int32_t t) {
  int32_t at = 0;
#pragma unroll
  for (int32_t step = kThreads / 2; step > 0; step >>= 1)
    if (numbers[at + step] <= t) at += step;
  return at;
}

template <bool MAP>
__global__ __launch_bounds__(kThreads) void plan_kernel(Plan a, Pool p) {
  __shared__ int64_t part[kThreads / 64];
  __shared__ int32_t begins[kThreads], firsts[kThreads], row_begins[MAP ? kThreads : 1], helds[MAP ? kThreads : 1];
  const int32_t count = min(max(*p.count, 0), p.pages), mask = (1 << p.shift) - 1;
  int64_t rows = 0, pages = 0;  // of the sequences before these
  for (int64_t s0 = 0; s0 < a.sequences; s0 += kThreads) {
    const int64_t s = s0 + threadIdx.x;
    const bool live = s < a.sequences;
    const int32_t held = live ? min(max(a.held[s], 0), kMostPositions) : 0;
    const int32_t asked = live ? min(max(a.fresh[s], 0), a.tokens) : 0;
    int64_t total;
    const int64_t before = rows + sum_before(asked, part, total);
    rows += total;
    const int32_t begin = (int32_t)min(before, (int64_t)a.tokens), fresh = min(asked, a.tokens - begin);
    // the pages that begin among the new positions, as far as the table goes (all sequences' together: fewer than their tokens
    // and one each)
    const int32_t length = held + fresh, first = min((held + mask) >> p.shift, a.width);
    const int32_t wanted = min((length + mask) >> p.shift, a.width) - first;
    begins[threadIdx.x] = (int32_t)sum_before(wanted, part, total);
    firsts[threadIdx.x] = first;
    if (MAP) row_begins[threadIdx.x] = live ? begin : INT32_MAX, helds[threadIdx.x] = held;
    if (live) {
      a.starts[s] = begin;
      a.lengths[s] = length;
    }
    __syncthreads();
    for (int32_t i = threadIdx.x; i < (int32_t)total; i += kThreads) {
      const int32_t w = last_up_to(begins, i);
      const int64_t at = pages + i;
      a.table[(s0 + w) * a.width + firsts[w] + (i - begins[w])] = at < count ? p.free[count - 1 - at] : -1;
    }
    pages += total;
  }
  const int32_t end = (int32_t)min(rows, (int64_t)a.tokens);
  if (threadIdx.x == 0) {
    a.starts[a.sequences] = end;
    *p.left = (int32_t)max(count - pages, (int64_t)0);
    if (p.missing) *p.missing = (int32_t)max(pages - count, (int64_t)0);
  }
  if (!MAP) return;
  __syncthreads();  // (the table's entries are written)
  for (int32_t t = threadIdx.x; t < a.tokens; t += kThreads) {
    const int32_t s = t < end ? last_up_to(row_begins, t) : -1;
    map_row(a, p, t, s, s < 0 ? 0 : helds[s] + (t - row_begins[s]));
  }
}

// A block has 1024 of the starts in LDS, evenly; what lies between two of them is searched in memory.
__global__ __launch_bounds__(kThreads) void map_kernel(Plan a, Pool p) {
  __shared__ int32_t begins[kThreads];
  const int32_t each = (a.sequences - 1) / kThreads + 1, mine = threadIdx.x * each;
  const int32_t end = a.starts[a.sequences];
  begins[threadIdx.x] = (int32_t)threadIdx.x < (a.sequences - 1) / each + (a.sequences > 0) ? a.starts[mine] : INT32_MAX;
  __syncthreads();
  const int32_t t = blockIdx.x * kThreads + threadIdx.x;
  if (t >= a.tokens) return;
  if (t >= end) return map_row(a, p, t, -1, 0);
  // starts[lo] <= t < starts[hi]
  int32_t lo = last_up_to(begins, t) * each, hi = lo + min(each, a.sequences - lo);
  while (hi - lo > 1) {
    const int32_t mid = (lo + hi) >> 1;
    if (a.starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  map_row(a, p, t, lo, a.lengths[lo] - (a.starts[lo + 1] - t));
}

__global__ __launch_bounds__(kThreads) void give_kernel(Pool p, int32_t *table, int32_t sequences, int32_t width, const int32_t *from,
                                                        const int32_t *to) {
  __shared__ int64_t part[kThreads / 64];
  int64_t count = min(max(*p.count, 0), p.pages);
  for (int32_t s = 0; s < sequences; s++) {
    const int32_t first = from ? max(from[s], 0) : 0, last = to ? min(to[s], width) : width;
    for (int32_t e0 = first; e0 < last; e0 += kThreads) {
      const int32_t e = e0 + threadIdx.x;
      int32_t *entry = table + (int64_t)s * width + min(e, width - 1);
      const int32_t page = e < last ? *entry : -1;
      const bool given = (uint32_t)page < (uint32_t)p.pages;
      int64_t total;
      const int64_t at = count + sum_before(given, part, total);
      if (given) {
        *entry = -1;
        if (at < p.pages) p.free[at] = page;
      }
      count += total;
    }
  }
  if (threadIdx.x == 0) *p.left = (int32_t)min(count, (int64_t)p.pages);
}

}  // namespace

hipError_t launch_plan(const Plan &a, const Pool &p, hipStream_t s) {
  const bool map = a.tokens > 0 && (a.sequence || a.position || a.slot);
  if (map && a.sequences <= kThreads && a.tokens <= kFew) {
    hipLaunchKernelGGL(plan_kernel<true>, dim3(1), dim3(kThreads), 0, s, a, p);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(plan_kernel<false>, dim3(1), dim3(kThreads), 0, s, a, p);
  if (const hipError_t e = hipGetLastError()) return e;
  if (!map) return hipSuccess;
  hipLaunchKernelGGL(map_kernel, dim3((uint32_t)(((int64_t)a.tokens + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, a, p);
  return hipGetLastError();
}

hipError_t launch_give(const Pool &p, int32_t *table, int32_t sequences, int32_t width, const int32_t *from, const int32_t *to,
                       hipStream_t s) {
  hipLaunchKernelGGL(give_kernel, dim3(1), dim3(kThreads), 0, s, p, table, sequences, width, from, to);
  return hipGetLastError();
}

}  // namespace hq
