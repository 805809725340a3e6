// plan.hip — what a step's new tokens make of a paged batch, on the device: starts, lengths and the page table, the pages taken
// from a stack, and for each token its sequence, position and slot; and pages given back to the stack.
//
// Two sums in a row: of the new tokens (a sequence's start), then of the pages that the tokens which fit need (where in the stack
// its pages are).  One block takes the sequences 1024 at a time; a second launch finds each row's sequence in the starts.
#include "paged.hpp"

namespace hq {

namespace {

constexpr int kThreads = 1024;

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

__global__ __launch_bounds__(kThreads) void plan_kernel(Plan a, Pool p) {
  __shared__ int64_t part[kThreads / 64];
  const int32_t count = min(max(*p.count, 0), p.pages), mask = (1 << p.shift) - 1;
  int64_t rows = 0, pages = 0;  // of the sequences before these
  for (int32_t s0 = 0; s0 < a.sequences; s0 += kThreads) {
    const int32_t s = s0 + threadIdx.x;
    const bool live = s < a.sequences;
    const int32_t held = live ? min(max(a.held[s], 0), kMostPositions) : 0;
    const int32_t asked = live ? min(max(a.fresh[s], 0), a.tokens) : 0;
    int64_t total;
    const int64_t before = rows + sum_before(asked, part, total);
    rows += total;
    const int32_t begin = (int32_t)min(before, (int64_t)a.tokens), fresh = min(asked, a.tokens - begin);
    // the pages that begin among the new positions, as far as the table goes
    const int32_t length = held + fresh, first = min((held + mask) >> p.shift, a.width);
    const int32_t wanted = min((length + mask) >> p.shift, a.width) - first;
    const int64_t at = pages + sum_before(wanted, part, total);
    pages += total;
    if (!live) continue;
    a.starts[s] = begin;
    a.lengths[s] = length;
#pragma clang loop unroll(disable) vectorize(disable)
    for (int32_t i = 0; i < wanted; i++)
      a.table[(int64_t)s * a.width + first + i] = at + i < count ? p.free[count - 1 - (at + i)] : -1;
  }
  if (threadIdx.x == 0) {
    a.starts[a.sequences] = (int32_t)min(rows, (int64_t)a.tokens);
    *p.left = (int32_t)max(count - pages, (int64_t)0);
    if (p.missing) *p.missing = (int32_t)max(pages - count, (int64_t)0);
  }
}

__global__ __launch_bounds__(256) void map_kernel(Plan a, Pool p) {
  const int32_t t = blockIdx.x * 256 + threadIdx.x;
  if (t >= a.tokens) return;
  // the last sequence whose first token is not behind t
  int32_t lo = 0, hi = a.sequences;  // starts[lo] <= t < starts[hi], where any sequence has t
  while (hi - lo > 1) {
    const int32_t mid = (lo + hi) >> 1;
    if (a.starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  if (t >= a.starts[a.sequences]) {  // (no sequence has it)
    if (a.sequence) a.sequence[t] = -1;
    if (a.position) a.position[t] = -1;
    if (a.slot) a.slot[t] = -1;
    return;
  }
  const int32_t position = a.lengths[lo] - (a.starts[lo + 1] - t), entry = position >> p.shift;
  if (a.sequence) a.sequence[t] = lo;
  if (a.position) a.position[t] = position;
  if (!a.slot) return;
  const int32_t page = entry < a.width ? a.table[(int64_t)lo * a.width + entry] : -1;
  a.slot[t] = (uint32_t)page < (uint32_t)p.pages ? ((int64_t)page << p.shift) + (position & ((1 << p.shift) - 1)) : -1;
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
  hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(kThreads), 0, s, a, p);
  if (const hipError_t e = hipGetLastError()) return e;
  if (a.tokens <= 0 || (!a.sequence && !a.position && !a.slot)) return hipSuccess;
  hipLaunchKernelGGL(map_kernel, dim3((uint32_t)((a.tokens + 255) / 256)), dim3(256), 0, s, a, p);
  return hipGetLastError();
}

hipError_t launch_give(const Pool &p, int32_t *table, int32_t sequences, int32_t width, const int32_t *from, const int32_t *to,
                       hipStream_t s) {
  hipLaunchKernelGGL(give_kernel, dim3(1), dim3(kThreads), 0, s, p, table, sequences, width, from, to);
  return hipGetLastError();
}

}  // namespace hq
