// paged.hpp — the paged key/value cache and a batch of new tokens, as the kernels of cache.hip and attention.hip see them.
//
// Every number that comes from device memory (starts, lengths, page numbers) is clamped before it addresses anything: a
// batch that contradicts itself gives wrong numbers, never an access out of the buffers.
#pragma once
#include "common.hpp"
#include "launch.hpp"

namespace hq {

struct Sequence {
  int32_t begin, count, length;  // its first new token, how many there are, and its positions with them
};

HQ_DEV Sequence sequence_of(const Batch &b, int32_t s) {
  Sequence q;
  q.begin = min(max(b.starts[s], 0), b.tokens);
  q.count = min(max(b.starts[s + 1], q.begin), b.tokens) - q.begin;
  q.length = max(b.lengths[s], 0);
  return q;
}

// the same of a sequence that the whole wave asks for
HQ_DEV Sequence wave_sequence_of(const Batch &b, int32_t s) {
  Sequence q = sequence_of(b, s);
  q.begin = __builtin_amdgcn_readfirstlane(q.begin);
  q.count = __builtin_amdgcn_readfirstlane(q.count);
  q.length = __builtin_amdgcn_readfirstlane(q.length);
  return q;
}

// the page that holds position `at` of sequence s, or -1: none (a position before the first or past the table, an entry that
// is no page)
HQ_DEV int32_t page_of(const Batch &b, const Cache &c, int32_t s, int32_t at) {
  const int32_t i = at >> c.shift;
  if (at < 0 || i >= b.width) return -1;
  const int32_t p = b.table[(int64_t)s * b.width + i];
  return (uint32_t)p < (uint32_t)c.pages ? p : -1;
}

// the first of a (page, head)'s vectors
HQ_DEV int64_t vectors_of(const Cache &c, int32_t page, int32_t head) {
  return ((int64_t)page * c.heads + head) << c.shift;
}

// The sequence whose items a launch's `at`-th are, and which of them: sequence s has its tokens / 64 + 2 of the tokens / 64 +
// 2 sequences items, from starts[s] / 64 + 2 s on (no sums over the sequences are needed), of which it may use fewer.  A lane a
// sequence, 64 at a time; every lane of the wave calls it; s is -1 where no sequence has the item.
struct Place {
  int32_t s, rest;
  Sequence q;
};
HQ_DEV Place place_of(const Batch &b, int32_t at) {
  const int lane = threadIdx.x & 63;
  for (int32_t s0 = 0; s0 < b.sequences; s0 += 64) {
    const int32_t s = min(s0 + lane, b.sequences - 1);
    const Sequence q = sequence_of(b, s);
    const int32_t first = (q.begin >> 6) + 2 * s, end = ((q.begin + q.count) >> 6) + 2 * s + 2;
    const uint64_t in = __ballot(s0 + lane < b.sequences && at >= first && at < end);
    if (!in) continue;
    const int l = __ffsll((unsigned long long)in) - 1;
    return {s0 + l, at - __builtin_amdgcn_readlane(first, l),
            {__builtin_amdgcn_readlane(q.begin, l), __builtin_amdgcn_readlane(q.count, l), __builtin_amdgcn_readlane(q.length, l)}};
  }
  return {-1, 0, {0, 0, 0}};
}

}  // namespace hq
