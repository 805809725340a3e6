// paged.hpp — the paged key/value cache and a batch of new tokens, as the kernels of cache.hip and attention.hip see them.
//
// Every number that comes from device memory (starts, lengths, page numbers) is clamped before it addresses anything: a
// batch that contradicts itself gives wrong numbers, never an access out of the buffers.
#pragma once
#include "common.hpp"
#include "launch.hpp"

namespace hq {

// (a table holds 2^30 positions at most and a batch 2^24 tokens: from a longer sequence all of its new tokens are past its table)
constexpr int32_t kMostPositions = (1 << 30) + (1 << 25);

struct Sequence {
  int32_t begin, count, length;  // its first new token, how many there are, and its positions with them
};

HQ_DEV Sequence sequence_of(const Batch &b, int32_t s) {
  Sequence q;
  q.begin = min(max(b.starts[s], 0), b.tokens);
  q.count = min(max(b.starts[s + 1], q.begin), b.tokens) - q.begin;
  q.length = min(max(b.lengths[s], 0), kMostPositions);
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

// The table's entry for position `at` of sequence s (the nearest one where it has none), and the page that it means: -1 where
// there is no such position (before the first or past the table) or the entry is no page.  The entry is loaded without a branch:
// a load in one is waited for at its end, with every load before it.
HQ_DEV int32_t entry_of(const Batch &b, const Cache &c, int32_t s, int32_t at) {
  return b.table[(int64_t)s * b.width + max(min(at >> c.shift, b.width - 1), 0)];
}
HQ_DEV int32_t page_in(const Batch &b, const Cache &c, int32_t entry, int32_t at) {
  return at >= 0 && (at >> c.shift) < b.width && (uint32_t)entry < (uint32_t)c.pages ? entry : -1;
}
HQ_DEV int32_t page_of(const Batch &b, const Cache &c, int32_t s, int32_t at) {
  return page_in(b, c, entry_of(b, c, s, at), at);
}

// the first of a (page, head)'s vectors
HQ_DEV int64_t vectors_of(const Cache &c, int32_t page, int32_t head) {
  return ((int64_t)page * c.heads + head) << c.shift;
}

// The sequence whose items (of 64 tokens, or 1 << SHIFT) a launch's `at`-th are, and which of them: sequence s has its tokens / 64 + 2
// of the tokens / 64 + 2 sequences items, from starts[s] / 64 + 2 s on (no sums over the sequences are needed), of which it may
// use fewer.  A lane a sequence, 64 at a time; every lane of the wave calls it; s is -1 where no sequence has the item.
struct Place {
  int32_t s, rest;
  Sequence q;
};
template <int SHIFT = 6>
HQ_DEV Place place_of(const Batch &b, int32_t at) {
  const int lane = threadIdx.x & 63;
  for (int32_t s0 = 0; s0 < b.sequences; s0 += 64) {
    const int32_t s = min(s0 + lane, b.sequences - 1);
    const Sequence q = sequence_of(b, s);
    const int32_t first = (q.begin >> SHIFT) + 2 * s, end = ((q.begin + q.count) >> SHIFT) + 2 * s + 2;
    const uint64_t in = __ballot(s0 + lane < b.sequences && at >= first && at < end);
    if (!in) continue;
    const int l = __ffsll((unsigned long long)in) - 1;
    return {s0 + l, at - __builtin_amdgcn_readlane(first, l),
            {__builtin_amdgcn_readlane(q.begin, l), __builtin_amdgcn_readlane(q.count, l), __builtin_amdgcn_readlane(q.length, l)}};
  }
  return {-1, 0, {0, 0, 0}};
}

}  // namespace hq
