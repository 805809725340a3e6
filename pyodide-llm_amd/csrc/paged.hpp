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

// Which sequence the `at`-th of all their items is in, count_of(s) items a sequence, and its place there: 64 sequences at a
// time, a lane each.  Every lane of the wave calls it; s is -1 where there are fewer items.
struct Place {
  int32_t s, rest;
};
template <typename Count>
HQ_DEV Place place_of(int32_t sequences, int32_t at, Count count_of) {
  const int lane = threadIdx.x & 63;
  for (int32_t s0 = 0; s0 < sequences; s0 += 64) {
    const int32_t mine = s0 + lane < sequences ? count_of(s0 + lane) : 0;
    int32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int32_t v = __shfl_up(upto, o, 64);
      if (lane >= o) upto += v;
    }
    const uint64_t past = __ballot(upto > at);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      return {s0 + l, __builtin_amdgcn_readlane(mine, l) - __builtin_amdgcn_readlane(upto, l) + at};
    }
    at -= __builtin_amdgcn_readlane(upto, 63);
  }
  return {-1, 0};
}

}  // namespace hq
