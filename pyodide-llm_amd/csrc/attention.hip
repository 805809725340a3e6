// attention.hip — attention of new tokens over the paged cache.
//
//   out = sum_j softmax_j(s_j) v_j,  s_j = scale q.k_j  (cap > 0: cap tanh(s_j / cap)), over the positions j that the token
//   sees: not past its own, within its window, on a page; zeros where there is none
//
// Rows.  The query heads that share a key/value head share its reads: a sequence's rows of that head are (token i, query head
// g), row i G + g.  A tile of 16 rows is one side of every matrix instruction, positions the other.
//
// Arithmetic.  An element of the cache, int8 or float16, is exact as a float16, so the products run on the float16 matrix
// instructions with float32 sums; what multiplies it, a query value or a weight, is held as two float16 (its rounding and the
// rounding of what is left: 22 bits), two instructions a product.  A row of queries is first scaled by the power of two that
// brings its largest |value| into [2^13, 2^14), so that the second half keeps its bits.  A position's scales multiply its score (up to
// 2^38 before) and its weight; the row's power of two is taken back before the key's scale multiplies (many rows: in steps with a scale
// of 2^64 and more, else with the rest of the score's factor), so that a score of ordinary size stays one whatever its factors' size.
//
// One pass over the positions holds a running maximum m and sum l of a softmax in base 2:
//   p_j = 2^(u_j - m + 7),  u_j = s_j log2(e),   l = sum p_j,   acc = sum (p_j vs_j 2^-E) v_j
// m, a whole number, moves only where a score passes it by 7 (p_j stays below 2^14), so that acc is seldom rescaled.
//
// A weight times its scale has to lie high in float16's range: below 1 its second half, of 2^-24 at least, holds less than 24 bits.
// While the scales of all positions loaded so far lie within 2^4 of each other, E is the largest one's exponent, the same for all
// rows: a row's largest p_j vs_j 2^-E is at least 2^2 then, and each is held to 2^-25 of the row's largest and better.  Where they
// lie further apart, or one is 0 (kApart), a row has an exponent of its own, from the largest p_j vs_j that it sees itself: what a row
// does not see, or gives no weight, takes nothing from it.  That costs a logarithm a weight more (apart_weights).
//
// Layout.  S^T = K Q^T and out^T = V^T P^T: rows are the instructions' columns, so that a lane holds one row's scores (lane % 16)
// and its maximum, sum and rescaling need no layout change, and the scores' registers are, with the keys taken in the right
// order, already the second product's operand.  V lies dimension by dimension in its pages and is its other operand as read.
#include <algorithm>
#include <climits>

#include "paged.hpp"

namespace hq {

namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kFewRows = 16;       // a tile's rows
constexpr float kRoom = 7.0f, kShift = 7.0f;  // how far a score may pass the maximum; p = 2^(u - m + kShift)
constexpr int kBand = 4;          // how far the exponents of the scales that share one E may lie apart
constexpr int kNoScale = -101;    // E before the first scale (a cache stores 2^-100 and more)
constexpr int kMostScale = 126;   // E's largest (2^-E is a float32)
constexpr int kApart = INT_MAX;   // in E's place: every row has its own
constexpr uint32_t kLargeScale = (uint32_t)(64 + 127) << 23;  // 2^64's bits
constexpr int kHeld = 14;         // powers of 2 that p and l lose at an item's end: acc is then no larger than the values' sum

// ---- rows, positions and shares ---------------------------------------------------------------------------------
struct Share {
  int32_t blocks;     // blocks that share the work
  int32_t rows;       // of a tile
  int32_t log;        // of a block's step's positions, to base 2
  int32_t group;      // query heads that share a key/value head
  uint32_t per;       // ceil(2^32 / group) (0: group is 1): the token of a row without a division
  int32_t tiles;      // there can be
  bool shared;        // whether an item can have more than one step
  // few_kernel: 0, or how many row tiles a sequence has a block a head for, which takes its tile's positions whole
  int32_t whole;
  int64_t parts;      // where in the workspace the shared items' parts are
  int64_t bytes;      // the workspace
  bool countable;     // whether its numbers fit their types
};

// what a kernel is called with
struct Call {
  Attention a;
  Cache c;
  Batch b;
  Share sh;
};

// row / group: exact while row group < 2^32, which the host makes sure of
HQ_DEV int32_t token_of(const Share &sh, int32_t row) { return sh.per ? (int32_t)__umulhi((uint32_t)row, sh.per) : row; }

// a tile's rows r0 .. r1 - 1 of a sequence, the positions from .. to - 1 that some of them see, and the steps that hold
// these: first .. first + steps - 1 (one at least: rows that see nothing are written too)
struct Tile {
  int32_t r0, r1, from, to, first, steps;
};
HQ_DEV Tile tile_of(const Call &k, const Sequence &q, int32_t rt) {
  Tile t;
  t.r0 = rt * k.sh.rows;
  t.r1 = min(t.r0 + k.sh.rows, q.count * k.sh.group);
  const int32_t before = q.length - q.count, reach = k.b.width << k.c.shift;
  t.to = min(max(before + token_of(k.sh, t.r1 - 1) + 1, 0), reach);
  t.from = k.a.window ? max(before + token_of(k.sh, t.r0) + 1 - k.a.window, 0) : 0;
  t.first = t.from >> k.sh.log;
  t.steps = max((int32_t)(((int64_t)t.to + (1 << k.sh.log) - 1) >> k.sh.log) - t.first, 1);
  return t;
}

// the steps of a sequence's tiles over all heads
HQ_DEV int32_t steps_of(const Call &k, const Sequence &q) {
  const int32_t rows = q.count * k.sh.group;
  int32_t n = 0;
  for (int32_t rt = 0; rt * kFewRows < rows; rt++) n += tile_of(k, q, rt).steps;
  return n * k.c.heads;
}

// All steps in a row: sequences, their row tiles, the heads, the steps.  Where a step is.
struct Spot {
  int32_t s, rt, h, step;
  Sequence q;
  Tile t;
};

// the sums up to each lane's value; INT32_MAX where they pass it (which sequences that overlap could make them)
template <int CTRL, int ROWS>
HQ_DEV int32_t plus_dpp(int32_t v) {
  const uint32_t w = (uint32_t)__builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
  return (int32_t)min((uint32_t)v + w, (uint32_t)INT32_MAX);
}
HQ_DEV int32_t wave_sums_of(int32_t v) {
  v = plus_dpp<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8: within a row of 16
  v = plus_dpp<0x112, 0xf>(v);
  v = plus_dpp<0x114, 0xf>(v);
  v = plus_dpp<0x118, 0xf>(v);
  v = plus_dpp<0x142, 0xa>(v);  // row_bcast 15: the row before, into rows 1 and 3
  return plus_dpp<0x143, 0xc>(v);  // row_bcast 31: the first half, into the second
}

HQ_DEV int32_t share_start(int32_t steps, int32_t block, int32_t blocks) {
  return (int32_t)((int64_t)steps * block / blocks);
}


// The block's share [u, end) of all steps, and where its first is (u < end): one look at every 64 sequences, two where there are
// more of them.
HQ_DEV void find_share(const Call &k, int32_t block, int32_t &all, int32_t &u, int32_t &end, Spot &o) {
  const int lane = threadIdx.x & 63;
  const int32_t n = k.b.sequences;
  Sequence q;
  int32_t mine, upto;
  const auto look = [&](int32_t s0) {  // at 64 sequences
    q = sequence_of(k.b, min(s0 + lane, n - 1));
    mine = s0 + lane < n ? steps_of(k, q) : 0;
    upto = wave_sums_of(mine);
  };
  uint32_t total = 0;
  for (int32_t s0 = 64; s0 < n; s0 += 64) {
    look(s0);
    total = min(total + (uint32_t)__builtin_amdgcn_readlane(upto, 63), (uint32_t)INT32_MAX);
  }
  look(0);
  total = min(total + (uint32_t)__builtin_amdgcn_readlane(upto, 63), (uint32_t)INT32_MAX);
  all = total < (uint32_t)INT32_MAX ? (int32_t)total : 0;
  u = share_start(all, block, k.sh.blocks), end = share_start(all, block + 1, k.sh.blocks);
  if (u >= end) return;
  int32_t rest = u, s0 = 0;
  uint64_t past;
  while (!(past = __ballot(upto > rest))) {  // (all steps are more than u: one chunk has it)
    rest -= __builtin_amdgcn_readlane(upto, 63);
    s0 += 64;
    look(s0);
  }
  const int l = __ffsll((unsigned long long)past) - 1;
  rest -= __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(mine, l);
  o.s = s0 + l, o.rt = 0;
  o.q.begin = __builtin_amdgcn_readlane(q.begin, l), o.q.count = __builtin_amdgcn_readlane(q.count, l);
  o.q.length = __builtin_amdgcn_readlane(q.length, l);
  for (;; o.rt++) {
    o.t = tile_of(k, o.q, o.rt);
    if (rest < o.t.steps * k.c.heads || (o.rt + 1) * kFewRows >= o.q.count * k.sh.group) break;
    rest -= o.t.steps * k.c.heads;
  }
  o.h = rest / o.t.steps;
  o.step = rest - o.h * o.t.steps;
}

// What join_kernel needs of the item whose start a block has and whose end it has not: its rows' first token and row there, how many
// rows, the head, the item's last step (-1: the block has no such item), and all steps
struct Tail {
  int32_t begin, r0, rows, h, last, all, pad[2];
};

// ---- arithmetic ---------------------------------------------------------------------------------------------------
HQ_DEV float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
HQ_DEV float power_of_2(int e) { return __int_as_float((e + 127) << 23); }
// v of lanes l and l ^ 32 (l ^ 16), in either order
HQ_DEV void pair32(float v, float &x, float &y) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  x = __uint_as_float(r[0]), y = __uint_as_float(r[1]);
}
HQ_DEV void pair16(float v, float &x, float &y) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  x = __uint_as_float(r[0]), y = __uint_as_float(r[1]);
}
HQ_DEV float max_pair(float v) {
  float x, y;
  pair32(v, x, y);
  return fmaxf(x, y);
}
HQ_DEV float sum_pair(float v) {
  float x, y;
  pair32(v, x, y);
  return x + y;
}
// the bits of the scales from which on, and below which, a scale is outside [2^low, 2^(high + 1))
HQ_DEV uint32_t above_bits(int high) { return (uint32_t)(high + 128) << 23; }
HQ_DEV uint32_t below_bits(int low) { return (uint32_t)(low + 127) << 23; }
// 2^e, for whatever e came of: 0 below its range
HQ_DEV float power_within(float e) { return __builtin_amdgcn_ldexpf(1.0f, (int)fminf(fmaxf(e, -300.0f), 100.0f)); }
// x 2^(from - to + e), from and to whole numbers or -infinity, in one step: neither factor alone need be a float32
HQ_DEV v4f shifted(v4f x, float from, float to, int e) {
  const int by = (int)fmaxf(from - to, -1000.0f) + e;
  return v4f{__builtin_amdgcn_ldexpf(x[0], by), __builtin_amdgcn_ldexpf(x[1], by), __builtin_amdgcn_ldexpf(x[2], by),
             __builtin_amdgcn_ldexpf(x[3], by)};
}

// over the lanes l, l ^ 16, l ^ 32, l ^ 48: a row's
HQ_DEV float max_row(float v) {
  float x, y;
  pair16(v, x, y);
  return max_pair(fmaxf(x, y));
}
HQ_DEV float sum_row(float v) {
  float x, y;
  pair16(v, x, y);
  return sum_pair(x + y);
}

// x, of which the compiler knows nothing: what a loop derives from it is formed in the loop, not held in scalar registers
HQ_DEV int32_t opaque(int32_t x) {
  asm volatile("" : "+s"(x));
  return x;
}

HQ_DEV float opaque(float x) {
  asm volatile("" : "+s"(x));
  return x;
}
HQ_DEV uint32_t opaque_lane(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

// A kernel's arguments, read anew: what only the start and the end of an item need is not held in scalar registers through the
// steps between (the kernel's one argument is a Call)
HQ_DEV const Call *call_again() {
  auto p = (const __attribute__((address_space(4))) Call *)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return (const Call *)p;
}

// tanh without a branch: 1 - 2 / (e^2|x| + 1), and below 0.55 its Taylor series to x^15 (the next term is 4e-8 of it)
HQ_DEV float tanh_of(float x, float bend, float twice) {  // bend 0.55, twice 2 log2(e): the caller's, of opaque()
  const float y = fabsf(x), z = x * x;
  const float big = 1.0f - 2.0f * __builtin_amdgcn_rcpf(exp2_of(y * twice) + 1.0f);
  float t = fmaf(z, -1.4558343870513182e-3f, 3.5921280365724810e-3f);
  t = fmaf(z, t, -8.8632355299021966e-3f);
  t = fmaf(z, t, 2.1869488536155203e-2f);
  t = fmaf(z, t, -5.3968253968253968e-2f);
  t = fmaf(z, t, 1.3333333333333333e-1f);
  t = fmaf(z, t, -3.3333333333333333e-1f);
  return y < bend ? fmaf(x * z, t, x) : copysignf(big, x);
}

// bits lo .. hi - 1 (of 0 .. 31)
HQ_DEV uint32_t bits_between(int32_t lo, int32_t hi) {
  const uint32_t below = (1u << min(max(lo, 0), 31)) - 1u, upto = (1u << min(max(hi, 0), 31)) - 1u;
  return upto & ~below;
}
// x where bit e of `bits` is set, else the float of the bits `other`
HQ_DEV float kept(float x, uint32_t bits, int e, uint32_t other) {
  const uint32_t m = (uint32_t)((int32_t)(bits << (31 - e)) >> 31);
  return __uint_as_float((__float_as_uint(x) & m) | (other & ~m));
}

// 4 int8 as 4 float16 (exact): 1024 + b + 128 is the half whose low byte is b with its sign flipped
HQ_DEV void widen4(uint32_t w, v2h &lo, v2h &hi) {
  const uint32_t x = w ^ 0x80808080u;
  const v2h bias = {(_Float16)-1152.0f, (_Float16)-1152.0f};
  lo = __builtin_bit_cast(v2h, perm(0x64646464u, x, 0x04010400u)) + bias;
  hi = __builtin_bit_cast(v2h, perm(0x64646464u, x, 0x04030402u)) + bias;
}
HQ_DEV v8h widen8(uint32_t w0, uint32_t w1) {
  v2h a, b, c, d;
  widen4(w0, a, b);
  widen4(w1, c, d);
  return v8h{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// the two float16 of 8 float32
HQ_DEV void halves_of(const float *x, v8h &hi, v8h &lo) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const v2f two = {x[j], x[j + 1]};
    const v2h h = __builtin_convertvector(two, v2h);
    // what is left of each: the mixed-precision multiply-add reads the float16 as it is
    v2f rest;
    float r0, r1;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r0) : "v"(h), "v"(two[0]));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r1) : "v"(h), "v"(two[1]));
    rest = v2f{r0, r1};
    const v2h l = __builtin_convertvector(rest, v2h);
    hi[j] = h[0], hi[j + 1] = h[1];
    lo[j] = l[0], lo[j + 1] = l[1];
  }
}

// A row's products (times 2^up) take 2^-up first, then a key's scale, so that nothing passes a float32 that the score itself does not
// pass: `first`, and the rest of the row's factor (with a large query's power of two: there the score does), in base 2 or a cap's.
HQ_DEV float first_of_large(int32_t up) { return power_of_2(-max(up, 0)); }
HQ_DEV float factor_of_large(int32_t up, float scale, float cap) {
  const float rowf = scale * power_of_2(-min(up, 0));
  return cap > 0.0f ? rowf / cap : rowf * kLog2e;
}

// A row whose positions' scales lie apart: its weights are p vs 2^-x, and top is log2 of the largest p vs so far, as p counts now
struct Apart {
  float top;
  int32_t x;
};
// ... where all shared E until now: whoever made m had p of 2^(kShift - 1) and more, and a scale of 2^(E - kBand) and more
HQ_DEV Apart apart_from(int exponent, float m) {
  return {m == -INFINITY || exponent == kNoScale ? -INFINITY : (float)(exponent + (int)kShift - 1 - kBand), exponent};
}
// N scores p (-infinity: not seen; times rowf in base 2) of such a row, whose scales vs are, enter: m, l and the row's exponent move, and
// its sums are to be multiplied by what comes back.  most: the row's largest score; row_most: the largest over the row's lanes.
template <int N, class RowMost>
HQ_DEV float apart_moves(const float (&p)[N], const float (&vs)[N], float rowf, float most, float &m, float &l, Apart &own, RowMost row_most) {
  const float was = m;
  if (most > m + kRoom) m = fmaxf(m, ceilf(most));
  const float drop = was == -INFINITY ? 0.0f : m - was, less = (m == -INFINITY ? 0.0f : m) - kShift;
  l *= exp2_of(-drop);
  float top = -INFINITY;
#pragma unroll
  for (int e = 0; e < N; e++)
    top = fmaxf(top, __builtin_fmaf(p[e], rowf, -less) + __builtin_amdgcn_logf(vs[e]));  // (log2; of 0 it is -infinity)
  own.top = fmaxf(own.top - drop, row_most(top));
  const float over = own.top - (float)own.x;
  const int x = own.x;
  // the largest weight to 2^7, and again only where it has left [1, 2^13]  (a top below -240: all weights are 0 in float32 anyway)
  if (own.top >= -240.0f && (over > 13.0f || over < 0.0f)) own.x = (int)rintf(own.top) - 7;
  return power_within((float)(x - own.x) - drop);
}
// ... and become weights p vs 2^-x
template <int N>
HQ_DEV void apart_weights(float (&p)[N], const float (&vs)[N], float rowf, float m, float &l, int32_t x) {
  const float less = (m == -INFINITY ? 0.0f : m) - kShift;
#pragma unroll
  for (int e = 0; e < N; e++) {
    p[e] = exp2_of(__builtin_fmaf(p[e], rowf, -less));
    l += p[e];
    p[e] = vs[e] == 0.0f ? 0.0f : __builtin_amdgcn_ldexpf(p[e], -x) * vs[e];
  }
}

// N consecutive elements of the cache (16 or 8)
template <int F16, int N>
struct Elements {
  static constexpr int kWords = N * (F16 ? 2 : 1) / 4;
  uint32_t w[kWords];
  HQ_DEV void load(const char *p) {
    if (kWords == 2) *(uint2 *)w = *(const uint2 *)p;
#pragma unroll
    for (int i = 0; i < kWords / 4; i++) ((uint4 *)w)[i] = ((const uint4 *)p)[i];
  }
  HQ_DEV v8h half(int i) const {  // elements 8 i .. 8 i + 7
    if (F16) return __builtin_bit_cast(v8h, ((const uint4 *)w)[i]);
    return widen8(w[2 * i], w[2 * i + 1]);
  }
};

// ---- a few rows: 16 a block, the positions split over its waves and over blocks ----------------------------------------
// Bound by the cache's bytes.  A token each of 32 sequences of 1200 to 8000 positions (32 query heads, 8 of keys, 128 values, int8:
// 320 MB) 70 us, one token over 131072 positions in float16 (545 MB) 100 us: 6.1 TB/s while all blocks run, where reading alone
// reaches 7.1, after 9 us until the first scores are there; 5 tokens each of 8 sequences of 4100 positions (71 MB, each read for
// two tiles) 28 us.  A second block's worth of loads a compute unit hides neither more nor less (half the positions a step: 78 us for
// the 72 that the first took then; twice the shares: 81 for 75), nor does another priority.  A wave takes 4 NP positions a step: lane l (m = l % 16, q = l / 16) holds 16 dimensions of a key
// at a time (row m of an instruction is the position NP (m / 4) + 4 t + m % 4 of its t-th 16, so that the lane's scores are those
// of the NP positions from NP q on), and of dimension 16 d + m the values of those NP positions.  Everything goes from
// memory to registers: the waves share nothing, and the next step's keys are on their way while this one's weights are formed.
// Steps of all (sequence, rows, head) are shared evenly among as many blocks as the GPU holds, whatever the lengths; what a
// block finds of an item that it does not have whole goes to `work` and join_kernel.
constexpr int few_np(int d, int f16) { return f16 || d <= 64 ? 8 : 16; }
constexpr int few_blocks_a_cu(int d, int) { return d <= 64 ? 3 : d <= 128 ? 2 : 1; }
template <int D, int F16>
__global__ __launch_bounds__(256, few_blocks_a_cu(D, F16)) void few_kernel(Call) {
  constexpr int ES = F16 ? 2 : 1, DB = D / 64, DT = D / 16, PITCH = D + 4, NP = few_np(D, F16), WK = 4 * NP, STEP = 4 * WK;
  __shared__ float sums[4][kFewRows][PITCH];
  __shared__ float stats[2][4][kFewRows];
  __shared__ Apart apart[4][kFewRows];
  __shared__ float firsts[4][kFewRows];  // first_of_large of the rows
  __shared__ int32_t parked[4][14];  // a wave's numbers that its steps do not need
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m16 = lane & 15, q4 = lane >> 4;
  int32_t u, end;
  Spot o;
  const Call *k = call_again();
  if (k->sh.whole) {
    o.s = blockIdx.x, o.rt = blockIdx.y, o.h = blockIdx.z, o.step = 0;
    o.q = wave_sequence_of(k->b, o.s);
    if (o.rt * kFewRows >= o.q.count * k->sh.group) return;
    o.t = tile_of(*k, o.q, o.rt);
    u = 0, end = o.t.steps;
  } else {
    int32_t all;
    find_share(*k, blockIdx.x, all, u, end, o);
    // (no tail yet: the share's last item says whether it has one)
    if (threadIdx.x == 0) ((Tail *)k->a.work)[blockIdx.x].all = all, ((Tail *)k->a.work)[blockIdx.x].last = -1;
    if (u >= end) return;
  }
  while (true) {
    const Call *call = call_again();
    const Attention &a = call->a;
    const Cache c = call->c;
    const Batch b = call->b;
    const Share sh = call->sh;
    const int32_t group = sh.group, reach = b.width << c.shift, mask = (1 << c.shift) - 1;
    const int32_t steps = min(o.t.steps - o.step, end - u);
    // ---- the rows' queries
    const int32_t row = o.t.r0 + m16, before = o.q.length - o.q.count;
    const bool live = row < o.t.r1;
    const int32_t token = token_of(sh, live ? row : o.t.r0), g = (live ? row : o.t.r0) - token * group;
    const float *x = (const float *)(a.q + (o.q.begin + token) * a.q_stride) + (int64_t)(o.h * group + g) * c.dim;
    float4 raw[DB][4];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int at = 64 * d + 16 * q4 + 4 * i;
        raw[d][i] = live && at < c.dim ? *(const float4 *)(x + at) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    // ---- the wave's positions: WK from base on, every STEP; their first loads are on their way before the queries are used
    int32_t base = (o.t.first + o.step) * STEP + WK * wave;
    const int32_t stop = min((o.t.first + o.step + steps) * STEP, o.t.to);
    while (base + WK <= o.t.from) base += STEP;
    const int32_t next0 = base + STEP < stop ? base + STEP : base;  // (the last step loads itself again)
    // the table's entries of the step's positions, for the keys' lanes (1) and the others' (2)
    const int32_t entry1 = entry_of(b, c, o.s, base + NP * (m16 >> 2));
    const int32_t entry2 = entry_of(b, c, o.s, base + NP * q4);
    // (Loads come back in order: an entry asked for after a step's values would be waited for with all of them, so that those of the
    // step after the next are asked for before this one's scores.)
    int32_t next = next0, next1 = entry_of(b, c, o.s, next + NP * (m16 >> 2)), next2 = entry_of(b, c, o.s, next + NP * q4);
    int32_t page2 = page_in(b, c, entry2, base + NP * q4);
    // Registers are loaded for the next step as soon as this one has used them: keys after the scores, scales after the weights,
    // values after their products, so that a step's bytes are always on their way.
    Elements<F16, 16> kk[NP / 4][DB];
    Elements<F16, NP> vv[DT];
    float ks[NP], vs[NP];
    const auto load_keys = [&](int32_t at, int32_t page) {
      const int64_t vec = vectors_of(c, max(page, 0), o.h) + ((at + NP * (m16 >> 2)) & mask) + (m16 & 3);
      const int32_t dim = opaque(c.dim);
      const char *p = c.k + vec * dim * ES;
#pragma unroll
      for (int t = 0; t < NP / 4; t++)
#pragma unroll
        for (int d = 0; d < DB; d++)
          // (dimensions past dim: the row's first, times zeros)
          kk[t][d].load(p + (t * 4 * dim + (64 * d + 16 * q4 < dim ? 64 * d + 16 * q4 : 0)) * ES);
    };
    // the lane's NP positions from at + NP q4 on, on `page`
    const auto load_scales = [&](int32_t at, int32_t page) {
      const int64_t vec = vectors_of(c, max(page, 0), o.h) + ((at + NP * q4) & mask);
#pragma unroll
      for (int i = 0; i < NP / 4; i++) {
        *(float4 *)(ks + 4 * i) = *(const float4 *)(c.ks + vec + 4 * i);
        *(float4 *)(vs + 4 * i) = *(const float4 *)(c.vs + vec + 4 * i);
      }
    };
    const auto values_at = [&](int32_t at, int32_t page) {
      return c.v + (vectors_of(c, max(page, 0), o.h) * c.dim + (m16 << c.shift) + ((at + NP * q4) & mask)) * ES;
    };
    const auto value_row = [&](int d, int32_t dim, int32_t shift) { return (min(d * 16, dim - 16) << shift) * ES; };  // (past dim: the last again)
    if (base < stop) {
      load_keys(base, page_in(b, c, entry1, base + NP * (m16 >> 2)));
      load_scales(base, page2);
      const char *p = values_at(base, page2);
#pragma unroll
      for (int d = 0; d < DT; d++) vv[d].load(p + value_row(d, c.dim, c.shift));
    }
    v8h qh[DB][2], ql[DB][2];
    float rowf;
    {
      float most = 0.0f;
#pragma unroll
      for (int d = 0; d < DB; d++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          most = fmaxf(fmaxf(most, fmaxf(fabsf(raw[d][i].x), fabsf(raw[d][i].y))), fmaxf(fabsf(raw[d][i].z), fabsf(raw[d][i].w)));
      most = max_row(most);
      const int up = most > 0.0f ? min(140 - (int)(__float_as_uint(most) >> 23), 126) : 0;
      const float by = power_of_2(up);
      firsts[wave][m16] = first_of_large(up), rowf = factor_of_large(up, a.scale, a.cap);
#pragma unroll
      for (int d = 0; d < DB; d++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const float4 e0 = raw[d][2 * i], e1 = raw[d][2 * i + 1];
          const float e[8] = {e0.x * by, e0.y * by, e0.z * by, e0.w * by, e1.x * by, e1.y * by, e1.z * by, e1.w * by};
          halves_of(e, qh[d][i], ql[d][i]);
        }
    }
    // a score is its product times first, its key's scale and rowf, in base 2; with a cap that is the tanh's argument
    const float cap = a.cap;
    const int32_t sees = before + token + 1;
    const int32_t to = min(sees, reach), from = a.window ? sees - a.window : 0;  // the lane's row's own positions
    // the positions that every row sees lie in [every_from, every_to)
    const int32_t every_to = min(before + token_of(sh, o.t.r0) + 1, reach);
    const int32_t every_from = a.window ? before + token_of(sh, o.t.r1 - 1) + 1 - a.window : 0;
    {
      const int32_t now[14] = {u, end, o.rt, o.step, o.h, steps, o.t.steps, o.t.r0, o.t.r1, o.q.begin, o.q.count, o.q.length, o.t.first, 0};
#pragma unroll
      for (int i = 0; i < 13; i++) parked[wave][i] = now[i];
    }
    float m = -INFINITY, l = 0.0f;
    int exponent = kNoScale, low = kNoScale;  // the largest and the smallest scale's
    v4f acc[DT] = {};
    if (base < stop) {
      while (true) {
        const bool more = base + STEP < stop;
        const int32_t after_next = next + STEP < stop ? next + STEP : next;
        const int32_t after1 = entry_of(b, c, o.s, after_next + NP * (m16 >> 2)), after2 = entry_of(b, c, o.s, after_next + NP * q4);
        // ---- scores
        v4f s[NP / 4] = {};
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
          for (int i = 0; i < 2; i++)
#pragma unroll
            for (int t = 0; t < NP / 4; t++) {
              const v8h k8 = kk[t][d].half(i);
              s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, ql[d][i], s[t], 0, 0, 0);
              s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, qh[d][i], s[t], 0, 0, 0);
            }
        load_keys(next, page_in(b, c, next1, next + NP * (m16 >> 2)));
        const int32_t next_page2 = page_in(b, c, next2, next + NP * q4);
        float p[NP];
        float by_row = rowf;
        const float first = firsts[wave][m16];
#pragma unroll
        for (int e = 0; e < NP; e++) p[e] = s[e >> 2][e & 3] * first * ks[e];
        if (cap > 0.0f) {
          const float bend = opaque(0.55f), twice = opaque(2.0f * kLog2e);
#pragma unroll
          for (int e = 0; e < NP; e++) p[e] = cap * kLog2e * tanh_of(p[e] * by_row, bend, twice);
          by_row = 1.0f;
        }
        const bool edge = base + WK > every_to || base < every_from || __any(page2 < 0);
        uint32_t seen = ~0u;
        if (edge) {
          // what the row does not see has no score; what no row sees may hold anything: its scale becomes one of the others', its values 0
          const int32_t at = base + NP * q4;
          seen = page2 < 0 ? 0u : bits_between(from - at, to - at);
          const uint32_t any = page2 < 0 ? 0u : bits_between(o.t.from - at, o.t.to - at);
          const uint32_t other = (uint32_t)((exponent == kApart ? 0 : exponent) + 127) << 23;
#pragma unroll
          for (int e = 0; e < NP; e++) {
            p[e] = kept(p[e], seen, e, 0xff800000u);
            vs[e] = kept(vs[e], any, e, other);
          }
          if (F16) {
#pragma unroll
            for (int j = 0; j < NP / 2; j++) {
              const uint32_t two = any >> (2 * j), keep = (two & 1u) * 0xffffu | (two & 2u) * 0x7fff8000u;
#pragma unroll
              for (int d = 0; d < DT; d++) vv[d].w[F16 ? j : 0] &= keep;
            }
          }
        }
        // ---- the running maximum and the scales' exponent
        float most = p[0];
        uint32_t most_scale = __float_as_uint(vs[0]), least_scale = most_scale;
#pragma unroll
        for (int e = 1; e < NP; e++) {
          most = fmaxf(most, p[e]);
          most_scale = max(most_scale, __float_as_uint(vs[e])), least_scale = min(least_scale, __float_as_uint(vs[e]));
        }
        most = max_row(most) * by_row;
        if (exponent != kApart && __any(most_scale >= above_bits(exponent) || least_scale < below_bits(low))) {
          // a scale outside those so far (or a NaN, which says nothing)
          float high = 0.0f, least = INFINITY;
#pragma unroll
          for (int e = 0; e < NP; e++) high = fmaxf(high, vs[e]), least = fminf(least, vs[e]);
          high = max_row(high), least = -max_row(-least);
          if (least <= high) {
            const int h1 = max(__builtin_amdgcn_readfirstlane((int)(__float_as_uint(high) >> 23) - 127), exponent);
            const int l0 = __builtin_amdgcn_readfirstlane((int)(__float_as_uint(least) >> 23) - 127);
            const int l1 = exponent == kNoScale ? l0 : min(l0, low);
            if (h1 - l1 <= kBand && h1 <= kMostScale) {
              if (h1 > exponent) {
                const float by = power_of_2(max(exponent - h1, -126));
#pragma unroll
                for (int d = 0; d < DT; d++) acc[d] *= by;
              }
              exponent = h1, low = l1;
            } else {
              apart[wave][m16] = apart_from(exponent, m);
              exponent = kApart;
            }
          }
        }
        if (exponent == kApart) {
          Apart own = apart[wave][m16];
          const float rescale = apart_moves(p, vs, by_row, most, m, l, own, [](float v) { return max_row(v); });
          apart[wave][m16] = own;
          if (__any(rescale != 1.0f)) {
#pragma unroll
            for (int d = 0; d < DT; d++) acc[d] *= rescale;
          }
          apart_weights(p, vs, by_row, m, l, own.x);
        } else {
          if (__any(most > m + kRoom)) {  // (the first that is seen too: m is -infinity before it)
            const float m1 = fmaxf(m, ceilf(most));
            const float alpha = m1 == -INFINITY ? 0.0f : exp2_of(m - m1);
            m = m1;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; d++) acc[d] *= alpha;
          }
          const float less = (m == -INFINITY ? 0.0f : m) - kShift, by = power_of_2(-exponent);
#pragma unroll
          for (int e = 0; e < NP; e++) {
            p[e] = exp2_of(__builtin_fmaf(p[e], by_row, -less));
            l += p[e];
            p[e] = p[e] * (vs[e] * by);
          }
        }
        if (edge) {
#pragma unroll
          for (int e = 0; e < NP; e++)
            p[e] = kept(p[e], seen, e, 0u);  // (a NaN scale that others see)
        }
        load_scales(next, next_page2);
        // ---- out += weights times values
        v8h ph[NP / 8], pl[NP / 8];
#pragma unroll
        for (int i = 0; i < NP / 8; i++) halves_of(p + 8 * i, ph[i], pl[i]);
        const char *v_next = values_at(next, next_page2);
        const int32_t dim = opaque(c.dim), shift = opaque(c.shift);
#pragma unroll
        for (int d = 0; d < DT; d++) {
          v8h v8[NP / 8];
#pragma unroll
          for (int i = 0; i < NP / 8; i++) v8[i] = vv[d].half(i);
#pragma unroll
          for (int i = 0; i < NP / 8; i++) {
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8[i], pl[i], acc[d], 0, 0, 0);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8[i], ph[i], acc[d], 0, 0, 0);
          }
          vv[d].load(v_next + value_row(d, dim, shift));
        }
        if (!more) break;
        base = next, page2 = next_page2;
        next = after_next, next1 = after1, next2 = after2;
      }
    }
    l = __builtin_amdgcn_ldexpf(sum_row(l), -kHeld);
    const int own_exponent = (exponent == kApart ? apart[wave][m16].x : exponent) - kHeld;
    // ---- the four waves together
    const Call *after = call_again();
    const int32_t heads = after->c.heads, shared = after->sh.group;
    int32_t back[13];
#pragma unroll
    for (int i = 0; i < 13; i++) back[i] = __builtin_amdgcn_readfirstlane(parked[wave][i]);
    u = back[0], end = back[1], o.rt = back[2], o.step = back[3], o.h = back[4], o.t.steps = back[6], o.t.r0 = back[7];
    o.t.r1 = back[8], o.q.begin = back[9], o.q.count = back[10], o.q.length = back[11], o.t.first = back[12];
    const int32_t done = back[5];
    const bool whole = done == o.t.steps;
    if (q4 == 0) stats[0][wave][m16] = m, stats[1][wave][m16] = l;
    __syncthreads();
    const float m0 = stats[0][0][m16], m1 = stats[0][1][m16], m2 = stats[0][2][m16], m3 = stats[0][3][m16];
    const float mm = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)), ref = mm == -INFINITY ? 0.0f : mm;
    const float ll = stats[1][0][m16] * exp2_of(m0 - ref) + stats[1][1][m16] * exp2_of(m1 - ref) +
                     stats[1][2][m16] * exp2_of(m2 - ref) + stats[1][3][m16] * exp2_of(m3 - ref);
#pragma unroll
    for (int d = 0; d < DT; d++) {
      *(v4f *)&sums[wave][m16][d * 16 + q4 * 4] = shifted(acc[d], m, ref, own_exponent);
    }
    __syncthreads();
    const int32_t slot = o.step > 0 ? 0 : 1;
    float *part = (float *)(after->a.work + after->sh.parts) + (int64_t)(blockIdx.x * 2 + slot) * kFewRows * (D + 2);
    if (!whole && threadIdx.x < kFewRows) part[m16 * 2] = mm, part[m16 * 2 + 1] = ll;
    for (int i = threadIdx.x; i < kFewRows * (D / 4); i += 256) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      if (o.t.r0 + r >= o.t.r1) break;
      v4f v = *(v4f *)&sums[0][r][d] + *(v4f *)&sums[1][r][d] + *(v4f *)&sums[2][r][d] + *(v4f *)&sums[3][r][d];
      if (!whole) {
        *(v4f *)(part + kFewRows * 2 + r * D + d) = v;
      } else if (d < after->c.dim) {
        // the row's sum, from the stats of its column
        const float a0 = stats[0][0][r], a1 = stats[0][1][r], a2 = stats[0][2][r], a3 = stats[0][3][r];
        const float am = fmaxf(fmaxf(a0, a1), fmaxf(a2, a3)), ar = am == -INFINITY ? 0.0f : am;
        const float sum = stats[1][0][r] * exp2_of(a0 - ar) + stats[1][1][r] * exp2_of(a1 - ar) +
                          stats[1][2][r] * exp2_of(a2 - ar) + stats[1][3][r] * exp2_of(a3 - ar);
        const int32_t i0 = token_of(after->sh, o.t.r0 + r), gg = o.t.r0 + r - i0 * shared;
        v = sum != 0.0f ? v / sum : v4f{0.f, 0.f, 0.f, 0.f};
        *(v4f *)(after->a.out + (o.q.begin + i0) * after->a.out_stride + ((int64_t)(o.h * shared + gg) * after->c.dim + d) * 4) = v;
      }
    }
    u += done;
    if (after->sh.whole) {
      // (a sequence may have more tiles than it has blocks)
      o.rt += after->sh.whole;
      if (o.rt * kFewRows >= o.q.count * shared) break;
      __syncthreads();
      o.t = tile_of(*after, o.q, o.rt);
      u = 0, end = o.t.steps;
      continue;
    }
    if (u >= end) {
      if (threadIdx.x == 0) {
        Tail &tail = ((Tail *)after->a.work)[blockIdx.x];
        tail.begin = o.q.begin, tail.r0 = o.t.r0, tail.rows = o.t.r1 - o.t.r0, tail.h = o.h;
        tail.last = o.step == 0 && !whole ? end - done + o.t.steps - 1 : -1;
      }
      break;
    }
    __syncthreads();
    // ---- the next item: the next head, row tile or sequence (one more step is left, so there is one)
    o.step = 0;
    if (++o.h == heads) {
      o.h = 0, o.rt++;
      if (o.rt * kFewRows >= o.q.count * shared) {
        o.rt = 0;
        do {
          if (++o.s >= after->b.sequences) return;
          o.q = wave_sequence_of(after->b, o.s);
        } while (!o.q.count);
      }
      o.t = tile_of(*after, o.q, o.rt);
    }
  }
}

// The items that blocks share: the block whose share an item starts in (and does not end in) has its rows' parts joined here, a
// thread 4 values of a row over every SLICES-th part, the slices together in the end: the largest of the maxima so far, their sum.
// A chain of loads, so that four parts are on their way at once, and where an item has few rows, it has many parts, which are
// sliced: one token over 131072 positions (4 rows an item, 64 parts) 10.0 us in one slice, 8.6 in 4, 8.0 in 8, which cost short
// items 1 us; 8 sequences of 5 tokens (20 rows) 5.1 us in one slice, 7.1 in 4.  A block's parts are two of (rows' (m, l) pairs,
// rows of D): what its first item's end and its last item's start gave.  edge: the shares' edges (NULL: even shares of all steps).
constexpr int kMostBlocks = 4096;  // of a launch that shares its items
template <int D, int SLICES>
__global__ __launch_bounds__(256) void join_kernel(Call k, const int32_t *edge) {
  constexpr int COLS = D / 4, ROWS = 256 / COLS / SLICES;  // rows at a time
  __shared__ int32_t of[kMostBlocks];  // the blocks that have a part
  __shared__ int32_t found;
  __shared__ v4f sums[SLICES > 1 ? 256 : 1];
  __shared__ float2 stats[SLICES > 1 ? 256 : 1];
  const Tail t = ((const Tail *)k.a.work)[blockIdx.x];
  if (t.last < 0 || (int32_t)blockIdx.y * ROWS >= t.rows) return;
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    const auto start_of = [&](int32_t i) { return edge ? edge[i] : share_start(t.all, i, k.sh.blocks); };
    int32_t n = 0;
    for (int32_t b0 = blockIdx.x; b0 < k.sh.blocks; b0 += 64) {
      const int32_t mine = b0 + lane, start = mine < k.sh.blocks ? start_of(mine) : INT32_MAX;
      const bool in = start <= t.last, some = in && start_of(mine + 1) > start;  // (a share may have no step)
      const uint64_t with = __ballot(some);
      if (some) of[n + __popcll(with & (((uint64_t)1 << lane) - 1))] = 2 * mine + (mine == (int32_t)blockIdx.x ? 1 : 0);
      n += __popcll(with);
      if (!__all(in)) break;
    }
    if (lane == 0) found = n;
  }
  __syncthreads();
  const int n = found, col = threadIdx.x % COLS * 4, slice = threadIdx.x / COLS % SLICES;
  const int64_t size = (int64_t)k.sh.rows * (D + 2);
  const float *parts = (const float *)(k.a.work + k.sh.parts);
  for (int r0 = blockIdx.y * ROWS; r0 < t.rows; r0 += ROWS * gridDim.y) {
    const int r = r0 + threadIdx.x / (COLS * SLICES), row = min(r, t.rows - 1);
    float m = -INFINITY, l = 0.0f;
    v4f acc = {};
    for (int i0 = slice; i0 < n; i0 += 4 * SLICES) {
      float2 ml[4];
      v4f v[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float *part = parts + of[min(i0 + SLICES * j, n - 1)] * size;
        ml[j] = *(const float2 *)(part + 2 * row);
        v[j] = *(const v4f *)(part + 2 * k.sh.rows + row * D + col);
      }
      float most = m;
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (i0 + SLICES * j < n) most = fmaxf(most, ml[j].x);
      // (a part's sums can be as large as its weight is small: they are moved in one step)
      const float ref = most == -INFINITY ? 0.0f : most;
      l *= exp2_of(m - ref), acc = shifted(acc, m, ref, 0);
      m = most;
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (i0 + SLICES * j < n) {
          l += ml[j].y * exp2_of(ml[j].x - ref);
          acc += shifted(v[j], ml[j].x, ref, 0);
        }
    }
    if (SLICES > 1) {
      __syncthreads();  // (the rows before)
      sums[threadIdx.x] = acc, stats[threadIdx.x] = make_float2(m, l);
      __syncthreads();
      if (slice) continue;
      for (int i = 1; i < SLICES; i++) m = fmaxf(m, stats[threadIdx.x + COLS * i].x);
      const float ref = m == -INFINITY ? 0.0f : m;
      l = 0.0f, acc = v4f{};
      for (int i = 0; i < SLICES; i++) {
        const float2 other = stats[threadIdx.x + COLS * i];
        l += other.y * exp2_of(other.x - ref);
        acc += shifted(sums[threadIdx.x + COLS * i], other.x, ref, 0);
      }
    }
    if (r >= t.rows) continue;
    const int32_t i0 = token_of(k.sh, t.r0 + r), g = t.r0 + r - i0 * k.sh.group;
    float *out = (float *)(k.a.out + (t.begin + i0) * k.a.out_stride) + (int64_t)(t.h * k.sh.group + g) * k.c.dim;
    if (col < k.c.dim) *(v4f *)(out + col) = l != 0.0f ? acc / l : v4f{0.f, 0.f, 0.f, 0.f};
  }
}

// ---- prompts: 128 rows a block, 32 a wave, over 64 positions a step -----------------------------------------------------
// Bound by the matrix cores and the softmax's vector instructions, whose times add up here.  2048 tokens behind 6144 (32 query heads, 8
// of keys, 128 values, int8): a call takes 520 us back to back, this kernel all of it but the plan's and the join's 22 (579 us in a
// profiled run, whose clock is lower): 480 TFLOP/s of the formula's products, twice that of the instructions' (a library's float16 matrix
// product reaches 1271).  A batch of prompts with heads of 64 float16 values: a call takes 94 us, 224 TFLOP/s (85 us of this kernel in a
// profiled run).  Where value scales lie apart in every step: 654 and 112 us for 529 and 93 in the same run.
//
// A wave's 32 rows are the columns of 32 x 32 x 16 instructions: lane l (row l % 32, h = l / 32) holds of the step's scores those of the
// positions 32 k + 16 c + 8 h + e (e < 8), which are its operand of the second product for the positions 32 k + 16 c .. + 15.  The block's keys and values go through LDS as float16, two steps' room, each element widened
// once a block; keys in rows whose number has bits 2 and 3 swapped (the instruction's row 8 j + 4 h + i is position
// 16 (j / 2) + 8 h + 4 (j % 2) + i), 16-byte chunks XORed with the row so that 8 lanes read 8 bank quads.
//
// Which block does what is worked out once a call (plan_kernel): steps of all (sequence, head, row tile) in a row, shared evenly,
// a share's end moved to an item's end that is near, so that few items are shared and their parts joined (join_kernel).
constexpr int kRows = 128, kPositions = 64, kAnyLarge = 16;

// where in the row of all steps: sequence, row tile, head and step of the item
struct Start {
  int32_t s, k, h, step;  // (k: the place of the row tile in its sequence's order)
};
// A sequence's row tiles in order: the first, the last, the second, the last but one ...  Later rows see more positions, so that two
// neighbours together take about the same time and a share of one tile's size ends near every second tile's end.
HQ_DEV int32_t tile_at(int32_t k, int32_t tiles) { return k & 1 ? tiles - 1 - (k >> 1) : k >> 1; }
// the plan, in a call's workspace: the shares' tails, their edges (blocks + 1 numbers), the place of each share's first step, and the
// steps of one head: of all sequences up to s, of the tiles up to a tile of its sequence (tiles[s] of them from base[s] on)
struct Plan {
  Tail *tail;
  int32_t *edge;
  Start *first;
  int32_t *upto, *base, *tiles, *tile;
};
__host__ __device__ inline Plan plan_of(char *work, int32_t blocks, int32_t sequences) {
  Plan p;
  p.tail = (Tail *)work;
  p.first = (Start *)(p.tail + blocks);
  p.edge = (int32_t *)(p.first + blocks);
  p.upto = p.edge + blocks + 1;
  p.base = p.upto + sequences;
  p.tiles = p.base + sequences;
  p.tile = p.tiles + sequences;
  return p;
}
int64_t plan_bytes(int64_t blocks, int64_t sequences, int64_t tiles) {
  return blocks * (int64_t)(sizeof(Tail) + sizeof(Start)) + (blocks + 1 + 3 * sequences + tiles) * 4;
}

// inclusive sums over a block of 1024 threads
HQ_DEV int64_t sum_upto(int32_t each, int64_t *wave_sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t v = wave_sums_of(each);
  __syncthreads();
  if (lane == 63) wave_sums[wave] = v;
  __syncthreads();
  for (int i = 0; i < wave; i++) v += wave_sums[i];
  return v;
}

constexpr int kPlanSequences = 1024, kPlanTiles = 4096;
__global__ __launch_bounds__(1024) void plan_kernel(Call k) {
  const Share &sh = k.sh;
  const Cache &c = k.c;
  const Batch &b = k.b;
  __shared__ int64_t wave_sums[16], carry;
  __shared__ int32_t near_upto[kPlanSequences], near_base[kPlanSequences], near_tiles[kPlanSequences], near_tile[kPlanTiles];
  Plan p = plan_of(k.a.work, sh.blocks, b.sequences);
  const int32_t group = sh.group, n = b.sequences;
  // the sums, which only this kernel reads, in LDS where they fit: the searches below are chains of loads
  if (n <= kPlanSequences && sh.tiles <= kPlanTiles) p.upto = near_upto, p.base = near_base, p.tiles = near_tiles, p.tile = near_tile;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // a sequence's first tile
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  for (int32_t s0 = 0; s0 < n; s0 += 1024) {
    const int32_t s = s0 + threadIdx.x;
    const int32_t tiles = s < n ? (sequence_of(b, s).count * group + sh.rows - 1) / sh.rows : 0;
    const int64_t upto = sum_upto(tiles, wave_sums) + carry;
    // (sequences that overlap could have more tiles than there is room for: those past it have none)
    if (s < n) p.base[s] = (int32_t)upto - tiles, p.tiles[s] = upto <= sh.tiles ? tiles : 0;
    __syncthreads();
    if (threadIdx.x == 1023) carry = upto;
    __syncthreads();
  }
  // a tile's steps and those of the sequence's before it, a wave a sequence
  for (int32_t s = wave; s < n; s += 16) {
    const Sequence q = sequence_of(b, s);
    const int32_t tiles = p.tiles[s];
    int32_t before = 0;
    for (int32_t t0 = 0; t0 < tiles; t0 += 64) {
      const int32_t v = wave_sums_of(t0 + lane < tiles ? tile_of(k, q, tile_at(t0 + lane, tiles)).steps : 0);
      if (t0 + lane < tiles) p.tile[p.base[s] + t0 + lane] = before + v;
      before += __builtin_amdgcn_readlane(v, 63);
    }
    if (lane == 0) p.upto[s] = before;
  }
  __syncthreads();
  // the sequences' steps up to each
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  for (int32_t s0 = 0; s0 < n; s0 += 1024) {
    const int32_t s = s0 + threadIdx.x;
    const int64_t upto = sum_upto(s < n ? p.upto[s] : 0, wave_sums) + carry;
    if (s < n) p.upto[s] = (int32_t)upto;
    __syncthreads();
    if (threadIdx.x == 1023) carry = upto;
    __syncthreads();
  }
  // An edge that near to an item's is moved there: what a block begins and does not end costs it more than the steps.  A 32nd of a
  // share, and a step where shares have more than one and a half (heads of 128 int8, 64 tokens behind 4000 positions, two steps a
  // share: 97 us without it, 71 with it; shares of one step, 512 tokens: 48 as they are, 53 as two steps)
  const int32_t all = (int32_t)carry * c.heads;
  const int32_t near = max(all / sh.blocks / 32, all > sh.blocks + sh.blocks / 2 ? 1 : 0);
  // where step `at` is; first and size: its item's
  const auto find = [&](int32_t at, int32_t &first, int32_t &size) {
    int32_t lo = 0, hi = n - 1;
    while (lo < hi) {  // the first sequence whose steps reach past it
      const int32_t mid = (lo + hi) >> 1;
      if (p.upto[mid] * c.heads > at) hi = mid;
      else lo = mid + 1;
    }
    Start o;
    o.s = lo;
    const int32_t before = lo ? p.upto[lo - 1] : 0, total = p.upto[lo] - before;
    int32_t rest = at - before * c.heads;
    o.h = rest / total;
    rest -= o.h * total;
    const int32_t *tile = p.tile + p.base[lo];
    int32_t t0 = 0, t1 = p.tiles[lo] - 1;
    while (t0 < t1) {
      const int32_t mid = (t0 + t1) >> 1;
      if (tile[mid] > rest) t1 = mid;
      else t0 = mid + 1;
    }
    const int32_t begin = t0 ? tile[t0 - 1] : 0;
    o.k = t0;
    o.step = rest - begin;
    first = at - o.step;
    size = tile[t0] - begin;
    return o;
  };
  for (int32_t i = threadIdx.x; i <= sh.blocks; i += 1024) {
    int32_t at = share_start(all, i, sh.blocks), first, size;
    if (at < all) {
      Start o = find(at, first, size);
      if (at - first <= near) {
        at = first, o.step = 0;
      } else if (first + size - at <= near) {
        at = first + size;
        if (at < all) o = find(at, first, size);
      }
      if (i < sh.blocks) p.first[i] = o;
    }
    p.edge[i] = at;
    if (i < sh.blocks) p.tail[i].last = -1;
  }
}

// the largest of a wave's numbers
HQ_DEV uint32_t wave_max(uint32_t m) {
  m = max8(m);
  m = max(m, (uint32_t)dpp<0x140>((int32_t)m));  // row_mirror
  auto r = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  m = max(r[0], r[1]);
  r = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  return __builtin_amdgcn_readfirstlane(max(r[0], r[1]));
}

HQ_DEV uint32_t key_row(uint32_t r) { return (r & ~12u) | ((r & 4u) << 1) | ((r & 8u) >> 1); }  // bits 2 and 3 swapped

typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int rows_blocks_a_cu(int d) { return d <= 64 ? 3 : d <= 128 ? 2 : 1; }
// WHOLE: a step's 64 positions are on one page (pages of 64 and more), whose addresses the scalar unit then forms: a 2048-token chunk
// 626 -> 611 us.  (For the other dims it does not fit the scalar registers.)
template <int D, int F16, bool WHOLE>
__global__ __launch_bounds__(256, rows_blocks_a_cu(D)) void rows_kernel(Call) {
  constexpr int ES = F16 ? 2 : 1, KS = D / 16, DT = D / 32;
  constexpr int PIECES = D * ES / 64;  // 16-byte pieces of keys, and of values, a thread stages
  constexpr bool BOTH = D <= 128;      // whether the registers hold a step's keys and values at once
  __shared__ __align__(16) char keys[2][kPositions * D * 2];
  __shared__ __align__(16) char values[2][kPositions * D * 2];
  __shared__ __align__(16) float scales[2][2][kPositions];  // of keys, of values (times 2^-exponent, or as they are: kApart)
  __shared__ int32_t info[2][2];  // the exponent or kApart; a bit for each 16 positions on a page, and one where a key's scale is large
  __shared__ Apart apart[kRows];
  __shared__ int32_t ups[kRows];  // the power of two that a row's queries are multiplied by
  __shared__ int32_t parked[4][10];                         // a wave's numbers that its steps do not need
  // neighbouring shares on one XCD (blocks go round its 8): they read the same keys and values
  int32_t block, u, end;
  Start o;
  {
    const Call *k = call_again();
    const int32_t blocks = k->sh.blocks;
    block = blocks % 8 ? blockIdx.x : (blockIdx.x % 8) * (blocks / 8) + blockIdx.x / 8;
    const Plan p = plan_of(k->a.work, blocks, k->b.sequences);
    u = __builtin_amdgcn_readfirstlane(p.edge[block]);
    end = __builtin_amdgcn_readfirstlane(p.edge[block + 1]);
    if (u >= end) return;
    o.s = __builtin_amdgcn_readfirstlane(p.first[block].s), o.k = __builtin_amdgcn_readfirstlane(p.first[block].k);
    o.h = __builtin_amdgcn_readfirstlane(p.first[block].h), o.step = __builtin_amdgcn_readfirstlane(p.first[block].step);
  }
  while (true) {
    const Call *call = call_again();
    const Attention &a = call->a;
    const Cache c = call->c;
    const Batch b = call->b;
    const Share sh = call->sh;
    const int32_t group = sh.group, reach = b.width << c.shift, mask = (1 << c.shift) - 1;
    const Sequence q = wave_sequence_of(b, o.s);
    const int32_t tiles = (q.count * group + kRows - 1) / kRows;
    const Tile tile = tile_of(*call, q, tile_at(o.k, tiles));
    const int32_t steps = min(tile.steps - o.step, end - u);
    // ---- the rows' queries
    const int thread = opaque_lane(threadIdx.x), m32 = thread & 31, h2 = (thread >> 5) & 1;
    const int wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const int32_t r0 = tile.r0 + 32 * wave, r1 = min(r0 + 32, tile.r1), before = q.length - q.count;
    const bool some = r0 < tile.r1, live = r0 + m32 < r1;
    const int32_t row = live ? r0 + m32 : tile.r0;
    const int32_t token = token_of(sh, row), g = row - token * group;
    const int32_t sees = before + token + 1;
    const int32_t to = min(sees, reach), from = a.window ? sees - a.window : 0;  // the lane's row's own positions
    // what some of the wave's rows see lies before any_to, what all of them see in [every_from, every_to)
    const int32_t any_to = some ? min(before + token_of(sh, r1 - 1) + 1, reach) : 0;
    const int32_t every_to = some ? min(before + token_of(sh, r0) + 1, reach) : 0;
    const int32_t every_from = some && a.window ? before + token_of(sh, r1 - 1) + 1 - a.window : 0;
    v8h qh[KS], ql[KS];
    float rowf;
    {
      const float *x = (const float *)(a.q + (q.begin + token) * a.q_stride) + (int64_t)(o.h * group + g) * c.dim;
      float most = 0.0f;
      for (int i = 8 * h2; i < c.dim; i += 16) {
        const float4 e0 = *(const float4 *)(x + i), e1 = *(const float4 *)(x + i + 4);
        most = fmaxf(fmaxf(most, fmaxf(fabsf(e0.x), fabsf(e0.y))), fmaxf(fabsf(e0.z), fabsf(e0.w)));
        most = fmaxf(fmaxf(most, fmaxf(fabsf(e1.x), fabsf(e1.y))), fmaxf(fabsf(e1.z), fabsf(e1.w)));
      }
      most = max_pair(most);
      const int up = most > 0.0f ? min(140 - (int)(__float_as_uint(most) >> 23), 126) : 0;
      const float by = live ? power_of_2(up) : 0.0f;
      rowf = a.scale * power_of_2(-up);
      ups[32 * wave + m32] = up;
#pragma unroll
      for (int k = 0; k < KS; k++) {
        const int at = 16 * k + 8 * h2;
        float4 e0 = make_float4(0.f, 0.f, 0.f, 0.f), e1 = e0;
        if (16 * k < c.dim) e0 = *(const float4 *)(x + at), e1 = *(const float4 *)(x + at + 4);
        const float e[8] = {e0.x * by, e0.y * by, e0.z * by, e0.w * by, e1.x * by, e1.y * by, e1.z * by, e1.w * by};
        halves_of(e, qh[k], ql[k]);
      }
    }
    // (as in few_kernel)
    const float cap = a.cap;
    rowf = cap > 0.0f ? rowf / cap : rowf * kLog2e;
    // ---- staging: the wave's 16 keys (consecutive in memory), the thread's 16 (8) positions of some dimensions, a scale a lane
    // (what the thread's number gives is formed anew in every step: registers are what the rows leave few of)
    constexpr int ROW = D * ES / 16, PARTS = F16 ? 8 : 4, EACH = kPositions / PARTS;
    uint4 reg[BOTH ? 2 * PIECES : PIECES];  // the next step's keys and its values, or one after the other
    constexpr int V0 = BOTH ? PIECES : 0;
    float sreg;
    const float *scale_at = wave ? c.vs : c.ks;  // (waves 0 and 1)
    int32_t kentry, ventry, sentry;  // the table's entries for the step to load next (WHOLE: all one)
    const auto entries_at = [&](int32_t base) {
      if (WHOLE) {
        const int64_t at = (int64_t)o.s * b.width + max(min(base >> c.shift, b.width - 1), 0);
        kentry = *(const __attribute__((address_space(4))) int32_t *)(uintptr_t)(b.table + at);
        return;
      }
      const uint32_t tid = opaque_lane(threadIdx.x);
      const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
      kentry = entry_of(b, c, o.s, base + 16 * wave);
      ventry = entry_of(b, c, o.s, base + EACH * (int32_t)(tid % PARTS));
      sentry = entry_of(b, c, o.s, base + (int32_t)(tid & 63));
    };
    const auto load_keys = [&](int32_t base) {
      const uint32_t tid = opaque_lane(threadIdx.x), ln = tid & 63;
      const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
      const uint32_t row_pieces = (uint32_t)(opaque(c.dim) * ES) / 16;
      const int32_t kpage = page_in(b, c, kentry, base + 16 * wave);
      const int64_t kvec = vectors_of(c, max(kpage, 0), o.h) + ((base + 16 * wave) & mask);
      const char *kp = c.k + kvec * c.dim * ES;
      if (D <= 128 && c.dim == D) {
#pragma unroll
        for (int i = 0; i < PIECES; i++) reg[i] = *(const uint4 *)(kp + (16 * ln + 1024 * i));
        return;
      }
#pragma unroll
      for (int i = 0; i < PIECES; i++) {
        const uint32_t at = ln + 64 * i, col = min(at % ROW, row_pieces - 1);  // (past dim: the last again)
        reg[i] = *(const uint4 *)(kp + (at / ROW * row_pieces + col) * 16);
      }
    };
    uint32_t on_page = 0;     // which 16 positions of the loaded step are on a page
    uint32_t keep_bits = 0;   // which of the thread's (float16) positions may be looked at
    int32_t left_over = 0;    // (WHOLE: 0 or more where all of the step's may be)
    uint32_t scale_bits = 0;  // all where the lane's position has a scale
    const auto load_values = [&](int32_t base) {
      const uint32_t tid = opaque_lane(threadIdx.x), ln = tid & 63;
      const int32_t part_at = EACH * (int32_t)(tid % PARTS);
      if (WHOLE) {
        const int32_t page = page_in(b, c, kentry, base), left = page >= 0 ? tile.to - base : 0;
        const int64_t vec = vectors_of(c, max(page, 0), o.h);
        const char *vp = c.v + (vec * c.dim + (base & mask)) * ES;
        const uint32_t lane_at = (((tid / PARTS) << c.shift) + part_at) * ES;
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
          // (past dim: the last again)
          const uint32_t at = c.dim == D ? lane_at + (uint32_t)(((i * (256 / PARTS)) << c.shift) * ES)
                                         : (uint32_t)(((min((int)(tid / PARTS) + i * (256 / PARTS), c.dim - 1) << c.shift) + part_at) * ES);
          reg[V0 + i] = *(const uint4 *)(vp + at);
        }
        sreg = (scale_at + vec + (base & mask))[ln];
        scale_bits = opaque_lane((int32_t)ln < left ? ~0u : 0u);
        on_page = page >= 0 ? 15 : 0;
        if (F16) left_over = left - kPositions, keep_bits = bits_between(0, left - part_at) & 0xffu;
        return;
      }
      const int32_t slot = (base + part_at) & mask;
      const int32_t vpage = page_in(b, c, ventry, base + part_at), spage = page_in(b, c, sentry, base + (int32_t)ln);
      const char *vp = c.v + (vectors_of(c, max(vpage, 0), o.h) * c.dim + slot) * ES;
#pragma unroll
      for (int i = 0; i < PIECES; i++) {
        const int d = (int)(tid / PARTS) + i * (256 / PARTS);
        reg[V0 + i] = *(const uint4 *)(vp + (min(d, c.dim - 1) << c.shift) * ES);  // (past dim: the last again)
      }
      const int32_t at = base + (int32_t)ln;
      const bool there = spage >= 0 && at < tile.to;
      sreg = scale_at[vectors_of(c, max(spage, 0), o.h) + (at & mask)];
      scale_bits = opaque_lane(there ? ~0u : 0u);
      const uint64_t mapped = __ballot(spage >= 0);
      on_page = (uint32_t)((mapped & 1) | (mapped >> 15 & 2) | (mapped >> 30 & 4) | (mapped >> 45 & 8));
      if (F16) keep_bits = vpage >= 0 ? bits_between(0, tile.to - (base + part_at)) & 0xffu : 0u;
    };
    const auto store_keys = [&](int buf) {
      const uint32_t tid = opaque_lane(threadIdx.x), ln = tid & 63;
      const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
#pragma unroll
      for (int i = 0; i < PIECES; i++) {
        const uint32_t at = ln + 64 * i, piece = at % ROW, lr = key_row(16 * wave + at / ROW), swap = lr & (D == 64 ? 7 : 15);
        if (c.dim < D && (int32_t)(16 * piece) >= c.dim * ES) reg[i] = make_uint4(0, 0, 0, 0);
        char *to_row = keys[buf] + lr * (D * 2);
        if (F16) {
          *(uint4 *)(to_row + 16 * (piece ^ swap)) = reg[i];
        } else {
          *(v8h *)(to_row + 16 * ((2 * piece) ^ swap)) = widen8(reg[i].x, reg[i].y);
          *(v8h *)(to_row + 16 * ((2 * piece + 1) ^ swap)) = widen8(reg[i].z, reg[i].w);
        }
      }
    };
    // (wave 1's, in one scalar register: the exponent of the largest scale times 8, and how far below it the smallest's is)
    int band_run = kNoScale * 8;
    const auto store_values = [&](int buf) {
      const uint32_t tid = opaque_lane(threadIdx.x), ln = tid & 63, part = tid % PARTS;
      const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
#pragma unroll
      for (int i = 0; i < PIECES; i++) {
        const int d = (int)(tid / PARTS) + i * (256 / PARTS);
        char *to_row = values[buf] + d * (kPositions * 2);
        if (F16) {
          uint4 w = reg[V0 + i];
          if (WHOLE ? left_over < 0 : keep_bits != 0xffu) {
            uint32_t *e = (uint32_t *)&w;
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const uint32_t two = keep_bits >> (2 * j);
              e[j] &= (two & 1u) * 0xffffu | (two & 2u) * 0x7fff8000u;
            }
          }
          *(uint4 *)(to_row + 16 * (part ^ (d & 7))) = w;
        } else {
          *(v8h *)(to_row + 16 * ((2 * part) ^ (d & 7))) = widen8(reg[V0 + i].x, reg[V0 + i].y);
          *(v8h *)(to_row + 16 * ((2 * part + 1) ^ (d & 7))) = widen8(reg[V0 + i].z, reg[V0 + i].w);
        }
      }
      sreg = __uint_as_float(__float_as_uint(sreg) & scale_bits);
      if (wave == 0) {
        scales[buf][0][ln] = sreg;
        const bool any_large = __any(__float_as_uint(sreg) >= kLargeScale);  // (or a NaN)
        if (ln == 0) info[buf][1] = on_page | (any_large ? kAnyLarge : 0);
      }
      if (wave == 1) {
        const uint32_t bits = __float_as_uint(sreg);
        if (band_run != kApart) {
          const int run = band_run >> 3, low = run - (band_run & 7);
          if (__any(bits >= above_bits(run) || (bits < below_bits(low) && scale_bits))) {
            // a scale outside those so far (or a NaN, which says nothing)
            const bool finite = scale_bits && bits < 0x7f800000u;
            const uint32_t high = wave_max(finite ? bits : 0u), least = ~wave_max(finite ? ~bits : 0u);
            if (least <= high) {
              const int h1 = max((int)(high >> 23) - 127, run), l0 = (int)(least >> 23) - 127;
              const int l1 = run == kNoScale ? l0 : min(l0, low);
              band_run = h1 - l1 <= kBand && h1 <= kMostScale ? 8 * h1 + (h1 - l1) : kApart;
            }
          }
        }
        const int exponent_run = band_run == kApart ? kApart : band_run >> 3;
        scales[buf][1][ln] = exponent_run == kApart ? sreg : sreg * power_of_2(-exponent_run);
        if (ln == 0) info[buf][0] = exponent_run;
      }
    };
    {
      const int32_t now[10] = {u, end, block, o.k, o.step, steps, tile.steps, q.begin, q.count, o.h};
#pragma unroll
      for (int i = 0; i < 10; i++) parked[wave][i] = now[i];
    }
    // ---- the steps
    float m = -INFINITY, l = 0.0f;
    int exponent = kNoScale;
    v16f acc[DT] = {};
    int32_t base = (tile.first + o.step) * kPositions;
    const int32_t stop = base < tile.to ? base + steps * kPositions : base;  // (rows that see nothing: a step without positions)
    if (base < stop) {
      entries_at(base);
      load_keys(base);
      store_keys(0);
      load_values(base);
      store_values(0);
      entries_at(base + kPositions);
    }
    __syncthreads();
    for (int buf = 0; base < stop; base += kPositions, buf ^= 1) {
      const bool more = base + kPositions < stop;
      if (more) {
        load_keys(base + kPositions);
        if (BOTH) {
          load_values(base + kPositions);
          entries_at(base + 2 * kPositions);
        }
      }
      // 32 positions at a time, as the registers allow
#pragma unroll 1
      for (int t = 0; t < 2; t++) {
        const int32_t at32 = base + 32 * t;
        if (at32 < any_to) {
          // ---- scores
          v16f s = {};
          // (the chunk 2 k + h2 of a row, XORed, is its place XOR 32 k)
          const uint32_t kat = opaque_lane((32 * t + m32) * (D * 2) + 16 * (h2 ^ (m32 & (D == 64 ? 7 : 15))));
#pragma unroll
          for (int k = 0; k < KS; k++) {
            const v8h k8 = *(const v8h *)(keys[buf] + (kat ^ (32 * k)));
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8, ql[k], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8, qh[k], s, 0, 0, 0);
          }
          float p[16];
          const int32_t flags = __builtin_amdgcn_readfirstlane(info[buf][1]), pages_here = flags >> (2 * t) & 3;
          const float *sc = &scales[buf][0][32 * t + 8 * h2];
          float by_row = rowf;
          v4f ks[4];
#pragma unroll
          for (int i = 0; i < 4; i++) ks[i] = *(const v4f *)(sc + 16 * (i >> 1) + 4 * (i & 1));
          if (flags & kAnyLarge) {
            const int32_t up = ups[32 * wave + m32];
            const float first = first_of_large(up);
#pragma unroll
            for (int e = 0; e < 16; e++) p[e] = s[e] * first * ks[e >> 2][e & 3];
            by_row = factor_of_large(up, call_again()->a.scale, cap);
          } else {
#pragma unroll
            for (int e = 0; e < 16; e++) p[e] = s[e] * ks[e >> 2][e & 3];
          }
          if (cap > 0.0f) {
            const float bend = opaque(0.55f), twice = opaque(2.0f * kLog2e);
#pragma unroll
            for (int e = 0; e < 16; e++) p[e] = cap * kLog2e * tanh_of(p[e] * by_row, bend, twice);
            by_row = 1.0f;
          }
          const bool edge = at32 + 32 > every_to || at32 < every_from || pages_here != 3;
          uint32_t seen = ~0u;
          if (edge) {
            const int32_t at = at32 + 8 * h2;
            seen = (pages_here & 1 ? bits_between(from - at, to - at) & 0xffu : 0u) |
                   (pages_here & 2 ? (bits_between(from - at - 16, to - at - 16) & 0xffu) << 8 : 0u);
#pragma unroll
            for (int e = 0; e < 16; e++) p[e] = kept(p[e], seen, e, 0xff800000u);
          }
          float most = p[0];
#pragma unroll
          for (int e = 1; e < 16; e++) most = fmaxf(most, p[e]);
          most = max_pair(most) * by_row;
          const int e1 = __builtin_amdgcn_readfirstlane(info[buf][0]);
          const auto value_scales = [&](float (&vs)[16]) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const v4f v0 = *(const v4f *)(sc + kPositions + 16 * i), v1 = *(const v4f *)(sc + kPositions + 16 * i + 4);
#pragma unroll
              for (int e = 0; e < 8; e++) vs[8 * i + e] = e < 4 ? v0[e & 3] : v1[e & 3];
            }
          };
          if (__any(most > m + kRoom) || e1 != exponent || e1 == kApart) {
            float rescale = 1.0f;
            if (e1 == kApart) {
              Apart own = exponent == kApart ? apart[32 * wave + m32] : apart_from(exponent, m);
              float vs[16];
              value_scales(vs);
              rescale = apart_moves(p, vs, by_row, most, m, l, own, [](float v) { return max_pair(v); });
              apart[32 * wave + m32] = own;
            } else {
              if (__any(most > m + kRoom)) {
                const float m1 = fmaxf(m, ceilf(most));
                rescale = m1 == -INFINITY ? 0.0f : exp2_of(m - m1);
                m = m1;
                l *= rescale;
              }
              rescale *= power_of_2(max(exponent - e1, -126));
            }
#pragma unroll
            for (int d = 0; d < DT; d++) acc[d] *= rescale;
            exponent = e1;
          }
          if (e1 == kApart) {
            float vs[16];
            value_scales(vs);
            apart_weights(p, vs, by_row, m, l, apart[32 * wave + m32].x);
          } else {
            const float less = (m == -INFINITY ? 0.0f : m) - kShift;
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const v4f v0 = *(const v4f *)(sc + kPositions + 16 * i), v1 = *(const v4f *)(sc + kPositions + 16 * i + 4);
#pragma unroll
              for (int e = 0; e < 8; e++) {
                const float w = exp2_of(__builtin_fmaf(p[8 * i + e], by_row, -less));
                l += w;
                p[8 * i + e] = w * (e < 4 ? v0[e & 3] : v1[e & 3]);
              }
            }
          }
          if (edge) {
#pragma unroll
            for (int e = 0; e < 16; e++) p[e] = kept(p[e], seen, e, 0u);  // (a NaN scale that others see)
          }
          v8h ph[2], pl[2];
#pragma unroll
          for (int i = 0; i < 2; i++) halves_of(p + 8 * i, ph[i], pl[i]);
          // ---- out += weights times values
          const uint32_t vat = opaque_lane(m32 * (kPositions * 2) + 16 * ((4 * t + h2) ^ (m32 & 7)));
#pragma unroll
          for (int i = 0; i < 2; i++) {
#pragma unroll
            for (int d = 0; d < DT; d++) {
              const v8h v8 = *(const v8h *)(values[buf] + d * (32 * kPositions * 2) + (vat ^ (32 * i)));
              acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v8, pl[i], acc[d], 0, 0, 0);
              acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v8, ph[i], acc[d], 0, 0, 0);
            }
          }
        }
        if (!BOTH && more && t == 0) {
          store_keys(buf ^ 1);
          load_values(base + kPositions);
          entries_at(base + 2 * kPositions);
        }
      }
      if (more) {
        if (BOTH) store_keys(buf ^ 1);
        store_values(buf ^ 1);
      }
      __syncthreads();
    }
    l = __builtin_amdgcn_ldexpf(sum_pair(l), -kHeld);
    // ---- the rows out, or to be joined
    const Call *after = call_again();
    int32_t kept_back[10];
#pragma unroll
    for (int i = 0; i < 10; i++) kept_back[i] = __builtin_amdgcn_readfirstlane(parked[wave][i]);
    u = kept_back[0], end = kept_back[1], block = kept_back[2], o.k = kept_back[3], o.step = kept_back[4], o.h = kept_back[9];
    const int32_t done = kept_back[5], begin = kept_back[7], count = kept_back[8];
    const bool whole = done == kept_back[6];
    if (live) {
      const int thread = opaque_lane(threadIdx.x), m32 = thread & 31, h2 = (thread >> 5) & 1, wave = thread >> 6;
      const int own_exponent = (exponent == kApart ? apart[32 * wave + m32].x : exponent) - kHeld;
      if (whole) {
        const int32_t shared = after->sh.group, dim = after->c.dim;
        const float per = l != 0.0f ? 1.0f / l : 0.0f;
        float *out = (float *)(after->a.out + (begin + token) * after->a.out_stride) + (int64_t)(o.h * shared + g) * dim;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const int at = 32 * d + 8 * j + 4 * h2;
            v4f v = {acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]};
            if (32 * d + 8 * j < dim) *(v4f *)(out + at) = shifted(v * per, 0.0f, 0.0f, own_exponent);
          }
      } else {
        float *part = (float *)(after->a.work + after->sh.parts) + (int64_t)(block * 2 + (o.step > 0 ? 0 : 1)) * kRows * (D + 2);
        const int r = 32 * wave + m32;
        if (h2 == 0) part[r * 2] = m, part[r * 2 + 1] = l;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            v4f v = {acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]};
            *(v4f *)(part + kRows * 2 + r * D + 32 * d + 8 * j + 4 * h2) = shifted(v, 0.0f, 0.0f, own_exponent);
          }
      }
    }
    u += done;
    if (u >= end) {
      if (threadIdx.x == 0 && o.step == 0 && !whole) {
        Tail &tail = ((Tail *)after->a.work)[block];
        const int32_t rows = count * after->sh.group, r0 = kRows * tile_at(o.k, (rows + kRows - 1) / kRows);
        tail.begin = begin, tail.r0 = r0, tail.rows = min(kRows, rows - r0), tail.h = o.h;
        tail.last = end - done + kept_back[6] - 1;
      }
      break;
    }
    // ---- the next item: the next row tile, head or sequence (one more step is left, so there is one)
    o.step = 0;
    if (++o.k * kRows >= count * after->sh.group) {
      o.k = 0;
      if (++o.h == after->c.heads) {
        o.h = 0;
        do {
          if (++o.s >= after->b.sequences) return;
        } while (!wave_sequence_of(after->b, o.s).count);
      }
    }
  }
}

int padded(int32_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// How a call's steps are shared: by as many blocks as the GPU holds, or as there can be steps.
Share share_of(const Cache &c, const Batch &b, int32_t heads, int32_t a_cu, int32_t rows_of_a_tile, int32_t log, bool plan) {
  Share sh{};
  sh.rows = rows_of_a_tile, sh.log = log, sh.group = heads / c.heads;
  sh.per = sh.group > 1 ? (uint32_t)((((uint64_t)1 << 32) + sh.group - 1) / sh.group) : 0;
  const int64_t rows = (int64_t)b.tokens * sh.group;
  const int64_t tiles = std::min(rows, rows / rows_of_a_tile + b.sequences);
  const int64_t steps = std::max<int64_t>((((int64_t)b.width << c.shift) + (1 << log) - 1) >> log, 1);
  sh.blocks = (int32_t)std::min<int64_t>(std::min(a_cu * cu_count(), kMostBlocks), tiles * c.heads * steps);
  sh.tiles = (int32_t)tiles;
  sh.shared = steps > 1 && sh.blocks > 1;
  sh.parts = ((plan ? plan_bytes(sh.blocks, b.sequences, tiles) : sh.blocks * (int64_t)sizeof(Tail)) + 255) / 256 * 256;
  sh.bytes = sh.parts + (int64_t)sh.blocks * 2 * rows_of_a_tile * (padded(c.dim) + 2) * 4;
  // (steps are counted in 32 bits, and a row's token is row ceil(2^32 / group) / 2^32)
  sh.countable = tiles * c.heads * steps < INT32_MAX && rows * sh.group < (int64_t)1 << 32;
  return sh;
}
// Where a sequence has room for four steps at most, a block takes a tile whole: the shares and the second launch that joins them
// cost more than three more steps.  For eight, where the sequences and heads alone give every compute unit a block.  Measured, whole /
// shared (us), one token a sequence, heads of 128 int8 (a step: 256 positions), 8 of keys: 250 positions of 1 sequence 10.2 / 13.3, of
// 32 sequences 12.0 / 16.6; 500 of 32 12.7 / 19.8; 1000 of 32 16.7 / 23.0; 1800 of 1 20.4 / 13.6, of 8 22.3 / 18.9, of 32 30.1 / 34.8,
// of 100 87.7 / 90.6.  (Longer ones gain 2 us and more, too, but lose as much as 15 where one sequence is longer than the others.)
constexpr int kWholeSteps = 4;
Share few_share(const Cache &c, const Batch &b, int32_t heads) {
  const int32_t d = padded(c.dim);
  Share sh = share_of(c, b, heads, few_blocks_a_cu(d, c.f16), kFewRows, few_np(d, c.f16) == 16 ? 8 : 7, false);
  const int64_t most = (int64_t)b.sequences * c.heads >= cu_count() ? 2 * kWholeSteps : kWholeSteps;
  if (((int64_t)b.width << c.shift) <= most << sh.log && b.sequences < 1 << 20) {
    sh.whole = (b.longest * sh.group + kFewRows - 1) / kFewRows;
    sh.shared = false;
  }
  return sh;
}
Share rows_share(const Cache &c, const Batch &b, int32_t heads) {
  return share_of(c, b, heads, rows_blocks_a_cu(padded(c.dim)), kRows, 6, true);
}

// Whether few_kernel takes the call: no sequence has more rows of a head than six of its tiles (three where a head has 64 values
// or fewer).  It reads a step's positions again for every tile, rows_kernel fills tiles of 128 rows with them.  Measured, few / rows
// (us): heads of 128 int8, 8 sequences over 4100 positions, 20 rows 34 / 59, 48 rows 51 / 73, 64 rows 55 / 80, 96 rows 77 / 91, 192
// rows 126 / 123; 32 over 1000, 64 rows 49 / 69, 256 rows 183 / 104; 256 int8, 96 rows 75 / 111; 64 float16, 48 rows 46 / 49, 64
// rows 53 / 51.
bool few_rows(const Cache &c, const Batch &b, int32_t heads) {
  return (int64_t)b.longest * (heads / c.heads) <= (padded(c.dim) > 64 ? 6 : 3) * kFewRows;
}

template <int D>
hipError_t launch(const Attention &a, const Cache &c, const Batch &b, hipStream_t s) {
  const bool few = few_rows(c, b, a.heads);
  Call call{a, c, b, few ? few_share(c, b, a.heads) : rows_share(c, b, a.heads)};
  // (a window past all positions is none; a position less the window then stays above 32 bits' lowest, 2^24 before the first too)
  call.a.window = std::min(a.window, kMostPositions);
  const dim3 blocks = call.sh.whole ? dim3(b.sequences, call.sh.whole, c.heads) : dim3(call.sh.blocks);
  const int32_t *edge = nullptr;
  if (few) {
    hipLaunchKernelGGL((c.f16 ? few_kernel<D, 1> : few_kernel<D, 0>), blocks, dim3(256), 0, s, call);
  } else {
    edge = plan_of(a.work, call.sh.blocks, b.sequences).edge;
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(1024), 0, s, call);
    if (D == 128 && c.shift >= 6)
      hipLaunchKernelGGL((c.f16 ? rows_kernel<D, 1, D == 128> : rows_kernel<D, 0, D == 128>), blocks, dim3(256), 0, s, call);
    else
      hipLaunchKernelGGL((c.f16 ? rows_kernel<D, 1, false> : rows_kernel<D, 0, false>), blocks, dim3(256), 0, s, call);
  }
  // (few rows: their parts sliced)
  constexpr int SLICES = 4;
  const int64_t rows = std::min<int64_t>((int64_t)b.longest * call.sh.group, call.sh.rows);
  if (call.sh.shared && rows <= 4)
    hipLaunchKernelGGL((join_kernel<D, SLICES>), dim3(call.sh.blocks, (rows * D * SLICES + 1023) / 1024), dim3(256), 0, s, call, edge);
  else if (call.sh.shared)
    hipLaunchKernelGGL((join_kernel<D, 1>), dim3(call.sh.blocks, std::min<int64_t>((rows * D + 1023) / 1024, 8)), dim3(256), 0, s, call, edge);
  return hipGetLastError();
}

}  // namespace

int64_t attention_work_bytes(const Cache &c, const Batch &b, int32_t heads) {
  if (b.tokens <= 0 || b.sequences <= 0) return 0;
  const Share few = few_share(c, b, heads), rows = rows_share(c, b, heads);
  if (!few.countable || !rows.countable) return -1;
  return few_rows(c, b, heads) ? few.bytes : rows.bytes;
}

hipError_t launch_attention(const Attention &a, const Cache &c, const Batch &b, hipStream_t s) {
  if (b.tokens <= 0 || b.sequences <= 0) return hipSuccess;
  switch (padded(c.dim)) {
  case 64: return launch<64>(a, c, b, s);
  case 128: return launch<128>(a, c, b, s);
  default: return launch<256>(a, c, b, s);
  }
}

}  // namespace hq
