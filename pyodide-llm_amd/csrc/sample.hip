// sample.hip — the next token of each row of logits from a given random number: temperature, top-k, top-p, min-p.
//
// A logit is held as its key, a 32-bit number that orders as the float does (0: never drawn).  What top-k and top-p leave is a
// smallest key t and how many of the logits equal to it (the first by index); both are found by histograms over the keys,
// round by round in the bin where the count (or the weight) passes the line, until a bin holds one key.  Weights in
// histograms are whole numbers (steps of a power of two below the largest weight), so that no order of additions changes them.
// The token is then found by a sum over the kept weights in index order, in 64 bits.
//
// Rows of up to 8192 logits: a block a row, whose keys stay in LDS.  Longer rows: every wave of a first launch takes
// 2048 logits of a row and hands on those above a line of its own, some 90 at most (with what they sum to, where the settings
// ask for the row's whole sum); a block a row of a second launch finds t among what was handed on, and goes to the row itself
// only where t lies below one of these lines.  A wave's logits are 32 grains of 64 over the whole row: words that stand out
// often have neighbouring numbers.
//
// Where top-p is asked for, three launches more: a row whose line lies below the list (a flat row, a high temperature) has its
// weights tallied and its line found by 16 blocks (tally, wide), and drawn by one (end); other rows leave them at once (1.6 to
// 4 us a launch).  One block for such a row takes as long however few there are.
//
// Measured: 256 rows of 128256 with their own settings: hand 49.4 us (131 MB, 2.7 TB/s: its waves wait for loads
// half of their time and to issue a third), join 29.9 (waits, for barriers and LDS, are 63 % of it), tally 13.2, wide 16.2, end 26.9 (rows whose line is low); 32 rows: 12.2, 25.8, 4.6, 4.6,
// 3.9.  A block a row over everything: 505 us and 373.
#include <algorithm>
#include <cmath>

#include "common.hpp"
#include "launch.hpp"

namespace hq {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = kThreads;
constexpr int kStep = 256;               // logits a wave takes at a time, 4 a lane
constexpr int kBatch = 8;                // steps whose loads are on their way together
constexpr int kHeld = 8192;              // the longest row that a block takes alone, in LDS
constexpr int kGrain = 64;               // neighbouring logits that the first launch gives to one wave
constexpr int kGrains = kBatch * kStep / kGrain;
constexpr int kHand = 192;               // logits that a wave of the first launch can hand on
constexpr int kList = 7680;              // and what the second launch takes of a row (62 KB of its 115: one block a compute unit)
constexpr int kFew = 64;                 // keys that one wave finishes with
constexpr uint32_t kLowest = 0x00800000u;  // the key of the lowest finite number

HQ_DEV uint32_t key_of(float v) {
  const uint32_t bits = __float_as_uint(fadd(v, 0.0f));  // (-0 orders as 0)
  return v > -__builtin_huge_valf() ? bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u) : 0u;
}
HQ_DEV float value_of(uint32_t key) { return __uint_as_float(key ^ ((uint32_t)((int32_t)~key >> 31) | 0x80000000u)); }

// 2^(i / 64)
__device__ const double kRoots[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0,
};

// e^x for x = d c ln 2 / 64, d c <= 0: 2^(n / 64) from the table, times the series of what is left (|rest| < 0.0055: its sixth power
// over 720 is below 2^-54), scaled by whole powers of two; within 2^-50 of it.  Whole numbers come and go as the low bits of a sum
// with 1.5 2^52: conversions of 64-bit numbers take several times an addition.
HQ_DEV double power(double d, double c, const double *roots) {
  const double y = fmax(d * c, -70000.0), sum = y + 6755399441055744.0, f = y - (sum - 6755399441055744.0);
  const int n = (int)(uint32_t)__builtin_bit_cast(uint64_t, sum);
  double s = fma(f, 0x1.5d87fe78a6731p-40, 0x1.3b2ab6fba4e77p-31);
  s = fma(f, s, 0x1.c6b08d704a0c0p-23);
  s = fma(f, s, 0x1.ebfbdff82c58fp-15);
  s = fma(f, s, 0x1.62e42fefa39efp-7);
  const double root = roots[n & 63];
  return ldexp(fma(root, f * s, root), n >> 6);
}
HQ_DEV double slope_of(double temperature) { return 92.332482616893656877 / temperature; }  // 64 / ln 2 of it

// a row's largest key and temperature: its weights
struct Weights {
  uint32_t top;
  double most, slope, by;  // the largest logit; by: 1 / step, a power of two up to 2^51
  const double *roots;
  HQ_DEV double of(uint32_t key) const {
    const double x = power((double)value_of(key) - most, slope, roots);
    return key == top ? 1.0 : key ? x : 0.0;
  }
  HQ_DEV uint64_t steps_of(double x) const { return __builtin_bit_cast(uint64_t, x * by + 0x1p52) - 0x4330000000000000u; }
  HQ_DEV uint64_t steps(uint32_t key) const { return steps_of(of(key)); }
};

HQ_DEV float range_of(const Weights &w) { return (float)fmin(40.0 * 92.332482616893656877 / w.slope, 3e38); }

struct Settings {
  double temperature, top_p, min_p, u;
  int32_t top_k, vocab;  // (0: all)
  HQ_DEV bool all() const { return !top_k && !(top_p < 1.0) && !(min_p > 0.0); }
  HQ_DEV bool whole_sum() const { return !top_k && (top_p < 1.0 || !(min_p > 0.0)); }  // the row's whole sum is needed
};
HQ_DEV Settings settings_of(const Sample &a, int64_t row) {
  // (all of them loaded before the first is looked at: an array that is not there is u's)
  const float u = a.u[row], temperature = (a.temperature ? a.temperature : a.u)[row];
  const float top_p = (a.top_p ? a.top_p : a.u)[row], min_p = (a.min_p ? a.min_p : a.u)[row];
  const int32_t top_k = (a.top_k ? a.top_k : (const int32_t *)a.u)[row];
  Settings o;
  o.vocab = a.vocab;
  o.temperature = a.temperature ? temperature : 1.0f;
  o.top_k = a.top_k && top_k > 0 && top_k < a.vocab ? top_k : 0;
  o.top_p = a.top_p ? top_p : 1.0f;
  o.min_p = a.min_p && min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f;
  // (1 or more: no sum passes it, so that the last that has any is drawn; times 1 a sum in another order might, by a rounding)
  o.u = u >= 1.0f ? __builtin_huge_val() : u >= 0.0f ? u : 0.0f;
  if (!(o.temperature > 0.0)) o.temperature = 1.0, o.top_k = 1;
  return o;
}

// ---- over a wave's lanes, by moves between registers ---------------------------------------------------------------
template <int CTRL, int ROWS, typename T>
HQ_DEV T moved(T v) {  // (0 for lanes that nothing comes to)
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int32_t, v), CTRL, ROWS, 0xf, true));
  } else {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int32_t)(uint32_t)u, CTRL, ROWS, 0xf, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int32_t)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, true);
    return __builtin_bit_cast(T, (uint64_t)lo | (uint64_t)hi << 32);
  }
}
// What lanes give each other is computed here, with all lanes, and not moved to where a few of them use it
template <typename T>
HQ_DEV T here(T v) {
  if constexpr (sizeof(T) == 4) {
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    asm volatile("" : "+v"(u));
    return __builtin_bit_cast(T, u);
  } else {
    uint64_t u = __builtin_bit_cast(uint64_t, v);
    asm volatile("" : "+v"(u));
    return __builtin_bit_cast(T, u);
  }
}
// the sum over the lanes up to and with this one, in rows of 16, then the rows before
template <typename T>
HQ_DEV T sum_row(T v) {
  v += moved<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  return here(v);
}
template <typename T>
HQ_DEV T sum_up_to(T v) {
  v = sum_row(v);
  v += moved<0x142, 0xa>(v);  // row_bcast 15 into rows 1 and 3, row_bcast 31 into rows 2 and 3
  v += moved<0x143, 0xc>(v);
  return here(v);
}
// lane l's value (l the same in all lanes)
template <typename T>
HQ_DEV T from_lane(T v, int l) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int32_t, v), l));
  } else {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int32_t)(uint32_t)u, l);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int32_t)(uint32_t)(u >> 32), l);
    return __builtin_bit_cast(T, (uint64_t)lo | (uint64_t)hi << 32);
  }
}
template <typename T>
HQ_DEV T wave_sum(T v) { return from_lane(sum_up_to(v), 63); }
HQ_DEV uint32_t wave_most(uint32_t v) {
  v = max(v, moved<0x111, 0xf>(v));
  v = max(v, moved<0x112, 0xf>(v));
  v = max(v, moved<0x114, 0xf>(v));
  v = max(v, moved<0x118, 0xf>(v));
  v = max(v, moved<0x142, 0xa>(v));
  v = max(v, moved<0x143, 0xc>(v));
  return from_lane(here(v), 63);
}

// ---- sums over a block ----------------------------------------------------------------------------------------------
// (every thread calls; `part`: kWaves doublewords of LDS that nothing else uses)
template <typename T>
HQ_DEV T block_sum(T v, T *part) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return from_lane(sum_row(part[threadIdx.x & (kWaves - 1)]), kWaves - 1);
}
HQ_DEV uint32_t block_most(uint32_t v, uint32_t *part) {
  v = wave_most(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return wave_most(part[threadIdx.x & (kWaves - 1)]);
}
// the sum over the threads before this one
template <typename T>
HQ_DEV T sum_before(T v, T *part, T &total) {
  const int wave = threadIdx.x >> 6;
  const T sum = sum_up_to(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) part[wave] = sum;
  __syncthreads();
  const T waves = sum_row(part[threadIdx.x & (kWaves - 1)]);  // (a lane a wave: the sums up to each)
  total = from_lane(waves, kWaves - 1);
  return (wave ? from_lane(waves, wave - 1) : (T)0) + (sum - v);
}

struct Scratch {
  double roots[64];
  uint64_t weight[kBins];
  uint32_t count[kBins], some[kBins];  // (a key of the bin)
  uint64_t part[kWaves];
  uint32_t part2[kWaves];
  uint64_t found[4];
  double sums[kWaves];
  uint32_t ties[kWaves];
  uint32_t few, few_keys[kFew];  // keys that a wave can finish with, their indexes, and how many
  int32_t few_at[kFew];
  uint64_t ahead[kFew];
  uint32_t rank[kFew], place[kFew];
};

// ---- where a row's keys are -----------------------------------------------------------------------------------------
// A wave takes a part of the row, `part` logits (whole steps) from wave * part on, a step's 4 a lane at a time, in order:
// sweep(f) calls f(keys, the first's place) until it returns false.

// 4 logits of each of BATCH steps, `stride` apart from the lane's own `from` on; -infinity from `to` on.  whole: all lie before `to`
template <bool WIDE, int BATCH>
HQ_DEV void load(const float *p, int32_t n, int32_t from, int32_t stride, int32_t to, bool whole, float v[4 * BATCH]) {
  if (whole) {
#pragma unroll
    for (int j = 0; j < BATCH; j++) {
      const float *q = p + from + j * stride;
      if (WIDE) {  // (rows that begin on 16 bytes)
        const float4 f = *(const float4 *)q;
        v[4 * j] = f.x, v[4 * j + 1] = f.y, v[4 * j + 2] = f.z, v[4 * j + 3] = f.w;
      } else {
#pragma unroll
        for (int c = 0; c < 4; c++) v[4 * j + c] = q[c];
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < BATCH; j++) {
    const int32_t i = from + j * stride;
#pragma unroll
    for (int c = 0; c < 4; c++) v[4 * j + c] = p[min(i + c, n - 1)];
#pragma unroll
    for (int c = 0; c < 4; c++)
      if (i + c >= to) v[4 * j + c] = -__builtin_huge_valf();
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <bool WIDE, int BATCH = kBatch>
struct Row {  // a row, or the part of one from `base` on, in memory
  const float *p;
  int32_t n, part, base;
  HQ_DEV Row(const float *row, int32_t n_, int32_t base_ = 0)
      : p(row + base_), n(n_), part((n_ + kWaves * kStep - 1) / (kWaves * kStep) * kStep), base(base_) {}
  HQ_DEV int32_t index(int32_t i) const { return base + i; }
  template <typename F>
  HQ_DEV void sweep(F f) const {
    const int32_t from = (int32_t)(threadIdx.x >> 6) * part, to = min(from + part, n);
    for (int32_t i0 = from; i0 < to; i0 += BATCH * kStep) {
      float v[4 * BATCH];
      load<WIDE, BATCH>(p, n, i0 + 4 * (int32_t)(threadIdx.x & 63), kStep, to, i0 + BATCH * kStep <= to, v);
#pragma unroll
      for (int j = 0; j < BATCH; j++) {
        uint32_t keys[4];
#pragma unroll
        for (int c = 0; c < 4; c++) keys[c] = key_of(v[4 * j + c]);
        if (i0 + j * kStep < to && !f(keys, i0 + j * kStep + 4 * (int32_t)(threadIdx.x & 63))) return;
        __builtin_amdgcn_sched_barrier(0);  // (one step's numbers at a time: registers)
      }
    }
  }
};

template <bool ALL>
struct List {  // a row, or what was handed on of one (with each key's index), in LDS; zeros up to a whole step
  const uint32_t *keys;
  const int32_t *at;
  int32_t n, part;
  HQ_DEV List(const uint32_t *keys_, const int32_t *at_, int32_t n_)
      : keys(keys_), at(at_), n(n_), part((n_ + kWaves * kStep - 1) / (kWaves * kStep) * kStep) {}
  HQ_DEV int32_t index(int32_t i) const { return ALL ? i : at[i]; }
  template <typename F>
  HQ_DEV void sweep(F f) const {
    const int32_t from = (int32_t)(threadIdx.x >> 6) * part, to = min(from + part, n);
    for (int32_t i0 = from; i0 < to; i0 += kStep) {
      const int32_t i = i0 + 4 * (int32_t)(threadIdx.x & 63);
      const uint4 q = *(const uint4 *)(keys + i);
      const uint32_t k[4] = {q.x, q.y, q.z, q.w};
      if (!f(k, i)) return;
    }
  }
};

// ---- the line -------------------------------------------------------------------------------------------------------
// Where in falling order of keys a count or a weight is reached: the key, what lies before its first, and how many are equal to it.
struct Line {
  uint32_t key;
  uint64_t before;
  uint32_t equal;
};

// the smallest key of lo .. hi for which `holds` (it does for hi and then for every larger one); the whole wave calls it
template <typename F>
HQ_DEV uint32_t first_key(uint32_t lo, uint32_t hi, F holds) {
  while (lo < hi) {
    const uint32_t step = (hi - lo) / 64 + 1;
    const uint64_t at = (uint64_t)lo + (uint64_t)(threadIdx.x & 63) * step;
    const uint64_t in = __ballot(at >= hi || holds((uint32_t)at));
    const int f = in ? __ffsll((unsigned long long)in) - 1 : 64;
    if (f < 64) hi = (uint32_t)min((uint64_t)hi, (uint64_t)lo + (uint64_t)f * step);
    if (f > 0) lo += (uint32_t)(f - 1) * step + 1;
  }
  return lo;
}

// A search for the line: rounds of histograms over the keys of lo .. hi, each in the bin of the one before in which the line lies.  The
// first round's bins lie evenly over `range` below the largest value, the rest in the last (logits on both sides of 0 would
// crowd a few bins of keys), those after it evenly over the keys.
struct Search {
  const Weights &w;
  uint32_t lo, hi;
  float most, per;
  bool values;
  int shift;
  // of the round: the line's bin, the count (weight) before it and in it, its keys and those before it too, one of them
  int bin;
  uint64_t before = 0, own;
  uint32_t equal, through, some;

  HQ_DEV Search(const Weights &w_, uint32_t lo_, float range) : w(w_), lo(lo_), hi(w_.top), most((float)w_.most), per((kBins - 0.5f) / range) {
    values = most < __builtin_huge_valf() && range > 0.0f && per > 0.0f && per < __builtin_huge_valf();
  }
  HQ_DEV int value_bin(uint32_t key) const { return (int)fminf((most - value_of(key)) * per, kBins - 1.0f); }
  HQ_DEV int bin_of(uint32_t key) const { return values ? value_bin(key) : (int)((hi - key) >> shift); }
  HQ_DEV bool inside(uint32_t key) const { return key >= lo && key <= hi; }

  // the round's histogram in m
  template <bool WEIGHT, typename Source>
  HQ_DEV void tally(const Source &source, Scratch &m) {
    shift = max(22 - (int)__builtin_clz((hi - lo) | 1u), 0);  // hi - lo in 10 bits
    __syncthreads();
    m.count[threadIdx.x] = 0;
    if (WEIGHT) m.weight[threadIdx.x] = 0;
    __syncthreads();
    source.sweep([&](const uint32_t keys[4], int32_t) {
#pragma unroll
      for (int c = 0; c < 4; c++) {
        if (!inside(keys[c])) continue;
        const int b = bin_of(keys[c]);
        atomicAdd(&m.count[b], 1u);
        if (WEIGHT) atomicAdd((unsigned long long *)&m.weight[b], (unsigned long long)w.steps(keys[c]));
        m.some[b] = keys[c];
      }
      return true;
    });
    __syncthreads();
  }
  // the line's bin by it; false: there is no key
  template <bool WEIGHT>
  HQ_DEV bool find(double target, Scratch &m) {
    const uint32_t count = m.count[threadIdx.x];
    const uint64_t mine = WEIGHT ? m.weight[threadIdx.x] : (uint64_t)count;
    // the sums over the bins before this thread's, of the line's measure and of keys
    const int wave = threadIdx.x >> 6;
    const uint64_t sum = sum_up_to(mine);
    const uint32_t keys = sum_up_to(count);
    if ((threadIdx.x & 63) == 63) m.part[wave] = sum, m.part2[wave] = keys;
    __syncthreads();
    const uint64_t sums = sum_row(m.part[threadIdx.x & (kWaves - 1)]);
    const uint32_t all = sum_row(m.part2[threadIdx.x & (kWaves - 1)]);
    const uint64_t ahead = before + (wave ? from_lane(sums, wave - 1) : 0) + (sum - mine);
    const uint32_t up_to = (wave ? from_lane(all, wave - 1) : 0) + keys;
    // the last bin with anything in it that begins before the line
    const uint64_t begun = __ballot(count && (double)ahead < target);
    if ((threadIdx.x & 63) == 0) m.ties[wave] = begun ? threadIdx.x + 64 - __clzll((long long)begun) : 0;
    __syncthreads();
    bin = (int)wave_most(m.ties[threadIdx.x & (kWaves - 1)]) - 1;
    if ((int)threadIdx.x == bin) m.found[1] = ahead, m.found[2] = up_to;
    __syncthreads();
    if (bin < 0) return false;
    before = m.found[1], own = WEIGHT ? m.weight[bin] : (uint64_t)m.count[bin];
    through = (uint32_t)m.found[2], equal = m.count[bin], some = m.some[bin];
    return true;
  }

  template <bool WEIGHT, typename Source>
  HQ_DEV bool round(const Source &source, double target, Scratch &m) {
    tally<WEIGHT>(source, m);
    return find<WEIGHT>(target, m);
  }
  // a key that none of the round's bin or before it lies below (the bins' edge, and a bin's width for what rounding does)
  HQ_DEV uint32_t edge() const {
    if (!values) return max(lo, hi - min(hi, ((uint32_t)bin << shift) | ((1u << shift) - 1)));
    return bin >= kBins - 1 ? lo : max(lo, key_of(most - (float)(bin + 2) / per));
  }

  // the round's bin as the next round's keys; false: it is one key
  HQ_DEV bool narrow() {
    if (values) {
      const uint32_t from = first_key(lo, hi, [&](uint32_t key) { return value_bin(key) <= bin; });
      if (bin > 0) hi = first_key(lo, hi, [&](uint32_t key) { return value_bin(key) < bin; }) - 1;
      lo = from;
      values = false;
    } else {
      if (shift == 0) return false;
      const uint32_t top = hi - ((uint32_t)bin << shift), width = (1u << shift) - 1;
      lo = top - lo > width ? top - width : lo;
      hi = top;
    }
    return lo < hi;
  }
};

// How far below the largest value top-p's line can lie: the tokens from it on, n at most, have 1 - p of all weights (`sum`) or more, so
// that it has w >= (1 - p) sum / n itself; and a little for roundings
HQ_DEV float reach_of(const Weights &w, double top_p, double sum, double n) {
  const double nats = log(n / ((1.0 - top_p) * sum)) + 0.01;
  return (float)fmin(fmin(fmax(nats, 0.5), 40.0) * 92.332482616893656877 / w.slope, 3e38);
}
// and the lowest key that it can be
HQ_DEV uint32_t floor_of(const Weights &w, float reach) {
  return w.most < 3e38 ? max(key_of((float)w.most - reach), 9u) - 8u : 1u;
}

// the keys from `edge` on that `takes` says, up to kFew of them, in any order
template <typename Source, typename F>
HQ_DEV uint32_t gather(const Source &source, uint32_t edge, Scratch &m, F takes) {
  __syncthreads();
  if (threadIdx.x == 0) m.few = 0;
  __syncthreads();
  source.sweep([&](const uint32_t keys[4], int32_t i) {
    if (!__any(max(max(keys[0], keys[1]), max(keys[2], keys[3])) >= edge)) return true;
#pragma unroll
    for (int c = 0; c < 4; c++) {
      if (keys[c] < edge || !takes(keys[c])) continue;
      const uint32_t to = atomicAdd(&m.few, 1u);
      if (to < kFew) m.few_keys[to] = keys[c], m.few_at[to] = source.index(i + c);
    }
    return true;
  });
  __syncthreads();
  return m.few;
}

// Of each of the n gathered keys, a few of them a wave: the measure (a count, or steps of weight) of those before it in falling order
// (of equals: by index), how many these are, and its place by index, in m.ahead, m.rank and m.place
template <bool WEIGHT>
HQ_DEV void order(const Weights &w, int n, Scratch &m) {
  const int lane = threadIdx.x & 63;
  const uint32_t key = lane < n ? m.few_keys[lane] : 0u;
  const int32_t at = lane < n ? m.few_at[lane] : INT32_MAX;
  const uint64_t mine = WEIGHT && lane < n ? w.steps(key) : 0;
  for (int i = threadIdx.x >> 6; i < n; i += kWaves) {
    const uint32_t its = m.few_keys[i];
    const int32_t its_at = m.few_at[i];
    const bool first = key > its || (key == its && at < its_at);
    const uint32_t rank = (uint32_t)__popcll(__ballot(first)), place = (uint32_t)__popcll(__ballot(at < its_at));
    const uint64_t ahead = WEIGHT ? wave_sum(first ? mine : 0) : rank;
    if (lane == 0) m.rank[i] = rank, m.place[i] = place, m.ahead[i] = ahead;
  }
  __syncthreads();
}

// The line, the search's first round done: up to and with the equals of its key the count (the weight) of the keys is `target` or more.
// Not reached: the smallest key there is.
template <bool WEIGHT, typename Source>
HQ_DEV Line line_of(const Source &source, Search &f, double target, Scratch &m) {
  while (true) {
    if (f.equal == 1) return Line{f.some, f.before, 1};
    if (f.equal <= kFew) {
      const int n = (int)gather(source, f.edge(), m, [&](uint32_t key) { return f.inside(key) && f.bin_of(key) == f.bin; });
      order<WEIGHT>(f.w, n, m);
      const int lane = threadIdx.x & 63;
      const uint32_t key = lane < n ? m.few_keys[lane] : 0u;
      const uint64_t ahead = f.before + (lane < n ? m.ahead[lane] : 0);
      // (of equals the first begins before the line when any does)
      const uint32_t least = ~wave_most(lane < n && (double)ahead < target ? ~key : 0u);
      const uint64_t equal = __ballot(lane < n && key == least);
      const uint32_t before = ~wave_most(lane < n && key == least ? ~m.rank[lane] : 0u);
      const uint64_t first = __ballot(lane < n && key == least && m.rank[lane] == before);
      return Line{least, from_lane(ahead, __ffsll((unsigned long long)first) - 1), (uint32_t)__popcll(equal)};
    }
    if (!f.narrow()) return Line{f.some, f.before, f.equal};
    if (!f.template round<WEIGHT>(source, target, m)) return Line{f.some, f.before, f.equal};
  }
}

// what top-k, top-p and min-p leave: keys above t, and the first `ties` of those equal to it; weights below min_p not
struct Kept {
  uint32_t t, ties;
};
constexpr uint32_t kAllTies = UINT32_MAX;

// ties j = 0, 1, .. of a line with before + j each < target, of `equal`: at least one
HQ_DEV uint32_t ties_of(const Line &p, uint32_t equal, double each, double target) {
  const double room = (target - (double)p.before) / each;
  uint32_t ties = room < (double)equal ? (uint32_t)ceil(room) : equal;
  while (ties > 1 && !((double)p.before + (double)(ties - 1) * each < target)) ties--;
  return max(ties, 1u);
}

// ---- the token ------------------------------------------------------------------------------------------------------
// The first by index whose kept weights up to it are more than u times all.  Each wave sums its part, then the wave in whose part the
// sum is reached goes through it again.  of_all: the source is a part of a row whose kept weights are that, `lead` of them before it.
template <typename Source>
HQ_DEV void draw(const Source &source, const Weights &w, const Settings &set, const Kept &kept, int32_t *token, float *chance,
                 Scratch &m, double of_all = 0.0, double lead = 0.0) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const double edge = w.of(kept.t);  // the weight of one that is equal to t
  const uint32_t most = edge >= set.min_p || kept.t == w.top ? kept.ties : 0;
  const auto weight = [&](uint32_t key) {
    if (key <= kept.t) return 0.0;
    const double x = w.of(key);
    return x >= set.min_p ? x : 0.0;
  };
  double sum = 0.0;
  uint32_t tied = 0;
  source.sweep([&](const uint32_t k[4], int32_t) {
#pragma unroll
    for (int c = 0; c < 4; c++) {
      if (k[c] > kept.t) sum += weight(k[c]);
      tied += k[c] == kept.t && k[c];
    }
    return true;
  });
  sum = wave_sum(sum), tied = wave_sum(tied);
  __syncthreads();
  if (lane == 0) m.sums[wave] = sum, m.ties[wave] = tied;
  __syncthreads();
  double total = 0.0, of_wave[kWaves];
  uint32_t seen = 0;
#pragma unroll
  for (int i = 0; i < kWaves; i++) {
    of_wave[i] = m.sums[i] + (double)min(m.ties[i], most - min(most, seen)) * edge;
    total += of_wave[i], seen += m.ties[i];
  }
  if (of_all > 0.0) total = of_all;
  const double target = set.u * total;
  // the wave whose sum passes the target (none: the last that has any)
  double before = lead, run = lead;
  uint32_t tied_before = 0;
  int which = -1;
  bool passed = false;
  seen = 0;
#pragma unroll
  for (int i = 0; i < kWaves; i++) {
    if (!passed && of_wave[i] > 0.0) {
      which = i, run = before, tied_before = seen;
      passed = before + of_wave[i] > target;
    }
    before += of_wave[i], seen += m.ties[i];
  }
  if (wave != which) return;
  int32_t last = -1;
  float last_chance = 0.0f;
  source.sweep([&](const uint32_t k[4], int32_t i) {
    uint64_t equal[4];
    uint32_t rank = tied_before;
#pragma unroll
    for (int c = 0; c < 4; c++) {
      equal[c] = __ballot(k[c] == kept.t && k[c]);
      rank += __popcll(equal[c] & (((uint64_t)1 << lane) - 1));
    }
    double mine[4], sum = 0.0;
#pragma unroll
    for (int c = 0; c < 4; c++) {
      mine[c] = weight(k[c]);
      if (k[c] == kept.t && k[c]) mine[c] = rank++ < most ? edge : 0.0;
      sum += mine[c];
    }
    const double up_to = sum_up_to(sum);
    // the lane in whose four the target is passed, or the last that has any
    const uint64_t over = __ballot(sum > 0.0 && run + up_to > target), any = __ballot(sum > 0.0);
    if (over || any) {
      const int l = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)any);
      double at = run + (up_to - sum);
      int32_t c_at = -1;
      double w_at = 0.0;
#pragma unroll
      for (int c = 0; c < 4; c++) {
        // (the first that passes the target, or the last of all)
        if (mine[c] > 0.0 && (c_at < 0 || !over || !(at > target))) c_at = c, w_at = mine[c];
        at += mine[c];
      }
      last = from_lane(i + c_at, l);
      last_chance = (float)(from_lane(w_at, l) / total);
      if (over) return false;
    }
    run += from_lane(up_to, 63);
#pragma unroll
    for (int c = 0; c < 4; c++) tied_before += __popcll(equal[c]);
    return true;
  });
  if (lane == 0) {
    *token = last < 0 ? -1 : source.index(last);
    if (chance) *chance = last_chance;
  }
}

// The same of up to 64 gathered keys that are the first of the row in falling order (all that can be kept among them), by one wave:
// target: the weight that top-p keeps (0: of what top-k leaves)
HQ_DEV void draw_few(const Weights &w, const Settings &set, uint32_t n, double target, int32_t *token, float *chance, Scratch &m) {
  order<true>(w, (int)n, m);
  if (threadIdx.x >= 64) return;
  const int lane = threadIdx.x;
  const bool there = lane < (int)n;
  const uint32_t key = there ? m.few_keys[lane] : 0u, rank = there ? m.rank[lane] : 0u;
  const uint64_t ahead = there ? m.ahead[lane] : 0;
  const double x = there ? w.of(key) : 0.0;
  const uint64_t mine = w.steps_of(x);
  bool kept = there && (!set.top_k || rank < (uint32_t)set.top_k);
  if (set.top_p < 1.0) {
    const uint64_t all = wave_sum(kept ? mine : 0);
    if (!(target > 0.0)) target = fmax(set.top_p * (double)all, 0.5);
    kept = kept && ((double)ahead < target || rank == 0);
  }
  kept = kept && (x >= set.min_p || key == w.top);
  // by index (what is not kept as 0)
  const int to = there ? (int)m.place[lane] : lane;
  const uint64_t bits = __builtin_bit_cast(uint64_t, kept ? x : 0.0);
  const uint32_t lo = here((uint32_t)__builtin_amdgcn_ds_permute(4 * to, (int32_t)(uint32_t)bits));
  const uint32_t hi = here((uint32_t)__builtin_amdgcn_ds_permute(4 * to, (int32_t)(uint32_t)(bits >> 32)));
  const int32_t place = here(__builtin_amdgcn_ds_permute(4 * to, there ? m.few_at[lane] : -1));
  const double own = __builtin_bit_cast(double, (uint64_t)lo | (uint64_t)hi << 32);
  const double up_to = sum_up_to(own), total = from_lane(up_to, 63), line = set.u * total;
  const uint64_t over = __ballot(own > 0.0 && up_to > line), any = __ballot(own > 0.0);
  const int l = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)any);
  if (lane == l) {
    *token = place;
    if (chance) *chance = (float)(own / total);
  }
}

// A row's token from a source that has all of the row's keys from lo on, `keys` of them (lo 1: all there are); sum: the row's whole
// sum of weights (below 0: not known, the source has all).  false: what is kept may lie below lo.
template <typename Source>
HQ_DEV bool answer(const Source &source, const Weights &w, const Settings &set, uint32_t lo, uint32_t keys, double sum, int32_t *token,
                   float *chance, Scratch &m) {
  if (set.top_k == 1) {  // the lowest index of the largest
    uint32_t first = 0;
    source.sweep([&](const uint32_t k[4], int32_t i) {
#pragma unroll
      for (int c = 0; c < 4; c++)
        if (k[c] == w.top) first = max(first, ~(uint32_t)source.index(i + c));
      return true;
    });
    first = ~block_most(first, (uint32_t *)m.part);
    if (threadIdx.x == 0) {
      *token = (int32_t)first;
      if (chance) *chance = 1.0f;
    }
    return true;
  }
  Kept kept{lo, kAllTies};
  const float range = range_of(w);
  bool cut = false;  // top-k or top-p leave something out
  if (set.top_k) {
    if (keys < (uint32_t)set.top_k && lo > 1) return false;
    Search f(w, lo, range);
    f.template round<false>(source, set.top_k, m);
    if (f.through <= kFew) {
      const uint32_t n = gather(source, f.edge(), m, [&](uint32_t key) { return f.inside(key) && f.bin_of(key) <= f.bin; });
      draw_few(w, set, n, 0.0, token, chance, m);
      return true;
    }
    const Line k = line_of<false>(source, f, set.top_k, m);
    kept = Kept{k.key, (uint32_t)min((uint64_t)set.top_k - k.before, (uint64_t)k.equal)};
    cut = true;
  }
  if (set.top_p < 1.0) {
    double steps = sum * w.by;
    if (set.top_k || sum < 0.0) {
      uint64_t all = 0;
      source.sweep([&](const uint32_t k[4], int32_t) {
#pragma unroll
        for (int c = 0; c < 4; c++) all += k[c] > kept.t || (k[c] == kept.t && kept.ties == kAllTies) ? w.steps(k[c]) : 0;
        return true;
      });
      all = block_sum(all, m.part);
      if (kept.ties != kAllTies) all += kept.ties * w.steps(kept.t);
      steps = (double)all;
    }
    // (the first token is kept whatever its share)
    const double target = fmax(set.top_p * steps, 0.5);
    const float reach = reach_of(w, set.top_p, steps / w.by, set.top_k ? set.top_k : set.vocab);
    Search f(w, max(kept.t, floor_of(w, reach)), reach);
    f.template round<true>(source, target, m);
    // (the source ends before the line: all of it is kept)
    if (lo <= 1 || set.top_k || (double)(f.before + f.own) >= target) {
      if (f.through <= kFew) {
        const uint32_t n = gather(source, f.edge(), m, [&](uint32_t key) { return f.inside(key) && f.bin_of(key) <= f.bin; });
        draw_few(w, set, n, target, token, chance, m);
        return true;
      }
      const Line p = line_of<true>(source, f, target, m);
      const uint32_t equal = p.key == kept.t ? min(p.equal, kept.ties) : p.equal;
      kept = Kept{p.key, ties_of(p, equal, (double)w.steps(p.key), target)};
      cut = true;
    }
  }
  if (!cut && lo > 1 && !(w.of(lo) < set.min_p)) return false;  // (what the source lacks may have min_p)
  if (!cut && set.min_p > 0.0) {
    // (no float below this has it: a logarithm's and the difference's roundings are far below a millionth)
    const float least = (float)(w.most + (log(set.min_p) * 1.000001 - 1e-6) * 92.332482616893656877 / w.slope);
    const uint32_t edge = least > -3e38f && w.most < 3e38 ? max(key_of(least - fabsf(least) * 1e-6f), 1u) : 1u;
    const uint32_t n = gather(source, edge, m, [&](uint32_t key) { return key && (w.of(key) >= set.min_p || key == w.top); });
    if (n <= kFew) {
      Settings none = set;
      none.top_p = 1.0;  // (all of these are within it)
      draw_few(w, none, n, 0.0, token, chance, m);
      return true;
    }
  }
  draw(source, w, set, kept, token, chance, m);
  return true;
}

// ---- a row a block --------------------------------------------------------------------------------------------------
HQ_DEV void none(const Sample &a, int64_t row) {
  if (threadIdx.x == 0) {
    a.tokens[row] = -1;
    if (a.chance) a.chance[row] = 0.0f;
  }
}

template <bool WIDE>
__global__ __launch_bounds__(kThreads) void row_kernel(Sample a, double by) {
  __shared__ Scratch m;
  __shared__ uint32_t keys[kHeld];
  const int64_t row = blockIdx.x;
  const Settings set = settings_of(a, row);
  if (threadIdx.x < 64) m.roots[threadIdx.x] = kRoots[threadIdx.x];
  const Row<WIDE, 2> from((const float *)(a.logits + row * a.stride), a.vocab);
  uint32_t top = 0;
  from.sweep([&](const uint32_t k[4], int32_t i) {
    *(uint4 *)(keys + i) = make_uint4(k[0], k[1], k[2], k[3]);
    top = max(max(top, max(k[0], k[1])), max(k[2], k[3]));
    return true;
  });
  top = block_most(top, (uint32_t *)m.part);
  if (!top) return none(a, row);
  const List<true> source(keys, nullptr, a.vocab);
  const Weights w{top, (double)value_of(top), slope_of(set.temperature), by, m.roots};
  answer(source, w, set, 1u, 0, -1.0, a.tokens + row, a.chance ? a.chance + row : nullptr, m);
}

// ---- a row over many blocks -----------------------------------------------------------------------------------------
// What a wave of the first launch leaves: its largest key, its line (it handed on all from there on; 1: all that there are), how
// many it handed on, and of each of its grains (grain 4 j + s in counts[s][j & 1], byte 3 - j / 2), its weights' sum relative to its largest, and each grain's,
// where nothing is cut off
struct alignas(16) Note {
  uint32_t counts[4][2];
  uint32_t top, line, handed;
  double sum, sums[kGrains];
};
struct Pair {
  uint32_t key, at;  // (the index, and from bit 20 on how many of its grain come before it)
};
static_assert(kMostVocab <= 1 << 20 && kGrain <= 1 << 12, "a pair's index");
// A row whose top-p reaches below what was handed on, spread over the whole vocabulary: the histogram over all of it, the keys of
// the bin in which top-p's line lies (kBand at most), and the sums of the parts' weights before that bin
constexpr int kParts = 16, kBand = 1024;
struct alignas(16) Wide {
  uint64_t weight[kBins];
  uint32_t count[kBins], keys[kBand], at[kBand];
  double sums[kParts], sum;
  float reach;
  uint32_t top, band;
};
struct Split {
  Wide *wide;       // [rows]
  uint32_t *rows;   // how many rows are wide, then which
  Note *notes;   // [rows][chunks]
  Pair *handed;  // [rows][chunks][kHand]
  int32_t chunks, lanes;  // waves a row; the lanes whose largest are to pass a wave's line
};

// What is computed from these four from here on is not kept from before, nor begun earlier: registers
HQ_DEV void anew(float v[4]) { asm volatile("" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3])); }

template <bool WIDE>
__global__ __launch_bounds__(256) void hand_kernel(Sample a, Split sp) {
  __shared__ double roots[64];
  const int lane = threadIdx.x & 63;
  const int32_t chunk = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int64_t row = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  if (row >= a.rows) return;
  // the lane's logits: 4 of grain (4 j + s) chunks + chunk of the row, s its 16 lanes
  const int32_t stride = 4 * sp.chunks * kGrain, from = (lane >> 4) * (stride / 4) + chunk * kGrain + 4 * (lane & 15);
  float v[4 * kBatch];
  if (chunk < sp.chunks)
    load<WIDE, kBatch>((const float *)(a.logits + row * a.stride), a.vocab, from, stride, a.vocab,
               ((kGrains - 1) * sp.chunks + chunk + 1) * kGrain <= a.vocab, v);
  if (row == 0 && blockIdx.x == 0 && threadIdx.x == 0) sp.rows[0] = 0;
  const Settings set = settings_of(a, row);
  if (set.whole_sum()) {
    if (threadIdx.x < 64) roots[threadIdx.x] = kRoots[threadIdx.x];
    __syncthreads();
  }
  if (chunk >= sp.chunks) return;
  Note *note = sp.notes + row * sp.chunks + chunk;
  float mine = -__builtin_huge_valf();
#pragma unroll
  for (int i = 0; i < 4 * kBatch; i++) mine = fmaxf(mine, v[i]);  // (NaN: the other)
  const uint32_t key = key_of(mine);
  const uint32_t top = wave_most(key);
  if (set.all()) {
    if (lane == 0) note->top = top;
  } else {
    // the line: so many lanes' largest are at or above it (the row's top_k, spread evenly, four times over)
    const int lanes = set.top_k == 1 ? 1 : set.top_k ? min(sp.lanes, 12 + 2 * (set.top_k / sp.chunks)) : sp.lanes;
    // (bits that all lanes' largest have in common are the line's)
    const uint32_t apart = top ^ ~wave_most(~key);
    uint32_t line = apart ? top & ~(UINT32_MAX >> __clz((int)apart)) : top;
    for (uint32_t bit = apart ? 1u << 31 >> __clz((int)apart) : 0u; bit; bit >>= 1) {
      const int above = __popcll(__ballot(key >= (line | bit)));
      if (above >= lanes) line |= bit;
      if (above == lanes) break;
    }
    line = line < kLowest ? 1u : line;
    // a bit for each of the lane's logits from the line on, the first the highest
    const auto mask_of = [&](float least) {
      uint32_t mask = 0;
#pragma unroll
      for (int i = 0; i < 4 * kBatch; i++) mask = 2 * mask + (v[i] >= least);
      return mask;
    };
    uint32_t mask = mask_of(value_of(max(line, kLowest)));
    uint32_t up_to = sum_up_to((uint32_t)__popc(mask)), total = from_lane(up_to, 63);
    if (total > kHand) {  // (equal ones by the dozen: those above them, if these are fewer)
      line = max(line, kLowest) + 1;
      mask = line <= top ? mask_of(value_of(line)) : 0u;
      up_to = sum_up_to((uint32_t)__popc(mask)), total = from_lane(up_to, 63);
      if (line > top || total > kHand) line = UINT32_MAX, mask = 0, total = 0;
    }
    // how many of each step's 4, in bytes (steps 0, 2, 4, 6 and 1, 3, 5, 7 from the top), then of its grain's before the lane's
    uint32_t pairs = mask - ((mask >> 1) & 0x55555555u);
    pairs = (pairs & 0x33333333u) + ((pairs >> 2) & 0x33333333u);
    const uint32_t even = (pairs >> 4) & 0x0f0f0f0fu, odd = pairs & 0x0f0f0f0fu;
    const uint32_t even_to = sum_row(even), odd_to = sum_row(odd), even_from = even_to - even, odd_from = odd_to - odd;
    const float *p = (const float *)(a.logits + row * a.stride);
    const uint32_t mask_all = mask;
    Pair *to = sp.handed + (row * sp.chunks + chunk) * kHand + (mask ? up_to - __popc(mask) : 0);
    while (mask) {
      const int bit = __clz((int)mask), j = bit >> 2;  // logit bit & 3 of step j
      const int32_t i = from + j * stride + (bit & 3);
      const uint32_t grain = ((j & 1 ? odd_from : even_from) >> (24 - 8 * (j >> 1))) & 0xffu;
      const uint32_t step = mask_all >> (28 - 4 * j) & 15u;  // (the step's 4 bits)
      *to++ = Pair{key_of(p[i]), (uint32_t)i | (grain + __popc(step >> (4 - (bit & 3)))) << 20};
      mask &= ~(0x80000000u >> bit);
    }
    if ((lane & 15) == 15) *(uint2 *)note->counts[lane >> 4] = make_uint2(even_to, odd_to);
    if (lane == 0) note->top = top, note->line = line, note->handed = total;
  }
  if (!set.whole_sum()) return;
  const double slope = slope_of(set.temperature), most = (double)value_of(top);
  double sum = 0.0;
#pragma unroll
  for (int j = 0; j < kBatch; j++) {
    anew(v + 4 * j);
    double s = 0.0;
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const float x = v[4 * j + c];
      const double e = power((double)x - most, slope, roots);
      s += x == value_of(top) ? 1.0 : x > -__builtin_huge_valf() ? e : 0.0;
    }
    if (set.all()) {  // (the 16 lanes' last has their sum)
      const double grain = sum_row(s);
      if ((lane & 15) == 15) note->sums[4 * j + (lane >> 4)] = top ? grain : 0.0;
    }
    sum += s;
    __builtin_amdgcn_sched_barrier(0);
  }
  sum = wave_sum(sum);
  if (lane == 0) note->sum = top ? sum : 0.0;
}

struct Joint {
  Scratch m;
  uint16_t offset[kMostVocab / kGrain + kGrains];  // a grain's place in the list
  uint32_t keys[kList + kStep];
  int32_t at[kList + kStep];
};

// nothing is cut off: the grain in which the sum is reached by what the first launch summed, then its 64 logits
template <bool WIDE>
HQ_DEV void draw_of_all(const Sample &a, const Split &sp, int64_t row, const Weights &w, double u, Scratch &m) {
  const Note *notes = sp.notes + row * sp.chunks;
  const int32_t grains = kGrains * sp.chunks, each = (grains + kThreads - 1) / kThreads, first = threadIdx.x * each;
  const auto sum_of = [&](int32_t i) {
    if (i >= grains) return 0.0;
    const Note &n = notes[i % sp.chunks];
    return n.top ? n.sums[i / sp.chunks] * w.of(n.top) : 0.0;
  };
  double mine = 0.0, total;
  for (int32_t i = first; i < first + each; i++) mine += sum_of(i);
  const double before = sum_before(mine, (double *)m.part, total), target = u * total;
  // the thread in whose grains the target is passed, or the last that has any
  if (threadIdx.x == 0) m.found[0] = UINT64_MAX, m.found[1] = 0;
  __syncthreads();
  if (mine > 0.0) {
    atomicMax((unsigned long long *)&m.found[1], (unsigned long long)threadIdx.x);
    if (before + mine > target) atomicMin((unsigned long long *)&m.found[0], (unsigned long long)threadIdx.x);
  }
  __syncthreads();
  const bool passed = m.found[0] != UINT64_MAX;
  if (threadIdx.x == (passed ? m.found[0] : m.found[1])) {
    double run = before, start = before;
    int32_t which = -1;
    for (int32_t i = first; i < first + each; i++) {
      const double s = sum_of(i);
      if (s > 0.0 && (which < 0 || !passed || !(run > target))) which = i, start = run;
      run += s;
    }
    m.found[2] = (uint64_t)which;
    m.sums[0] = start;
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const int lane = threadIdx.x;
  const float *p = (const float *)(a.logits + row * a.stride);
  // (a grain whose sum is some smallest number may have no weight that is one: then the next, or the one before)
  for (int32_t g = (int32_t)m.found[2]; g >= 0 && g < grains; g += passed ? 1 : -1) {
    const int32_t i = g * kGrain + lane;
    const float v = p[min(i, a.vocab - 1)];
    const double x = i < a.vocab ? w.of(key_of(v)) : 0.0, up_to = sum_up_to(x);
    const uint64_t over = __ballot(x > 0.0 && m.sums[0] + up_to > target), any = __ballot(x > 0.0);
    if (!any) continue;
    if (lane == (over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)any))) {
      a.tokens[row] = i;
      if (a.chance) a.chance[row] = (float)(x / total);
    }
    return;
  }
}

template <bool WIDE>
__global__ __launch_bounds__(kThreads) void join_kernel(Sample a, Split sp, double by) {
  __shared__ Joint s;
  Scratch &m = s.m;
  const int64_t row = blockIdx.x;
  const Settings set = settings_of(a, row);
  const Note *notes = sp.notes + row * sp.chunks;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // the first of what the first chunks handed on, or whatever lies there, on its way before anything is known
  constexpr int kEarly = 4;
  const Pair *handed = sp.handed + row * sp.chunks * kHand;
  const auto handed_by = [&](int32_t c) { return (int32_t)notes[c].handed; };
  Pair early[kEarly];
  int32_t early_n[kEarly];
#pragma unroll
  for (int i = 0; i < kEarly; i++) {
    const int32_t c = min(wave + i * kWaves, sp.chunks - 1);
    early[i] = handed[c * kHand + lane];
    early_n[i] = handed_by(c);
  }
  if (threadIdx.x < 64) m.roots[threadIdx.x] = kRoots[threadIdx.x];
  // (grains in order of the row: number (4 j + s) chunks + c is chunk c's grain 4 j + s)
  const int32_t grains = kGrains * sp.chunks;
  uint32_t top = 0, line = 0;  // the largest key, and the highest line
  for (int32_t c = threadIdx.x; c < sp.chunks; c += kThreads) {
    top = max(top, notes[c].top);
    if (set.all()) continue;
    line = max(line, notes[c].line);
    const uint4 q[2] = {*(const uint4 *)notes[c].counts[0], *(const uint4 *)notes[c].counts[2]};
    const uint32_t d[8] = {q[0].x, q[0].y, q[0].z, q[0].w, q[1].x, q[1].y, q[1].z, q[1].w};
#pragma unroll
    for (int g = 0; g < kGrains; g++)
      s.offset[g * sp.chunks + c] = (uint16_t)((d[2 * (g & 3) + ((g >> 2) & 1)] >> (24 - 8 * (g >> 3))) & 0xffu);
  }
  top = block_most(top, (uint32_t *)m.part);
  line = block_most(line, (uint32_t *)m.part + kWaves);
  if (!top) return none(a, row);
  const Weights w{top, (double)value_of(top), slope_of(set.temperature), by, m.roots};
  if (set.all()) return draw_of_all<WIDE>(a, sp, row, w, set.u, m);
  double sum = -1.0;  // the row's sum of weights, by its chunks' largest
  if (set.whole_sum()) {
    sum = 0.0;
    for (int32_t c = threadIdx.x; c < sp.chunks; c += kThreads)
      if (notes[c].top) sum += notes[c].sum * w.of(notes[c].top);
    sum = block_sum(sum, (double *)m.part);
  }
  // each grain's place in the list
  const int32_t each = (grains + kThreads - 1) / kThreads, first = min((int32_t)threadIdx.x * each, grains), last = min(first + each, grains);
  uint32_t mine = 0, total;
  for (int32_t i = first; i < last; i++) mine += s.offset[i];
  uint32_t before = sum_before(mine, (uint32_t *)m.part, total);
  for (int32_t i = first; i < last; i++) {
    const uint32_t n = s.offset[i];
    s.offset[i] = (uint16_t)before;  // (where it does not fit, neither does the list)
    before += n;
  }
  __syncthreads();
  const int32_t n = (int32_t)total;
  if (n <= kList && line <= top) {
    uint32_t keys = 0;
    const auto place = [&](const Pair &pair) {
      const int32_t i = (int32_t)(pair.at & (kMostVocab - 1));
      const uint32_t to = s.offset[i / kGrain] + (pair.at >> 20);
      s.keys[to] = pair.key >= line ? pair.key : 0u;
      s.at[to] = i;
      keys += pair.key >= line;
    };
#pragma unroll
    for (int i = 0; i < kEarly; i++) {
      const int32_t c = wave + i * kWaves;
      if (c >= sp.chunks) break;
      if (lane < early_n[i]) place(early[i]);
      for (int32_t e = lane + 64; e < early_n[i]; e += 64) place(handed[c * kHand + e]);
    }
    for (int32_t c = wave + kEarly * kWaves; c < sp.chunks; c += kWaves)
      for (int32_t e = lane, n = handed_by(c); e < n; e += 64) place(handed[c * kHand + e]);
    if ((int32_t)threadIdx.x < kStep) s.keys[n + threadIdx.x] = 0;
    keys = block_sum(keys, (uint32_t *)m.part);
    const List<false> source(s.keys, s.at, n);
    if (answer(source, w, set, max(line, 1u), keys, sum, a.tokens + row, a.chance ? a.chance + row : nullptr, m)) return;
  }
  if (!set.top_k && set.top_p < 1.0) {  // the wide kernels go on
    Wide &wide = sp.wide[row];
    wide.weight[threadIdx.x] = 0, wide.count[threadIdx.x] = 0;
    if (threadIdx.x == 0) {
      wide.sum = sum, wide.reach = reach_of(w, set.top_p, sum, a.vocab), wide.top = top, wide.band = 0;
      sp.rows[1 + atomicAdd(&sp.rows[0], 1u)] = (uint32_t)row;
    }
    return;
  }
  __syncthreads();
  const Row<WIDE> source((const float *)(a.logits + row * a.stride), a.vocab);
  answer(source, w, set, 1u, 0, sum, a.tokens + row, a.chance ? a.chance + row : nullptr, m);
}

// ---- wide rows: a part of one a block at a time ---------------------------------------------------------------------
template <bool WIDE>
using Part = Row<WIDE, 2>;
// (parts begin on whole steps; the last may be short, or empty)
HQ_DEV int32_t part_of(int32_t vocab) { return (vocab + kParts * kStep - 1) / (kParts * kStep) * kStep; }

struct Item {  // a wide row's part
  int64_t row;
  int32_t part, from, n;
};
HQ_DEV Item item_of(const Sample &a, const Split &sp, uint32_t item) {
  Item o;
  o.row = sp.rows[1 + item / kParts], o.part = (int32_t)(item % kParts);
  o.from = min(o.part * part_of(a.vocab), a.vocab);
  o.n = min(part_of(a.vocab), a.vocab - o.from);
  return o;
}
HQ_DEV Weights weights_of(const Wide &wide, const Settings &set, double by, const double *roots) {
  return Weights{wide.top, (double)value_of(wide.top), slope_of(set.temperature), by, roots};
}

template <bool WIDE>
__global__ __launch_bounds__(kThreads) void tally_kernel(Sample a, Split sp, double by) {
  __shared__ Scratch m;
  if (threadIdx.x < 64) m.roots[threadIdx.x] = kRoots[threadIdx.x];
  const uint32_t items = sp.rows[0] * kParts;
  for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
    const Item it = item_of(a, sp, item);
    Wide &wide = sp.wide[it.row];
    const Weights w = weights_of(wide, settings_of(a, it.row), by, m.roots);
    Search f(w, floor_of(w, wide.reach), wide.reach);
    f.template tally<true>(Part<WIDE>((const float *)(a.logits + it.row * a.stride), it.n, it.from), m);
    if (m.count[threadIdx.x]) {
      atomicAdd(&wide.count[threadIdx.x], m.count[threadIdx.x]);
      atomicAdd((unsigned long long *)&wide.weight[threadIdx.x], (unsigned long long)m.weight[threadIdx.x]);
    }
  }
}

struct Band {
  Scratch m;
  uint32_t keys[kBand + kStep];
  int32_t at[kBand + kStep];
  uint32_t sorted[kBand];
  int32_t sorted_at[kBand];
  double starts[kParts + 1], sums[kParts];  // the band's kept weights before each part, the parts' before the band
  uint32_t tied[kParts + 1], any[kParts];  // (and how many of its equals of the line; whether the part keeps one of its keys)
};

// the search of a wide row, its first round done (the histogram is brought into m)
HQ_DEV void find_in(const Wide &wide, Search &f, double target, Scratch &m) {
  f.shift = max(22 - (int)__builtin_clz((f.hi - f.lo) | 1u), 0);
  __syncthreads();
  m.weight[threadIdx.x] = wide.weight[threadIdx.x], m.count[threadIdx.x] = wide.count[threadIdx.x];
  __syncthreads();
  f.template find<true>(target, m);
}
HQ_DEV double target_of(const Wide &wide, const Settings &set, double by) { return fmax(set.top_p * (wide.sum * by), 0.5); }

// of a wide row the sum of each part's weights before the line's bin, and that bin's keys
template <bool WIDE>
__global__ __launch_bounds__(kThreads) void wide_kernel(Sample a, Split sp, double by) {
  __shared__ Scratch m;
  if (threadIdx.x < 64) m.roots[threadIdx.x] = kRoots[threadIdx.x];
  const uint32_t items = sp.rows[0] * kParts;
  for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
    const Item it = item_of(a, sp, item);
    Wide &wide = sp.wide[it.row];
    const Settings set = settings_of(a, it.row);
    const Weights w = weights_of(wide, set, by, m.roots);
    const float *p = (const float *)(a.logits + it.row * a.stride);
    Search f(w, floor_of(w, wide.reach), wide.reach);
    find_in(wide, f, target_of(wide, set, by), m);
    const uint32_t edge = f.edge();
    double sum = 0.0;
    const Part<WIDE> source(p, it.n, it.from);
    source.sweep([&](const uint32_t k[4], int32_t i) {
#pragma unroll
      for (int c = 0; c < 4; c++) {
        if (k[c] < edge || !f.inside(k[c])) continue;
        const int bin = f.bin_of(k[c]);
        if (bin < f.bin) {
          const double x = w.of(k[c]);
          sum += x >= set.min_p || k[c] == w.top ? x : 0.0;
        } else if (bin == f.bin) {
          const uint32_t to = atomicAdd(&wide.band, 1u);
          if (to < kBand) wide.keys[to] = k[c], wide.at[to] = (uint32_t)source.index(i + c);
        }
      }
      return true;
    });
    sum = block_sum(sum, (double *)m.part);
    if (threadIdx.x == 0) wide.sums[it.part] = sum;
  }
}

// of a wide row the line among its bin's keys, then the token
template <bool WIDE>
__global__ __launch_bounds__(kThreads) void end_kernel(Sample a, Split sp, double by) {
  __shared__ Band b;
  Scratch &m = b.m;
  if (threadIdx.x < 64) m.roots[threadIdx.x] = kRoots[threadIdx.x];
  if (blockIdx.x >= sp.rows[0]) return;
  const int64_t row = sp.rows[1 + blockIdx.x];
  const Wide &wide = sp.wide[row];
  const Settings set = settings_of(a, row);
  const Weights w = weights_of(wide, set, by, m.roots);
  const float *p = (const float *)(a.logits + row * a.stride);
  const double target = target_of(wide, set, by);
  Search f(w, floor_of(w, wide.reach), wide.reach);
  find_in(wide, f, target, m);
  const int32_t n = (int32_t)wide.band;
  for (int i = threadIdx.x; i < kBand + kStep; i += kThreads) {
    b.keys[i] = i < n && i < kBand ? wide.keys[i] : 0u;
    b.at[i] = i < n && i < kBand ? (int32_t)wide.at[i] : INT32_MAX;
  }
  if (threadIdx.x < kParts) b.sums[threadIdx.x] = wide.sums[threadIdx.x], b.any[threadIdx.x] = 0;
  __syncthreads();
  f.some = b.keys[0];  // (a bin of one key)
  const bool fits = n <= kBand;  // (else equal ones by the thousand: the whole row again)
  Line line;
  if (fits) {
    line = line_of<true>(List<false>(b.keys, b.at, n), f, target, m);
  } else {
    while (f.narrow() && f.template round<true>(Part<WIDE>(p, a.vocab), target, m)) {}
    line = Line{f.some, f.before, f.equal};
  }
  Kept kept{line.key, ties_of(line, line.equal, (double)w.steps(line.key), target)};
  int32_t from = 0, to = a.vocab;
  double total = 0.0, lead = 0.0;
  if (fits) {
    // the bin's keys by index
    if ((int)threadIdx.x < n) {
      const int32_t at = b.at[threadIdx.x];
      int rank = 0;
#pragma unroll 2
      for (int i = 0; i < n; i += 4) {
        const int4 q = *(const int4 *)(b.at + i);
        rank += (q.x < at) + (q.y < at) + (q.z < at) + (q.w < at);
      }
      b.sorted[rank] = b.keys[threadIdx.x], b.sorted_at[rank] = at;
    }
    __syncthreads();
    const bool there = (int)threadIdx.x < n;
    const uint32_t key = there ? b.sorted[threadIdx.x] : 0u;
    uint32_t ties;
    const uint32_t tied = sum_before((uint32_t)(there && key == kept.t), (uint32_t *)m.part, ties);
    const double x = w.of(key);
    const bool in = there && (key > kept.t || (key == kept.t && tied < kept.ties)) && (x >= set.min_p || key == w.top);
    const double before = sum_before(in ? x : 0.0, m.sums, total);
    // what comes before each part
    const int32_t per = part_of(a.vocab);
    const int part = there ? b.sorted_at[threadIdx.x] / per : kParts;
    const int part_before = threadIdx.x && (int)threadIdx.x <= n ? b.sorted_at[threadIdx.x - 1] / per : -1;
    if (in && x > 0.0) b.any[part] = 1;
    if ((int)threadIdx.x <= n)
      for (int q = part_before + 1; q <= part; q++) b.starts[q] = before, b.tied[q] = tied;
    if (n == kBand && threadIdx.x == kThreads - 1)
      for (int q = part + 1; q <= kParts; q++) b.starts[q] = total, b.tied[q] = ties;
    __syncthreads();
#pragma unroll 1
    for (int q = 0; q < kParts; q++) total += b.sums[q];
    // the part in which the sum is reached (none: the last that has any)
    double run = 0.0;
    int which = 0;
    bool passed = false;
#pragma unroll 1
    for (int q = 0; q < kParts; q++) {
      // (not by starts' difference: two sums over the same keys may differ by a rounding)
      if (!passed && (b.sums[q] > 0.0 || b.any[q])) which = q, lead = run + b.starts[q], passed = run + b.sums[q] + b.starts[q + 1] > set.u * total;
      run += b.sums[q];
    }
    from = min(which * per, a.vocab), to = min(from + per, a.vocab);
    kept.ties -= min(b.tied[which], kept.ties);
  }
  __syncthreads();
  draw(Part<WIDE>(p, to - from, from), w, set, kept, a.tokens + row, a.chance ? a.chance + row : nullptr, m, total, lead);
}

int32_t chunks_of(int32_t vocab) { return (int32_t)(((int64_t)vocab + kBatch * kStep - 1) / (kBatch * kStep)); }
int64_t notes_bytes(int64_t rows, int32_t vocab) { return (rows * chunks_of(vocab) * (int64_t)sizeof(Note) + 255) / 256 * 256; }

}  // namespace

int64_t sample_work_bytes(int32_t rows, int32_t vocab) {
  if (vocab <= kHeld) return 0;
  return notes_bytes(rows, vocab) + (int64_t)rows * (chunks_of(vocab) * kHand * (int64_t)sizeof(Pair) + (int64_t)sizeof(Wide) + 4) + 4;
}

hipError_t launch_sample(const Sample &a, hipStream_t s) {
  if (a.rows <= 0 || a.vocab <= 0) return hipSuccess;
  // (a weight's steps stay below 2^52, a row's below 2^62)
  int bits = 0;
  while (((int64_t)1 << bits) < a.vocab) bits++;
  const double by = (double)((int64_t)1 << std::min(51, 62 - bits));
  const bool wide = a.vocab >= 4 && (uintptr_t)a.logits % 16 == 0 && (a.rows == 1 || a.stride % 16 == 0);
  if (a.vocab <= kHeld) {
    hipLaunchKernelGGL(wide ? row_kernel<true> : row_kernel<false>, dim3((uint32_t)a.rows), dim3(kThreads), 0, s, a, by);
    return hipGetLastError();
  }
  Split sp{};
  sp.chunks = chunks_of(a.vocab);
  sp.notes = (Note *)a.work;
  sp.handed = (Pair *)(a.work + notes_bytes(a.rows, a.vocab));
  sp.wide = (Wide *)(sp.handed + (int64_t)a.rows * sp.chunks * kHand);
  sp.rows = (uint32_t *)(sp.wide + a.rows);
  // The lanes whose largest of 32 logits pass a wave's line, so that evenly spread logits hand on some 5500 of a row: of a share q of
  // the logits above the line, a lane has one with chance 1 - (1 - q)^32.  At most 48, which hand on 90 of a wave's 2048.
  const double share = std::min(1.0, 5500.0 / ((double)sp.chunks * kBatch * kStep));
  sp.lanes = std::min(48, std::max(1, (int)(64.0 * (1.0 - std::pow(1.0 - share, 4.0 * kBatch)))));
  const uint32_t wide_rows = (uint32_t)std::min(a.rows, 32768);
  const dim3 grid((uint32_t)((sp.chunks + 3) / 4), wide_rows, ((uint32_t)a.rows + wide_rows - 1) / wide_rows);
  hipLaunchKernelGGL(wide ? hand_kernel<true> : hand_kernel<false>, grid, dim3(256), 0, s, a, sp);
  if (const hipError_t e = hipGetLastError()) return e;
  hipLaunchKernelGGL(wide ? join_kernel<true> : join_kernel<false>, dim3((uint32_t)a.rows), dim3(kThreads), 0, s, a, sp, by);
  if (const hipError_t e = hipGetLastError()) return e;
  if (!a.top_p) return hipSuccess;
  // rows that top-p leaves wide: how many is known there; a block a compute unit, which ends at once where there are none
  const dim3 blocks((uint32_t)std::min<int64_t>(cu_count(), (int64_t)a.rows * kParts));
  hipLaunchKernelGGL(wide ? tally_kernel<true> : tally_kernel<false>, blocks, dim3(kThreads), 0, s, a, sp, by);
  if (const hipError_t e = hipGetLastError()) return e;
  hipLaunchKernelGGL(wide ? wide_kernel<true> : wide_kernel<false>, blocks, dim3(kThreads), 0, s, a, sp, by);
  if (const hipError_t e = hipGetLastError()) return e;
  hipLaunchKernelGGL(wide ? end_kernel<true> : end_kernel<false>, dim3((uint32_t)a.rows), dim3(kThreads), 0, s, a, sp, by);
  return hipGetLastError();
}

}  // namespace hq
