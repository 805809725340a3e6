// sample.hip — the next token of each row of logits from a given random number: temperature, top-k, top-p, min-p.
//
// A logit is held as its key, a 32-bit number that orders as the float does (0: never drawn).  What top-k and top-p leave is a
// smallest key t and how many of the logits equal to it (the first by index); both are found by histograms over the keys,
// round by round in the bin where the count (or the weight) passes the line, until a bin holds one key.  Weights in
// histograms are whole numbers (steps of a power of two below the largest weight), so that no order of additions changes them.
// The token is then found by a sum over the kept weights in index order, in 64 bits.
//
// Rows of up to 32768 logits: a block a row, whose keys stay in LDS.  Longer rows: every wave of a first launch takes
// 2048 logits of a row and hands on those above a line of its own, some 90 at most (with what they sum to, where the settings
// ask for the row's whole sum); a block a row of a second launch finds t among what was handed on, and goes to the row itself
// only where t lies below one of these lines.  A wave's logits are 8 stripes of 256 over the whole row: words that stand out
// often have neighbouring numbers.
#include <algorithm>
#include <cmath>

#include "common.hpp"
#include "launch.hpp"

namespace hq {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = kThreads;
constexpr int kStep = 256;               // logits a wave takes at a time, 4 a lane
constexpr int kBatch = 8;                // steps whose loads are on their way together
constexpr int kHeld = 32768, kSmall = 8192;  // the longest rows that a block holds in LDS (alone on its compute unit, beside others)
constexpr int kHand = 128;               // logits that a wave of the first launch can hand on
constexpr int kList = 7680;              // and what the second launch takes of a row (two blocks a compute unit)
constexpr uint32_t kLowest = 0x00800000u;  // the key of the lowest finite number

HQ_DEV uint32_t key_of(float v) {
  const uint32_t bits = __float_as_uint(fadd(v, 0.0f));  // (-0 orders as 0)
  return v > -__builtin_huge_valf() ? bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u) : 0u;
}
HQ_DEV float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

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
// over 720 is below 2^-54), scaled by whole powers of two.  A third of the library's instructions; within 2^-50 of it.
HQ_DEV double power(double d, double c, const double *roots) {
  const double y = fmax(d * c, -70000.0), whole = rint(y), f = y - whole;
  const int n = (int)whole;
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
  double most, slope, by;  // the largest logit; by: 1 / step
  const double *roots;
  HQ_DEV double of(uint32_t key) const {
    const double x = power((double)value_of(key) - most, slope, roots);
    return key == top ? 1.0 : key ? x : 0.0;
  }
  HQ_DEV uint64_t steps(uint32_t key) const { return (uint64_t)(of(key) * by + 0.5); }
};

struct Settings {
  double temperature, top_p, min_p, u;
  int32_t top_k;  // (0: all)
  HQ_DEV bool all() const { return !top_k && !(top_p < 1.0) && !(min_p > 0.0); }
  HQ_DEV bool whole_sum() const { return !top_k && (top_p < 1.0 || !(min_p > 0.0)); }  // the row's whole sum is needed
};
HQ_DEV Settings settings_of(const Sample &a, int64_t row) {
  Settings o;
  o.temperature = a.temperature ? a.temperature[row] : 1.0f;
  o.top_k = a.top_k ? max(a.top_k[row], 0) : 0;
  if (o.top_k >= a.vocab) o.top_k = 0;
  o.top_p = a.top_p ? a.top_p[row] : 1.0f;
  o.min_p = a.min_p ? a.min_p[row] : 0.0f;
  o.min_p = o.min_p > 0.0 ? fmin(o.min_p, 1.0) : 0.0;
  o.u = a.u[row];
  if (!(o.u >= 0.0)) o.u = 0.0;
  if (!(o.temperature > 0.0)) o.temperature = 1.0, o.top_k = 1;
  return o;
}

// ---- sums over a block ----------------------------------------------------------------------------------------------
// (every thread calls; `part`: kWaves doublewords of LDS that nothing else uses)
template <typename T, typename Op>
HQ_DEV T block_all(T v, T *part, Op op) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = op(v, (T)__shfl_xor(v, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[threadIdx.x & (kWaves - 1)];
#pragma unroll
  for (int o = kWaves / 2; o > 0; o >>= 1) v = op(v, (T)__shfl_xor(v, o, kWaves));
  return v;
}
struct Add {
  template <typename T> HQ_DEV T operator()(T x, T y) const { return x + y; }
};
struct Most {
  template <typename T> HQ_DEV T operator()(T x, T y) const { return x > y ? x : y; }
};

// the sum over the threads before this one
template <typename T>
HQ_DEV T sum_before(T v, T *part, T &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T sum = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T other = __shfl_up(sum, o, 64);
    if (lane >= o) sum += other;
  }
  __syncthreads();
  if (lane == 63) part[wave] = sum;
  __syncthreads();
  // (a lane a wave: the sums up to each)
  T waves = part[lane & (kWaves - 1)];
#pragma unroll
  for (int o = 1; o < kWaves; o <<= 1) {
    const T other = __shfl_up(waves, o, kWaves);
    if ((lane & (kWaves - 1)) >= o) waves += other;
  }
  total = __shfl(waves, kWaves - 1, kWaves);
  const T before = wave ? __shfl(waves, wave - 1, kWaves) : (T)0;
  return before + (sum - v);
}

struct Scratch {
  double roots[64];
  union {
    struct {
      uint64_t weight[kBins];
      uint32_t count[kBins], some[kBins];  // (a key of the bin)
    };
    uint32_t offset[4 * kBins];  // (the second launch: a step's place in the list)
  };
  uint64_t part[kWaves];
  uint64_t found[4];
  double sums[kWaves];
  uint32_t ties[kWaves];
};

// ---- where a row's keys are -----------------------------------------------------------------------------------------
// A wave takes a part of the row, `part` logits (whole steps) from wave * part on, a step's 4 a lane at a time, in order:
// sweep(f) calls f(keys, the first's place) until it returns false.

// 8 steps of logits, `stride` apart from `from` on; -infinity from `to` on
template <bool WIDE>
HQ_DEV void load(const float *p, int32_t n, int32_t from, int32_t stride, int32_t to, float v[4 * kBatch]) {
  const int lane = threadIdx.x & 63;
  if (from + (kBatch - 1) * stride + kStep <= to) {
#pragma unroll
    for (int j = 0; j < kBatch; j++) {
      const float *q = p + from + j * stride + 4 * lane;
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
  for (int j = 0; j < kBatch; j++) {
    const int32_t i = from + j * stride + 4 * lane;
#pragma unroll
    for (int c = 0; c < 4; c++) v[4 * j + c] = p[min(i + c, n - 1)];
#pragma unroll
    for (int c = 0; c < 4; c++)
      if (i + c >= to) v[4 * j + c] = -__builtin_huge_valf();
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <bool WIDE>
struct Row {  // a row in memory
  const float *p;
  int32_t n, part;
  HQ_DEV Row(const float *p_, int32_t n_) : p(p_), n(n_), part((n_ + kWaves * kStep - 1) / (kWaves * kStep) * kStep) {}
  HQ_DEV int32_t index(int32_t i) const { return i; }
  template <typename F>
  HQ_DEV void sweep(F f) const {
    const int32_t from = (int32_t)(threadIdx.x >> 6) * part, to = min(from + part, n);
    for (int32_t i0 = from; i0 < to; i0 += kBatch * kStep) {
      float v[4 * kBatch];
      load<WIDE>(p, n, i0, kStep, to, v);
#pragma unroll
      for (int j = 0; j < kBatch; j++) {
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

// The first key, from the top downward, up to and with whose equals the count (the weight) of the keys is `target` or more; those below
// lo do not count.  Not reached: the smallest key there is.  The first round's bins lie evenly over `range` below the
// largest value, the rest in the last (logits on both sides of 0 would crowd a few bins of keys), those after it evenly over the keys.
template <bool WEIGHT, typename Source>
HQ_DEV Line line_of(const Source &source, const Weights &w, uint32_t lo, float range, double target, Scratch &m) {
  uint32_t hi = w.top;
  Line o{hi, 0, 0};
  const float most = (float)w.most, per = (kBins - 0.5f) / range;
  bool values = most < __builtin_huge_valf() && range > 0.0f && per > 0.0f && per < __builtin_huge_valf();
  const auto value_bin = [&](uint32_t key) { return (int)fminf((most - value_of(key)) * per, kBins - 1.0f); };
  while (true) {
    const int shift = max(22 - (int)__builtin_clz((hi - lo) | 1u), 0);  // hi - lo in 10 bits
    __syncthreads();
    m.count[threadIdx.x] = 0;
    if (WEIGHT) m.weight[threadIdx.x] = 0;
    if (threadIdx.x == 0) m.found[0] = 0;
    __syncthreads();
    source.sweep([&](const uint32_t keys[4], int32_t) {
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const uint32_t key = keys[c];
        if (key < lo || key > hi) continue;
        const int bin = values ? value_bin(key) : (int)((hi - key) >> shift);
        atomicAdd(&m.count[bin], 1u);
        if (WEIGHT) atomicAdd((unsigned long long *)&m.weight[bin], (unsigned long long)w.steps(key));
        m.some[bin] = key;
      }
      return true;
    });
    __syncthreads();
    const uint32_t count = m.count[threadIdx.x];
    uint64_t all;
    const uint64_t before = o.before + sum_before(WEIGHT ? m.weight[threadIdx.x] : (uint64_t)count, m.part, all);
    // the last bin with anything in it that begins before the line
    if (count && (double)before < target) atomicMax((unsigned long long *)&m.found[0], (unsigned long long)threadIdx.x + 1);
    __syncthreads();
    const int bin = (int)m.found[0] - 1;
    if (bin < 0) return o;
    if ((int)threadIdx.x == bin) m.found[1] = before;
    __syncthreads();
    o.before = m.found[1];
    o.equal = m.count[bin];
    o.key = m.some[bin];
    if (o.equal == 1) return o;
    if (values) {
      const uint32_t from = first_key(lo, hi, [&](uint32_t key) { return value_bin(key) <= bin; });
      if (bin > 0) hi = first_key(lo, hi, [&](uint32_t key) { return value_bin(key) < bin; }) - 1;
      lo = from;
      values = false;
    } else {
      if (shift == 0) return o;
      const uint32_t top = hi - ((uint32_t)bin << shift), width = (1u << shift) - 1;
      lo = top - lo > width ? top - width : lo;
      hi = top;
    }
    if (lo == hi) return o;
  }
}

// what top-k, top-p and min-p leave: keys above t, and the first `ties` of those equal to it; weights below min_p not
struct Kept {
  uint32_t t, ties;
  bool known;  // (false: t may lie below the keys that the source has)
};
constexpr uint32_t kAllTies = UINT32_MAX;

// lo: the source has all of the row's keys from lo on, `keys` of them (lo 1: all there are); sum: the row's whole sum of weights
// (below 0: not known, the source has all)
template <typename Source>
HQ_DEV Kept kept_of(const Source &source, const Weights &w, const Settings &set, uint32_t lo, int64_t keys, double sum, Scratch &m) {
  Kept o{lo, kAllTies, true};
  if (set.top_k == 1) return Kept{w.top, 1, true};
  const float range = (float)fmin(40.0 * 92.332482616893656877 / w.slope, 3e38);
  if (set.top_k) {
    if (keys < set.top_k && lo > 1) return Kept{0, 0, false};
    const Line k = line_of<false>(source, w, lo, range, (double)set.top_k, m);
    o.t = k.key, o.ties = (uint32_t)min((uint64_t)set.top_k - k.before, (uint64_t)k.equal);
  }
  // nothing that the source lacks can have min_p or more
  const bool low = lo <= 1 || set.top_k || w.of(lo) < set.min_p;
  if (!(set.top_p < 1.0)) return Kept{o.t, o.ties, low};
  double steps = sum * w.by;
  if (set.top_k || sum < 0.0) {
    uint64_t all = 0;
    source.sweep([&](const uint32_t k[4], int32_t) {
#pragma unroll
      for (int c = 0; c < 4; c++) all += k[c] > o.t || (k[c] == o.t && o.ties == kAllTies) ? w.steps(k[c]) : 0;
      return true;
    });
    all = block_all(all, m.part, Add());
    if (o.ties != kAllTies) all += o.ties * w.steps(o.t);
    steps = (double)all;
  }
  // (the first token is kept whatever its share)
  const double target = fmax(set.top_p * steps, 0.5);
  const Line p = line_of<true>(source, w, max(o.t, 1u), range, target, m);
  const uint32_t equal = p.key == o.t ? min(p.equal, o.ties) : p.equal;
  const uint64_t each = w.steps(p.key);
  if (lo > 1 && !set.top_k && (double)(p.before + equal * each) < target) return Kept{o.t, o.ties, low};  // (all of the source is kept)
  // ties j = 0, 1, .. with before + j each < target
  const double room = (target - (double)p.before) / (double)each;
  uint32_t ties = room < (double)equal ? (uint32_t)ceil(room) : equal;
  while (ties > 1 && !((double)p.before + (double)(ties - 1) * (double)each < target)) ties--;
  return Kept{p.key, max(ties, 1u), true};
}

// ---- the token ------------------------------------------------------------------------------------------------------
// The first by index whose kept weights up to it are more than u times all.  Each wave sums its part, then the wave in whose part the
// sum is reached goes through it again.
template <typename Source>
HQ_DEV void draw(const Source &source, const Weights &w, const Settings &set, const Kept &kept, int32_t *token, float *chance,
                 Scratch &m) {
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
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64), tied += __shfl_xor(tied, o, 64);
  __syncthreads();
  if (lane == 0) m.sums[wave] = sum, m.ties[wave] = tied;
  __syncthreads();
  double total = 0.0;
  uint32_t seen = 0;
  for (int i = 0; i < kWaves; i++) {
    total += m.sums[i] + (double)min(m.ties[i], most - min(most, seen)) * edge;
    seen += m.ties[i];
  }
  const double target = set.u * total;
  // the wave whose sum passes the target (none: the last that has any)
  double before = 0.0, run = 0.0;
  uint32_t tied_before = 0;
  int which = -1;
  bool passed = false;
  seen = 0;
  for (int i = 0; i < kWaves; i++) {
    const double own = m.sums[i] + (double)min(m.ties[i], most - min(most, seen)) * edge;
    if (!passed && own > 0.0) {
      which = i, run = before, tied_before = seen;
      passed = before + own > target;
    }
    before += own, seen += m.ties[i];
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
    double up_to = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double other = __shfl_up(up_to, o, 64);
      if (lane >= o) up_to += other;
    }
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
      last = __shfl(i + c_at, l, 64);
      last_chance = (float)(__shfl(w_at, l, 64) / total);
      if (over) return false;
    }
    run += __shfl(up_to, 63, 64);
#pragma unroll
    for (int c = 0; c < 4; c++) tied_before += __popcll(equal[c]);
    return true;
  });
  if (lane == 0) {
    *token = last < 0 ? -1 : source.index(last);
    if (chance) *chance = last_chance;
  }
}

// ---- a row a block --------------------------------------------------------------------------------------------------
HQ_DEV void none(const Sample &a, int64_t row) {
  if (threadIdx.x == 0) {
    a.tokens[row] = -1;
    if (a.chance) a.chance[row] = 0.0f;
  }
}

template <bool WIDE, int MOST>
__global__ __launch_bounds__(kThreads) void row_kernel(Sample a, double by) {
  __shared__ Scratch m;
  __shared__ uint32_t keys[MOST];
  const int64_t row = blockIdx.x;
  const Settings set = settings_of(a, row);
  if (threadIdx.x < 64) m.roots[threadIdx.x] = kRoots[threadIdx.x];
  const Row<WIDE> from((const float *)(a.logits + row * a.stride), a.vocab);
  uint32_t top = 0;
  from.sweep([&](const uint32_t k[4], int32_t i) {
    *(uint4 *)(keys + i) = make_uint4(k[0], k[1], k[2], k[3]);
    top = max(max(top, max(k[0], k[1])), max(k[2], k[3]));
    return true;
  });
  top = (uint32_t)block_all((uint64_t)top, m.part, Most());
  if (!top) return none(a, row);
  const List<true> source(keys, nullptr, a.vocab);
  const Weights w{top, (double)value_of(top), slope_of(set.temperature), by, m.roots};
  const Kept kept = kept_of(source, w, set, 1u, 0, -1.0, m);
  draw(source, w, set, kept, a.tokens + row, a.chance ? a.chance + row : nullptr, m);
}

// ---- a row over many blocks -----------------------------------------------------------------------------------------
// What a wave of the first launch leaves: its largest key, its line (it handed on all from there on; 1: all that there are), how
// many of each of its steps it handed on, and the sums of each step's weights relative to its largest
struct alignas(16) Note {
  uint16_t counts[kBatch];
  double sums[kBatch];
  uint32_t top, line;
};
struct Pair {
  uint32_t key;
  int32_t at;
};
struct Split {
  Note *notes;   // [rows][chunks]
  Pair *handed;  // [rows][chunks][kHand]
  int32_t chunks, lanes;  // waves a row; the lanes whose largest are to pass a wave's line
};

// What is computed from these four from here on is not kept from before, nor begun earlier: registers
HQ_DEV void anew(float v[4]) { asm volatile("" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3])); }

template <bool WIDE>
__global__ __launch_bounds__(256) void hand_kernel(Sample a, Split sp) {
  __shared__ double roots[64];
  if (threadIdx.x < 64) roots[threadIdx.x] = kRoots[threadIdx.x];
  __syncthreads();
  const int lane = threadIdx.x & 63;
  const int32_t chunk = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int64_t row = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  if (chunk >= sp.chunks || row >= a.rows) return;
  const Settings set = settings_of(a, row);
  const int32_t stripe = sp.chunks * kStep;
  float v[4 * kBatch];
  load<WIDE>((const float *)(a.logits + row * a.stride), a.vocab, chunk * kStep, stripe, a.vocab, v);
  Note *note = sp.notes + row * sp.chunks + chunk;
  float mine = -__builtin_huge_valf();
#pragma unroll
  for (int i = 0; i < 4 * kBatch; i++) mine = fmaxf(mine, v[i]);  // (NaN: the other)
  const uint32_t key = key_of(mine);
  uint32_t top = key;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor(top, o, 64));
  if (set.all()) {
    if (lane == 0) note->top = top;
  } else {
    // the line: so many lanes' largest are at or above it (the row's top_k, spread evenly, four times over)
    const int lanes = set.top_k == 1 ? 1 : set.top_k ? min(sp.lanes, 12 + 2 * (set.top_k / sp.chunks)) : sp.lanes;
    uint32_t line = 0;
    for (uint32_t bit = 1u << 31; bit; bit >>= 1) {
      const int above = __popcll(__ballot(key >= (line | bit)));
      if (above >= lanes) line |= bit;
      if (above == lanes) break;
    }
    uint16_t counts[kBatch];
    int total = 0;
    const auto count = [&](float from) {
      total = 0;
#pragma unroll
      for (int j = 0; j < kBatch; j++) {
        int n = 0;
#pragma unroll
        for (int c = 0; c < 4; c++) n += __popcll(__ballot(v[4 * j + c] >= from));
        counts[j] = (uint16_t)n, total += n;
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    line = line < kLowest ? 1u : line;
    float from = value_of(max(line, kLowest));
    count(from);
    if (total > kHand) {  // (equal ones by the dozen: those above them, if these are fewer)
      line = max(line, kLowest) + 1;
      from = value_of(line);
      if (line <= top) count(from);
      if (line > top || total > kHand) {
        line = UINT32_MAX, total = 0;
#pragma unroll
        for (int j = 0; j < kBatch; j++) counts[j] = 0;
      }
    }
    if (total) {
      Pair *to = sp.handed + (row * sp.chunks + chunk) * kHand;
#pragma unroll
      for (int j = 0; j < kBatch; j++) {
        if (!counts[j]) continue;
        anew(v + 4 * j);
        int before = 0, own = 0;
#pragma unroll
        for (int c = 0; c < 4; c++) {
          const uint64_t in = __ballot(v[4 * j + c] >= from);
          before += __popcll(in & (((uint64_t)1 << lane) - 1));
        }
#pragma unroll
        for (int c = 0; c < 4; c++)
          if (v[4 * j + c] >= from) to[before + own++] = Pair{key_of(v[4 * j + c]), chunk * kStep + j * stripe + 4 * lane + c};
        to += counts[j];
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (lane == 0) {
      note->top = top, note->line = line;
#pragma unroll
      for (int j = 0; j < kBatch; j++) note->counts[j] = counts[j];
    }
  }
  if (!set.whole_sum()) return;
  const double slope = slope_of(set.temperature), most = (double)value_of(top);
  double s[kBatch];
#pragma unroll
  for (int j = 0; j < kBatch; j++) {
    anew(v + 4 * j);
    s[j] = 0.0;
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const float x = v[4 * j + c];
      const double e = power((double)x - most, slope, roots);
      s[j] += x == value_of(top) ? 1.0 : x > -__builtin_huge_valf() ? e : 0.0;
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  // the eight sums over the lanes: halves of them change sides until a lane holds an eighth of one
#pragma unroll
  for (int half = kBatch / 2, mask = 32; half; half >>= 1, mask >>= 1) {
    const bool upper = lane & mask;
#pragma unroll
    for (int j = 0; j < half; j++) {
      const double give = upper ? s[j] : s[j + half], keep = upper ? s[j + half] : s[j];
      s[j] = keep + __shfl_xor(give, mask, 64);
    }
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) s[0] += __shfl_xor(s[0], o, 64);
  if ((lane & 7) == 0) note->sums[lane >> 3] = top ? s[0] : 0.0;
}

struct Joint {
  Scratch m;
  uint32_t keys[kList + kStep];
  int32_t at[kList + kStep];
};

// nothing is cut off: the step in which the sum is reached by what the first launch summed, then its 256 logits
template <bool WIDE>
HQ_DEV void draw_of_all(const Sample &a, const Split &sp, int64_t row, const Weights &w, double u, Scratch &m) {
  const Note *notes = sp.notes + row * sp.chunks;
  const int32_t steps = kBatch * sp.chunks, each = (steps + kThreads - 1) / kThreads, first = threadIdx.x * each;
  const auto sum_of = [&](int32_t i) {
    if (i >= steps) return 0.0;
    const Note &n = notes[i % sp.chunks];
    return n.top ? n.sums[i / sp.chunks] * w.of(n.top) : 0.0;
  };
  double mine = 0.0, total;
  for (int32_t i = first; i < first + each; i++) mine += sum_of(i);
  const double before = sum_before(mine, (double *)m.part, total), target = u * total;
  // the thread in whose steps the target is passed, or the last that has any
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
  // (a step whose sum is some smallest number may have no weight that is one: then the next, or the one before)
  for (int32_t i = (int32_t)m.found[2]; i >= 0 && i < steps; i += passed ? 1 : -1) {
    const int32_t from = i * kStep + 4 * lane;
    double x[4], sum = 0.0;
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const float v = p[min(from + c, a.vocab - 1)];
      x[c] = from + c < a.vocab ? w.of(key_of(v)) : 0.0;
      sum += x[c];
    }
    double up_to = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double other = __shfl_up(up_to, o, 64);
      if (lane >= o) up_to += other;
    }
    const uint64_t over = __ballot(sum > 0.0 && m.sums[0] + up_to > target), any = __ballot(sum > 0.0);
    if (!any) continue;
    const int l = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)any);
    double at = m.sums[0] + (up_to - sum), share = 0.0;
    int32_t found = -1;
#pragma unroll
    for (int c = 0; c < 4; c++) {
      if (x[c] > 0.0 && (found < 0 || !over || !(at > target))) found = from + c, share = x[c];
      at += x[c];
    }
    if (lane == l) {
      a.tokens[row] = found;
      if (a.chance) a.chance[row] = (float)(share / total);
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
  if (threadIdx.x < 64) m.roots[threadIdx.x] = kRoots[threadIdx.x];
  // (steps in order of the row: step j of chunk c is the row's j chunks + c; up to 4096, where the histograms will be)
  const int32_t steps = kBatch * sp.chunks;
  uint32_t *const offset = m.offset;
  uint64_t ends = 0;  // the largest key, and the highest line
  for (int32_t c = threadIdx.x; c < sp.chunks; c += kThreads) {
    ends = max(ends, (uint64_t)notes[c].top << 32);
    if (set.all()) continue;
    const uint32_t line = notes[c].line;
    const uint4 q = *(const uint4 *)notes[c].counts;
    const uint32_t d[4] = {q.x, q.y, q.z, q.w};
    ends = max(ends & ~(uint64_t)UINT32_MAX, (uint64_t)notes[c].top << 32) | max((uint32_t)ends, line);
#pragma unroll
    for (int j = 0; j < kBatch; j++) offset[j * sp.chunks + c] = (d[j >> 1] >> (16 * (j & 1))) & 0xffffu;
  }
  ends = block_all(ends, m.part, [](uint64_t x, uint64_t y) {
    return max(x & ~(uint64_t)UINT32_MAX, y & ~(uint64_t)UINT32_MAX) | max((uint32_t)x, (uint32_t)y);
  });
  const uint32_t top = (uint32_t)(ends >> 32), line = (uint32_t)ends;
  if (!top) return none(a, row);
  const Weights w{top, (double)value_of(top), slope_of(set.temperature), by, m.roots};
  if (set.all()) return draw_of_all<WIDE>(a, sp, row, w, set.u, m);
  // the row's sum of weights
  double sum = -1.0;
  if (set.whole_sum()) {
    sum = 0.0;
    for (int32_t c = threadIdx.x; c < sp.chunks; c += kThreads) {
      double own = 0.0;
#pragma unroll
      for (int j = 0; j < kBatch; j++) own += notes[c].sums[j];
      if (notes[c].top) sum += own * w.of(notes[c].top);
    }
    sum = block_all(sum, (double *)m.part, Add());
  }
  // each step's place in the list
  const int32_t each = (steps + kThreads - 1) / kThreads, first = min((int32_t)threadIdx.x * each, steps), last = min(first + each, steps);
  uint32_t mine = 0, total;
  for (int32_t i = first; i < last; i++) mine += offset[i];
  uint32_t before = sum_before(mine, (uint32_t *)m.part, total);
  for (int32_t i = first; i < last; i++) {
    const uint32_t n = offset[i];
    offset[i] = before;
    before += n;
  }
  __syncthreads();
  const int32_t n = (int32_t)total;
  if (n <= kList && line <= top) {
    uint64_t keys = 0;
    for (int32_t c = wave; c < sp.chunks; c += kWaves) {
      const Pair *from = sp.handed + (row * sp.chunks + c) * kHand;
      const uint4 q = *(const uint4 *)notes[c].counts;
      const uint32_t d[4] = {q.x, q.y, q.z, q.w};
      uint32_t start[kBatch + 1];
      start[0] = 0;
#pragma unroll
      for (int j = 0; j < kBatch; j++) start[j + 1] = start[j] + ((d[j >> 1] >> (16 * (j & 1))) & 0xffffu);
      for (uint32_t e = lane; e < start[kBatch]; e += 64) {
        const Pair pair = from[e];
        uint32_t to = 0;
#pragma unroll
        for (int j = 0; j < kBatch; j++)
          if (e >= start[j] && e < start[j + 1]) to = offset[j * sp.chunks + c] + (e - start[j]);
        s.keys[to] = pair.key >= line ? pair.key : 0u;
        s.at[to] = pair.at;
        keys += pair.key >= line;
      }
    }
    if ((int32_t)threadIdx.x < kStep) s.keys[n + threadIdx.x] = 0;
    keys = block_all(keys, m.part, Add());
    const List<false> source(s.keys, s.at, n);
    const Kept kept = kept_of(source, w, set, max(line, 1u), (int64_t)keys, sum, m);
    if (kept.known) return draw(source, w, set, kept, a.tokens + row, a.chance ? a.chance + row : nullptr, m);
  }
  __syncthreads();
  const Row<WIDE> source((const float *)(a.logits + row * a.stride), a.vocab);
  const Kept kept = kept_of(source, w, set, 1u, 0, sum, m);
  draw(source, w, set, kept, a.tokens + row, a.chance ? a.chance + row : nullptr, m);
}

int32_t chunks_of(int32_t vocab) { return (int32_t)(((int64_t)vocab + kBatch * kStep - 1) / (kBatch * kStep)); }
int64_t notes_bytes(int64_t rows, int32_t vocab) { return (rows * chunks_of(vocab) * (int64_t)sizeof(Note) + 255) / 256 * 256; }

}  // namespace

int64_t sample_work_bytes(int32_t rows, int32_t vocab) {
  if (vocab <= kHeld) return 0;
  return notes_bytes(rows, vocab) + (int64_t)rows * chunks_of(vocab) * kHand * (int64_t)sizeof(Pair);
}

hipError_t launch_sample(const Sample &a, hipStream_t s) {
  if (a.rows <= 0 || a.vocab <= 0) return hipSuccess;
  // (a row's steps stay below 2^62)
  int bits = 0;
  while (((int64_t)1 << bits) < a.vocab) bits++;
  const double by = (double)((int64_t)1 << (62 - bits));
  const bool wide = a.vocab >= 4 && (uintptr_t)a.logits % 16 == 0 && (a.rows == 1 || a.stride % 16 == 0);
  if (a.vocab <= kHeld) {
    const auto kernel = a.vocab <= kSmall ? wide ? row_kernel<true, kSmall> : row_kernel<false, kSmall>
                                          : wide ? row_kernel<true, kHeld> : row_kernel<false, kHeld>;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)a.rows), dim3(kThreads), 0, s, a, by);
    return hipGetLastError();
  }
  Split sp{};
  sp.chunks = chunks_of(a.vocab);
  sp.notes = (Note *)a.work;
  sp.handed = (Pair *)(a.work + notes_bytes(a.rows, a.vocab));
  // The lanes whose largest of 32 logits pass a wave's line, so that evenly spread logits hand on some 5500 of a row: of a share q of
  // the logits above the line, a lane has one with chance 1 - (1 - q)^32.  At most 48, which hand on 90 of a wave's 2048.
  const double share = std::min(1.0, 5500.0 / ((double)sp.chunks * kBatch * kStep));
  sp.lanes = std::min(48, std::max(1, (int)(64.0 * (1.0 - std::pow(1.0 - share, 4.0 * kBatch)))));
  const uint32_t wide_rows = (uint32_t)std::min(a.rows, 32768);
  const dim3 grid((uint32_t)((sp.chunks + 3) / 4), wide_rows, ((uint32_t)a.rows + wide_rows - 1) / wide_rows);
  hipLaunchKernelGGL(wide ? hand_kernel<true> : hand_kernel<false>, grid, dim3(256), 0, s, a, sp);
  if (const hipError_t e = hipGetLastError()) return e;
  hipLaunchKernelGGL(wide ? join_kernel<true> : join_kernel<false>, dim3((uint32_t)a.rows), dim3(kThreads), 0, s, a, sp, by);
  return hipGetLastError();
}

}  // namespace hq
