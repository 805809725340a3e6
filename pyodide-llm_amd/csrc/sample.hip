// sample.hip — the next token of each row of logits from a given random number: temperature, top-k, top-p, min-p.
//
// A logit is held as its key, a 32-bit number that orders as the float does (0: never drawn).  What top-k and top-p leave is a
// smallest key t and how many of the logits equal to it (the first by index); both are found by histograms over the keys,
// round by round in the bin where the count (or the weight) passes the line, until a bin holds one key.  Weights in
// histograms are whole numbers (steps of a power of two below the largest weight), so that no order of additions changes them.
// The token is then found by a sum over the kept weights in index order, in 64 bits.
//
// A block takes a row.
#include "common.hpp"
#include "launch.hpp"

namespace hq {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = kThreads;

HQ_DEV uint32_t key_of(float v) {
  const uint32_t bits = __float_as_uint(fadd(v, 0.0f));  // (-0 orders as 0)
  return v > -__builtin_huge_valf() ? bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u) : 0u;
}
HQ_DEV float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

// sums and maxima over a block (every thread calls; `part`: kWaves doublewords of LDS that nothing else uses)
template <typename T, typename Op>
HQ_DEV T block_all(T v, T *part, Op op) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = op(v, (T)__shfl_xor(v, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int i = 1; i < kWaves; i++) v = op(v, part[i]);
  return v;
}

// the sum over the threads before this one
HQ_DEV uint64_t sum_before(uint64_t v, uint64_t *part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t sum = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t other = __shfl_up(sum, o, 64);
    if (lane >= o) sum += other;
  }
  __syncthreads();
  if (lane == 63) part[wave] = sum;
  __syncthreads();
  // (a lane a wave: the sums up to each)
  uint64_t waves = part[lane & 15];
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    const uint64_t other = __shfl_up(waves, o, 16);
    if ((lane & 15) >= o) waves += other;
  }
  const uint64_t before = wave ? __shfl(waves, wave - 1, 16) : 0;
  return before + sum - v;
}

struct Scratch {
  uint64_t weight[kBins];
  uint32_t count[kBins], some[kBins];  // (a key of the bin)
  uint64_t part[kWaves];
  uint64_t found[4];
};

// a row's largest key and temperature: its weights
struct Weights {
  uint32_t top;
  double most, by;  // the largest logit, 1 / step
  double temperature;
  HQ_DEV double of(uint32_t key) const {
    if (key == top) return 1.0;
    return key ? exp(((double)value_of(key) - most) / temperature) : 0.0;
  }
  HQ_DEV uint64_t steps(uint32_t key) const { return (uint64_t)(of(key) * by + 0.5); }
};

// a row of logits in memory
struct Row {
  const float *p;
  int32_t n;
  HQ_DEV uint32_t key(int32_t i) const { return i < n ? key_of(p[i]) : 0u; }
  template <typename F>
  HQ_DEV void each(F f) const {
    for (int32_t i = threadIdx.x; i < n; i += kThreads) f(key_of(p[i]));
  }
};

// Where in falling order of keys a count or a weight is reached: the key, what lies before its first, and how many are equal to it.
struct Line {
  uint32_t key;
  uint64_t before, equal;
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

// The first key, from hi downward, up to and with whose equals the row's count (its weight) is `target` or more; all keys of the row
// that count lie in lo .. hi, and `target` is reached within them.  The first round's bins lie evenly over the values (logits that
// lie on both sides of 0 crowd a few bins of their keys), those after it evenly over the keys.
template <bool WEIGHT, typename Source>
HQ_DEV Line line_of(const Source &source, const Weights &w, uint32_t lo, uint32_t hi, double range, double target, Scratch &m) {
  Line o{hi, 0, 0};
  bool values = range > 0.0 && range < 1e300;
  while (true) {
    const double per = (kBins - 0.5) / range;
    const auto value_bin = [&](uint32_t key) { return (int)fmin((w.most - (double)value_of(key)) * per, kBins - 1.0); };
    const int shift = max(22 - (int)__builtin_clz((hi - lo) | 1u), 0);  // hi - lo in 10 bits
    __syncthreads();
    m.count[threadIdx.x] = 0;
    if (WEIGHT) m.weight[threadIdx.x] = 0;
    if (threadIdx.x == 0) m.found[0] = 0;
    __syncthreads();
    source.each([&](uint32_t key) {
      if (key < lo || key > hi) return;
      const int bin = values ? value_bin(key) : (int)((hi - key) >> shift);
      atomicAdd(&m.count[bin], 1u);
      if (WEIGHT) atomicAdd((unsigned long long *)&m.weight[bin], (unsigned long long)w.steps(key));
      m.some[bin] = key;
    });
    __syncthreads();
    const uint64_t mine = WEIGHT ? m.weight[threadIdx.x] : m.count[threadIdx.x];
    const uint64_t before = o.before + sum_before(mine, m.part);
    // (no bin passes the line where rounding puts it behind the last: the last bin with anything in it then)
    if (m.count[threadIdx.x] && (double)before < target) atomicMax((unsigned long long *)&m.found[0], (unsigned long long)threadIdx.x + 1);
    __syncthreads();
    const int bin = (int)m.found[0] - 1;
    if (bin < 0) return o;
    if ((int)threadIdx.x == bin) m.found[2] = before;
    __syncthreads();
    o.before = m.found[2];
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

struct Settings {
  double temperature, top_p, min_p, u;
  int32_t top_k;  // (0: all)
};
HQ_DEV Settings settings_of(const Sample &a, int64_t row) {
  Settings o;
  o.temperature = a.temperature ? a.temperature[row] : 1.0f;
  o.top_k = a.top_k ? max(a.top_k[row], 0) : 0;
  o.top_p = a.top_p ? a.top_p[row] : 1.0f;
  o.min_p = a.min_p ? a.min_p[row] : 0.0f;
  o.min_p = o.min_p > 0.0 ? fmin(o.min_p, 1.0) : 0.0;
  o.u = a.u[row];
  if (!(o.u >= 0.0)) o.u = 0.0;
  if (!(o.temperature > 0.0)) o.temperature = 1.0, o.top_k = 1;
  return o;
}

// what top-k, top-p and min-p leave: keys above t, and the first `ties` of those equal to it; weights below min_p not
struct Kept {
  uint32_t t;
  uint64_t ties;
};

// keys: how many of the row are not 0; least: the smallest of these
template <typename Source>
HQ_DEV Kept kept_of(const Source &source, const Weights &w, const Settings &set, uint64_t keys, uint32_t least, Scratch &m) {
  Kept o{1, UINT64_MAX};
  uint32_t lo = least;
  const bool finite = w.most < __builtin_huge_val();
  const double all = finite ? w.most - (double)value_of(least) : 0.0;
  if (set.top_k > 0 && (uint64_t)set.top_k < keys) {
    const Line k = line_of<false>(source, w, lo, w.top, all, (double)set.top_k, m);
    o.t = lo = k.key, o.ties = (uint64_t)set.top_k - k.before;
  }
  if (!(set.top_p < 1.0)) return o;
  uint64_t sum = 0;
  source.each([&](uint32_t key) { sum += key > o.t || (key == o.t && o.ties == UINT64_MAX) ? w.steps(key) : 0; });
  sum = block_all(sum, m.part, [](uint64_t x, uint64_t y) { return x + y; });
  if (o.ties != UINT64_MAX) sum += o.ties * w.steps(o.t);
  // (the first token is kept whatever its share)
  const double target = fmax(set.top_p * (double)sum, 0.5);
  const double range = finite ? fmin(w.most - (double)value_of(lo), 40.0 * w.temperature) : 0.0;
  const Line p = line_of<true>(source, w, lo, w.top, range, target, m);
  const double each = (double)w.steps(p.key), room = (target - (double)p.before) / each;
  const uint64_t equal = p.key == o.t ? min(p.equal, o.ties) : p.equal;
  // ties j = 0, 1, .. with before + j each < target
  uint64_t ties = room < (double)equal ? (uint64_t)ceil(room) : equal;
  while (ties > 1 && !((double)p.before + (double)(ties - 1) * each < target)) ties--;
  return Kept{p.key, ties > 1 ? ties : 1};
}

// The token: the first by index whose kept weights up to it are more than u times all.  Each wave sums its part of the row, then
// the wave in whose part the sum is reached goes through it again.
template <typename Source>
HQ_DEV void draw(const Source &source, const Weights &w, const Settings &set, const Kept &kept, int32_t *token, float *chance,
                 Scratch &m) {
  __shared__ double sums[kWaves];
  __shared__ uint64_t ties[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int32_t part = (source.n + kWaves * 64 - 1) / (kWaves * 64) * 64, from = wave * part, to = min(from + part, source.n);
  const double edge = kept.t > 1 ? w.of(kept.t) : 0.0;  // the weight of one that is equal to t
  const uint64_t most = edge >= set.min_p || kept.t == w.top ? kept.ties : 0;
  const auto weight = [&](uint32_t key) {
    if (!key || key < kept.t) return 0.0;
    const double x = w.of(key);
    return x >= set.min_p ? x : 0.0;
  };
  double sum = 0.0;
  uint64_t tied = 0;
  for (int32_t i = from + lane; i < to; i += 64) {
    const uint32_t key = source.key(i);
    if (key == kept.t) tied++;
    else sum += weight(key);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64), tied += __shfl_xor(tied, o, 64);
  __syncthreads();
  if (lane == 0) sums[wave] = sum, ties[wave] = tied;
  __syncthreads();
  double total = 0.0;
  uint64_t seen = 0;
#pragma unroll
  for (int i = 0; i < kWaves; i++) {
    const uint64_t mine = min(ties[i], most - min(most, seen));
    total += sums[i] + (double)mine * edge;
    seen += ties[i];
  }
  const double target = set.u * total;
  // the wave whose sum passes the target (none: the last that has any)
  double before = 0.0, start = 0.0;
  uint64_t tied_before = 0;
  int which = -1;
  bool passed = false;
  seen = 0;
#pragma unroll
  for (int i = 0; i < kWaves; i++) {
    const uint64_t mine = min(ties[i], most - min(most, seen));
    const double own = sums[i] + (double)mine * edge;
    if (!passed && own > 0.0) {
      which = i, start = before, tied_before = seen;
      passed = before + own > target;
    }
    before += own, seen += ties[i];
  }
  if (wave != which) return;
  double run = start;
  int32_t last = -1;
  float last_chance = 0.0f;
  for (int32_t i0 = from; i0 < to; i0 += 64) {
    const int32_t i = i0 + lane;
    const uint32_t key = i < to ? source.key(i) : 0u;
    const uint64_t equal = __ballot(key == kept.t && key != 0);
    const uint64_t rank = tied_before + __popcll(equal & (((uint64_t)1 << lane) - 1));
    const double mine = key == kept.t ? (key && rank < most ? edge : 0.0) : weight(key);
    double sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double other = __shfl_up(sum, o, 64);
      if (lane >= o) sum += other;
    }
    const uint64_t over = __ballot(mine > 0.0 && run + sum > target), any = __ballot(mine > 0.0);
    if (over || any) {
      const int l = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)any);
      last = i0 + l;
      last_chance = (float)(__shfl(mine, l, 64) / total);
      if (over) break;
    }
    run += __shfl(sum, 63, 64);
    tied_before += __popcll(equal);
  }
  if (lane == 0) {
    *token = last;
    if (chance) *chance = last_chance;
  }
}

__global__ __launch_bounds__(kThreads) void sample_kernel(Sample a, double by) {
  __shared__ Scratch m;
  const int64_t row = blockIdx.x;
  const Row source{(const float *)(a.logits + row * a.stride), a.vocab};
  const Settings set = settings_of(a, row);
  uint32_t top = 0, least = UINT32_MAX;
  uint64_t keys = 0;
  source.each([&](uint32_t key) {
    if (!key) return;
    top = max(top, key), least = min(least, key), keys++;
  });
  top = (uint32_t)block_all((uint64_t)top, m.part, [](uint64_t x, uint64_t y) { return x > y ? x : y; });
  least = (uint32_t)block_all((uint64_t)least, m.part, [](uint64_t x, uint64_t y) { return x < y ? x : y; });
  keys = block_all(keys, m.part, [](uint64_t x, uint64_t y) { return x + y; });
  if (!top) {
    if (threadIdx.x == 0) {
      a.tokens[row] = -1;
      if (a.chance) a.chance[row] = 0.0f;
    }
    return;
  }
  const Weights w{top, (double)value_of(top), by, set.temperature};
  const Kept kept = kept_of(source, w, set, keys, least, m);
  draw(source, w, set, kept, a.tokens + row, a.chance ? a.chance + row : nullptr, m);
}

}  // namespace

int64_t sample_work_bytes(int32_t rows, int32_t vocab) { return 0; }

hipError_t launch_sample(const Sample &a, hipStream_t s) {
  if (a.rows <= 0 || a.vocab <= 0) return hipSuccess;
  // (a row's steps stay below 2^62)
  int bits = 0;
  while (((int64_t)1 << bits) < a.vocab) bits++;
  const double by = (double)((int64_t)1 << (62 - bits));
  hipLaunchKernelGGL(sample_kernel, dim3((uint32_t)a.rows), dim3(kThreads), 0, s, a, by);
  return hipGetLastError();
}

}  // namespace hq
