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
// brings its largest |value| into [2^13, 2^14), so that the second half keeps its bits.  A position's scales multiply its score and
// its weight.  One pass over the positions holds a running maximum m and sum l of a softmax in base 2:
//   p_j = 2^(u_j - m + 6),  u_j = s_j log2(e),   l = sum p_j,   acc = sum (p_j vs_j 2^-E) v_j
// m moves only where a score passes it by 8 (p_j stays below 2^14), so that acc is seldom rescaled; E, the largest exponent of
// a position's scale so far, keeps a weight times its scale within float16's range whatever the values' size.
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
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kFewRows = 16;       // a tile's rows
constexpr float kRoom = 8.0f, kShift = 6.0f;  // how far a score may pass the maximum; p = 2^(u - m + kShift)
constexpr int kLeast = -100;  // the exponent of the smallest scale a cache stores (and E's start)

// ---- rows, positions and shares ---------------------------------------------------------------------------------
struct Share {
  int32_t blocks;     // blocks that share the work
  int32_t rows;       // of a tile
  int32_t positions;  // of a block's step
  int32_t tiles;      // there can be
  int64_t parts;      // where in the workspace the shared items' parts are
  int64_t bytes;      // the workspace
  int64_t most;       // steps there can be
};

// a tile's rows r0 .. r1 - 1 of a sequence, the positions from .. to - 1 that some of them see, and the steps that hold
// these: first .. first + steps - 1 (one at least: rows that see nothing are written too)
struct Tile {
  int32_t r0, r1, from, to, first, steps;
};
HQ_DEV Tile tile_of(const Attention &a, const Cache &c, const Batch &b, const Share &sh, const Sequence &q, int32_t group,
                    int32_t rt) {
  Tile t;
  t.r0 = rt * sh.rows;
  t.r1 = min(t.r0 + sh.rows, q.count * group);
  const int32_t before = q.length - q.count, reach = b.width << c.shift;
  t.to = min(max(before + (t.r1 - 1) / group + 1, 0), reach);
  t.from = a.window ? max(before + t.r0 / group + 1 - a.window, 0) : 0;
  t.first = t.from / sh.positions;
  t.steps = max((t.to + sh.positions - 1) / sh.positions - t.first, 1);
  return t;
}

HQ_DEV int32_t steps_of(const Attention &a, const Cache &c, const Batch &b, const Share &sh, int32_t s) {
  const Sequence q = sequence_of(b, s);
  const int32_t group = a.heads / c.heads, rows = q.count * group;
  int32_t n = 0;
  for (int32_t rt = 0; rt * kFewRows < rows; rt++) n += tile_of(a, c, b, sh, q, group, rt).steps;
  return n * c.heads;
}

// All steps in a row: sequences, their row tiles, the heads, the steps.  Where step `at` is.
struct Spot {
  int32_t s, rt, h, step;
  Sequence q;
  Tile t;
};
HQ_DEV Spot spot_of(const Attention &a, const Cache &c, const Batch &b, const Share &sh, int32_t at) {
  const Place p = place_of(b.sequences, at, [&](int32_t s) { return steps_of(a, c, b, sh, s); });
  Spot o;
  o.s = p.s, o.rt = 0;
  o.q = wave_sequence_of(b, max(p.s, 0));
  const int32_t group = a.heads / c.heads;
  int32_t rest = p.rest;
  for (;; o.rt++) {
    o.t = tile_of(a, c, b, sh, o.q, group, o.rt);
    if (rest < o.t.steps * c.heads || (o.rt + 1) * kFewRows >= o.q.count * group) break;
    rest -= o.t.steps * c.heads;
  }
  o.h = rest / o.t.steps;
  o.step = rest - o.h * o.t.steps;
  return o;
}

// (sequences that overlap could have more steps than 32 bits count, which the host has made sure of for others: none then)
HQ_DEV int32_t all_steps(const Attention &a, const Cache &c, const Batch &b, const Share &sh) {
  int64_t n = 0;
  for (int32_t s = threadIdx.x & 63; s < b.sequences; s += 64) n += steps_of(a, c, b, sh, s);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  return __builtin_amdgcn_readfirstlane(n <= INT32_MAX ? (int32_t)n : 0);
}
HQ_DEV int32_t share_start(int32_t steps, int32_t block, int32_t blocks) {
  return (int32_t)((int64_t)steps * block / blocks);
}

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
struct Call {
  Attention a;
  Cache c;
  Batch b;
  Share sh;
};
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
  for (int j = 0; j < 8; j++) {
    hi[j] = (_Float16)x[j];
    lo[j] = (_Float16)(x[j] - (float)hi[j]);
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
// Bound by the cache's bytes.  A wave takes 4 NP positions a step: lane l (m = l % 16, q = l / 16) holds 16 dimensions of a key
// at a time (row m of an instruction is the position NP (m / 4) + 4 t + m % 4 of its t-th 16, so that the lane's scores are those
// of the NP positions from NP q on), and of dimension 16 d + m the values of those NP positions.  Everything goes from
// memory to registers: the waves share nothing, and the next step's keys are on their way while this one's weights are formed.
// Steps of all (sequence, rows, head) are shared evenly among as many blocks as the GPU holds, whatever the lengths; what a
// block finds of an item that it does not have whole goes to `work` and join_kernel.
constexpr int few_np(int, int f16) { return f16 ? 8 : 16; }
constexpr int few_blocks_a_cu(int d, int) { return d <= 64 ? 3 : d <= 128 ? 2 : 1; }
template <int D, int F16>
__global__ __launch_bounds__(256, few_blocks_a_cu(D, F16)) void few_kernel(Call) {
  constexpr int ES = F16 ? 2 : 1, DB = D / 64, DT = D / 16, PITCH = D + 4, NP = few_np(D, F16), WK = 4 * NP, STEP = 4 * WK;
  __shared__ float sums[4][kFewRows][PITCH];
  __shared__ float stats[2][4][kFewRows];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m16 = lane & 15, q4 = lane >> 4;
  int32_t u, end;
  Spot o;
  {
    const Call *k = call_again();
    const int32_t all = all_steps(k->a, k->c, k->b, k->sh);
    u = share_start(all, blockIdx.x, k->sh.blocks);
    end = share_start(all, blockIdx.x + 1, k->sh.blocks);
    if (u >= end) return;
    o = spot_of(k->a, k->c, k->b, k->sh, u);
  }
  while (true) {
    const Call *call = call_again();
    const Attention &a = call->a;
    const Cache c = call->c;
    const Batch b = call->b;
    const int32_t group = a.heads / c.heads, reach = b.width << c.shift, mask = (1 << c.shift) - 1;
    const int32_t steps = min(o.t.steps - o.step, end - u);
    const bool whole = steps == o.t.steps;
    // ---- the rows' queries
    const int32_t row = o.t.r0 + m16, before = o.q.length - o.q.count;
    const bool live = row < o.t.r1;
    const int32_t token = (live ? row : o.t.r0) / group, g = (live ? row : o.t.r0) - token * group;
    const float *x = (const float *)(a.q + (o.q.begin + token) * a.q_stride) + (int64_t)(o.h * group + g) * c.dim;
    v8h qh[DB][2], ql[DB][2];
    float rowf;
    {
      float4 f[DB][4];
      float most = 0.0f;
#pragma unroll
      for (int d = 0; d < DB; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int at = 64 * d + 16 * q4 + 4 * i;
          f[d][i] = live && at < c.dim ? *(const float4 *)(x + at) : make_float4(0.f, 0.f, 0.f, 0.f);
          most = fmaxf(fmaxf(most, fmaxf(fabsf(f[d][i].x), fabsf(f[d][i].y))), fmaxf(fabsf(f[d][i].z), fabsf(f[d][i].w)));
        }
      most = max_row(most);
      const int up = most > 0.0f ? min(140 - (int)(__float_as_uint(most) >> 23), 126) : 0;
      const float by = power_of_2(up);
      rowf = a.scale * power_of_2(-up);
#pragma unroll
      for (int d = 0; d < DB; d++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const float4 e0 = f[d][2 * i], e1 = f[d][2 * i + 1];
          const float e[8] = {e0.x * by, e0.y * by, e0.z * by, e0.w * by, e1.x * by, e1.y * by, e1.z * by, e1.w * by};
          halves_of(e, qh[d][i], ql[d][i]);
        }
    }
    if (a.cap == 0.0f) rowf *= kLog2e;
    const float cap = a.cap, per_cap = 1.0f / cap;
    const int32_t sees = before + token + 1;
    const int32_t to = min(sees, reach), from = a.window ? sees - a.window : 0;  // the lane's row's own positions
    // the positions that every row sees lie in [every_from, every_to)
    const int32_t every_to = min(before + o.t.r0 / group + 1, reach);
    const int32_t every_from = a.window ? before + (o.t.r1 - 1) / group + 1 - a.window : 0;
    // ---- the wave's positions: WK from base on, every STEP
    float m = -INFINITY, l = 0.0f;
    int exponent = kLeast;
    v4f acc[DT] = {};
    int32_t base = (o.t.first + o.step) * STEP + WK * wave;
    const int32_t stop = min((o.t.first + o.step + steps) * STEP, o.t.to);
    while (base + WK <= o.t.from) base += STEP;
    if (base < stop) {
      Elements<F16, 16> kk[NP / 4][DB];
      int32_t page1 = page_of(b, c, o.s, base + NP * (m16 >> 2)), page2 = page_of(b, c, o.s, base + NP * q4);
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
      load_keys(base, page1);
      while (true) {
        const int32_t next = base + STEP;
        const bool more = next < stop;
        const int32_t at1 = (more ? next : base) + NP * (m16 >> 2), at2 = (more ? next : base) + NP * q4;
        const int32_t next1 = page_of(b, c, o.s, at1), next2 = page_of(b, c, o.s, at2);
        // ---- values and scales of the lane's 16 positions
        const int64_t vec = vectors_of(c, max(page2, 0), o.h);
        const int32_t slot = (base + NP * q4) & mask;
        Elements<F16, NP> vv[DT];
        float ks[NP], vs[NP];
#pragma unroll
        for (int i = 0; i < NP / 4; i++) {
          *(float4 *)(ks + 4 * i) = *(const float4 *)(c.ks + vec + slot + 4 * i);
          *(float4 *)(vs + 4 * i) = *(const float4 *)(c.vs + vec + slot + 4 * i);
        }
        {
          const int32_t dim = opaque(c.dim), shift = opaque(c.shift);
          const char *p = c.v + (vec * dim + (m16 << shift) + slot) * ES;
#pragma unroll
          for (int d = 0; d < DT; d++) vv[d].load(p + (min(d * 16, dim - 16) << shift) * ES);  // (past dim: the last again)
        }
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
        load_keys(more ? next : base, next1);
        float p[NP];
#pragma unroll
        for (int e = 0; e < NP; e++) p[e] = s[e >> 2][e & 3] * ks[e] * rowf;
        if (cap > 0.0f) {
          const float bend = opaque(0.55f), twice = opaque(2.0f * kLog2e);
#pragma unroll
          for (int e = 0; e < NP; e++) p[e] = cap * kLog2e * tanh_of(p[e] * per_cap, bend, twice);
        }
        const bool edge = base + WK > every_to || base < every_from || __any(page2 < 0);
        uint32_t seen = ~0u;
        if (edge) {
          // what the row does not see has no score; what no row sees may hold anything: its scale and values become zeros
          const int32_t at = base + NP * q4;
          seen = page2 < 0 ? 0u : bits_between(from - at, to - at);
          const uint32_t any = page2 < 0 ? 0u : bits_between(o.t.from - at, o.t.to - at);
#pragma unroll
          for (int e = 0; e < NP; e++) {
            p[e] = kept(p[e], seen, e, 0xff800000u);
            vs[e] = kept(vs[e], any, e, 0u);
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
        float most = p[0], wide = vs[0];
#pragma unroll
        for (int e = 1; e < NP; e++) most = fmaxf(most, p[e]), wide = fmaxf(wide, vs[e]);
        most = max_row(most), wide = max_row(wide);
        if (__any(most > m + kRoom)) {  // (the first that is seen too: m is -infinity before it)
          const float m1 = fmaxf(m, most);
          const float alpha = m1 == -INFINITY ? 0.0f : exp2_of(m - m1);
          m = m1;
          l *= alpha;
#pragma unroll
          for (int d = 0; d < DT; d++) acc[d] *= alpha;
        }
        const int e1 = __builtin_amdgcn_readfirstlane((int)(__float_as_uint(wide) >> 23) - 127);
        if (e1 > exponent && e1 < 128) {  // (128: nothing but NaN)
          const float by = power_of_2(max(exponent - e1, -126));
#pragma unroll
          for (int d = 0; d < DT; d++) acc[d] *= by;
          exponent = e1;
        }
        const float less = (m == -INFINITY ? 0.0f : m) - kShift, by = power_of_2(-exponent);
#pragma unroll
        for (int e = 0; e < NP; e++) {
          p[e] = exp2_of(p[e] - less);
          l += p[e];
          p[e] = p[e] * (vs[e] * by);
        }
        if (edge) {
#pragma unroll
          for (int e = 0; e < NP; e++)
            p[e] = kept(p[e], seen, e, 0u);  // (a NaN scale that others see)
        }
        // ---- out += weights times values
        v8h ph[NP / 8], pl[NP / 8];
#pragma unroll
        for (int i = 0; i < NP / 8; i++) halves_of(p + 8 * i, ph[i], pl[i]);
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
          for (int i = 0; i < NP / 8; i++) {
            const v8h v8 = vv[d].half(i);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, pl[i], acc[d], 0, 0, 0);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, ph[i], acc[d], 0, 0, 0);
          }
        if (!more) break;
        base = next, page1 = next1, page2 = next2;
      }
    }
    l = sum_row(l);
    // ---- the four waves together
    const Call *after = call_again();
    const int32_t heads = after->c.heads, shared = after->a.heads / heads;
    if (q4 == 0) stats[0][wave][m16] = m, stats[1][wave][m16] = l;
    __syncthreads();
    const float m0 = stats[0][0][m16], m1 = stats[0][1][m16], m2 = stats[0][2][m16], m3 = stats[0][3][m16];
    const float mm = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)), ref = mm == -INFINITY ? 0.0f : mm;
    const float f = exp2_of(m - ref) * power_of_2(exponent);
    const float ll = stats[1][0][m16] * exp2_of(m0 - ref) + stats[1][1][m16] * exp2_of(m1 - ref) +
                     stats[1][2][m16] * exp2_of(m2 - ref) + stats[1][3][m16] * exp2_of(m3 - ref);
#pragma unroll
    for (int d = 0; d < DT; d++) {
      const v4f v = acc[d] * f;
      *(v4f *)&sums[wave][m16][d * 16 + q4 * 4] = v;
    }
    __syncthreads();
    const int32_t slot = o.step > 0 ? 0 : 1;
    float *part = (float *)after->a.work + (int64_t)(blockIdx.x * 2 + slot) * kFewRows * (D + 2);
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
        const int32_t i0 = (o.t.r0 + r) / shared, gg = o.t.r0 + r - i0 * shared;
        v = sum != 0.0f ? v / sum : v4f{0.f, 0.f, 0.f, 0.f};
        *(v4f *)(after->a.out + (o.q.begin + i0) * after->a.out_stride + ((int64_t)(o.h * shared + gg) * after->c.dim + d) * 4) = v;
      }
    }
    u += steps;
    if (u >= end) break;
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
      o.t = tile_of(after->a, after->c, after->b, after->sh, o.q, shared, o.rt);
    }
  }
}

// The items that blocks share: the block whose share an item starts in (and does not end in) has its rows' parts joined here, a
// wave a row.
template <int D>
__global__ __launch_bounds__(256) void join_kernel(Attention a, Cache c, Batch b, Share sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int32_t group = a.heads / c.heads;
  const int32_t all = all_steps(a, c, b, sh);
  const int32_t start = share_start(all, blockIdx.x, sh.blocks), end = share_start(all, blockIdx.x + 1, sh.blocks);
  if (start >= end || end >= all) return;
  const Spot o = spot_of(a, c, b, sh, end - 1);
  const int32_t first = end - 1 - o.step, last = first + o.t.steps - 1;  // the item's steps
  if (first < start || last < end) return;
  const int r = blockIdx.y * 4 + wave;
  if (o.t.r0 + r >= o.t.r1) return;
  const int64_t size = kFewRows * (D + 2);
  const float *work = (const float *)a.work;
  float m = -INFINITY, l = 0.0f;
  float acc[D / 64] = {};
  int32_t at = blockIdx.x, slot = 1;
  while (true) {
    if (share_start(all, at + 1, sh.blocks) > share_start(all, at, sh.blocks)) {  // (a block may have no step)
      const float *part = work + (int64_t)(at * 2 + slot) * size;
      const float pm = part[r * 2], pl = part[r * 2 + 1];
      const float m1 = fmaxf(m, pm), ref = m1 == -INFINITY ? 0.0f : m1;
      const float f0 = exp2_of(m - ref), f1 = exp2_of(pm - ref);
      m = m1;
      l = l * f0 + pl * f1;
#pragma unroll
      for (int i = 0; i < D / 64; i++) acc[i] = acc[i] * f0 + part[kFewRows * 2 + r * D + lane + 64 * i] * f1;
    }
    slot = 0;
    if (share_start(all, at + 1, sh.blocks) > last || ++at >= sh.blocks) break;
  }
  const int32_t i0 = (o.t.r0 + r) / group, g = o.t.r0 + r - i0 * group;
  float *out = (float *)(a.out + (o.q.begin + i0) * a.out_stride) + (int64_t)(o.h * group + g) * c.dim;
#pragma unroll
  for (int i = 0; i < D / 64; i++)
    if (lane + 64 * i < c.dim) out[lane + 64 * i] = l != 0.0f ? acc[i] / l : 0.0f;
}

// ---- prompts: 128 rows a block, 32 a wave, over 64 positions a step -----------------------------------------------------
// Bound by the matrix cores.  A wave's 32 rows are the columns of 32 x 32 x 16 instructions: lane l (row l % 32, h = l / 32) holds
// of the step's scores those of the positions 32 k + 16 c + 8 h + e (e < 8), which are its operand of the second product for the
// positions 32 k + 16 c .. + 15.  The block's keys and values go through LDS as float16, two steps' room, each element widened
// once a block; keys in rows whose number has bits 2 and 3 swapped (the instruction's row 8 j + 4 h + i is position
// 16 (j / 2) + 8 h + 4 (j % 2) + i), 16-byte chunks XORed with the row so that 8 lanes read 8 bank quads.
//
// Which block does what is worked out once a call (plan_kernel): steps of all (sequence, head, row tile) in a row, shared evenly,
// a share's end moved to an item's end that is near, so that few items are shared and their parts joined (join_kernel).
constexpr int kRows = 128, kPositions = 64;

// where in the row of all steps: sequence, row tile, head and step of the item
struct Start {
  int32_t s, rt, h, step;
};
// the plan, in a call's workspace: the shares' edges (blocks + 1 numbers), the place of each share's first and last step, and the
// steps of one head: of all sequences up to s, of the tiles up to a tile of its sequence (tiles from base[s] on)
struct Plan {
  int32_t *edge;
  Start *first, *last;
  int32_t *upto, *base, *tile;
};
HQ_DEV Plan plan_of(char *work, int32_t blocks, int32_t sequences) {
  Plan p;
  p.first = (Start *)work;
  p.last = p.first + blocks;
  p.edge = (int32_t *)(p.last + blocks);
  p.upto = p.edge + blocks + 1;
  p.base = p.upto + sequences;
  p.tile = p.base + sequences;
  return p;
}
int64_t plan_bytes(int64_t blocks, int64_t sequences, int64_t tiles) {
  return ((2 * blocks * (int64_t)sizeof(Start) + (blocks + 1 + 2 * sequences + tiles) * 4) + 255) / 256 * 256;
}

// inclusive sums over a block of 1024 threads
HQ_DEV int64_t sum_upto(int64_t v, int64_t *wave_sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t w = __shfl_up(v, o, 64);
    if (lane >= o) v += w;
  }
  __syncthreads();
  if (lane == 63) wave_sums[wave] = v;
  __syncthreads();
  for (int i = 0; i < wave; i++) v += wave_sums[i];
  return v;
}

__global__ __launch_bounds__(1024) void plan_kernel(Attention a, Cache c, Batch b, Share sh) {
  __shared__ int64_t wave_sums[16], carry;
  const Plan p = plan_of(a.work, sh.blocks, b.sequences);
  const int32_t group = a.heads / c.heads, n = b.sequences;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // a sequence's first tile
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  for (int32_t s0 = 0; s0 < n; s0 += 1024) {
    const int32_t s = s0 + threadIdx.x;
    const int32_t tiles = s < n ? (sequence_of(b, s).count * group + sh.rows - 1) / sh.rows : 0;
    const int64_t upto = sum_upto(tiles, wave_sums) + carry;
    // (sequences that overlap could have more tiles than there is room for: those past it have none)
    if (s < n) p.base[s] = upto <= sh.tiles ? (int32_t)upto - tiles : -1;
    __syncthreads();
    if (threadIdx.x == 1023) carry = upto;
    __syncthreads();
  }
  // a tile's steps and those of the sequence's before it, a wave a sequence
  for (int32_t s = wave; s < n; s += 16) {
    const Sequence q = sequence_of(b, s);
    const int32_t tiles = p.base[s] < 0 ? 0 : (q.count * group + sh.rows - 1) / sh.rows;
    int32_t before = 0;
    for (int32_t t0 = 0; t0 < tiles; t0 += 64) {
      int32_t v = t0 + lane < tiles ? tile_of(a, c, b, sh, q, group, t0 + lane).steps : 0;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int32_t w = __shfl_up(v, o, 64);
        if (lane >= o) v += w;
      }
      if (t0 + lane < tiles) p.tile[p.base[s] + t0 + lane] = before + v;
      before += __shfl(v, 63, 64);
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
  const int32_t all = (int32_t)carry * c.heads, near = all / sh.blocks / 8;
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
    int32_t t0 = 0, t1 = (sequence_of(b, lo).count * group + sh.rows - 1) / sh.rows - 1;
    while (t0 < t1) {
      const int32_t mid = (t0 + t1) >> 1;
      if (tile[mid] > rest) t1 = mid;
      else t0 = mid + 1;
    }
    const int32_t begin = t0 ? tile[t0 - 1] : 0;
    o.rt = t0;
    o.step = rest - begin;
    first = at - o.step;
    size = tile[t0] - begin;
    return o;
  };
  for (int32_t i = threadIdx.x; i <= sh.blocks; i += 1024) {
    int32_t at = share_start(all, i, sh.blocks), first, size;
    if (at < all) {
      find(at, first, size);
      if (at - first <= near) at = first;
      else if (first + size - at <= near) at = first + size;
    }
    p.edge[i] = at;
  }
  __syncthreads();
  for (int32_t i = threadIdx.x; i < sh.blocks; i += 1024) {
    int32_t first, size;
    if (p.edge[i] >= p.edge[i + 1]) continue;
    p.first[i] = find(p.edge[i], first, size);
    p.last[i] = find(p.edge[i + 1] - 1, first, size);
  }
}

HQ_DEV uint32_t key_row(uint32_t r) { return (r & ~12u) | ((r & 4u) << 1) | ((r & 8u) >> 1); }  // bits 2 and 3 swapped

typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int rows_blocks_a_cu(int d) { return d <= 64 ? 3 : d <= 128 ? 2 : 1; }
template <int D, int F16>
__global__ __launch_bounds__(256, rows_blocks_a_cu(D)) void rows_kernel(Call) {
  constexpr int ES = F16 ? 2 : 1, KS = D / 16, DT = D / 32;
  constexpr int PIECES = D * ES / 64;  // 16-byte pieces of keys, and of values, a thread stages
  __shared__ __align__(16) char keys[2][kPositions * D * 2];
  __shared__ __align__(16) char values[2][kPositions * D * 2];
  __shared__ __align__(16) float scales[2][2][kPositions];  // of keys, of values (times 2^-exponent)
  __shared__ int32_t info[2][2];                            // the exponent, which 16 positions are on a page
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
    o.s = __builtin_amdgcn_readfirstlane(p.first[block].s), o.rt = __builtin_amdgcn_readfirstlane(p.first[block].rt);
    o.h = __builtin_amdgcn_readfirstlane(p.first[block].h), o.step = __builtin_amdgcn_readfirstlane(p.first[block].step);
  }
  while (true) {
    const Call *call = call_again();
    const Attention &a = call->a;
    const Cache c = call->c;
    const Batch b = call->b;
    const int32_t group = a.heads / c.heads, reach = b.width << c.shift, mask = (1 << c.shift) - 1;
    const Sequence q = wave_sequence_of(b, o.s);
    const Tile tile = tile_of(a, c, b, call->sh, q, group, o.rt);
    const int32_t steps = min(tile.steps - o.step, end - u);
    // ---- the rows' queries
    const int thread = opaque_lane(threadIdx.x), m32 = thread & 31, h2 = (thread >> 5) & 1;
    const int wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const int32_t r0 = tile.r0 + 32 * wave, r1 = min(r0 + 32, tile.r1), before = q.length - q.count;
    const bool some = r0 < tile.r1, live = r0 + m32 < r1;
    const int32_t row = live ? r0 + m32 : tile.r0;
    const int32_t token = row / group, g = row - token * group;
    const int32_t sees = before + token + 1;
    const int32_t to = min(sees, reach), from = a.window ? sees - a.window : 0;  // the lane's row's own positions
    // what some of the wave's rows see lies before any_to, what all of them see in [every_from, every_to)
    const int32_t any_to = some ? min(before + (r1 - 1) / group + 1, reach) : 0;
    const int32_t every_to = some ? min(before + r0 / group + 1, reach) : 0;
    const int32_t every_from = some && a.window ? before + (r1 - 1) / group + 1 - a.window : 0;
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
      rowf = a.scale * power_of_2(-up) * (a.cap == 0.0f ? kLog2e : 1.0f);
#pragma unroll
      for (int k = 0; k < KS; k++) {
        const int at = 16 * k + 8 * h2;
        float4 e0 = make_float4(0.f, 0.f, 0.f, 0.f), e1 = e0;
        if (16 * k < c.dim) e0 = *(const float4 *)(x + at), e1 = *(const float4 *)(x + at + 4);
        const float e[8] = {e0.x * by, e0.y * by, e0.z * by, e0.w * by, e1.x * by, e1.y * by, e1.z * by, e1.w * by};
        halves_of(e, qh[k], ql[k]);
      }
    }
    const float cap = a.cap, per_cap = 1.0f / cap;
    // ---- staging: the wave's 16 keys (consecutive in memory), the thread's 16 (8) positions of some dimensions, a scale a lane
    // (what the thread's number gives is formed anew in every step: registers are what the rows leave few of)
    constexpr int ROW = D * ES / 16, PARTS = F16 ? 8 : 4, EACH = kPositions / PARTS;
    uint4 reg[PIECES];  // the next step's keys, then its values
    float sreg;
    const float *scale_at = wave ? c.vs : c.ks;  // (waves 0 and 1)
    int32_t kpage, vpage, spage;  // of the step to load next
    const auto pages_at = [&](int32_t base) {
      const uint32_t tid = opaque_lane(threadIdx.x);
      const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
      kpage = page_of(b, c, o.s, base + 16 * wave);
      vpage = page_of(b, c, o.s, base + EACH * (int32_t)(tid % PARTS));
      spage = page_of(b, c, o.s, base + (int32_t)(tid & 63));
    };
    const auto load_keys = [&](int32_t base) {
      const uint32_t tid = opaque_lane(threadIdx.x), ln = tid & 63;
      const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
      const uint32_t row_pieces = (uint32_t)(opaque(c.dim) * ES) / 16;
      const int64_t kvec = vectors_of(c, max(kpage, 0), o.h) + ((base + 16 * wave) & mask);
      const char *kp = c.k + kvec * c.dim * ES;
#pragma unroll
      for (int i = 0; i < PIECES; i++) {
        const uint32_t at = ln + 64 * i, col = min(at % ROW, row_pieces - 1);  // (past dim: the last again)
        reg[i] = *(const uint4 *)(kp + (at / ROW * row_pieces + col) * 16);
      }
    };
    uint32_t on_page = 0, keep_bits = 0;  // of the loaded step
    const auto load_values = [&](int32_t base) {
      const uint32_t tid = opaque_lane(threadIdx.x), ln = tid & 63;
      const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
      const int32_t part_at = EACH * (int32_t)(tid % PARTS), slot = (base + part_at) & mask;
      const char *vp = c.v + (vectors_of(c, max(vpage, 0), o.h) * c.dim + slot) * ES;
#pragma unroll
      for (int i = 0; i < PIECES; i++) {
        const int d = (int)(tid / PARTS) + i * (256 / PARTS);
        reg[i] = *(const uint4 *)(vp + (min(d, c.dim - 1) << c.shift) * ES);  // (past dim: the last again)
      }
      const int32_t at = base + (int32_t)ln;
      const bool there = spage >= 0 && at >= tile.from && at < tile.to;
      sreg = 0.0f;
      if (wave < 2 && there) sreg = scale_at[vectors_of(c, spage, o.h) + (at & mask)];
      const uint64_t mapped = __ballot(spage >= 0);
      on_page = (uint32_t)((mapped & 1) | (mapped >> 15 & 2) | (mapped >> 30 & 4) | (mapped >> 45 & 8));
      if (F16) keep_bits = vpage >= 0 ? bits_between(tile.from - (base + part_at), tile.to - (base + part_at)) & 0xffu : 0u;
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
    int exponent_run = kLeast;  // (wave 1's)
    const auto store_values = [&](int buf) {
      const uint32_t tid = opaque_lane(threadIdx.x), ln = tid & 63, part = tid % PARTS;
      const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
#pragma unroll
      for (int i = 0; i < PIECES; i++) {
        const int d = (int)(tid / PARTS) + i * (256 / PARTS);
        char *to_row = values[buf] + d * (kPositions * 2);
        if (F16) {
          uint4 w = reg[i];
          if (keep_bits != 0xffu) {
            uint32_t *e = (uint32_t *)&w;
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const uint32_t two = keep_bits >> (2 * j);
              e[j] &= (two & 1u) * 0xffffu | (two & 2u) * 0x7fff8000u;
            }
          }
          *(uint4 *)(to_row + 16 * (part ^ (d & 7))) = w;
        } else {
          *(v8h *)(to_row + 16 * ((2 * part) ^ (d & 7))) = widen8(reg[i].x, reg[i].y);
          *(v8h *)(to_row + 16 * ((2 * part + 1) ^ (d & 7))) = widen8(reg[i].z, reg[i].w);
        }
      }
      if (wave == 0) scales[buf][0][ln] = sreg;
      if (wave == 1) {
        float wide = sreg;
#pragma unroll
        for (int i = 32; i > 0; i >>= 1) wide = fmaxf(wide, __shfl_xor(wide, i, 64));
        const int e1 = __builtin_amdgcn_readfirstlane((int)(__float_as_uint(wide) >> 23) - 127);
        if (e1 > exponent_run && e1 < 128) exponent_run = e1;  // (128: nothing but NaN)
        scales[buf][1][ln] = sreg * power_of_2(-exponent_run);
        if (ln == 0) info[buf][0] = exponent_run, info[buf][1] = on_page;
      }
    };
    {
      const int32_t now[10] = {u, end, block, o.rt, o.step, steps, tile.steps, q.begin, q.count, o.h};
#pragma unroll
      for (int i = 0; i < 10; i++) parked[wave][i] = now[i];
    }
    // ---- the steps
    float m = -INFINITY, l = 0.0f;
    int exponent = kLeast;
    v16f acc[DT] = {};
    int32_t base = (tile.first + o.step) * kPositions;
    const int32_t stop = base < tile.to ? base + steps * kPositions : base;  // (rows that see nothing: a step without positions)
    if (base < stop) {
      pages_at(base);
      load_keys(base);
      store_keys(0);
      load_values(base);
      store_values(0);
      pages_at(base + kPositions);
    }
    __syncthreads();
    for (int buf = 0; base < stop; base += kPositions, buf ^= 1) {
      const bool more = base + kPositions < stop;
      if (more) load_keys(base + kPositions);
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
          const int32_t pages_here = __builtin_amdgcn_readfirstlane(info[buf][1]) >> (2 * t) & 3;
          const float *sc = &scales[buf][0][32 * t + 8 * h2];
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const v4f k0 = *(const v4f *)(sc + 16 * i), k1 = *(const v4f *)(sc + 16 * i + 4);
#pragma unroll
            for (int e = 0; e < 8; e++) p[8 * i + e] = s[8 * i + e] * (e < 4 ? k0[e & 3] : k1[e & 3]) * rowf;
          }
          if (cap > 0.0f) {
            const float bend = opaque(0.55f), twice = opaque(2.0f * kLog2e);
#pragma unroll
            for (int e = 0; e < 16; e++) p[e] = cap * kLog2e * tanh_of(p[e] * per_cap, bend, twice);
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
          most = max_pair(most);
          if (__any(most > m + kRoom)) {
            const float m1 = fmaxf(m, most);
            const float alpha = m1 == -INFINITY ? 0.0f : exp2_of(m - m1);
            m = m1;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; d++) acc[d] *= alpha;
          }
          const int e1 = __builtin_amdgcn_readfirstlane(info[buf][0]);
          if (e1 > exponent) {
            const float by = power_of_2(max(exponent - e1, -126));
#pragma unroll
            for (int d = 0; d < DT; d++) acc[d] *= by;
            exponent = e1;
          }
          const float less = (m == -INFINITY ? 0.0f : m) - kShift;
          v8h ph[2], pl[2];
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const v4f v0 = *(const v4f *)(sc + kPositions + 16 * i), v1 = *(const v4f *)(sc + kPositions + 16 * i + 4);
#pragma unroll
            for (int e = 0; e < 8; e++) {
              const float w = exp2_of(p[8 * i + e] - less);
              l += w;
              p[8 * i + e] = w * (e < 4 ? v0[e & 3] : v1[e & 3]);
            }
            if (edge) {
#pragma unroll
              for (int e = 0; e < 8; e++) p[8 * i + e] = kept(p[8 * i + e], seen, 8 * i + e, 0u);  // (a NaN scale that others see)
            }
            halves_of(p + 8 * i, ph[i], pl[i]);
          }
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
        if (more && t == 0) {
          store_keys(buf ^ 1);
          load_values(base + kPositions);
          pages_at(base + 2 * kPositions);
        }
      }
      if (more) store_values(buf ^ 1);
      __syncthreads();
    }
    l = sum_pair(l);
    // ---- the rows out, or to be joined
    const Call *after = call_again();
    int32_t kept_back[10];
#pragma unroll
    for (int i = 0; i < 10; i++) kept_back[i] = __builtin_amdgcn_readfirstlane(parked[wave][i]);
    u = kept_back[0], end = kept_back[1], block = kept_back[2], o.rt = kept_back[3], o.step = kept_back[4], o.h = kept_back[9];
    const int32_t done = kept_back[5], begin = kept_back[7], count = kept_back[8];
    const bool whole = done == kept_back[6];
    if (live) {
      const int thread = opaque_lane(threadIdx.x), m32 = thread & 31, h2 = (thread >> 5) & 1, wave = thread >> 6;
      const float by = power_of_2(exponent);
      if (whole) {
        const int32_t heads = after->a.heads, shared = heads / after->c.heads, dim = after->c.dim;
        const float per = l != 0.0f ? by / l : 0.0f;
        float *out = (float *)(after->a.out + (begin + token) * after->a.out_stride) + (int64_t)(o.h * shared + g) * dim;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const int at = 32 * d + 8 * j + 4 * h2;
            v4f v = {acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]};
            if (32 * d + 8 * j < dim) *(v4f *)(out + at) = v * per;
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
            *(v4f *)(part + kRows * 2 + r * D + 32 * d + 8 * j + 4 * h2) = v * by;
          }
      }
    }
    u += done;
    if (u >= end) break;
    // ---- the next item: the next row tile, head or sequence (one more step is left, so there is one)
    o.step = 0;
    if (++o.rt * kRows >= count * (after->a.heads / after->c.heads)) {
      o.rt = 0;
      if (++o.h == after->c.heads) {
        o.h = 0;
        do {
          if (++o.s >= after->b.sequences) return;
        } while (!wave_sequence_of(after->b, o.s).count);
      }
    }
  }
}

// what blocks found of an item that they shared, a wave a row: the block whose share it starts in joins the parts
template <int D>
__global__ __launch_bounds__(256) void rows_join_kernel(Attention a, Cache c, Batch b, Share sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int32_t group = a.heads / c.heads;
  const Plan p = plan_of(a.work, sh.blocks, b.sequences);
  const int32_t start = p.edge[blockIdx.x], end = p.edge[blockIdx.x + 1];
  if (start >= end || end >= p.edge[sh.blocks]) return;
  const Start o = p.last[blockIdx.x];
  const Sequence q = sequence_of(b, o.s);
  const Tile t = tile_of(a, c, b, sh, q, group, o.rt);
  const int32_t first = end - 1 - o.step, last = first + t.steps - 1;  // the item's steps
  if (first < start || last < end) return;
  const int r = blockIdx.y * 4 + wave;
  if (t.r0 + r >= t.r1) return;
  const int64_t size = kRows * (D + 2);
  const float *parts = (const float *)(a.work + sh.parts);
  float m = -INFINITY, l = 0.0f;
  float acc[D / 64] = {};
  for (int32_t at = blockIdx.x, slot = 1; at < sh.blocks && p.edge[at] <= last; at++, slot = 0) {
    if (p.edge[at + 1] <= p.edge[at]) {  // (a share without steps)
      continue;
    }
    const float *part = parts + (int64_t)(at * 2 + slot) * size;
    const float pm = part[r * 2], pl = part[r * 2 + 1];
    const float m1 = fmaxf(m, pm), ref = m1 == -INFINITY ? 0.0f : m1;
    const float f0 = exp2_of(m - ref), f1 = exp2_of(pm - ref);
    m = m1;
    l = l * f0 + pl * f1;
#pragma unroll
    for (int i = 0; i < D / 64; i++) acc[i] = acc[i] * f0 + part[kRows * 2 + r * D + lane + 64 * i] * f1;
  }
  const int32_t i0 = (t.r0 + r) / group, g = t.r0 + r - i0 * group;
  float *out = (float *)(a.out + (q.begin + i0) * a.out_stride) + (int64_t)(o.h * group + g) * c.dim;
#pragma unroll
  for (int i = 0; i < D / 64; i++)
    if (lane + 64 * i < c.dim) out[lane + 64 * i] = l != 0.0f ? acc[i] / l : 0.0f;
}

int padded(int32_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// How a call's steps are shared: by as many blocks as the GPU holds, or as there can be steps.
Share few_share(const Cache &c, const Batch &b, int32_t heads) {
  const int32_t d = padded(c.dim), positions = 16 * few_np(d, c.f16);
  const int64_t rows = (int64_t)b.tokens * (heads / c.heads);
  const int64_t tiles = std::min(rows, rows / kFewRows + b.sequences);
  const int64_t steps = (((int64_t)b.width << c.shift) + positions - 1) / positions + 1;
  const int32_t blocks = (int32_t)std::min<int64_t>(few_blocks_a_cu(d, c.f16) * 256, tiles * c.heads * steps);
  return {blocks, kFewRows, positions, (int32_t)tiles, 0, (int64_t)blocks * 2 * kFewRows * (d + 2) * 4, tiles * c.heads * steps};
}
Share rows_share(const Cache &c, const Batch &b, int32_t heads) {
  const int32_t d = padded(c.dim);
  const int64_t rows = (int64_t)b.tokens * (heads / c.heads);
  const int64_t tiles = std::min(rows, rows / kRows + b.sequences);
  const int64_t steps = (((int64_t)b.width << c.shift) + kPositions - 1) / kPositions + 1;
  const int32_t blocks = (int32_t)std::min<int64_t>(rows_blocks_a_cu(d) * 256, tiles * c.heads * steps);
  const int64_t plan = plan_bytes(blocks, b.sequences, tiles);
  return {blocks, kRows, kPositions, (int32_t)tiles, plan, plan + (int64_t)blocks * 2 * kRows * (d + 2) * 4, tiles * c.heads * steps};
}

// whether few_kernel takes the call: no sequence has more rows of a head than two of its tiles (8 sequences of 5 tokens, 20 rows,
// over 4100 positions: 43 us in its tiles, 74 in rows_kernel's)
bool few_rows(const Cache &c, const Batch &b, int32_t heads) { return (int64_t)b.longest * (heads / c.heads) <= 2 * kFewRows; }

template <int D>
hipError_t launch(const Attention &a, const Cache &c, const Batch &b, hipStream_t s) {
  if (few_rows(c, b, a.heads)) {
    const Share sh = few_share(c, b, a.heads);
    hipLaunchKernelGGL((c.f16 ? few_kernel<D, 1> : few_kernel<D, 0>), dim3(sh.blocks), dim3(256), 0, s, Call{a, c, b, sh});
    if (sh.blocks > 1) hipLaunchKernelGGL(join_kernel<D>, dim3(sh.blocks, kFewRows / 4), dim3(256), 0, s, a, c, b, sh);
  } else {
    const Share sh = rows_share(c, b, a.heads);
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(1024), 0, s, a, c, b, sh);
    hipLaunchKernelGGL((c.f16 ? rows_kernel<D, 1> : rows_kernel<D, 0>), dim3(sh.blocks), dim3(256), 0, s, Call{a, c, b, sh});
    if (sh.blocks > 1) hipLaunchKernelGGL(rows_join_kernel<D>, dim3(sh.blocks, kRows / 4), dim3(256), 0, s, a, c, b, sh);
  }
  return hipGetLastError();
}

}  // namespace

int64_t attention_work_bytes(const Cache &c, const Batch &b, int32_t heads) {
  if (b.tokens <= 0 || b.sequences <= 0) return 0;
  const Share few = few_share(c, b, heads), rows = rows_share(c, b, heads);
  if (few.most > INT32_MAX || rows.most > INT32_MAX) return -1;  // (steps are counted in 32 bits)
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
