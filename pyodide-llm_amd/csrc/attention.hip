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
  int32_t positions;  // of a block's step
  int32_t most_rows;  // sequences of more rows are not this kernel's
};

// a tile's rows r0 .. r1 - 1 of a sequence, the positions from .. to - 1 that some of them see, and the steps that hold
// these: first .. first + steps - 1 (one at least: rows that see nothing are written too)
struct Tile {
  int32_t r0, r1, from, to, first, steps;
};
HQ_DEV Tile tile_of(const Attention &a, const Cache &c, const Batch &b, const Share &sh, const Sequence &q, int32_t group,
                    int32_t rt) {
  Tile t;
  t.r0 = rt * kFewRows;
  t.r1 = min(t.r0 + kFewRows, q.count * group);
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
  if (!rows || rows > sh.most_rows) return 0;
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
  o.q = sequence_of(b, max(p.s, 0));
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

HQ_DEV int32_t all_steps(const Attention &a, const Cache &c, const Batch &b, const Share &sh) {
  int32_t n = 0;
  for (int32_t s = threadIdx.x & 63; s < b.sequences; s += 64) n += steps_of(a, c, b, sh, s);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  return __builtin_amdgcn_readfirstlane(n);
}
HQ_DEV int32_t share_start(int32_t steps, int32_t block, int32_t blocks) {
  return (int32_t)((int64_t)steps * block / blocks);
}

// ---- arithmetic ---------------------------------------------------------------------------------------------------
HQ_DEV float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
HQ_DEV float power_of_2(int e) { return __int_as_float((e + 127) << 23); }
// over the lanes l, l ^ 16, l ^ 32, l ^ 48: a row's
HQ_DEV float max_row(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
HQ_DEV float sum_row(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// x, of which the compiler knows nothing: what a loop derives from it is formed in the loop, not held in scalar registers
HQ_DEV int32_t opaque(int32_t x) {
  asm volatile("" : "+s"(x));
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
HQ_DEV float tanh_of(float x) {
  const float y = fabsf(x), z = x * x;
  const float big = 1.0f - 2.0f * __builtin_amdgcn_rcpf(exp2_of(y * (2.0f * kLog2e)) + 1.0f);
  float t = fmaf(z, -1.4558343870513182e-3f, 3.5921280365724810e-3f);
  t = fmaf(z, t, -8.8632355299021966e-3f);
  t = fmaf(z, t, 2.1869488536155203e-2f);
  t = fmaf(z, t, -5.3968253968253968e-2f);
  t = fmaf(z, t, 1.3333333333333333e-1f);
  t = fmaf(z, t, -3.3333333333333333e-1f);
  return y < 0.55f ? fmaf(x * z, t, x) : copysignf(big, x);
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
#pragma unroll
          for (int e = 0; e < NP; e++) p[e] = cap * kLog2e * tanh_of(p[e] * per_cap);
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
          o.q = sequence_of(after->b, o.s);
        } while (!o.q.count || o.q.count * shared > after->sh.most_rows);
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

int padded(int32_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// how many blocks share the steps, as many as the GPU holds or as there can be steps, and a step's positions
Share few_share(const Cache &c, const Batch &b, int32_t heads) {
  const int32_t d = padded(c.dim), positions = 16 * few_np(d, c.f16);
  const int64_t rows = (int64_t)b.tokens * (heads / c.heads);
  const int64_t tiles = std::min(rows, rows / kFewRows + b.sequences);
  const int64_t steps = (((int64_t)b.width << c.shift) + positions - 1) / positions + 1;
  return {(int32_t)std::min<int64_t>(few_blocks_a_cu(d, c.f16) * 256, tiles * c.heads * steps), positions, INT32_MAX};
}

template <int D>
hipError_t launch_few(const Attention &a, const Cache &c, const Batch &b, hipStream_t s) {
  const Share sh = few_share(c, b, a.heads);
  const auto kernel = c.f16 ? few_kernel<D, 1> : few_kernel<D, 0>;
  hipLaunchKernelGGL(kernel, dim3(sh.blocks), dim3(256), 0, s, Call{a, c, b, sh});
  if (sh.blocks > 1) hipLaunchKernelGGL(join_kernel<D>, dim3(sh.blocks, kFewRows / 4), dim3(256), 0, s, a, c, b, sh);
  return hipGetLastError();
}

}  // namespace

int64_t attention_work_bytes(const Cache &c, const Batch &b, int32_t heads) {
  if (b.tokens <= 0 || b.sequences <= 0) return 0;
  return (int64_t)few_share(c, b, heads).blocks * 2 * kFewRows * (padded(c.dim) + 2) * 4;
}

hipError_t launch_attention(const Attention &a, const Cache &c, const Batch &b, hipStream_t s) {
  if (b.tokens <= 0 || b.sequences <= 0) return hipSuccess;
  switch (padded(c.dim)) {
  case 64: return launch_few<64>(a, c, b, s);
  case 128: return launch_few<128>(a, c, b, s);
  default: return launch_few<256>(a, c, b, s);
  }
}

}  // namespace hq
