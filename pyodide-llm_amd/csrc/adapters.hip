// adapters.hip — low-rank adapters of many requests beside the products of one input.
//
//   low[t] = a[w] x[t]  (rank numbers a projection);  y[t] = from[t] + scales[w] b[w] low[t],  w = which[t's sequence]
//
// Two launches on the float32 matrix instructions (16 x 16 x 4): the low numbers of all projections, 16 tokens of a sequence a block whose
// waves (and, for few tokens, blocks) share the n values and add what they have in a fixed order; then each projection's rows, 16
// tokens and some rows a wave.  Factors widen to float32 exactly, so all that is rounded are float32's products and sums.
// Measured: 2048 tokens of a sequence, rank 64, n and rows 4096: down 22.6 us, up 27.4 (x, from and y are 100 MB, 20 us at a large
// copy's 5.1 TB/s); five prompts of rank 32, n 2048, two projections of 8192 rows: 15.9 and 41.0.  Four tiles of low
// numbers take 142 registers and 66 KB of LDS, one block a compute unit, whose barriers nobody covers: its waves wait to issue 54 % of
// their time (after a barrier all begin their matrix instructions, which are busy 30 %) and for loads and barriers 33 %.  The rows'
// waves wait for loads 59 to 73 %.  Four times the blocks, or rows of 16 x 128 bytes straight from memory, gain nothing.
// Where the batch says that each sequence has one token, a tile would be empty but for one: tokens then have kernels of their own.
#include <algorithm>
#include <type_traits>

#include "paged.hpp"

namespace hq {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 16, kShift = 4;
constexpr int kWaves = 8;      // of a block that makes low numbers: they share the n values,
constexpr int kSplits = 4;     // as do so many blocks at most
constexpr int kMostTiles = 4;  // tiles of 16 low numbers of a block

// factors' numbers as float32
template <int BF16>
HQ_DEV float widen(uint32_t h) {
  return BF16 ? __uint_as_float(h << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
template <int BF16>
HQ_DEV void widen2(uint32_t d, float *f) {
  f[0] = widen<BF16>(d & 0xffffu), f[1] = BF16 ? __uint_as_float(d & 0xffff0000u) : widen<0>(d >> 16);
}
HQ_DEV f32x4 mfma(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// the tokens of a block's tile, and their adapter (-1: none)
struct Tokens {
  int32_t first, count, adapter;
};
HQ_DEV Tokens tokens_of(const Adapters &a, const Batch &b, int32_t at) {
  const Place p = place_of<kShift>(b, at);
  if (p.s < 0) return {0, 0, -1};
  const int32_t rest = p.q.count - p.rest * kTile, w = a.which[p.s];
  return {p.q.begin + p.rest * kTile, min(max(rest, 0), kTile), (uint32_t)w < (uint32_t)a.adapters ? w : -1};
}

// A block takes its tokens' values 256 at a time, a token's kilobyte a wave's load (16 tokens' 128 bytes each reach 1.8 TB/s), into
// LDS, from where wave w takes the w-th 32 of them.  Lane l has column (token) or row l & 15 and of the 32 those from 8 (l / 16)
// on: instruction j of 8 takes value 8 (l / 16) + j of both operands.
constexpr int kChunk = 32 * kWaves, kPitch = kChunk + 4;

template <int TILES>
struct Loads {  // of a chunk: the wave's two tokens' values, and its factors
  f32x4 v0, v1;
  u32x4 h[TILES];
};

template <int BF16, int TILES>
__global__ __launch_bounds__(64 * kWaves) void down_kernel(Adapters a, Batch b, int32_t splits) {
  __shared__ float held[2][kTile][kPitch];
  __shared__ f32x4 part[kWaves][TILES][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, group = lane >> 4;
  const Tokens t = tokens_of(a, b, blockIdx.x);
  if (!t.count || t.adapter < 0) return;
  const int32_t numbers = a.count * a.rank, tile0 = blockIdx.z * TILES, split = blockIdx.y;
  const int32_t chunks = (a.n + kChunk - 1) / kChunk, from = chunks * split / splits, to = chunks * (split + 1) / splits;
  const char *f[TILES];
  f32x4 sum[TILES];
#pragma unroll
  for (int i = 0; i < TILES; i++) {
    const int32_t q = min((tile0 + i) * kTile + col, numbers - 1), target = q / a.rank, r = q - target * a.rank;
    f[i] = a.target[target].a + 2 * (((int64_t)t.adapter * a.rank + r) * a.n + 8 * group + 32 * wave);
    sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // the wave's two tokens (where there are fewer, the last), their values past the end the row's first
  const float *x0 = (const float *)(a.x + (t.first + min(2 * wave, t.count - 1)) * a.x_stride);
  const float *x1 = (const float *)(a.x + (t.first + min(2 * wave + 1, t.count - 1)) * a.x_stride);
  Loads<TILES> l0, l1, l2;  // three chunks on their way
  const int32_t n = a.n;    // (a lambda that takes `a` keeps all of it in memory)
  const auto begin = [&](Loads<TILES> &l, int32_t c) __attribute__((always_inline)) {
    const int32_t i = c * kChunk + 4 * lane, at = i < n ? i : 0;
    l.v0 = *(const f32x4 *)(x0 + at), l.v1 = *(const f32x4 *)(x1 + at);
    const int32_t mine = c * kChunk + 32 * wave < n ? c * kChunk : -32 * wave;
#pragma unroll
    for (int k = 0; k < TILES; k++) l.h[k] = *(const u32x4 *)(f[k] + 2 * (int64_t)mine);
  };
  const auto step = [&](Loads<TILES> &l, int32_t c) __attribute__((always_inline)) {
    float (*x)[kPitch] = held[c & 1];
    *(f32x4 *)&x[2 * wave][4 * lane] = l.v0, *(f32x4 *)&x[2 * wave + 1][4 * lane] = l.v1;
    float m[TILES][8];
#pragma unroll
    for (int i = 0; i < TILES; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) widen2<BF16>(l.h[i][j], m[i] + 2 * j);
    if (c + 3 < to) begin(l, c + 3);
    __syncthreads();  // (the other buffer is written when all have read this one: after the next of these)
    const f32x4 e0 = *(const f32x4 *)&x[col][32 * wave + 8 * group], e1 = *(const f32x4 *)&x[col][32 * wave + 8 * group + 4];
    if (c * kChunk + 32 * wave < n) {
#pragma unroll
      for (int j = 0; j < 8; j++)
#pragma unroll
        for (int i = 0; i < TILES; i++) sum[i] = mfma(m[i][j], j < 4 ? e0[j & 3] : e1[j & 3], sum[i]);
    }
  };
  if (from < to) {
    begin(l0, from);
    if (from + 1 < to) begin(l1, from + 1);
    if (from + 2 < to) begin(l2, from + 2);
    for (int32_t c = from; c < to; c += 3) {
      step(l0, c);
      if (c + 1 < to) step(l1, c + 1);
      if (c + 2 < to) step(l2, c + 2);
    }
  }
#pragma unroll
  for (int i = 0; i < TILES; i++) part[wave][i][lane] = sum[i];
  __syncthreads();
  // low numbers 4 group .. + 3 of a tile, of token `col`
  for (int i = wave; i < TILES; i += kWaves) {
    const int32_t q = (tile0 + i) * kTile + 4 * group;
    f32x4 all = part[0][i][lane];
#pragma unroll
    for (int k = 1; k < kWaves; k++) all += part[k][i][lane];
    if (q < numbers && col < t.count) *(f32x4 *)(a.work + ((int64_t)split * b.tokens + t.first + col) * numbers + q) = all;
  }
}

// the low numbers, or a row's factors, of a lane: of every 32 those from 8 group on, of 16 that are left from 4 group, of 8 from 2 group
template <int WHOLE, typename T>
struct Ranks {
  T whole[WHOLE ? WHOLE : 1][8], half[4], quarter[2];
};

constexpr int kSpan = 64;  // rows at a time

// WHOLE: 32s of the rank (8: up to so many); ROWS: a wave's rows in tiles of 16
template <int BF16, int WHOLE, int ROWS>
__global__ __launch_bounds__(256) void up_kernel(Adapters a, Batch b, int32_t splits) {
  const int lane = threadIdx.x & 63, col = lane & 15, group = lane >> 4;
  const Target &o = a.target[blockIdx.z];
  const int32_t row0 = __builtin_amdgcn_readfirstlane((blockIdx.y * 4 + (threadIdx.x >> 6)) * (kTile * ROWS));
  if (row0 >= o.rows) return;
  const Tokens t = tokens_of(a, b, blockIdx.x);
  if (!t.count) return;
  __shared__ float turned[4][kTile][kSpan + 4];
  float (*turn)[kSpan + 4] = turned[threadIdx.x >> 6];  // (the wave's own)
  const int64_t token = t.first + min(col, t.count - 1);
  const bool adapted = t.adapter >= 0, halves = a.rank & 16, quarters = a.rank & 8;
  const int32_t numbers = a.count * a.rank, whole = WHOLE < 8 ? WHOLE : a.rank >> 5;
  Ranks<WHOLE, float> low = {};
  if (adapted) {
#pragma unroll
    for (int s = 0; s < kSplits; s++) {
      if (s >= splits) break;
      const float *w = a.work + ((int64_t)s * b.tokens + token) * numbers + blockIdx.z * a.rank;
#pragma unroll
      for (int i = 0; i < WHOLE; i++) {
        if (i >= whole) break;
        const float4 w0 = *(const float4 *)(w + 32 * i + 8 * group), w1 = *(const float4 *)(w + 32 * i + 8 * group + 4);
        const float e[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int j = 0; j < 8; j++) low.whole[i][j] += e[j];
      }
      if (halves) {
        const float4 w0 = *(const float4 *)(w + 32 * whole + 4 * group);
        low.half[0] += w0.x, low.half[1] += w0.y, low.half[2] += w0.z, low.half[3] += w0.w;
      }
      if (quarters) {
        const float2 w0 = *(const float2 *)(w + (a.rank & ~15) + 2 * group);
        low.quarter[0] += w0.x, low.quarter[1] += w0.y;
      }
    }
  }
  const float scale = adapted && a.scales ? a.scales[t.adapter] : 1.0f;
  const char *f = o.b + 2 * (int64_t)max(t.adapter, 0) * o.rows * a.rank;
  // the product of 16 rows with these, the k-th 16 of a span
  const auto multiply = [&](const uint4 *h, const uint2 &h16, uint32_t h8, int k) {
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < WHOLE; i++) {
      if (WHOLE == 8 && i >= whole) break;
      float e[8];
      widen2<BF16>(h[i].x, e), widen2<BF16>(h[i].y, e + 2), widen2<BF16>(h[i].z, e + 4), widen2<BF16>(h[i].w, e + 6);
#pragma unroll
      for (int j = 0; j < 8; j++) sum = mfma(e[j], low.whole[i][j], sum);
    }
    if (halves) {
      float e[4];
      widen2<BF16>(h16.x, e), widen2<BF16>(h16.y, e + 2);
#pragma unroll
      for (int j = 0; j < 4; j++) sum = mfma(e[j], low.half[j], sum);
    }
    if (quarters) {
      float e[2];
      widen2<BF16>(h8, e);
      sum = mfma(e[0], low.quarter[0], sum);
      sum = mfma(e[1], low.quarter[1], sum);
    }
    *(f32x4 *)&turn[col][kTile * k + 4 * group] = sum;
  };
  const int32_t rows = min(o.rows - row0, kTile * ROWS);  // the wave's
  const bool aligned = !(((uintptr_t)o.from | (uintptr_t)o.y | (uint32_t)o.from_stride | (uint32_t)o.y_stride) & 15);  // (else a float at a time)
  // The products of 16 tokens and kSpan rows turn in LDS, so that a token's numbers are read and written 16 lanes (256 bytes) together
  const int32_t first = lane >> 4, at4 = 4 * col;  // (tokens first, first + 4, ..)
  for (int32_t r0 = 0; r0 < rows; r0 += kSpan) {
    const int32_t row = row0 + r0 + at4;
    const bool full = r0 + kSpan <= rows && aligned;
    f32x4 base[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      base[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (!o.from) continue;
      const float *from = (const float *)(o.from + (t.first + min(first + 4 * i, t.count - 1)) * o.from_stride);
      if (full) {
        base[i] = *(const f32x4 *)(from + row);
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++) base[i][j] = from[min(row + j, o.rows - 1)];
      }
    }
    if (adapted) {
      // (rows past the end are the last)
      uint4 h[kSpan / kTile][WHOLE ? WHOLE : 1];
      uint2 h16[kSpan / kTile];
      uint32_t h8[kSpan / kTile];
#pragma unroll
      for (int k = 0; k < kSpan / kTile; k++) {
        const char *m = f + 2 * (int64_t)min(row0 + r0 + kTile * k + col, o.rows - 1) * a.rank;
        h16[k] = make_uint2(0, 0), h8[k] = 0;
#pragma unroll
        for (int i = 0; i < WHOLE; i++)
          if (WHOLE < 8 || i < whole) h[k][i] = *(const uint4 *)(m + 64 * i + 16 * group);
        if (halves) h16[k] = *(const uint2 *)(m + 64 * whole + 8 * group);
        if (quarters) h8[k] = *(const uint32_t *)(m + 2 * (a.rank & ~15) + 4 * group);
        if (WHOLE == 8) multiply(h[k], h16[k], h8[k], k);
      }
      if (WHOLE < 8) {
#pragma unroll
        for (int k = 0; k < kSpan / kTile; k++) multiply(h[k], h16[k], h8[k], k);
      }
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int32_t mine = first + 4 * i;
      f32x4 sum = base[i];
      if (adapted) {
        const f32x4 add = *(const f32x4 *)&turn[mine][at4];
#pragma unroll
        for (int j = 0; j < 4; j++) sum[j] = fmaf(scale, add[j], sum[j]);
      }
      if (mine >= t.count) continue;
      float *y = (float *)(o.y + (int64_t)(t.first + mine) * o.y_stride);
      if (full) {
        *(f32x4 *)(y + row) = sum;
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (row + j < o.rows) y[row + j] = sum[j];
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// ---- single tokens ----------------------------------------------------------------------------------------------------
// A token's low numbers, four a wave; then its rows, one a thread: no tile waits for 15 tokens that are not there, and more waves
// have loads on their way

// the sequence that has row t (-1: none): the last whose first row is not behind t
HQ_DEV int32_t sequence_at(const Batch &b, int32_t t) {
  int32_t lo = 0, hi = b.sequences;
  while (hi - lo > 1) {
    const int32_t mid = (lo + hi) >> 1;
    if (b.starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  return b.starts[lo] <= t && t < b.starts[lo + 1] ? lo : -1;
}
template <int BF16>
HQ_DEV void widen8(const uint4 &v, float f[8]) {
  widen2<BF16>(v.x, f), widen2<BF16>(v.y, f + 2), widen2<BF16>(v.z, f + 4), widen2<BF16>(v.w, f + 6);
}

constexpr int kEach = 4;  // low numbers of a wave

template <int BF16>
__global__ __launch_bounds__(256) void token_down_kernel(Adapters a, Batch b, int32_t first) {
  const int32_t t = first + blockIdx.x, lane = threadIdx.x & 63;
  const int32_t low = __builtin_amdgcn_readfirstlane((blockIdx.y * 4 + (threadIdx.x >> 6)) * kEach);
  const int32_t s = sequence_at(b, t);
  if (s < 0 || low >= a.count * a.rank) return;
  const int32_t w = a.which[s];
  if ((uint32_t)w >= (uint32_t)a.adapters) return;
  const int32_t target = low / a.rank, r = low % a.rank;  // (rank is whole fours)
  const float *x = (const float *)(a.x + t * a.x_stride);
  const char *f = a.target[target].a + 2 * ((int64_t)w * a.rank + r) * a.n;
  float sum[kEach] = {0.f, 0.f, 0.f, 0.f};
  for (uint32_t i = lane * 8; i < (uint32_t)a.n; i += 512) {  // (a single token's row may end within 512 of 2^31)
    const float4 x0 = *(const float4 *)(x + i), x1 = *(const float4 *)(x + i + 4);
    const float e[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
    for (int k = 0; k < kEach; k++) {
      float m[8];
      widen8<BF16>(*(const uint4 *)(f + 2 * ((int64_t)k * a.n + i)), m);
#pragma unroll
      for (int j = 0; j < 8; j++) sum[k] = fmaf(m[j], e[j], sum[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < kEach; k++) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum[k] += __shfl_xor(sum[k], o, 64);
    if (lane == 0) a.work[(int64_t)t * a.count * a.rank + low + k] = sum[k];
  }
}

template <int BF16>
__global__ __launch_bounds__(256) void token_up_kernel(Adapters a, Batch b, int32_t first) {
  __shared__ float low[256];
  const int32_t t = first + blockIdx.x, row = blockIdx.y * 256 + threadIdx.x;
  const Target &o = a.target[blockIdx.z];
  if ((int32_t)blockIdx.y * 256 >= o.rows) return;
  const int32_t s = sequence_at(b, t);
  if (s < 0) return;
  const int32_t w = a.which[s];
  const bool adapted = (uint32_t)w < (uint32_t)a.adapters;
  if (adapted && (int32_t)threadIdx.x < a.rank)
    low[threadIdx.x] = a.work[((int64_t)t * a.count + blockIdx.z) * a.rank + threadIdx.x];
  __syncthreads();
  if (row >= o.rows) return;
  float y = o.from ? ((const float *)(o.from + t * o.from_stride))[row] : 0.0f;
  if (adapted) {
    float sum = 0.0f;
    const char *f = o.b + 2 * ((int64_t)w * o.rows + row) * a.rank;
    for (int32_t i = 0; i < a.rank; i += 8) {
      float m[8];
      widen8<BF16>(*(const uint4 *)(f + 2 * i), m);
#pragma unroll
      for (int j = 0; j < 8; j++) sum = fmaf(m[j], low[i + j], sum);
    }
    y = fmaf(a.scales ? a.scales[w] : 1.0f, sum, y);
  }
  ((float *)(o.y + t * o.y_stride))[row] = y;
}

int32_t tiles_of(int32_t count, int32_t rank) { return (count * rank + kTile - 1) / kTile; }
// blocks that share a tile's n values: about one a compute unit where there are few tokens
int32_t splits_of(int32_t count, int32_t rank, int32_t tokens) {
  const int64_t blocks = (int64_t)((tokens + kTile - 1) / kTile) * ((tiles_of(count, rank) + kMostTiles - 1) / kMostTiles);
  return (int32_t)std::max<int64_t>(1, std::min<int64_t>(kSplits, 256 / std::max<int64_t>(blocks, 1)));
}

}  // namespace

// What is written is `splits` times tokens x count x rank numbers, which may be more for fewer projections or tokens, as these are
// split more often.  A call may run fewer projections than it states (those without rows are left out), and a workspace is kept for
// steps of many sizes: this grows with each of the three and covers them all.  A launch that splits has 256 blocks at most, and a
// block writes at most 16 tokens' 16 kMostTiles numbers.
int64_t adapters_work_bytes(int32_t count, int32_t rank, int32_t tokens) {
  const int64_t numbers = (int64_t)tokens * count * rank, split = 256 * kTile * kTile * kMostTiles;
  return 4 * std::max(numbers, std::min(kSplits * numbers, split));
}

hipError_t launch_adapters(const Adapters &a, const Batch &b, hipStream_t s) {
  if (b.tokens <= 0 || b.sequences <= 0 || a.count <= 0) return hipSuccess;
  int32_t rows = 0;
  for (int i = 0; i < a.count; i++) rows = std::max(rows, a.target[i].rows);
  if (b.longest == 1) {  // 32 tokens of 3 projections, n 4096: 9.0 us of kernels, as tiles of one token 17.9
    const auto lows = a.bf16 ? token_down_kernel<1> : token_down_kernel<0>;
    const auto ups = a.bf16 ? token_up_kernel<1> : token_up_kernel<0>;
    constexpr int32_t kTokens = 1 << 23;  // of a launch (a dimension has fewer than 2^32 threads)
    for (int32_t first = 0; first < b.tokens; first += kTokens) {
      const uint32_t tokens = (uint32_t)std::min(b.tokens - first, kTokens);
      const dim3 down(tokens, (uint32_t)((a.count * a.rank + 4 * kEach - 1) / (4 * kEach)));
      if (a.adapters > 0) hipLaunchKernelGGL(lows, down, dim3(256), 0, s, a, b, first);
      if (const hipError_t e = hipGetLastError()) return e;
      const dim3 up(tokens, (uint32_t)((rows + 255) / 256), (uint32_t)a.count);
      if (rows) hipLaunchKernelGGL(ups, up, dim3(256), 0, s, a, b, first);
      if (const hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
  }
  const uint32_t items = (uint32_t)(b.tokens / kTile + 2 * b.sequences);
  const int32_t tiles = tiles_of(a.count, a.rank), splits = splits_of(a.count, a.rank, b.tokens);
  if (a.adapters > 0) {
    const int32_t each = std::min(tiles, kMostTiles);
    const dim3 grid(items, (uint32_t)splits, (uint32_t)((tiles + each - 1) / each));
    const auto kernel = a.bf16 ? each == 1 ? down_kernel<1, 1> : each == 2 ? down_kernel<1, 2> : each == 3 ? down_kernel<1, 3> : down_kernel<1, 4>
                               : each == 1 ? down_kernel<0, 1> : each == 2 ? down_kernel<0, 2> : each == 3 ? down_kernel<0, 3> : down_kernel<0, 4>;
    hipLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), 0, s, a, b, splits);
    if (const hipError_t e = hipGetLastError()) return e;
  }
  if (rows == 0) return hipSuccess;
  constexpr int32_t kRows = 4, block = 4 * kTile * kRows;  // a wave's rows are 64 (256 take a tenth longer: 30.0 us for 27.5 at 2048 tokens)
  const dim3 grid(items, (uint32_t)((rows + block - 1) / block), (uint32_t)a.count);
  const int32_t whole = a.rank >> 5;
  const auto launch = [&](auto bf16, auto most) {
    constexpr int B = decltype(bf16)::value, W = decltype(most)::value;
    const auto kernel = up_kernel<B, W, kRows>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, b, splits);
  };
  const auto pick = [&](auto bf16) {
    using std::integral_constant;
    if (whole == 0) launch(bf16, integral_constant<int, 0>());
    else if (whole == 1) launch(bf16, integral_constant<int, 1>());
    else if (whole == 2) launch(bf16, integral_constant<int, 2>());
    else launch(bf16, integral_constant<int, 8>());
  };
  if (a.bf16) pick(std::integral_constant<int, 1>());
  else pick(std::integral_constant<int, 0>());
  return hipGetLastError();
}

}  // namespace hq
