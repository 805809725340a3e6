// adapters.hip — low-rank adapters of many requests beside the products of one input.
//
//   low[t] = a[w] x[t]  (rank numbers a projection);  y[t] = from[t] + scales[w] b[w] low[t],  w = which[t's sequence]
//
// Two launches on the float32 matrix instructions (16 x 16 x 4): the low numbers of all projections, 16 tokens of a sequence a block whose
// waves (and, for few tokens, blocks) share the n values and add what they have in a fixed order; then each projection's rows, 16
// tokens and some rows a wave.  Factors widen to float32 exactly, so all that is rounded are float32's products and sums.
// A token alone has a tile of its own: what such calls take is their factors' bytes.
#include <algorithm>

#include "paged.hpp"

namespace hq {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 16, kShift = 4;
constexpr int kSplits = 8;   // blocks that share a tile's n values at most
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

// Lane l of a tile: column (token) l & 15, and of every 32 values those from 8 (l / 16) on: instruction j of 8 takes value 8 (l / 16) + j
// of both operands
template <int BF16, int TILES>
__global__ __launch_bounds__(256) void down_kernel(Adapters a, Batch b, int32_t splits) {
  __shared__ f32x4 part[4][TILES][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, group = lane >> 4;
  const Tokens t = tokens_of(a, b, blockIdx.x);
  if (!t.count || t.adapter < 0) return;
  const int32_t numbers = a.count * a.rank, tile0 = blockIdx.z * TILES, split = blockIdx.y;
  const int32_t steps = a.n >> 5, share = 4 * split + wave, shares = 4 * splits;
  const int32_t from = (int32_t)((int64_t)steps * share / shares), to = (int32_t)((int64_t)steps * (share + 1) / shares);
  const float *x = (const float *)(a.x + (t.first + min(col, t.count - 1)) * a.x_stride) + 8 * group;
  const char *f[TILES];
  f32x4 sum[TILES];
#pragma unroll
  for (int i = 0; i < TILES; i++) {
    const int32_t q = min((tile0 + i) * kTile + col, numbers - 1), target = q / a.rank, r = q - target * a.rank;
    f[i] = a.target[target].a + 2 * (((int64_t)t.adapter * a.rank + r) * a.n + 8 * group);
    sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll 2
  for (int32_t s = from; s < to; s++) {
    const float4 x0 = *(const float4 *)(x + 32 * (int64_t)s), x1 = *(const float4 *)(x + 32 * (int64_t)s + 4);
    uint4 h[TILES];
#pragma unroll
    for (int i = 0; i < TILES; i++) h[i] = *(const uint4 *)(f[i] + 64 * (int64_t)s);
    const float e[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
    for (int i = 0; i < TILES; i++) {
      float m[8];
      widen2<BF16>(h[i].x, m), widen2<BF16>(h[i].y, m + 2), widen2<BF16>(h[i].z, m + 4), widen2<BF16>(h[i].w, m + 6);
#pragma unroll
      for (int j = 0; j < 8; j++) sum[i] = mfma(m[j], e[j], sum[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < TILES; i++) part[wave][i][lane] = sum[i];
  __syncthreads();
  // low numbers 4 group .. + 3 of a tile, of token `col`
  for (int i = wave; i < TILES; i += 4) {
    const int32_t q = (tile0 + i) * kTile + 4 * group;
    const f32x4 all = part[0][i][lane] + part[1][i][lane] + part[2][i][lane] + part[3][i][lane];
    if (q < numbers && col < t.count) *(f32x4 *)(a.work + ((int64_t)split * b.tokens + t.first + col) * numbers + q) = all;
  }
}

// ROWS: a wave's rows in tiles of 16
template <int BF16, int RANK32, int ROWS>
__global__ __launch_bounds__(256) void up_kernel(Adapters a, Batch b, int32_t splits) {
  const int lane = threadIdx.x & 63, col = lane & 15, group = lane >> 4;
  const Target &o = a.target[blockIdx.z];
  const int32_t row0 = __builtin_amdgcn_readfirstlane((blockIdx.y * 4 + (threadIdx.x >> 6)) * (kTile * ROWS));
  if (blockIdx.y * (4 * kTile * ROWS) >= (uint32_t)o.rows) return;
  const Tokens t = tokens_of(a, b, blockIdx.x);
  if (!t.count || row0 >= o.rows) return;
  const bool there = col < t.count;
  const int64_t token = t.first + min(col, t.count - 1);
  const float *from = o.from ? (const float *)(o.from + token * o.from_stride) : nullptr;
  float *y = (float *)(o.y + token * o.y_stride);
  // the token's low numbers times the adapter's scale: 8 group .. of every 32, 4 group .. of 16 and 2 group .. of 8 that are left
  const bool adapted = t.adapter >= 0;
  const int32_t numbers = a.count * a.rank, whole = a.rank >> 5;
  float low[8 * RANK32], low16[4] = {0.f, 0.f, 0.f, 0.f}, low8[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 8 * RANK32; i++) low[i] = 0.f;
  if (adapted) {
    for (int32_t s = 0; s < splits; s++) {
      const float *w = a.work + ((int64_t)s * b.tokens + token) * numbers + blockIdx.z * a.rank;
#pragma unroll
      for (int i = 0; i < RANK32; i++) {
        if (i >= whole) break;
        const float4 w0 = *(const float4 *)(w + 32 * i + 8 * group), w1 = *(const float4 *)(w + 32 * i + 8 * group + 4);
        low[8 * i] += w0.x, low[8 * i + 1] += w0.y, low[8 * i + 2] += w0.z, low[8 * i + 3] += w0.w;
        low[8 * i + 4] += w1.x, low[8 * i + 5] += w1.y, low[8 * i + 6] += w1.z, low[8 * i + 7] += w1.w;
      }
      if (a.rank & 16) {
        const float4 w0 = *(const float4 *)(w + 32 * whole + 4 * group);
        low16[0] += w0.x, low16[1] += w0.y, low16[2] += w0.z, low16[3] += w0.w;
      }
      if (a.rank & 8) {
        const float2 w0 = *(const float2 *)(w + (a.rank & ~15) + 2 * group);
        low8[0] += w0.x, low8[1] += w0.y;
      }
    }
  }
  const float scale = adapted && a.scales ? a.scales[t.adapter] : 1.0f;
  const char *f = o.b + 2 * (int64_t)max(t.adapter, 0) * o.rows * a.rank;
#pragma unroll 4
  for (int r = 0; r < ROWS; r++) {
    const int32_t tile = row0 + kTile * r, row = tile + 4 * group;
    if (tile >= o.rows) break;
    const bool full = tile + kTile <= o.rows;
    float4 base = make_float4(0.f, 0.f, 0.f, 0.f);
    if (from) {
      if (full) {
        base = *(const float4 *)(from + row);
      } else {
        float *e = &base.x;
#pragma unroll
        for (int j = 0; j < 4; j++) e[j] = row + j < o.rows ? from[row + j] : 0.f;
      }
    }
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (adapted) {
      const char *m = f + 2 * (int64_t)min(tile + col, o.rows - 1) * a.rank;
#pragma unroll
      for (int i = 0; i < RANK32; i++) {
        if (i >= whole) break;
        const uint4 h = *(const uint4 *)(m + 64 * i + 16 * group);
        float e[8];
        widen2<BF16>(h.x, e), widen2<BF16>(h.y, e + 2), widen2<BF16>(h.z, e + 4), widen2<BF16>(h.w, e + 6);
#pragma unroll
        for (int j = 0; j < 8; j++) sum = mfma(e[j], low[8 * i + j], sum);
      }
      if (a.rank & 16) {
        const uint2 h = *(const uint2 *)(m + 64 * whole + 8 * group);
        float e[4];
        widen2<BF16>(h.x, e), widen2<BF16>(h.y, e + 2);
#pragma unroll
        for (int j = 0; j < 4; j++) sum = mfma(e[j], low16[j], sum);
      }
      if (a.rank & 8) {
        float e[2];
        widen2<BF16>(*(const uint32_t *)(m + 2 * (a.rank & ~15) + 4 * group), e);
        sum = mfma(e[0], low8[0], sum);
        sum = mfma(e[1], low8[1], sum);
      }
    }
    const float4 out = make_float4(fmaf(scale, sum[0], base.x), fmaf(scale, sum[1], base.y), fmaf(scale, sum[2], base.z),
                                   fmaf(scale, sum[3], base.w));
    if (!there) continue;
    if (full) {
      *(float4 *)(y + row) = out;
    } else {
      const float e[4] = {out.x, out.y, out.z, out.w};
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (row + j < o.rows) y[row + j] = e[j];
    }
  }
}

int32_t tiles_of(int32_t count, int32_t rank) { return (count * rank + kTile - 1) / kTile; }
// blocks that share a tile's n values: about two blocks a compute unit where there are few tokens
int32_t splits_of(int32_t count, int32_t rank, int32_t tokens) {
  const int64_t blocks = (int64_t)((tokens + kTile - 1) / kTile) * ((tiles_of(count, rank) + kMostTiles - 1) / kMostTiles);
  return (int32_t)std::max<int64_t>(1, std::min<int64_t>(kSplits, 512 / std::max<int64_t>(blocks, 1)));
}

}  // namespace

int64_t adapters_work_bytes(int32_t count, int32_t rank, int32_t tokens) {
  return 4 * (int64_t)splits_of(count, rank, tokens) * tokens * count * rank;
}

hipError_t launch_adapters(const Adapters &a, const Batch &b, hipStream_t s) {
  if (b.tokens <= 0 || b.sequences <= 0 || a.count <= 0) return hipSuccess;
  int32_t rows = 0;
  for (int i = 0; i < a.count; i++) rows = std::max(rows, a.target[i].rows);
  const uint32_t items = (uint32_t)(b.tokens / kTile + 2 * b.sequences);
  const int32_t tiles = tiles_of(a.count, a.rank), splits = splits_of(a.count, a.rank, b.tokens);
  if (a.adapters > 0) {
    const int32_t each = std::min(tiles, kMostTiles);
    const dim3 grid(items, (uint32_t)splits, (uint32_t)((tiles + each - 1) / each));
    const auto kernel = a.bf16 ? each == 1 ? down_kernel<1, 1> : each == 2 ? down_kernel<1, 2> : each == 3 ? down_kernel<1, 3> : down_kernel<1, 4>
                               : each == 1 ? down_kernel<0, 1> : each == 2 ? down_kernel<0, 2> : each == 3 ? down_kernel<0, 3> : down_kernel<0, 4>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, b, splits);
    if (const hipError_t e = hipGetLastError()) return e;
  }
  if (rows == 0) return hipSuccess;
  const bool many = b.tokens >= 512;  // (a wave's rows: 256 where there are tokens enough, else 64)
  const int32_t block = 4 * kTile * (many ? 16 : 4);
  const dim3 grid(items, (uint32_t)((rows + block - 1) / block), (uint32_t)a.count);
  const auto pick = [&](auto r2, auto r8) {
    constexpr int R2 = decltype(r2)::value, R8 = decltype(r8)::value;
    if (a.rank < 96) return a.bf16 ? many ? up_kernel<1, R2, 16> : up_kernel<1, R2, 4> : many ? up_kernel<0, R2, 16> : up_kernel<0, R2, 4>;
    return a.bf16 ? many ? up_kernel<1, R8, 16> : up_kernel<1, R8, 4> : many ? up_kernel<0, R8, 16> : up_kernel<0, R8, 4>;
  };
  hipLaunchKernelGGL(pick(std::integral_constant<int, 2>(), std::integral_constant<int, 8>()), grid, dim3(256), 0, s, a, b, splits);
  return hipGetLastError();
}

}  // namespace hq
