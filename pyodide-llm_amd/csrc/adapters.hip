// adapters.hip — low-rank adapters of many requests beside the products of one input.
//
//   low[t] = a[w] x[t]  (rank numbers a projection);  y[t] = from[t] + scales[w] b[w] low[t],  w = which[t's sequence]
//
// Two launches: the low products of all projections, then each projection's rows.
#include "paged.hpp"

namespace hq {

namespace {

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

// a factor's number as float32, exactly
template <int BF16>
HQ_DEV float widen(uint32_t h) {
  return BF16 ? __uint_as_float(h << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
template <int BF16>
HQ_DEV void widen8(const uint4 &v, float f[8]) {
  const uint32_t d[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; i++) f[2 * i] = widen<BF16>(d[i] & 0xffffu), f[2 * i + 1] = widen<BF16>(d[i] >> 16);
}

constexpr int kEach = 4;  // low numbers of a wave

template <int BF16>
__global__ __launch_bounds__(256) void down_kernel(Adapters a, Batch b) {
  const int32_t t = blockIdx.x, lane = threadIdx.x & 63;
  const int32_t low = __builtin_amdgcn_readfirstlane((blockIdx.y * 4 + (threadIdx.x >> 6)) * kEach);
  const int32_t s = sequence_at(b, t);
  if (s < 0 || low >= a.count * a.rank) return;
  const int32_t w = a.which[s];
  if ((uint32_t)w >= (uint32_t)a.adapters) return;
  const int32_t target = low / a.rank, r = low % a.rank;  // (rank is whole fours)
  const float *x = (const float *)(a.x + t * a.x_stride);
  const char *f = a.target[target].a + 2 * ((int64_t)w * a.rank + r) * a.n;
  float sum[kEach] = {0.f, 0.f, 0.f, 0.f};
  for (int32_t i = lane * 8; i < a.n; i += 512) {
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
__global__ __launch_bounds__(256) void up_kernel(Adapters a, Batch b) {
  __shared__ float low[256];
  const int32_t t = blockIdx.x, row = blockIdx.y * 256 + threadIdx.x;
  const Target &o = a.target[blockIdx.z];
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

}  // namespace

int64_t adapters_work_bytes(int32_t count, int32_t rank, int32_t tokens) {
  return 4 * (int64_t)tokens * count * rank;
}

hipError_t launch_adapters(const Adapters &a, const Batch &b, hipStream_t s) {
  if (b.tokens <= 0 || b.sequences <= 0 || a.count <= 0) return hipSuccess;
  int32_t rows = 0;
  for (int i = 0; i < a.count; i++) rows = rows > a.target[i].rows ? rows : a.target[i].rows;
  if (a.adapters > 0) {
    const dim3 grid((uint32_t)b.tokens, (uint32_t)((a.count * a.rank + 4 * kEach - 1) / (4 * kEach)));
    if (a.bf16) hipLaunchKernelGGL(down_kernel<1>, grid, dim3(256), 0, s, a, b);
    else hipLaunchKernelGGL(down_kernel<0>, grid, dim3(256), 0, s, a, b);
    if (const hipError_t e = hipGetLastError()) return e;
  }
  if (rows == 0) return hipSuccess;
  const dim3 grid((uint32_t)b.tokens, (uint32_t)((rows + 255) / 256), (uint32_t)a.count);
  if (a.bf16) hipLaunchKernelGGL(up_kernel<1>, grid, dim3(256), 0, s, a, b);
  else hipLaunchKernelGGL(up_kernel<0>, grid, dim3(256), 0, s, a, b);
  return hipGetLastError();
}

}  // namespace hq
