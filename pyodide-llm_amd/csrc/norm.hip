// norm.hip — the root-mean-square norm between two products: the residual's addition, the norm and the int8 activations
// the next products take, in one launch (norm_ready: the caller's add, norm and ready() of a layer).
//
//   r = x + d;  y_i = r_i w_i / sqrt(mean(r^2) + eps);  then quantize_x of y with what its packing takes (ready.hpp)
//
// The sum of squares, its root and y are held in 64 bits and y rounded once to float32: the products of two float32 are exact
// there, so whatever order the lanes add them in, y is the same float32 but for one value in some 10^8, and an int8 does not
// depend on how many tokens a launch has.  The 64-bit operations run at float32's rate here.
//
// Bound by memory: a block takes a row, whose values stay in registers between the sum and the products.  2048 rows of 4096 values
// with a residual, readied: 110 MB in 21.4 us a call back to back, 5.2 TB/s, as a copy (22.6 us in a profiled run, whose clock is
// lower); a row of 288 values 2.8 us of the GPU's time, 7.8 of the host's for the call.
#include <algorithm>

#include "common.hpp"
#include "launch.hpp"
#include "ready.hpp"

namespace hq {

namespace {

constexpr int kNormKeep = 4;  // passes of the block over the row that stay in registers

template <int MODE>
__global__ __launch_bounds__(1024) void norm_kernel(NormRows a, int32_t n, float eps, int32_t bias) {
  __shared__ double part[16];
  const int64_t t = blockIdx.x + (int64_t)blockIdx.y * gridDim.x;
  if (t >= a.count) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, step = blockDim.x * 4;
  const char *x = a.x + t * a.x_stride, *d = a.d ? a.d + t * a.d_stride : nullptr;
  char *r = a.r ? a.r + t * a.x_stride : nullptr;
  float4 kept[kNormKeep];
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < kNormKeep; i++) {
    const int at = i * step + threadIdx.x * 4;
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    if (at < n) {
      f = *(const float4 *)(x + 4 * (int64_t)at);
      if (d) {
        const float4 g = *(const float4 *)(d + 4 * (int64_t)at);
        f.x = fadd(f.x, g.x), f.y = fadd(f.y, g.y), f.z = fadd(f.z, g.z), f.w = fadd(f.w, g.w);
      }
      if (r) *(float4 *)(r + 4 * (int64_t)at) = f;
    }
    kept[i] = f;
    ss += (double)f.x * f.x + (double)f.y * f.y + ((double)f.z * f.z + (double)f.w * f.w);
  }
  for (int at = kNormKeep * step + threadIdx.x * 4; at < n; at += step) {
    float4 f = *(const float4 *)(x + 4 * (int64_t)at);
    if (d) {
      const float4 g = *(const float4 *)(d + 4 * (int64_t)at);
      f.x = fadd(f.x, g.x), f.y = fadd(f.y, g.y), f.z = fadd(f.z, g.z), f.w = fadd(f.w, g.w);
    }
    if (r) *(float4 *)(r + 4 * (int64_t)at) = f;
    ss += (double)f.x * f.x + (double)f.y * f.y + ((double)f.z * f.z + (double)f.w * f.w);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
  if (lane == 0) part[wave] = ss;
  __syncthreads();
  ss = 0.0;
  for (int i = 0; i < waves; i++) ss += part[i];
  const double inv = 1.0 / sqrt(ss / (double)n + (double)eps);
  char *y = a.y ? a.y + t * a.y_stride : nullptr;
  char *xq = a.xq ? a.xq + t * a.frame : nullptr, *xs = a.xs + t * a.frame;
  const int passes = (n + step - 1) / step;
  const auto finish = [&](int i, float4 f) {
    const int at = i * step + threadIdx.x * 4;
    const bool live = at < n;
    const float4 w = *(const float4 *)(a.w + 4 * (int64_t)(live ? at : 0));
    f.x = (float)((double)f.x * inv * w.x), f.y = (float)((double)f.y * inv * w.y);
    f.z = (float)((double)f.z * inv * w.z), f.w = (float)((double)f.w * inv * w.w);
    if (y && live) *(float4 *)(y + 4 * (int64_t)at) = f;
    if (xq) store_ready<MODE>(quantize4(f, bias), xq, xs, at, n, lane, live);
  };
#pragma unroll
  for (int i = 0; i < kNormKeep; i++)
    if (i < passes) finish(i, kept[i]);
  for (int i = kNormKeep; i < passes; i++) {  // what the lane itself wrote (or read) above, again
    const int at = i * step + threadIdx.x * 4;
    finish(i, *(const float4 *)((r ? r : x) + 4 * (int64_t)(at < n ? at : 0)));
  }
}

template <int MODE>
hipError_t launch_norm_mode(const NormRows &a, int32_t n, float eps, int32_t bias, hipStream_t s) {
  // 256 threads of 4 values and up to kNormKeep passes, then up to 1024 threads: several blocks a compute unit, so that some load
  // while others store (calls back to back, 2048 rows of 4096 values: 21.7 us, in one pass of 1024 threads 25.9; of 2048 values 13.4,
  // in one of 512 14.7; a single row 8.2 us either way).  By the row alone, so that a token's sums run in one order however many tokens there are
  const int32_t lanes = (n + 3) / 4, passes = std::max((lanes + 1023) / 1024, std::min((lanes + 255) / 256, kNormKeep));
  const int32_t threads = ((lanes + passes - 1) / passes + 63) / 64 * 64;
  const uint32_t wide = a.count < 65536 ? (uint32_t)a.count : 65536u;
  hipLaunchKernelGGL(norm_kernel<MODE>, dim3(wide, ((uint32_t)a.count + wide - 1) / wide), dim3(threads), 0, s, a, n, eps,
                     bias);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_norm(Ready mode, const NormRows &a, int32_t n, float eps, int32_t bias, hipStream_t s) {
  if (n <= 0 || a.count <= 0) return hipSuccess;
  switch (mode) {
  case kReadyPlanes: return launch_norm_mode<1>(a, n, eps, bias, s);
  case kReadySums: return launch_norm_mode<2>(a, n, eps, bias, s);
  default: return launch_norm_mode<0>(a, n, eps, bias, s);
  }
}

}  // namespace hq
