// embed.hip — embeddings of token ids from a packed table (the block types' are in blocks.hip, beside their reader).
//
//   out[t][i] = f(f(value(ids[t], i) scale(ids[t], i's group)) times)
//
// A thread takes 4 neighbouring weights of a row: a dword of int8 values, the low and the high bits of four int6 values, a byte
// of ternary codes, a nibble of binary signs, and one group's scale: a wave writes a kilobyte at once, and what bounds a large call is
// memory.  2048 int8 rows of 4096: 9.3 us a call (4.6 TB/s of a copy's 5.1); a row of 288: 1.7 us of kernel, the launch is the call.
#include "common.hpp"
#include "launch.hpp"

namespace hq {

namespace {

// weights 4 q .. 4 q + 3 of the row at v as integers
template <int PACKING>
HQ_DEV void four(const char *v, int32_t q, float e[4]) {
  if (PACKING == kPackInt8) {
    const uint32_t d = ((const uint32_t *)v)[q];
#pragma unroll
    for (int j = 0; j < 4; j++) e[j] = (float)(int32_t)(int8_t)(d >> (8 * j));
  } else if (PACKING == kPackInt6) {  // six_widen's dword i of a group's eight
    const char *g = v + (int64_t)(q >> 3) * 24;
    const int i = q & 7;
    const uint32_t low = *(const uint32_t *)(g + 4 * (i & 3)), top = *(const uint32_t *)(g + 16 + 4 * (i & 1));
    const uint32_t nibbles = i < 4 ? low << 2 : low >> 2, bits = top << (6 - 2 * (i >> 1));
    const uint32_t d = (nibbles & 0x3c3c3c3cu) | (bits & 0xc0c0c0c0u);
#pragma unroll
    for (int j = 0; j < 4; j++) e[j] = (float)(int32_t)(int8_t)(d >> (8 * j));
  } else if (PACKING == kPackTernary) {
    const uint32_t d = ((const uint8_t *)v)[q];
#pragma unroll
    for (int j = 0; j < 4; j++) e[j] = (float)((int32_t)((d >> (2 * j)) & 3u) - 1);
  } else {
    const uint32_t d = ((const uint8_t *)v)[((q >> 5) << 4) + (q & 15)] >> (4 * ((q >> 4) & 1));
#pragma unroll
    for (int j = 0; j < 4; j++) e[j] = (float)((int32_t)(((d >> j) & 1u) << 1) - 1);
  }
}

constexpr int64_t row_bytes(int packing, int64_t dim) {
  return packing == kPackInt8 ? dim : packing == kPackInt6 ? dim / 4 * 3 : packing == kPackTernary ? dim / 4 : dim / 8;
}

template <int PACKING>
__global__ __launch_bounds__(256) void embed_kernel(Embed e, int32_t group_shift) {
  const int32_t q = blockIdx.x * 256 + threadIdx.x;
  if (q >= (e.dim >> 2)) return;
  for (int64_t t = blockIdx.y; t < e.count; t += gridDim.y) {
    float4 *to = (float4 *)(e.out + t * e.out_stride) + q;
    const int32_t id = e.ids[t];
    if ((uint32_t)id >= (uint32_t)e.vocab) {
      *to = make_float4(0.f, 0.f, 0.f, 0.f);
      continue;
    }
    const int64_t g = (int64_t)id * (e.dim >> group_shift) + ((4 * q) >> group_shift);
    const float scale = PACKING >= kPackTernary ? half_to_float(((const uint16_t *)e.scales)[g]) : ((const float *)e.scales)[g];
    float v[4];
    four<PACKING>(e.values + id * row_bytes(PACKING, e.dim), q, v);
    *to = make_float4(fmul(fmul(v[0], scale), e.scale), fmul(fmul(v[1], scale), e.scale), fmul(fmul(v[2], scale), e.scale),
                      fmul(fmul(v[3], scale), e.scale));
  }
}

// int8 rows that are no whole dwords (groups of 1 or 2): a thread a weight
__global__ __launch_bounds__(256) void embed_odd_kernel(Embed e, int32_t group_shift) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;  // (a row may end within 256 of 2^31)
  if (i >= (uint32_t)e.dim) return;
  for (int64_t t = blockIdx.y; t < e.count; t += gridDim.y) {
    const int32_t id = e.ids[t];
    float x = 0.0f;
    if ((uint32_t)id < (uint32_t)e.vocab) {
      const float scale = ((const float *)e.scales)[(int64_t)id * (e.dim >> group_shift) + (i >> group_shift)];
      x = fmul(fmul((float)(int8_t)e.values[(int64_t)id * e.dim + i], scale), e.scale);
    }
    ((float *)(e.out + t * e.out_stride))[i] = x;
  }
}

}  // namespace

hipError_t launch_embed(int32_t packing, const Embed &e, int32_t group, hipStream_t s) {
  if (e.count <= 0 || e.dim <= 0) return hipSuccess;
  const int32_t shift = __builtin_ctz(group), lanes = e.dim % 4 ? e.dim : e.dim / 4;
  const dim3 grid((uint32_t)(((int64_t)lanes + 255) / 256), (uint32_t)(e.count < 65535 ? e.count : 65535));
  const auto kernel = e.dim % 4 ? embed_odd_kernel : packing == kPackInt8 ? embed_kernel<kPackInt8>
                    : packing == kPackInt6 ? embed_kernel<kPackInt6> : packing == kPackTernary ? embed_kernel<kPackTernary>
                    : embed_kernel<kPackBinary>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, e, shift);
  return hipGetLastError();
}

}  // namespace hq
