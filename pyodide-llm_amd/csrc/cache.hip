// cache.hip — the paged key/value cache: new tokens' vectors quantized as they are written, and read back as float32.
//
// Keys lie as they are multiplied with a query, a vector after the other ([page][head][slot][dim]); values lie dimension by
// dimension ([page][head][dim][slot]), so that attention's product over the positions reads consecutive positions of a
// dimension straight into a matrix instruction's registers.  An int8 vector is quantize_x's arithmetic over the whole head
// (scale = largest |x| / 127, the inverse rounded, the product rounded to even); a float16 one is scaled by the power of two
// that brings its largest |x| into [2^14, 2^15), so that it neither overflows nor loses small values to float16's range.
// One float32 scale a (position, head): attention multiplies a score and a weight by it after and before its products, where
// a scale for every 32 values would take an extra product each.
//
// A block takes up to 64 positions (a multiple of 64 on) of a sequence, one head, its keys or its values: the values turn in
// LDS, so that whole 64-byte lines of positions are written and read.
#include "paged.hpp"

namespace hq {

namespace {

constexpr int kChunk = 64;  // positions of a block
constexpr float kSmallest = 7.888609052210118e-31f;  // 2^-100: a smaller scale is stored as 0 and its vector as zeros

HQ_DEV int32_t chunks_of(const Batch &b, int32_t s) {
  const Sequence q = sequence_of(b, s);
  if (!q.count) return 0;
  return ((q.length - 1) >> 6) - ((q.length - q.count) >> 6) + 1;
}

// the largest bits over a row of 16 lanes
HQ_DEV uint32_t max16(uint32_t m) {
  m = max8(m);
  return max(m, (uint32_t)dpp<0x140>((int32_t)m));  // row_mirror
}

// a value's element of a vector whose scale is `scale`, 1 / scale `inv`
template <int F16>
HQ_DEV uint32_t element(float v, float inv) {
  if (F16) {
    const _Float16 h = (_Float16)fmul(v, inv);
    return __builtin_bit_cast(uint16_t, h);
  }
  return (uint32_t)(int32_t)rintf(fmul(v, inv)) & 0xffu;  // at most 127 either way: |x| / scale rounds to 127 at the largest
}

// the scale of a vector whose largest |x| has bits m, and its inverse (0: store zeros)
template <int F16>
HQ_DEV void scale_of(uint32_t m, float &scale, float &inv) {
  if (m >= 0x7f800000u) {  // an infinity or NaN: the whole vector is NaN
    scale = __uint_as_float(0x7fc00000u), inv = 0.0f;
    return;
  }
  // 2^(e - 14), 2^e <= x: the exponent's bits less 14 (x of 2^-126 and more; smaller ones are below kSmallest anyway)
  scale = F16 ? __uint_as_float(max((int32_t)(m & 0x7f800000u) - (14 << 23), 0)) : fdiv(__uint_as_float(m), 127.0f);
  if (scale < kSmallest) scale = 0.0f;
  inv = scale > 0.0f ? fdiv(1.0f, scale) : 0.0f;
}

template <int F16>
__global__ __launch_bounds__(256) void write_kernel(Cache c, Batch b, const char *k, const char *v, int64_t k_stride,
                                                    int64_t v_stride) {
  constexpr int ES = F16 ? 2 : 1, PITCH = kChunk * ES + 4;  // 17 (33) dwords: 16 lanes' dimensions fall into 16 banks
  __shared__ char turned[256 * PITCH];
  const Place place = place_of(b.sequences, blockIdx.x, [&](int32_t s) { return chunks_of(b, s); });
  if (place.s < 0) return;
  const int32_t h = blockIdx.y;
  const bool values = blockIdx.z;
  const Sequence q = wave_sequence_of(b, place.s);
  const int32_t first = q.length - q.count, base = ((first >> 6) + place.rest) * kChunk;
  const int32_t from = max(max(first, base), 0), to = min(q.length, base + kChunk);  // the positions to write
  const int row = threadIdx.x >> 4, l = threadIdx.x & 15;
  for (int p0 = base + ((from - base) & ~15); p0 < to; p0 += 16) {
    const int32_t at = p0 + row;
    const bool live = at >= from && at < to;
    const int32_t page = live ? page_of(b, c, place.s, at) : -1;
    // (a lane without a token reads the sequence's first)
    const int64_t t = q.begin + (live ? at - first : 0);
    const float *x = (const float *)((values ? v + t * v_stride : k + t * k_stride) + 4 * (int64_t)h * c.dim);
    float4 f[4];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int at4 = 64 * i + 4 * l;
      f[i] = at4 < c.dim ? *(const float4 *)(x + at4) : make_float4(0.f, 0.f, 0.f, 0.f);
      m = max(max(m, __float_as_uint(f[i].x) & 0x7fffffffu), __float_as_uint(f[i].y) & 0x7fffffffu);
      m = max(max(m, __float_as_uint(f[i].z) & 0x7fffffffu), __float_as_uint(f[i].w) & 0x7fffffffu);
    }
    float scale, inv;
    scale_of<F16>(max16(m), scale, inv);
    const bool zero = inv == 0.0f;  // (an infinity times 0 is no element)
    const int64_t vec = page >= 0 ? vectors_of(c, page, h) + (at & ((1 << c.shift) - 1)) : 0;
    if (page >= 0 && l == 0) (values ? c.vs : c.ks)[vec] = scale;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int at4 = 64 * i + 4 * l;
      if (at4 >= c.dim) continue;
      const float e[4] = {f[i].x, f[i].y, f[i].z, f[i].w};
      uint32_t u[4];
#pragma unroll
      for (int j = 0; j < 4; j++) u[j] = zero ? 0u : element<F16>(e[j], inv);
      if (values) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          char *to_lds = turned + (at4 + j) * PITCH + (at - base) * ES;
          if (F16) *(uint16_t *)to_lds = (uint16_t)u[j];
          else *(uint8_t *)to_lds = (uint8_t)u[j];
        }
      } else if (page >= 0) {
        char *to_mem = c.k + (vec * c.dim + at4) * ES;
        if (F16) *(uint2 *)to_mem = make_uint2(u[0] | (u[1] << 16), u[2] | (u[3] << 16));
        else *(uint32_t *)to_mem = u[0] | (u[1] << 8) | (u[2] << 16) | (u[3] << 24);
      }
    }
  }
  if (!values) return;
  __syncthreads();
  // 16 bytes of a dimension's positions a thread (16 or 8 of them: all in one page)
  constexpr int PARTS = kChunk * ES / 16, EACH = 16 / ES;
  for (int i = threadIdx.x; i < c.dim * PARTS; i += 256) {
    const int d = i / PARTS, part = i % PARTS, p0 = base + part * EACH;
    if (p0 + EACH <= from || p0 >= to) continue;
    const int32_t page = page_of(b, c, place.s, p0);
    if (page < 0) continue;
    char *to_mem = c.v + (((vectors_of(c, page, h) * c.dim) + ((int64_t)d << c.shift)) + (p0 & ((1 << c.shift) - 1))) * ES;
    const char *lds = turned + d * PITCH + part * 16;
    if (p0 >= from && p0 + EACH <= to) {
      const uint32_t *w = (const uint32_t *)lds;
      *(uint4 *)to_mem = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      for (int j = 0; j < EACH; j++) {
        if (p0 + j < from || p0 + j >= to) continue;
        if (F16) *(uint16_t *)(to_mem + 2 * j) = *(const uint16_t *)(lds + 2 * j);
        else *(uint8_t *)(to_mem + j) = *(const uint8_t *)(lds + j);
      }
    }
  }
}

template <int F16>
HQ_DEV float value_of(uint32_t u, float scale) {
  if (F16) return fmul((float)__builtin_bit_cast(_Float16, (uint16_t)u), scale);
  return fmul((float)(int32_t)(int8_t)(uint8_t)u, scale);
}

template <int F16>
__global__ __launch_bounds__(256) void read_kernel(Cache c, Batch b, char *k, char *v, int64_t k_stride, int64_t v_stride) {
  constexpr int ES = F16 ? 2 : 1, PITCH = kChunk * ES + 4;
  __shared__ char turned[256 * PITCH];
  const Place place = place_of(b.sequences, blockIdx.x, [&](int32_t s) { return chunks_of(b, s); });
  if (place.s < 0) return;
  const int32_t h = blockIdx.y;
  const bool values = blockIdx.z;
  const Sequence q = wave_sequence_of(b, place.s);
  const int32_t first = q.length - q.count, base = ((first >> 6) + place.rest) * kChunk;
  const int32_t from = max(first, base), to = min(q.length, base + kChunk);
  constexpr int PARTS = kChunk * ES / 16, EACH = 16 / ES;
  if (values) {
    for (int i = threadIdx.x; i < c.dim * PARTS; i += 256) {
      const int d = i / PARTS, part = i % PARTS, p0 = base + part * EACH;
      if (p0 + EACH <= from || p0 >= to) continue;
      const int32_t page = page_of(b, c, place.s, p0);
      if (page < 0) continue;
      const uint4 w = *(const uint4 *)(c.v + (((vectors_of(c, page, h) * c.dim) + ((int64_t)d << c.shift)) +
                                              (p0 & ((1 << c.shift) - 1))) * ES);
      uint32_t *lds = (uint32_t *)(turned + d * PITCH + part * 16);
      lds[0] = w.x, lds[1] = w.y, lds[2] = w.z, lds[3] = w.w;
    }
    __syncthreads();
  }
  const int row = threadIdx.x >> 4, l = threadIdx.x & 15;
  for (int p0 = base + ((from - base) & ~15); p0 < to; p0 += 16) {
    const int32_t at = p0 + row;
    if (at < from || at >= to) continue;
    const int32_t page = page_of(b, c, place.s, at);
    const int64_t t = q.begin + (at - first);
    float *x = (float *)((values ? v + t * v_stride : k + t * k_stride) + 4 * (int64_t)h * c.dim);
    const int64_t vec = page >= 0 ? vectors_of(c, page, h) + (at & ((1 << c.shift) - 1)) : 0;
    const float scale = page >= 0 ? (values ? c.vs : c.ks)[vec] : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int at4 = 64 * i + 4 * l;
      if (at4 >= c.dim) continue;
      uint32_t u[4] = {0, 0, 0, 0};
      if (page >= 0 && values) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const char *lds = turned + (at4 + j) * PITCH + (at - base) * ES;
          u[j] = F16 ? *(const uint16_t *)lds : *(const uint8_t *)lds;
        }
      } else if (page >= 0) {
        const char *mem = c.k + (vec * c.dim + at4) * ES;
        if (F16) {
          const uint2 w = *(const uint2 *)mem;
          u[0] = w.x & 0xffffu, u[1] = w.x >> 16, u[2] = w.y & 0xffffu, u[3] = w.y >> 16;
        } else {
          const uint32_t w = *(const uint32_t *)mem;
          u[0] = w & 0xffu, u[1] = (w >> 8) & 0xffu, u[2] = (w >> 16) & 0xffu, u[3] = w >> 24;
        }
      }
      *(float4 *)(x + at4) = make_float4(value_of<F16>(u[0], scale), value_of<F16>(u[1], scale),
                                         value_of<F16>(u[2], scale), value_of<F16>(u[3], scale));
    }
  }
}

// every chunk holds a new token, and a sequence's tokens touch two chunks more than they fill at most
dim3 grid_of(const Cache &c, const Batch &b) {
  const int64_t chunks = (int64_t)b.tokens / kChunk + 2 * (int64_t)b.sequences;
  return dim3((uint32_t)(chunks < b.tokens ? chunks : b.tokens), (uint32_t)c.heads, 2);
}

}  // namespace

hipError_t launch_cache_write(const Cache &c, const Batch &b, const char *k, const char *v, int64_t k_stride,
                              int64_t v_stride, hipStream_t s) {
  if (b.tokens <= 0 || b.sequences <= 0) return hipSuccess;
  const auto kernel = c.f16 ? write_kernel<1> : write_kernel<0>;
  hipLaunchKernelGGL(kernel, grid_of(c, b), dim3(256), 0, s, c, b, k, v, k_stride, v_stride);
  return hipGetLastError();
}

hipError_t launch_cache_read(const Cache &c, const Batch &b, char *k, char *v, int64_t k_stride, int64_t v_stride,
                             hipStream_t s) {
  if (b.tokens <= 0 || b.sequences <= 0) return hipSuccess;
  const auto kernel = c.f16 ? read_kernel<1> : read_kernel<0>;
  hipLaunchKernelGGL(kernel, grid_of(c, b), dim3(256), 0, s, c, b, k, v, k_stride, v_stride);
  return hipGetLastError();
}

}  // namespace hq
