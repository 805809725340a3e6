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
//
// Bound by memory where there is much of it, else by a launch and its chain of loads (the sequence's numbers, its page, the values).
// 8192 positions of 8 heads of 128 int8 values read in 16.5 us (84 MB: 5.1 TB/s, a copy reaches 5.2); 5 prompts of up to 2048
// tokens, 8 heads of 64 float16 values, written in 9.0 us and read in 8.3 (26 MB each: 2.9 and 3.1 TB/s); a token each of 32
// sequences written in 5.0 us and read in 4.2; 777 positions of 4 heads of 64 read in 5.0.
#include "paged.hpp"

namespace hq {

namespace {

constexpr int kChunk = 64;  // positions of a block
constexpr float kSmallest = 7.888609052210118e-31f;  // 2^-100: a smaller scale is stored as 0 and its vector as zeros

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

// the positions of the block's chunk: [from, to), from base on, the first new one `first`; none: to <= from
struct Chunk {
  Place place;
  int32_t first, base, from, to;
};
HQ_DEV Chunk chunk_of(const Batch &b, int32_t at) {
  Chunk o;
  o.place = place_of(b, at);
  o.first = o.place.q.length - o.place.q.count;
  o.base = ((o.first >> 6) + o.place.rest) * kChunk;
  o.from = max(o.first, o.base), o.to = o.place.s < 0 ? o.from : min(o.place.q.length, o.base + kChunk);
  return o;
}

// DIM: the head's values in 64s.  All of the block's loads are on their way before the first is used.
template <int F16, int DIM>
__global__ __launch_bounds__(256) void write_kernel(Cache c, Batch b, const char *k, const char *v, int64_t k_stride,
                                                    int64_t v_stride) {
  constexpr int ES = F16 ? 2 : 1, PITCH = kChunk * ES + 4;  // 17 (33) dwords: 16 lanes' dimensions fall into 16 banks
  constexpr int PARTS = kChunk * ES / 16, EACH = 16 / ES;   // 16 bytes of a dimension's positions
  __shared__ char turned[64 * DIM * PITCH];
  const Chunk o = chunk_of(b, blockIdx.x);
  if (o.to <= o.from || o.to <= 0) return;  // (no such chunk, or before position 0)
  const int32_t h = blockIdx.y, from = max(o.from, 0), to = o.to;
  const bool values = blockIdx.z;
  const int row = threadIdx.x >> 4, l = threadIdx.x & 15;
  float4 f[4][DIM];
  int32_t page[4];
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const int32_t at = o.base + 16 * r + row;
    const bool live = at >= from && at < to;
    page[r] = live ? page_of(b, c, o.place.s, at) : -1;
    const int64_t t = o.place.q.begin + (at - o.first);
    const float *x = (const float *)((values ? v + t * v_stride : k + t * k_stride) + 4 * (int64_t)h * c.dim);
#pragma unroll
    for (int i = 0; i < DIM; i++) {
      const int at4 = 64 * i + 4 * l;
      f[r][i] = live && at4 < c.dim ? *(const float4 *)(x + at4) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  // (the pages of the values' 16 bytes: the thread's part is the same for all its dimensions)
  const int part = threadIdx.x % PARTS, p0 = o.base + part * EACH;
  const int32_t part_page = values && p0 + EACH > from && p0 < to ? page_of(b, c, o.place.s, p0) : -1;
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const int32_t at = o.base + 16 * r + row;
    if (!__any(page[r] >= 0)) continue;
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < DIM; i++) {
      m = max(max(m, __float_as_uint(f[r][i].x) & 0x7fffffffu), __float_as_uint(f[r][i].y) & 0x7fffffffu);
      m = max(max(m, __float_as_uint(f[r][i].z) & 0x7fffffffu), __float_as_uint(f[r][i].w) & 0x7fffffffu);
    }
    float scale, inv;
    scale_of<F16>(max16(m), scale, inv);
    const bool zero = inv == 0.0f;  // (an infinity times 0 is no element)
    const int64_t vec = page[r] >= 0 ? vectors_of(c, page[r], h) + (at & ((1 << c.shift) - 1)) : 0;
    if (page[r] >= 0 && l == 0) (values ? c.vs : c.ks)[vec] = scale;
#pragma unroll
    for (int i = 0; i < DIM; i++) {
      const int at4 = 64 * i + 4 * l;
      if (at4 >= c.dim) continue;
      const float e[4] = {f[r][i].x, f[r][i].y, f[r][i].z, f[r][i].w};
      uint32_t u[4];
#pragma unroll
      for (int j = 0; j < 4; j++) u[j] = zero ? 0u : element<F16>(e[j], inv);
      if (values) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          char *to_lds = turned + (at4 + j) * PITCH + (16 * r + row) * ES;
          if (F16) *(uint16_t *)to_lds = (uint16_t)u[j];
          else *(uint8_t *)to_lds = (uint8_t)u[j];
        }
      } else if (page[r] >= 0) {
        char *to_mem = c.k + (vec * c.dim + at4) * ES;
        if (F16) *(uint2 *)to_mem = make_uint2(u[0] | (u[1] << 16), u[2] | (u[3] << 16));
        else *(uint32_t *)to_mem = u[0] | (u[1] << 8) | (u[2] << 16) | (u[3] << 24);
      }
    }
  }
  if (!values) return;
  __syncthreads();
  if (part_page < 0) return;
  char *to_part = c.v + (vectors_of(c, part_page, h) * c.dim + (p0 & ((1 << c.shift) - 1))) * ES;
  for (int d = threadIdx.x / PARTS; d < c.dim; d += 256 / PARTS) {
    char *to_mem = to_part + ((int64_t)d << c.shift) * ES;
    const char *lds = turned + d * PITCH + part * 16;
    if (p0 >= from && p0 + EACH <= to) {
      const uint32_t *w = (const uint32_t *)lds;
      *(uint4 *)to_mem = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      for (int j = max(from - p0, 0); j < min(to - p0, EACH); j++) {
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

template <int F16, int DIM>
__global__ __launch_bounds__(256) void read_kernel(Cache c, Batch b, char *k, char *v, int64_t k_stride, int64_t v_stride) {
  constexpr int ES = F16 ? 2 : 1, PITCH = kChunk * ES + 4, PARTS = kChunk * ES / 16, EACH = 16 / ES;
  constexpr int ROWS = 64 * DIM * PARTS / 256;  // dimensions whose 16 bytes a thread turns
  __shared__ char turned[64 * DIM * PITCH];
  const Chunk o = chunk_of(b, blockIdx.x);
  if (o.to <= o.from) return;
  const int32_t h = blockIdx.y;
  const bool values = blockIdx.z;
  const int row = threadIdx.x >> 4, l = threadIdx.x & 15;
  int32_t page[4];
  float scale[4];
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const int32_t at = o.base + 16 * r + row;
    page[r] = at >= o.from && at < o.to ? page_of(b, c, o.place.s, at) : -1;
  }
  uint2 w[4][DIM];  // the lane's 4 elements
  if (values) {
    const int part = threadIdx.x % PARTS, p0 = o.base + part * EACH, d0 = threadIdx.x / PARTS;
    const int32_t part_page = p0 + EACH > o.from && p0 < o.to ? page_of(b, c, o.place.s, p0) : -1;
    const char *from_part = c.v + (vectors_of(c, max(part_page, 0), h) * c.dim + (p0 & ((1 << c.shift) - 1))) * ES;
    uint4 q[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const int d = d0 + i * (256 / PARTS);
      q[i] = part_page >= 0 && d < c.dim ? *(const uint4 *)(from_part + ((int64_t)d << c.shift) * ES) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      uint32_t *lds = (uint32_t *)(turned + (d0 + i * (256 / PARTS)) * PITCH + part * 16);
      lds[0] = q[i].x, lds[1] = q[i].y, lds[2] = q[i].z, lds[3] = q[i].w;
    }
  }
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const int64_t vec = vectors_of(c, max(page[r], 0), h) + ((o.base + 16 * r + row) & ((1 << c.shift) - 1));
    scale[r] = page[r] >= 0 ? (values ? c.vs : c.ks)[vec] : 0.0f;
    if (values) continue;
#pragma unroll
    for (int i = 0; i < DIM; i++) {
      const int at4 = 64 * i + 4 * l;
      w[r][i] = make_uint2(0, 0);
      if (page[r] >= 0 && at4 < c.dim) {
        const char *mem = c.k + (vec * c.dim + at4) * ES;
        if (F16) w[r][i] = *(const uint2 *)mem;
        else w[r][i].x = *(const uint32_t *)mem;
      }
    }
  }
  if (values) __syncthreads();
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const int32_t at = o.base + 16 * r + row;
    if (at < o.from || at >= o.to) continue;
    const int64_t t = o.place.q.begin + (at - o.first);
    float *x = (float *)((values ? v + t * v_stride : k + t * k_stride) + 4 * (int64_t)h * c.dim);
#pragma unroll
    for (int i = 0; i < DIM; i++) {
      const int at4 = 64 * i + 4 * l;
      if (at4 >= c.dim) continue;
      uint32_t u[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const char *lds = turned + (at4 + j) * PITCH + (16 * r + row) * ES;
        if (values) u[j] = page[r] < 0 ? 0 : F16 ? *(const uint16_t *)lds : *(const uint8_t *)lds;
        else u[j] = F16 ? (j < 2 ? w[r][i].x : w[r][i].y) >> (16 * (j & 1)) : w[r][i].x >> (8 * j);
      }
      *(float4 *)(x + at4) = make_float4(value_of<F16>(u[0], scale[r]), value_of<F16>(u[1], scale[r]),
                                         value_of<F16>(u[2], scale[r]), value_of<F16>(u[3], scale[r]));
    }
  }
}

// as many items as place_of gives the sequences
dim3 grid_of(const Cache &c, const Batch &b) {
  return dim3((uint32_t)(b.tokens / kChunk + 2 * b.sequences), (uint32_t)c.heads, 2);
}

template <typename Kernel, typename... Args>
hipError_t run(const Cache &c, const Batch &b, hipStream_t s, Kernel kernel, Args... args) {
  hipLaunchKernelGGL(kernel, grid_of(c, b), dim3(256), 0, s, c, b, args...);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_cache_write(const Cache &c, const Batch &b, const char *k, const char *v, int64_t k_stride,
                              int64_t v_stride, hipStream_t s) {
  if (b.tokens <= 0 || b.sequences <= 0) return hipSuccess;
  if (c.dim <= 64) return run(c, b, s, c.f16 ? write_kernel<1, 1> : write_kernel<0, 1>, k, v, k_stride, v_stride);
  if (c.dim <= 128) return run(c, b, s, c.f16 ? write_kernel<1, 2> : write_kernel<0, 2>, k, v, k_stride, v_stride);
  return run(c, b, s, c.f16 ? write_kernel<1, 4> : write_kernel<0, 4>, k, v, k_stride, v_stride);
}

hipError_t launch_cache_read(const Cache &c, const Batch &b, char *k, char *v, int64_t k_stride, int64_t v_stride,
                             hipStream_t s) {
  if (b.tokens <= 0 || b.sequences <= 0) return hipSuccess;
  if (c.dim <= 64) return run(c, b, s, c.f16 ? read_kernel<1, 1> : read_kernel<0, 1>, k, v, k_stride, v_stride);
  if (c.dim <= 128) return run(c, b, s, c.f16 ? read_kernel<1, 2> : read_kernel<0, 2>, k, v, k_stride, v_stride);
  return run(c, b, s, c.f16 ? read_kernel<1, 4> : read_kernel<0, 4>, k, v, k_stride, v_stride);
}

}  // namespace hq
