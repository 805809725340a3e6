// attention.hip — attention of new tokens over the paged cache.
//
//   out = sum_j softmax_j(s_j) v_j,  s_j = scale q.k_j  (cap > 0: cap tanh(s_j / cap)), over the positions j that the token
//   sees: not past its own, within its window, on a page; zeros where there is none
//
// A wave a (token, query head): 64 positions at a time, a lane a score, then a lane a few dimensions of the values.
#include "paged.hpp"

namespace hq {

namespace {

template <int F16>
HQ_DEV float stored(const char *p) {
  if (F16) return (float)*(const _Float16 *)p;
  return (float)*(const int8_t *)p;
}

template <int F16>
__global__ __launch_bounds__(64) void attention_kernel(Attention a, Cache c, Batch b) {
  constexpr int ES = F16 ? 2 : 1;
  __shared__ float qs[256], ws[64];
  const int lane = threadIdx.x;
  const int32_t t = blockIdx.x, head = blockIdx.y, h = head / (a.heads / c.heads);
  int32_t s = -1;
  for (int32_t s0 = 0; s0 < b.sequences && s < 0; s0 += 64) {
    bool mine = false;
    if (s0 + lane < b.sequences) {
      const Sequence q = sequence_of(b, s0 + lane);
      mine = t >= q.begin && t - q.begin < q.count;
    }
    const uint64_t in = __ballot(mine);
    if (in) s = s0 + __ffsll((unsigned long long)in) - 1;
  }
  if (s < 0) return;
  const Sequence q = sequence_of(b, s);
  const int64_t reach = (int64_t)b.width << c.shift;
  const int32_t sees = q.length - q.count + (t - q.begin) + 1;  // the positions before this one, and its own
  const int32_t to = (int32_t)min((int64_t)sees, reach), from = a.window ? max(sees - a.window, 0) : 0;
  const float *x = (const float *)(a.q + t * (int64_t)a.q_stride) + (int64_t)head * c.dim;
  for (int d = lane; d < c.dim; d += 64) qs[d] = x[d];
  __syncthreads();
  float m = -INFINITY, l = 0.0f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int32_t base = from & ~63; base < to; base += 64) {
    const int32_t j = base + lane;
    const int32_t page = j >= from && j < to ? page_of(b, c, s, j) : -1;
    const int64_t vec = page >= 0 ? vectors_of(c, page, h) + (j & ((1 << c.shift) - 1)) : 0;
    float score = -INFINITY;
    if (page >= 0) {
      float dot = 0.0f;
      for (int d = 0; d < c.dim; d++) dot = fmaf(qs[d], stored<F16>(c.k + (vec * c.dim + d) * ES), dot);
      score = dot * c.ks[vec] * a.scale;
      if (a.cap > 0.0f) score = a.cap * tanhf(score / a.cap);
    }
    float most = score;
    for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
    const float m1 = fmaxf(m, most), ref = m1 == -INFINITY ? 0.0f : m1;
    const float alpha = expf(m - ref), p = page >= 0 ? expf(score - ref) : 0.0f;
    m = m1;
    l = l * alpha + p;
    ws[lane] = page >= 0 ? p * c.vs[vec] : 0.0f;
    __syncthreads();
    for (int i = 0; i < 4; i++) acc[i] *= alpha;
    for (int e = 0; e < 64; e++) {
      const int32_t pe = __shfl(page, e, 64);
      if (pe < 0) continue;
      const int64_t at = ((vectors_of(c, pe, h) * c.dim)) + ((base + e) & ((1 << c.shift) - 1));
      for (int i = 0; i < 4; i++) {
        const int d = lane + 64 * i;
        if (d < c.dim) acc[i] = fmaf(ws[e], stored<F16>(c.v + (at + ((int64_t)d << c.shift)) * ES), acc[i]);
      }
    }
    __syncthreads();
  }
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
  float *out = (float *)(a.out + t * (int64_t)a.out_stride) + (int64_t)head * c.dim;
  for (int i = 0; i < 4; i++)
    if (lane + 64 * i < c.dim) out[lane + 64 * i] = l != 0.0f ? acc[i] / l : 0.0f;  // (NaN stays)
}

}  // namespace

int64_t attention_work_bytes(const Cache &, const Batch &, int32_t) { return 0; }

hipError_t launch_attention(const Attention &a, const Cache &c, const Batch &b, hipStream_t s) {
  if (b.tokens <= 0 || b.sequences <= 0) return hipSuccess;
  const auto kernel = c.f16 ? attention_kernel<1> : attention_kernel<0>;
  hipLaunchKernelGGL(kernel, dim3((uint32_t)b.tokens, (uint32_t)a.heads), dim3(64), 0, s, a, c, b);
  return hipGetLastError();
}

}  // namespace hq
