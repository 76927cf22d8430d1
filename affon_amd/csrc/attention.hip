// Attention of drafted tokens over a paged cache.

#include <algorithm>

#include "paged.h"

namespace affon {
namespace {

constexpr int kThreads = 256;

// One workgroup for one head of one row: a key per thread and tile, the
// running maximum and sum of a softmax over the tiles, and a value of the
// output per thread.
template <typename T>
__global__ __launch_bounds__(kThreads) void row_kernel(AttentionProblem p) {
  __shared__ float q[256], score[kThreads], part[kThreads / 64];
  __shared__ int64_t line[kThreads];
  const int D = p.cache.head_dim;
  const int64_t row = blockIdx.x;
  const int head = blockIdx.y, kv = head / (p.heads / p.cache.kv_heads);
  const int b = static_cast<int>(row / p.batch.rows);
  const uint32_t i = static_cast<uint32_t>(row - static_cast<int64_t>(b) * p.batch.rows);
  const uint32_t length = committed(p.batch, b), count = drafted(p.batch, b);
  const uint32_t n = i < count ? length + count : 0;
  const int t = threadIdx.x;
  if (t < D) q[t] = T::load(p.query, row * p.query_stride + static_cast<int64_t>(head) * D + t);
  float m = -INFINITY, l = 0.0f, o = 0.0f;
  for (uint32_t first = 0; first < n; first += kThreads) {
    __syncthreads();
    const uint32_t at = first + t;
    int64_t where = at < n ? line_of(p.cache, p.batch, b, at) : -1;
    if (where >= 0 && at >= length) {
      const uint32_t j = at - length;
      const bool seen = p.mask != nullptr ? p.mask[row * p.mask_stride + j / 32] >> (j % 32) & 1 : j <= i;
      if (!seen) where = -1;
    }
    float s = -INFINITY;
    if (where >= 0) {
      where += static_cast<int64_t>(kv) * p.cache.page_size;
      s = 0.0f;
      for (int d = 0; d < D; ++d) s = fmaf(q[d], T::load(p.cache.keys, where * D + d), s);
      s *= p.scale;
    }
    line[t] = where;
    float top = s;
    for (int offset = 32; offset > 0; offset >>= 1) top = fmaxf(top, __shfl_xor(top, offset));
    if ((t & 63) == 0) part[t >> 6] = top;
    __syncthreads();
    top = m;
    for (int w = 0; w < kThreads / 64; ++w) top = fmaxf(top, part[w]);
    const float base = top == -INFINITY ? 0.0f : top;
    score[t] = where >= 0 ? expf(s - base) : 0.0f;
    const float keep = expf(m - base);
    m = top;
    l *= keep;
    o *= keep;
    __syncthreads();
    for (int k = 0; k < kThreads; ++k) {
      if (line[k] < 0) continue;
      l += score[k];
      if (t < D) o = fmaf(score[k], T::load(p.cache.values, line[k] * D + t), o);
    }
  }
  if (t >= D) return;
  const float out = l == 0.0f ? 0.0f : o / l;
  const int64_t to = (row * p.heads + head) * D + t;
  if constexpr (T::bytes == 2)
    reinterpret_cast<uint16_t*>(p.out)[to] = f32_to_bf16_bits(out);
  else
    reinterpret_cast<float*>(p.out)[to] = out;
}

}  // namespace

hipError_t attention_launch(const AttentionProblem& p, const Launch& l) {
  const dim3 grid(static_cast<unsigned>(p.batch.sequences * p.batch.rows), static_cast<unsigned>(p.heads));
  if (p.cache.dtype == AFFON_ROCM_BF16)
    hipLaunchKernelGGL(row_kernel<BF16>, grid, dim3(kThreads), 0, l.stream, p);
  else
    hipLaunchKernelGGL(row_kernel<F32>, grid, dim3(kThreads), 0, l.stream, p);
  return hipGetLastError();
}

}  // namespace affon
