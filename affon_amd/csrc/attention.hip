// Attention of drafted tokens over a paged cache: the choice of kernel and
// of the pieces that a long context is cut into, and the join of their
// results (attention.h holds the kernels).

#include <algorithm>
#include <cmath>

#include "attention.h"

namespace affon {
namespace attention {
namespace {

// out = sum_s 2^(m_s - m) sums_s / sum_s 2^(m_s - m) l_s over the splits that
// hold keys of the row's sequence; four values per thread.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(Args a) {
  const AttentionProblem& p = a.p;
  const int D = p.cache.head_dim, pieces = D / 4;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t slot = item / pieces;  // of [row][head]
  const int d = static_cast<int>(item - slot * pieces) * 4;
  const int64_t row = slot / p.heads;
  if (row >= static_cast<int64_t>(p.batch.sequences) * p.batch.rows) return;
  const int head = static_cast<int>(slot - row * p.heads), kv = head / a.group;
  const int b = static_cast<int>(row / p.batch.rows), t = static_cast<int>(row - static_cast<int64_t>(b) * p.batch.rows);
  const uint32_t count = drafted(p.batch, b);
  const uint32_t n = min(committed(p.batch, b) + count, p.batch.capacity);
  f32x4_t v{0, 0, 0, 0};
  if (t < static_cast<int>(count)) {
    const int used = min(static_cast<uint32_t>(a.splits), (n + a.chunk - 1) / a.chunk);
    const int64_t first = (static_cast<int64_t>(b) * p.cache.kv_heads + kv) * a.splits * a.row_slots + t * a.group +
                          head - kv * a.group;
    float top = kLowest, sum = 0.0f;
    for (int s = 0; s < used; ++s) top = fmaxf(top, a.stats[first + static_cast<int64_t>(s) * a.row_slots].x);
    for (int s = 0; s < used; ++s) {
      const int64_t at = first + static_cast<int64_t>(s) * a.row_slots;
      const float2 st = a.stats[at];
      const float keep = __builtin_amdgcn_exp2f(st.x - top);
      sum = fmaf(st.y, keep, sum);
      v += *reinterpret_cast<const f32x4_t*>(a.sums + at * D + d) * keep;
    }
    v = sum == 0.0f ? f32x4_t{0, 0, 0, 0} : v * (1.0f / sum);
  }
  const int64_t to = slot * D + d;
  if constexpr (T::bytes == 2) {
    auto* out = reinterpret_cast<uint16_t*>(p.out) + to;
    const u32x2_t h{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
    if (reinterpret_cast<uintptr_t>(p.out) % 8 == 0) {
      *reinterpret_cast<u32x2_t*>(out) = h;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = static_cast<uint16_t>(h[e / 2] >> (16 * (e % 2)));
    }
  } else {
    auto* out = reinterpret_cast<float*>(p.out) + to;
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = v[e];
  }
}

// Few rows: waves side by side over the keys; more: over the rows.
Shape shape_for(int rows) {
  if (rows <= 16) return {1, 1};
  if (rows <= 32) return {2, 1};
  if (rows <= 64) return {1, 4};
  return {2, 4};
}

}  // namespace
}  // namespace attention

hipError_t attention_launch(const AttentionProblem& p, const Launch& l) {
  using namespace attention;
  Args a{};
  a.p = p;
  a.group = p.heads / p.cache.kv_heads;
  const int64_t rows = static_cast<int64_t>(p.batch.rows) * a.group;
  if (rows > (int64_t(1) << 30)) return hipErrorInvalidValue;
  a.rows = static_cast<int>(rows);
  const Shape shape = shape_for(a.rows);
  a.row_groups = (a.rows + shape.rows() - 1) / shape.rows();
  a.row_slots = a.rows;
  a.log2_scale = p.scale == 0.0f ? 1.0f : std::fabs(p.scale) * 1.44269504088896340736f;
  a.sign = p.scale > 0.0f ? 1.0f : p.scale < 0.0f ? -1.0f : 0.0f;

  // Pieces of the context: enough workgroups for the GPU, none so short that
  // its results weigh against the keys it reads.
  const int64_t units = static_cast<int64_t>(p.batch.sequences) * p.cache.kv_heads;
  constexpr int64_t kWanted = 1024;
  const int64_t capacity = p.batch.capacity;
  int64_t splits = std::max<int64_t>(1, kWanted / (units * a.row_groups));
  const int64_t least = std::max<int64_t>(128, 8 * std::min(a.rows, shape.rows()));
  splits = std::min(splits, (capacity + least - 1) / least);
  a.chunk = static_cast<uint32_t>((capacity + splits - 1) / splits + 127) / 128 * 128;
  a.splits = static_cast<int>((capacity + a.chunk - 1) / a.chunk);
  if (a.splits > 1) {
    const size_t slots = static_cast<size_t>(units) * a.splits * a.row_slots;
    const size_t sums = (slots * p.cache.head_dim * sizeof(float) + 255) / 256 * 256;
    auto* scratch = static_cast<uint8_t*>(l.scratch(sums + slots * sizeof(float2)));
    if (scratch != nullptr) {
      a.sums = reinterpret_cast<float*>(scratch);
      a.stats = reinterpret_cast<float2*>(scratch + sums);
    } else {  // a captured stream whose workspace cannot grow
      a.splits = 1;
    }
  }
  const int64_t groups = units * a.splits;
  const int64_t blocks = (groups + 7) / 8 * 8 * a.row_groups;
  if (blocks > (int64_t(1) << 31) - 1) return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks));
  const bool half = p.cache.dtype == AFFON_ROCM_BF16;
  (half ? launch_bf16 : launch_f32)(a, shape, grid, l.stream);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  const int64_t items = static_cast<int64_t>(p.batch.sequences) * p.batch.rows * p.heads * (p.cache.head_dim / 4);
  const int64_t join_blocks = (items + 255) / 256;
  if (join_blocks > (int64_t(1) << 31) - 1) return hipErrorInvalidValue;
  if (half)
    hipLaunchKernelGGL(join_kernel<BF16>, dim3(static_cast<unsigned>(join_blocks)), dim3(256), 0, l.stream, a);
  else
    hipLaunchKernelGGL(join_kernel<F32>, dim3(static_cast<unsigned>(join_blocks)), dim3(256), 0, l.stream, a);
  return hipGetLastError();
}

}  // namespace affon
