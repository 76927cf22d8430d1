// Attention of sequences that share prefixes: each group's prefix once for
// all its rows, what follows it for each sequence, and the join of both.

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "attention.h"

namespace affon {
namespace attention {
namespace {

// Partial results of one part, as its kernels leave them.
struct Joined {
  Args prefix, own;
};

// head_dim / 4 threads for every row and head, which take the pieces of the
// prefix and then the own ones in their order; several rows and heads to a workgroup.
template <typename T>
__global__ __launch_bounds__(256) void join_parts_kernel(Joined j) {
  const AttentionProblem& p = j.own.p;
  const int D = p.cache.head_dim, pieces = D / 4, per = 256 / pieces;
  const int local = threadIdx.x / pieces, d = 4 * static_cast<int>(threadIdx.x - local * pieces);
  const int64_t slot = static_cast<int64_t>(blockIdx.x) * per + local;  // of [row][head]
  const int64_t row = slot / p.heads;
  if (local >= per || row >= static_cast<int64_t>(p.batch.sequences) * p.batch.rows) return;
  const int head = static_cast<int>(slot - row * p.heads), kv = head / j.own.group, g = head - kv * j.own.group;
  const int b = static_cast<int>(row / p.batch.rows);
  const int t = static_cast<int>(row - static_cast<int64_t>(b) * p.batch.rows);
  const int group = b / j.own.per;
  const uint32_t count = drafted(p.batch, b);
  const uint32_t n = min(committed(p.batch, b) + count, p.batch.capacity);
  const uint32_t prefix = prefix_tokens(j.own, p.batch, group);
  const bool takes = prefix > 0 && takes_prefix(j.own, p.batch, b, group);

  float top = kLowest, sum = 0.0f;
  f32x4_t v{0, 0, 0, 0};
  if (takes) {
    const uint32_t chunk = piece_of(prefix, j.prefix.splits, j.prefix.chunk);
    const int64_t r = static_cast<int64_t>(row - static_cast<int64_t>(group) * j.own.per * p.batch.rows) * j.own.group + g;
    const int64_t first = (static_cast<int64_t>(group) * p.cache.kv_heads + kv) * j.prefix.splits * j.prefix.row_slots + r;
    v = joined_sums<false>(j.prefix, first, d, D, 0, (prefix + chunk - 1) / chunk, 1, &top, &sum);
  }
  const uint32_t own = n - min(n, takes ? prefix : 0u);
  const uint32_t used = max(1u, (own + j.own.chunk - 1) / j.own.chunk);
  const int64_t first = (static_cast<int64_t>(b) * p.cache.kv_heads + kv) * j.own.splits * j.own.row_slots +
                        static_cast<int64_t>(t) * j.own.group + g;
  float own_top, own_sum;
  const f32x4_t w = joined_sums<false>(j.own, first, d, D, 0, used, 1, &own_top, &own_sum);
  const float peak = fmaxf(top, own_top);
  const float keep = __builtin_amdgcn_exp2f(top - peak), own_keep = __builtin_amdgcn_exp2f(own_top - peak);
  sum = fmaf(sum, keep, own_sum * own_keep);
  v = v * keep + w * own_keep;
  store_result<T>(p.out, slot * D + d, v, t < static_cast<int>(count) ? sum : 0.0f);
}

// Workgroups of a launch over `units` x row groups x splits.
int64_t blocks_of(const Args& a, int64_t units) { return (units * a.splits + 7) / 8 * 8 * a.row_groups; }

}  // namespace
}  // namespace attention

hipError_t shared_attention_launch(const AttentionProblem& p, const uint32_t* shared, int groups, const Launch& l) {
  using namespace attention;
  const bool half = p.cache.dtype == AFFON_ROCM_BF16;
  const int64_t capacity = p.batch.capacity, unit = half ? 128 : 64;
  constexpr int64_t kRound = 512;  // workgroups, two to a CU
  Joined j{};
  j.own.p = j.prefix.p = p;
  j.own.shared = j.prefix.shared = shared;
  j.own.per = j.prefix.per = p.batch.sequences / groups;
  j.prefix.p.batch.sequences = groups;
  j.prefix.p.mask = nullptr;
  const int64_t prefix_rows = static_cast<int64_t>(p.batch.rows) * j.own.per;
  if (prefix_rows * (p.heads / p.cache.kv_heads) > (int64_t(1) << 30)) return hipErrorInvalidValue;
  j.prefix.p.batch.rows = static_cast<int>(prefix_rows);
  Shape shapes[2];
  int tiles = 0;  // waves of the kernel for prefixes of many rows, or 0: the other one
  size_t bytes = 0, sums[2], stats[2];
  for (int part = 0; part < 2; ++part) {
    Args& a = part == 0 ? j.prefix : j.own;
    a.group = p.heads / p.cache.kv_heads;
    a.rows = a.p.batch.rows * a.group;
    a.row_slots = a.rows;
    shapes[part] = shape_for(a.rows, p.cache.head_dim);
    int64_t round = kRound;
    if (part == 0 && half && (p.cache.head_dim == 64 || p.cache.head_dim == 128) && a.rows > 64) {
      tiles = a.rows > 128 ? 8 : 4;
      if (tiles == 8) round /= 2;
    }
    const int group_rows = part == 0 && tiles > 0 ? 32 * tiles : shapes[part].rows();
    a.row_groups = (a.rows + group_rows - 1) / group_rows;
    a.log2_scale = p.scale == 0.0f ? 1.0f : std::min(std::fabs(p.scale) * 1.44269504088896340736f, FLT_MAX);
    a.sign = p.scale > 0.0f ? 1.0f : p.scale < 0.0f ? -1.0f : 0.0f;
    const int64_t units = static_cast<int64_t>(a.p.batch.sequences) * p.cache.kv_heads;
    int64_t splits = std::min(round / (units * a.row_groups), capacity / unit);
    splits = std::max<int64_t>(splits, 1);
    // The prefix is cut on the device, in pieces of `chunk` at least.
    a.chunk = part == 0 ? static_cast<uint32_t>(unit)
                        : static_cast<uint32_t>((capacity + splits - 1) / splits + unit - 1) / unit * unit;
    a.splits = part == 0 ? static_cast<int>(splits) : static_cast<int>((capacity + a.chunk - 1) / a.chunk);
    const size_t slots = static_cast<size_t>(units) * a.splits * a.row_slots;
    sums[part] = bytes;
    bytes += (slots * p.cache.head_dim * sizeof(float) + 255) / 256 * 256;
    stats[part] = bytes;
    bytes += (slots * sizeof(float2) + 255) / 256 * 256;
    if (blocks_of(a, units) > kMaxBlocks) return hipErrorInvalidValue;
  }
  auto* scratch = static_cast<uint8_t*>(l.scratch(bytes));
  // A captured stream whose workspace cannot grow: every sequence by itself.
  if (scratch == nullptr) return attention_launch(p, l);
  for (int part = 0; part < 2; ++part) {
    Args& a = part == 0 ? j.prefix : j.own;
    a.sums = reinterpret_cast<float*>(scratch + sums[part]);
    a.stats = reinterpret_cast<float*>(scratch + stats[part]);
    const dim3 grid(static_cast<unsigned>(blocks_of(a, static_cast<int64_t>(a.p.batch.sequences) * p.cache.kv_heads)));
    if (part == 0 && tiles > 0)
      launch_prefix_tiles(a, tiles, grid, l.stream);
    else if (part == 0)
      (half ? launch_prefix_bf16 : launch_prefix_f32)(a, shapes[part], grid, l.stream);
    else
      (half ? launch_own_bf16 : launch_own_f32)(a, shapes[part], grid, l.stream);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const int64_t per = 256 / (p.cache.head_dim / 4);
  const int64_t blocks = (static_cast<int64_t>(p.batch.sequences) * p.batch.rows * p.heads + per - 1) / per;
  if (blocks > kMaxBlocks) return hipErrorInvalidValue;
  if (half)
    hipLaunchKernelGGL(join_parts_kernel<BF16>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, l.stream, j);
  else
    hipLaunchKernelGGL(join_parts_kernel<F32>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, l.stream, j);
  return hipGetLastError();
}

}  // namespace affon
