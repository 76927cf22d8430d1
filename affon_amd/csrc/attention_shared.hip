// Attention of sequences that share prefixes: each group's prefix once for
// all its rows, what follows it for each sequence, and the join of both.

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "attention.h"
#include "join_thread.h"
#include "prefix_cut.h"

namespace affon {
namespace attention {
namespace {

// Joins the pieces of the prefix and the own ones, in their order: head_dim / 4
// threads for each of `shares` shares of the pieces of a row and head, which then
// meet in LDS; several rows and heads to a workgroup. Bound by the results it reads: 64
// sequences of 64 heads of 128 in 17 pieces, 36 MB, 11 us.
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void join_parts_kernel(Parts parts, int shares) {
  __shared__ __attribute__((aligned(16))) f32x4_t part[kJoinThreads];
  __shared__ float2 stats[kJoinThreads];
  const AttentionProblem& p = parts.p;
  const int D = p.cache.head_dim, pieces = D / 4;
  const JoinThread thread(threadIdx.x, pieces, shares);
  const int share = thread.share, d = 4 * thread.piece;
  const int64_t slot = static_cast<int64_t>(blockIdx.x) * thread.per + thread.local;  // of [row][head]
  const int64_t row = slot / p.heads;
  const bool there = thread.holds() && row < static_cast<int64_t>(p.batch.sequences) * p.batch.rows;
  const int head = static_cast<int>(slot - row * p.heads), kv = head / parts.group, g = head - kv * parts.group;
  const int b = there ? static_cast<int>(row / p.batch.rows) : 0;
  const int t = static_cast<int>(row - static_cast<int64_t>(b) * p.batch.rows);
  const uint32_t count = drafted(p.batch, b);
  float top = kLowest, sum = 0.0f;
  f32x4_t v{0, 0, 0, 0};
  if (there && t < static_cast<int>(count)) {
    const int group = b / parts.per;
    const uint32_t n = min(committed(p.batch, b) + count, p.batch.capacity);
    const uint32_t prefix = takes_prefix(parts, p.batch, b, group) ? prefix_tokens(parts, p.batch, group) : 0u;
    if (prefix > 0) {
      const Args a = parts.prefix();
      const uint32_t chunk = piece_of(prefix, a.splits, a.chunk);
      uint32_t used = (prefix + chunk - 1) / chunk;
      int64_t first = (static_cast<int64_t>(group) * p.cache.kv_heads + kv) * a.splits;
      if (a.plan != nullptr) {
        const uint2 plan = a.plan[group];
        used = plan.y;
        first = plan.x + static_cast<int64_t>(kv) * used;
      }
      const int64_t r = (row - static_cast<int64_t>(group) * parts.group_rows) * parts.group + g;
      if (share < static_cast<int>(used)) v = joined_sums<false>(a, first * a.row_slots + r, d, D, share, used, shares, &top, &sum);
    }
    const uint32_t chunk = piece_of(n - prefix, parts.splits, parts.chunk), used = max(1u, (n - prefix + chunk - 1) / chunk);
    const uint32_t own_share = static_cast<uint32_t>(shares - 1 - share);  // the prefix's last ones have fewer pieces
    if (own_share < used) {
      float own_top, own_sum;
      const f32x4_t w = joined_sums<false>(parts, (static_cast<int64_t>(b) * p.cache.kv_heads + kv) * parts.splits * parts.row_slots +
                                           static_cast<int64_t>(t) * parts.group + g, d, D, own_share, used, shares, &own_top, &own_sum);
      const float peak = fmaxf(top, own_top);
      const float keep = __builtin_amdgcn_exp2f(top - peak), own_keep = __builtin_amdgcn_exp2f(own_top - peak);
      sum = fmaf(sum, keep, own_sum * own_keep);
      v = v * keep + w * own_keep;
      top = peak;
    }
  }
  if (shares > 1) {
    part[threadIdx.x] = v;
    stats[threadIdx.x] = float2{top, sum};
    __syncthreads();
    if (!thread.adds_up()) return;
    for (int s = 1; s < shares; ++s) top = fmaxf(top, stats[threadIdx.x + s * pieces].x);
    v = f32x4_t{0, 0, 0, 0};
    sum = 0.0f;
    for (int s = 0; s < shares; ++s) {
      const float2 st = stats[threadIdx.x + s * pieces];
      const float keep = __builtin_amdgcn_exp2f(st.x - top);
      sum = fmaf(st.y, keep, sum);
      v += part[threadIdx.x + s * pieces] * keep;
    }
  }
  if (there) store_result<T>(p.out, slot * D + d, v, sum);
}

// Workgroups over `units` x row groups x splits.
int64_t blocks_of(int64_t units, int splits, int row_groups) { return (units * splits + 7) / 8 * 8 * row_groups; }

int64_t splits_for(int64_t round, int64_t groups, int64_t most) {
  return std::max<int64_t>(1, std::min((round + groups - 1) / groups, most));
}

}  // namespace
}  // namespace attention

hipError_t shared_attention_launch(const AttentionProblem& p, const uint32_t* shared, int groups, const Launch& l) {
  using namespace attention;
  const bool half = p.cache.dtype == AFFON_ROCM_BF16;
  const int D = p.cache.head_dim;
  const int64_t unit = half ? 128 : 64;  // the least keys of a piece
  constexpr int64_t kRound = 512;        // workgroups, two to a CU
  Parts parts{};
  parts.p = p;
  parts.shared = shared;
  parts.per = p.batch.sequences / groups;
  parts.group = p.heads / p.cache.kv_heads;
  parts.log2_scale = p.scale == 0.0f ? 1.0f : std::min(std::fabs(p.scale) * 1.44269504088896340736f, FLT_MAX);
  parts.sign = p.scale > 0.0f ? 1.0f : p.scale < 0.0f ? -1.0f : 0.0f;
  parts.groups = groups;
  const int64_t group_rows = static_cast<int64_t>(p.batch.rows) * parts.per, prefix_rows = group_rows * parts.group;
  if (prefix_rows > (int64_t(1) << 30)) return hipErrorInvalidValue;
  parts.group_rows = static_cast<int>(group_rows);
  parts.rows = parts.row_slots = p.batch.rows * parts.group;
  parts.prefix_rows = parts.prefix_slots = static_cast<int>(prefix_rows);

  // Waves of the kernel for prefixes of many rows, one workgroup to a CU, or 0: the
  // general one takes them, whose waves share 16 rows' keys. The whole call, 8 key
  // heads of 128, general and 4 waves (us): 16 rows of a key head after 2048
  // tokens 14.0 and 20.7, after 8192 26.2 and 25.6, after 32768 43.5 and 46.6; 32 rows
  // 23.1 and 21.6, 31.0 and 26.2, 48.6 and 47.3; 128 rows 30.0 and 28.8, 37.6
  // and 32.4, 58.3 and 52.5. 4 and 8 waves: 256 rows 29.1 and 37.8, 36.8 and
  // 41.6, 73.0 and 70.0; 192 rows 31.1 and 33.8, 34.9 and 38.6, 70.4 and 61.0.
  const bool takes = half ? D == 64 || D == 128 : D == 64 || D == 80 || D == 96 || D == 128;
  // f32, whose products bound both, from 129 rows on: one group's 128 rows of 80 after
  // 2048 tokens 44.7 us by the general one and 47.4, 32 rows of 64 after 16000 36.6 and
  // 41.7; 200 rows of 80 after 16000 151.3 and 144.5, of 64 114.3 and 111.3, and
  // where a third of the rows is not in use 102 and 92.
  const int tiles = !takes || prefix_rows <= (half ? 16 : 128) ? 0 : prefix_rows > 128 ? 8 : 4;
  const Shape own_shape = shape_for(parts.rows, D), prefix_shape = shape_for(parts.prefix_rows, D);
  const int64_t at_once = tiles > 0 ? 32 * tiles : prefix_shape.rows();
  parts.row_groups = (parts.rows + own_shape.rows() - 1) / own_shape.rows();
  parts.prefix_row_groups = static_cast<int>((prefix_rows + at_once - 1) / at_once);
  const int64_t units = static_cast<int64_t>(p.batch.sequences) * p.cache.kv_heads;
  const int64_t prefix_units = static_cast<int64_t>(groups) * p.cache.kv_heads;
  const int64_t most = std::max<int64_t>(1, p.batch.capacity / unit);
  parts.chunk = static_cast<uint32_t>(unit);
  parts.prefix_chunk = static_cast<uint32_t>(tiles > 0 ? 32 : unit);  // a step of the tiles' kernels
  parts.splits = static_cast<int>(splits_for(kRound, units * parts.row_groups, most));
  parts.prefix_splits = static_cast<int>(splits_for(tiles > 0 ? kRound / 2 : kRound, prefix_units * parts.prefix_row_groups, most));
  const int64_t own_blocks = blocks_of(units, parts.splits, parts.row_groups);
  // Pieces of all prefixes; cut over all groups, some have a few more.
  const int64_t prefix_pieces = tiles > 0 ? cut_most(groups, parts.prefix_splits) * p.cache.kv_heads : prefix_units * parts.prefix_splits;
  const int64_t prefix_blocks = blocks_of(prefix_pieces, 1, parts.prefix_row_groups);
  if (own_blocks + prefix_blocks > kMaxBlocks) return hipErrorInvalidValue;

  auto whole = [](size_t bytes) { return (bytes + 255) / 256 * 256; };
  const size_t own_slots = static_cast<size_t>(units) * parts.splits * parts.row_slots;
  const size_t prefix_slots = static_cast<size_t>(prefix_pieces) * parts.prefix_slots;
  const size_t sums = whole(own_slots * D * sizeof(float)), stats = whole(own_slots * sizeof(float2));
  const size_t prefix_sums = whole(prefix_slots * D * sizeof(float)), prefix_stats = whole(prefix_slots * sizeof(float2));
  const size_t plan = tiles > 0 ? groups * sizeof(uint2) : 0;
  auto* scratch = static_cast<uint8_t*>(l.scratch(sums + stats + prefix_sums + prefix_stats + plan));
  // A captured stream whose workspace cannot grow: every sequence by itself.
  if (scratch == nullptr) return attention_launch(p, l);
  parts.sums = reinterpret_cast<float*>(scratch);
  parts.stats = reinterpret_cast<float*>(scratch + sums);
  parts.prefix_sums = reinterpret_cast<float*>(scratch + sums + stats);
  parts.prefix_stats = reinterpret_cast<float*>(scratch + sums + stats + prefix_sums);
  if (tiles > 0) parts.prefix_plan = reinterpret_cast<uint2*>(scratch + sums + stats + prefix_sums + prefix_stats);

  auto launch = half ? launch_parts_bf16 : launch_parts_f32;
  auto run = [&](Shape shape, int64_t of_prefix, int64_t of_own) {
    parts.prefix_blocks = static_cast<unsigned>(of_prefix);
    launch(parts, shape, dim3(static_cast<unsigned>(of_prefix + of_own)), l.stream);
    return hipGetLastError();
  };
  hipError_t e = hipSuccess;
  if (tiles == 0 && prefix_shape.tiles == own_shape.tiles && prefix_shape.waves == own_shape.waves) {
    // One launch for both parts (four sequences of 40 tokens after 1008 12.7 us, in two launches 19.8).
    e = run(own_shape, prefix_blocks, own_blocks);
  } else {
    if (tiles > 0) {
      launch_prefix_tiles(parts.prefix(), tiles, dim3(static_cast<unsigned>(prefix_blocks)), l.stream);
      e = hipGetLastError();
    } else {
      e = run(prefix_shape, prefix_blocks, 0);
    }
    if (e == hipSuccess) e = run(own_shape, 0, own_blocks);
  }
  if (e != hipSuccess) return e;
  // A share takes the eight pieces that a thread has in flight, or fewer where
  // there are not enough workgroups.
  const int64_t results = static_cast<int64_t>(p.batch.sequences) * p.batch.rows * p.heads;
  const int threads = D / 4;
  int shares = std::min((std::max(parts.prefix_splits, parts.splits) + 7) / 8, kJoinThreads / threads);
  while (shares * 2 <= kJoinThreads / threads && shares * 2 <= parts.prefix_splits && results * threads * shares < 256 * 512) shares *= 2;
  const int64_t per = kJoinThreads / (threads * shares), blocks = (results + per - 1) / per;
  if (blocks > kMaxBlocks) return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (half)
    hipLaunchKernelGGL(join_parts_kernel<BF16>, grid, dim3(kJoinThreads), 0, l.stream, parts, shares);
  else
    hipLaunchKernelGGL(join_parts_kernel<F32>, grid, dim3(kJoinThreads), 0, l.stream, parts, shares);
  return hipGetLastError();
}

}  // namespace affon
