// Attention of drafted tokens over a paged cache: the choice of kernel and
// of the pieces that a long context is cut into, and the join of their
// results (attention.h holds the kernels).

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "attention.h"

namespace affon {
namespace attention {
namespace {

// Joins the splits, where the kernel's own workgroups do not: head_dim / 4
// threads for each of `shares` shares of the splits of a row and head, which
// then meet in LDS; several rows and heads to a workgroup.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(Args a, int shares) {
  __shared__ __attribute__((aligned(16))) f32x4_t part[256];
  __shared__ float2 stats[256];
  const AttentionProblem& p = a.p;
  const int D = p.cache.head_dim, pieces = D / 4, own = pieces * shares, per = 256 / own;
  const int local = threadIdx.x / own, share = (threadIdx.x - local * own) / pieces;
  const int piece = threadIdx.x % pieces, d = 4 * piece;
  const int64_t slot = static_cast<int64_t>(blockIdx.x) * per + local;  // of [row][head]
  const int64_t row = slot / p.heads;
  const bool there = local < per && row < static_cast<int64_t>(p.batch.sequences) * p.batch.rows;
  const int head = static_cast<int>(slot - row * p.heads), kv = head / a.group;
  const int b = there ? static_cast<int>(row / p.batch.rows) : 0;
  const int t = static_cast<int>(row - static_cast<int64_t>(b) * p.batch.rows);
  const uint32_t count = drafted(p.batch, b);
  const uint32_t n = min(committed(p.batch, b) + count, p.batch.capacity);
  const uint32_t used = (n + a.chunk - 1) / a.chunk;
  const bool works = there && used > 1;  // else the result is there
  f32x4_t v{0, 0, 0, 0};
  float top = kLowest, sum = 0.0f;
  if (works && share < static_cast<int>(used)) {
    const int64_t first = (static_cast<int64_t>(b) * p.cache.kv_heads + kv) * a.splits * a.row_slots + t * a.group +
                          head - kv * a.group;
    v = joined_sums<false>(a, first, d, D, share, used, shares, &top, &sum);
  }
  if (shares > 1) {
    part[threadIdx.x] = v;
    stats[threadIdx.x] = float2{top, sum};
    __syncthreads();
    if (share != 0 || local >= per) return;
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
  if (works) store_result<T>(p.out, slot * D + d, v, t < static_cast<int>(count) ? sum : 0.0f);
}

__global__ __launch_bounds__(256) void clear_kernel(uint32_t* words, int count) {
  for (int i = blockIdx.x * 256 + threadIdx.x; i < count; i += gridDim.x * 256) words[i] = 0;
}

// Few rows: waves side by side over the keys; more: over the rows, and where
// the keys of two waves do not fit in LDS twice to a CU. There two waves, as
// the ones past the last row still repeat its work: 32 sequences of one token
// over up to 4096, width 256, bf16 133 us in two waves and 169 in four, f32 306
// and 614.
Shape shape_for(int rows, int head_dim) {
  if (rows <= 16 && head_dim <= 128) return {1, 1};
  if (rows <= 32 && head_dim <= 128) return {2, 1};
  if (rows <= 32) return {1, 2};
  // Wide heads of odd sizes leave no registers for a second tile.
  if (rows <= 64 || (head_dim > 128 && head_dim != 256)) return {1, 4};
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
  const bool half = p.cache.dtype == AFFON_ROCM_BF16;
  const Shape shape = shape_for(a.rows, p.cache.head_dim);
  a.row_groups = (a.rows + shape.rows() - 1) / shape.rows();
  a.row_slots = a.rows;
  // Finite for every finite scale: infinite, it would make NaN of scores of 0.
  a.log2_scale = p.scale == 0.0f ? 1.0f : std::min(std::fabs(p.scale) * 1.44269504088896340736f, FLT_MAX);
  a.sign = p.scale > 0.0f ? 1.0f : p.scale < 0.0f ? -1.0f : 0.0f;

  // Pieces of the context: enough workgroups for the GPU, none so short that
  // its results weigh against the keys it reads. The lengths are on the device,
  // so pieces are cut from what the table holds; under a table wider than the
  // contexts they are longer and fewer, and the rest of the workgroups leave at
  // once (one token over 777 8.8 us under a table of 784 tokens, 10.9 of 8192
  // and 15.2 of 131072; 8 sequences of 2000 17.1 us, 17.3 and 28.8).
  const int64_t units = static_cast<int64_t>(p.batch.sequences) * p.cache.kv_heads;
  const int64_t capacity = p.batch.capacity;
  const int64_t own_rows = std::min(a.rows, shape.rows());
  // One round of workgroups, two to a CU: a second round of shorter ones costs
  // more in starts and joins than it evens out (32 sequences of one token over
  // up to 4096 tokens: 68.0 us in 512 workgroups, 76.8 in 768; trees of 24 of
  // 8 sequences 57.8 and 69.6). Much longer pieces leave the GPU uneven where
  // lengths differ, but the results of many rows weigh more (trees of 64 of
  // 16 sequences over up to 16384: 541 us in 512 workgroups, 445 in pieces of
  // 4096 keys, 463 of 2048). Pieces of fewer keys than rows cost more to join
  // than they read (trees of 64 of one sequence over 2000 tokens: 20.2 us in
  // pieces of as many keys as rows, 24.4 in twice that, 44.6 in eight times);
  // f32, whose products take eight times as long, is cut finer (trees of 32 of
  // 4 sequences over up to 2000 tokens 38.6 us against 51.5 with bf16's sizes).
  constexpr int64_t kRound = 512, kEven = 2048;
  const int64_t groups_whole = units * a.row_groups;
  // Four rounds of workgroups are even enough, and hold the partial results of no more.
  const int64_t even = std::min(capacity / std::max(kEven, 32 * own_rows), (4 * kRound + groups_whole - 1) / groups_whole);
  int64_t splits = std::max(kRound / groups_whole, even);
  const int64_t unit = half ? 128 : 64;  // keys, at least
  splits = std::min(splits, capacity / std::max<int64_t>(unit, half ? own_rows : own_rows / 2));
  splits = std::max<int64_t>(splits, 1);
  a.chunk = static_cast<uint32_t>((capacity + splits - 1) / splits + unit - 1) / unit * unit;
  a.splits = static_cast<int>((capacity + a.chunk - 1) / a.chunk);
  bool few = false;
  if (a.splits > 1) {
    const size_t slots = static_cast<size_t>(units) * a.splits * a.row_slots;
    const size_t sums = (slots * p.cache.head_dim * sizeof(float) + 255) / 256 * 256;
    auto* scratch = static_cast<uint8_t*>(l.scratch(sums + slots * sizeof(float2)));
    if (scratch != nullptr) {
      a.sums = reinterpret_cast<float*>(scratch);
      a.stats = reinterpret_cast<float*>(scratch + sums);
      bool fresh = false;
      // Few results are joined by the workgroup that is last to end (one token
      // over 777: 9.4 us against 11.8 with a second launch; 32 sequences 67.7
      // and 70.2), more by a launch of their own (one token over 32000, 129 KB
      // a head: 36.6 and 34.6; trees of 24 94 and 62). Captured calls get no
      // tickets, and join few results in a launch too, in the same order (one
      // token over 777 in a graph: 10.3 us against 8.3 with tickets).
      constexpr int64_t kJoined = 32768;
      few = own_rows * p.cache.head_dim * 4 * a.splits <= kJoined;
      if (few && units * a.row_groups <= Workspace::kTickets && l.workspace != nullptr)
        a.tickets = l.workspace->tickets(&fresh);
      if (fresh) hipLaunchKernelGGL(clear_kernel, dim3(64), dim3(256), 0, l.stream, a.tickets, Workspace::kTickets);
    } else {  // a captured stream whose workspace cannot grow
      a.splits = 1;
    }
  }
  const int64_t groups = units * a.splits;
  const int64_t blocks = (groups + 7) / 8 * 8 * a.row_groups;
  if (blocks > kMaxBlocks) return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks));
  (half ? launch_bf16 : launch_f32)(a, shape, grid, l.stream);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1 || a.tickets != nullptr) return e;
  // A share takes the eight splits that a thread has in flight.
  const int pieces = p.cache.head_dim / 4;
  const int shares = few ? 1 : std::min((a.splits + 7) / 8, 256 / pieces);
  const int64_t per = 256 / (pieces * shares);
  const int64_t join_blocks = (static_cast<int64_t>(p.batch.sequences) * p.batch.rows * p.heads + per - 1) / per;
  if (join_blocks > kMaxBlocks) return hipErrorInvalidValue;
  const dim3 join_grid(static_cast<unsigned>(join_blocks));
  if (half)
    hipLaunchKernelGGL(join_kernel<BF16>, join_grid, dim3(256), 0, l.stream, a, shares);
  else
    hipLaunchKernelGGL(join_kernel<F32>, join_grid, dim3(256), 0, l.stream, a, shares);
  return hipGetLastError();
}

}  // namespace affon
