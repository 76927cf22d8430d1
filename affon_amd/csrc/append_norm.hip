// The append with norms of the query and key heads, and with positions of
// several axes: for each head, n = x / sqrt(mean(x^2) + epsilon) * w, and each
// pair of n turned by the position of its axis, in one pass.
//
// Bound by memory where rows are many: 4096 rows of 80 heads of 128 (f32 to bf16
// pages) 50.4 us, 5.0 TB/s of 5.2 that a large copy reaches; 2738 rows of 48 heads (bf16,
// three axes) 15.6 us, 4.4 TB/s, where the instructions around 16 bytes a lane count too.
// One row of 48 heads 3.7 us, a launch and a chain of three loads.

#include <algorithm>

#include "lds_pipeline.h"
#include "paged.h"
#include "values.h"

namespace affon {
namespace {

// The sum over each group of 2^lanes_log lanes, in all of them.
__device__ __forceinline__ float group_sum(float v, int lanes_log) {
  if (lanes_log > 0) v = plus_lane<kNextLane>(v);
  if (lanes_log > 1) v = plus_lane<kNextPair>(v);
  if (lanes_log > 2) v = plus_lane<kOtherFour>(v);
  if (lanes_log > 3) v = plus_lane<kOtherEight>(v);
  if (lanes_log > 4) v += __shfl_xor(v, 16);
  if (lanes_log > 5) v += __shfl_xor(v, 32);
  return v;
}

template <typename C, int V>
__device__ __forceinline__ void store_rounded(uint8_t* base, int64_t at, const float (&v)[V]) {
  if constexpr (C::bytes == 2 && V == 8) {
    *reinterpret_cast<u32x4_t*>(base + at * 2) = u32x4_t{pipeline::pack_bf16(v[0], v[1]), pipeline::pack_bf16(v[2], v[3]),
                                                         pipeline::pack_bf16(v[4], v[5]), pipeline::pack_bf16(v[6], v[7])};
  } else if constexpr (C::bytes == 2 && V == 4) {
    *reinterpret_cast<u32x2_t*>(base + at * 2) = u32x2_t{pipeline::pack_bf16(v[0], v[1]), pipeline::pack_bf16(v[2], v[3])};
  } else {
    store_values<C, V>(base, at, v);
  }
}

// 2^lanes_log lanes hold a head, V pairs of it each (V = 1: two where a wave
// holds fewer than half the head's values): the first and the second value of
// the pairs are V consecutive ones each, interleaved pairs 2V consecutive
// values. A head's lanes meet in its sum of squares without LDS, and lanes past
// an odd head's end idle. `parts` workgroups take the heads of one row, one
// after the other in a group of lanes: what belongs to the row (its place, positions and
// pages) is in scalar registers, its cosines and sines are read once.
template <typename X, typename C, int V, bool INTERLEAVED>
__global__ __launch_bounds__(320) void append_norm_kernel(AppendNormProblem q, int lanes_log, uint32_t parts) {
  constexpr int kChunks = V == 1 ? 2 : 1;
  const AppendProblem& p = q.base;
  const int D = p.cache.head_dim, half = p.rotary_dim / 2;
  const uint32_t heads = p.heads, kv = p.cache.kv_heads, slots = heads + 2 * kv;
  const int64_t row = blockIdx.x / parts, rows = static_cast<int64_t>(p.batch.sequences) * p.batch.rows;
  const int b = static_cast<int>(row / p.batch.rows);
  const uint32_t i = static_cast<uint32_t>(row - static_cast<int64_t>(b) * p.batch.rows);
  const uint32_t groups = blockDim.x >> lanes_log;
  const uint32_t first_head = (blockIdx.x - static_cast<uint32_t>(row) * parts) * groups + (threadIdx.x >> lanes_log);
  const uint32_t stride = groups * parts;
  const int lane = threadIdx.x & ((1 << lanes_log) - 1);

  // Places in a query or key (its pairs, or the halves of its kept dims), and in a value (its halves).
  int w[kChunks], first[kChunks], second[kChunks];
  bool there[kChunks], turns[kChunks];
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    w[c] = ((c << lanes_log) + lane) * V;  // pairs before
    there[c] = w[c] < D / 2;
    turns[c] = w[c] < half;
    if (turns[c]) {
      first[c] = INTERLEAVED ? 2 * w[c] : w[c];
      second[c] = INTERLEAVED ? 2 * w[c] + V : half + w[c];
    } else {
      first[c] = p.rotary_dim + (w[c] - half);
      second[c] = first[c] + (D / 2 - half);
    }
  }
  const uint8_t* in[3] = {p.query + row * p.query_stride * X::bytes, p.key + row * p.key_stride * X::bytes,
                          p.value + row * p.value_stride * X::bytes};
  float x[kChunks][V], y[kChunks][V];
  auto load = [&](uint32_t head, float (&to_x)[kChunks][V], float (&to_y)[kChunks][V]) {
    const bool is_query = head < heads, is_value = head >= heads + kv;
    const uint32_t h = is_query ? head : is_value ? head - heads - kv : head - heads;
    const uint8_t* from = (is_query ? in[0] : is_value ? in[2] : in[1]) + h * static_cast<uint32_t>(D * X::bytes);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
#pragma unroll
      for (int e = 0; e < V; ++e) to_x[c][e] = to_y[c][e] = 0.0f;
      if (!there[c]) continue;
      load_values<X, V>(from, is_value ? w[c] : first[c], to_x[c]);
      load_values<X, V>(from, is_value ? D / 2 + w[c] : second[c], to_y[c]);
    }
  };
  if (first_head < slots) load(first_head, x, y);

  const uint32_t length = p.batch.lengths[b];
  const bool used = i < drafted(p.batch, b);
  const int64_t line = used && length < p.batch.capacity ? line_of(p.cache, p.batch, b, length + i) : -1;
  float cosine[kChunks][V], sine[kChunks][V];
  uint32_t axes[kChunks];  // two bits a pair, of a table of words in the arguments
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    axes[c] = 0;
    if (q.axes > 1) {
#pragma unroll
      for (int word = 0; word < kAxisWords; ++word)
        if (w[c] / 16 == word) axes[c] = q.axis[word];
      axes[c] >>= 2 * (w[c] % 16);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) cosine[c][e] = sine[c][e] = 0.0f;
  }
  uint32_t place[4];  // the row's positions
#pragma unroll
  for (int axis = 0; axis < 4; ++axis) {
    place[axis] = length + i;
    if (p.positions != nullptr && axis < q.axes) place[axis] = p.positions[axis * rows + row];
  }
  auto table_at = [&](uint32_t position, int c, float (&co)[V], float (&si)[V]) {
    if (position >= p.rotary_rows) return;  // zeros
    const auto* table = reinterpret_cast<const uint8_t*>(p.rotary + static_cast<int64_t>(position) * p.rotary_dim);
    load_values<F32, V>(table, w[c], co);
    load_values<F32, V>(table, half + w[c], si);
  };
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    constexpr uint32_t kPairs = (uint32_t(1) << 2 * V) - 1;
    const uint32_t axis = axes[c] & 3;
    if (__all((axes[c] & kPairs) == axis * (0x5555u & kPairs) || !turns[c])) {  // each lane's pairs have one axis
      const uint32_t position = axis < 2 ? (axis == 0 ? place[0] : place[1]) : (axis == 2 ? place[2] : place[3]);
      if (turns[c]) table_at(position, c, cosine[c], sine[c]);
      continue;
    }
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      bool any = false;
#pragma unroll
      for (int e = 0; e < V; ++e) any |= static_cast<int>(axes[c] >> (2 * e) & 3) == a;
      if (!any || !turns[c]) continue;
      float co[V] = {}, si[V] = {};
      table_at(place[a], c, co, si);
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (static_cast<int>(axes[c] >> (2 * e) & 3) == a) {
          cosine[c][e] = co[e];
          sine[c][e] = si[e];
        }
    }
  }

  auto finish = [&](uint32_t head, float (&hx)[kChunks][V], float (&hy)[kChunks][V]) {
    const bool is_query = head < heads, is_value = head >= heads + kv;
    const uint32_t h = is_query ? head : is_value ? head - heads - kv : head - heads;
    const uint8_t* weight = is_query ? q.query_norm.weight : q.key_norm.weight;
    if (!is_value && weight != nullptr) {
      const bool half_weight = (is_query ? q.query_norm.dtype : q.key_norm.dtype) == AFFON_ROCM_BF16;
      const uint32_t at = h * static_cast<uint32_t>(is_query ? q.query_norm.stride : q.key_norm.stride);
      float wx[kChunks][V], wy[kChunks][V], sum = 0.0f;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          wx[c][e] = wy[c][e] = 0.0f;
          sum = fmaf(hx[c][e], hx[c][e], fmaf(hy[c][e], hy[c][e], sum));
        }
        if (!there[c]) continue;
        if (half_weight) {
          load_values<BF16, V>(weight, at + first[c], wx[c]);
          load_values<BF16, V>(weight, at + second[c], wy[c]);
        } else {
          load_values<F32, V>(weight, at + first[c], wx[c]);
          load_values<F32, V>(weight, at + second[c], wy[c]);
        }
      }
      sum = group_sum(sum, lanes_log);
      const float scale = 1.0f / sqrtf(sum / static_cast<float>(D) + q.epsilon);
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          hx[c][e] = hx[c][e] * scale * wx[c][e];
          hy[c][e] = hy[c][e] * scale * wy[c][e];
        }
    }
    if (!is_query && line < 0) return;
    uint8_t* to = is_query   ? p.out + (row * heads + h) * D * C::bytes
                  : is_value ? p.cache.values + (line + static_cast<int64_t>(h) * p.cache.page_size) * D * C::bytes
                             : p.cache.keys + (line + static_cast<int64_t>(h) * p.cache.page_size) * D * C::bytes;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      if (!there[c]) continue;
      if (is_value) {
        store_rounded<C, V>(to, w[c], hx[c]);
        store_rounded<C, V>(to, D / 2 + w[c], hy[c]);
        continue;
      }
      if (!used) {  // a query: keys have left
#pragma unroll
        for (int e = 0; e < V; ++e) hx[c][e] = hy[c][e] = 0.0f;
      } else if (turns[c]) {
        float v[2 * V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          v[e] = hx[c][e];
          v[V + e] = hy[c][e];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
          // Interleaved: pair e is the two neighbours 2e, 2e + 1 of the 2V values.
          const int one = INTERLEAVED ? 2 * e : e, two = INTERLEAVED ? 2 * e + 1 : V + e;
          const float x1 = v[one], x2 = v[two];
          v[one] = x1 * cosine[c][e] - x2 * sine[c][e];
          v[two] = x2 * cosine[c][e] + x1 * sine[c][e];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
          hx[c][e] = v[e];
          hy[c][e] = v[V + e];
        }
      }
      store_rounded<C, V>(to, first[c], hx[c]);
      store_rounded<C, V>(to, second[c], hy[c]);
    }
  };
  for (uint32_t head = first_head; head < slots; head += stride) {
    finish(head, x, y);
    if (head + stride < slots) load(head + stride, x, y);
  }
}

// As the plain append: eight values at a time for many rows (four: 4096 rows of 80
// heads 58 us instead of 51; few rows then have too few lanes with loads on their way).
constexpr int64_t kManyRows = 64;

template <typename X, typename C, int V>
hipError_t launch_wide(const AppendNormProblem& q, hipStream_t stream) {
  const AppendProblem& p = q.base;
  const int64_t rows = static_cast<int64_t>(p.batch.sequences) * p.batch.rows;
  int lanes_log = 0;
  while (lanes_log < 6 && (V << lanes_log) < p.cache.head_dim / 2) ++lanes_log;
  // Few rows: a head to every group of lanes. Many: a workgroup of at most `most`
  // waves to a row, which take its heads in turns, and as few waves as need no more
  // turns. bf16 operands, where the instructions bound it, in more turns, to set
  // the row up less often: 2738 rows of 48 heads of 128 in two waves (three
  // turns) 16.2 us, in three (two turns) 17.8 (whole calls). f32, 4096 rows of 80 heads, in
  // two waves (five turns) 54.2, in five (two turns) 52.2.
  const int64_t waves = ((static_cast<int64_t>(p.heads + 2 * p.cache.kv_heads) << lanes_log) + 63) / 64;
  const int64_t most = X::bytes == 2 ? 2 : 5;
  const int64_t turns = rows < kManyRows ? 1 : (waves + most - 1) / most;
  const int64_t each = rows < kManyRows ? std::min<int64_t>(waves, 4) : (waves + turns - 1) / turns;
  const int64_t parts = rows < kManyRows ? (waves + each - 1) / each : 1;
  if (rows * parts * each > kMaxBlocks * 4) return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(rows * parts)), block(static_cast<unsigned>(64 * each));
  if (p.interleaved)
    hipLaunchKernelGGL((append_norm_kernel<X, C, V, true>), grid, block, 0, stream, q, lanes_log, static_cast<uint32_t>(parts));
  else
    hipLaunchKernelGGL((append_norm_kernel<X, C, V, false>), grid, block, 0, stream, q, lanes_log, static_cast<uint32_t>(parts));
  return hipGetLastError();
}

template <typename X, typename C>
hipError_t launch_typed(const AppendNormProblem& q, hipStream_t stream) {
  const AppendProblem& p = q.base;
  const int64_t rows = static_cast<int64_t>(p.batch.sequences) * p.batch.rows;
  const int D = p.cache.head_dim, half = p.rotary_dim / 2;
  // Eight or four values at a time where every row, half, weight and table row
  // starts at a multiple of them (16-byte accesses need no more than that), else one.
  const uint64_t starts = static_cast<uint64_t>(p.query_stride | p.key_stride | p.value_stride | half |
                                                (D / 2 - half) | p.rotary_dim);
  const uintptr_t bases = reinterpret_cast<uintptr_t>(p.query) | reinterpret_cast<uintptr_t>(p.key) |
                          reinterpret_cast<uintptr_t>(p.value);
  const uintptr_t outs = reinterpret_cast<uintptr_t>(p.out);
  auto weights_fit = [](const HeadNorm& n, int v) {
    const int size = n.dtype == AFFON_ROCM_BF16 ? 2 : 4;
    return reinterpret_cast<uintptr_t>(n.weight) % std::min(16, v * size) == 0;
  };
  auto fits = [&](int v) {
    return starts % v == 0 && bases % std::min(16, v * X::bytes) == 0 && outs % std::min(16, v * C::bytes) == 0 &&
           weights_fit(q.query_norm, v) && weights_fit(q.key_norm, v) &&
           reinterpret_cast<uintptr_t>(p.rotary) % 16 == 0 && D % (2 * v) == 0;
  };
  if (fits(8) && rows >= kManyRows) return launch_wide<X, C, 8>(q, stream);
  if (fits(4)) return launch_wide<X, C, 4>(q, stream);
  return launch_wide<X, C, 1>(q, stream);
}

}  // namespace

hipError_t append_norm_launch(const AppendNormProblem& q, hipStream_t stream) {
  const bool half = q.base.cache.dtype == AFFON_ROCM_BF16;
  if (q.base.x_dtype == AFFON_ROCM_BF16)
    return half ? launch_typed<BF16, BF16>(q, stream) : launch_typed<BF16, F32>(q, stream);
  return half ? launch_typed<F32, BF16>(q, stream) : launch_typed<F32, F32>(q, stream);
}

}  // namespace affon
