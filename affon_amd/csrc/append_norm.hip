// The append with norms of the query and key heads, and with positions of
// several axes: for each head, n = x / sqrt(mean(x^2) + epsilon) * w, and each
// pair of n turned by the position of its axis, in one pass.

#include <algorithm>

#include "paged.h"
#include "values.h"

namespace affon {
namespace {

// 2^lanes_log lanes hold a head, V pairs of it each (V = 1: two where a wave
// holds fewer than half the head's values): the first and the second value of the pairs are V consecutive
// ones each, interleaved pairs 2V consecutive values. A head's lanes meet in
// its sum of squares without LDS, and lanes past an odd head's end idle.
template <typename X, typename C, int V>
__global__ __launch_bounds__(256) void append_norm_kernel(AppendNormProblem q, int lanes_log) {
  constexpr int kChunks = V == 1 ? 2 : 1;
  const AppendProblem& p = q.base;
  const int D = p.cache.head_dim, heads = p.heads, kv = p.cache.kv_heads;
  const uint32_t slots = static_cast<uint32_t>(heads + 2 * kv);  // heads of a row
  const int lanes = 1 << lanes_log, lane = threadIdx.x & (lanes - 1);
  const uint32_t per = 256u >> lanes_log;
  int64_t row = static_cast<int64_t>(blockIdx.x) * per / slots;
  uint32_t head = static_cast<uint32_t>(static_cast<int64_t>(blockIdx.x) * per - row * slots) + (threadIdx.x >> lanes_log);
  if (head >= slots) {
    row += head / slots;
    head %= slots;
  }
  if (row >= static_cast<int64_t>(p.batch.sequences) * p.batch.rows) return;
  const int b = static_cast<int>(row / p.batch.rows);
  const uint32_t i = static_cast<uint32_t>(row - static_cast<int64_t>(b) * p.batch.rows);

  const int half = p.rotary_dim / 2;
  const bool is_query = head < static_cast<uint32_t>(heads), is_value = head >= static_cast<uint32_t>(heads + kv);
  const uint32_t h = is_query ? head : is_value ? head - heads - kv : head - heads;
  const uint8_t* in = is_query ? p.query + row * p.query_stride * X::bytes
                      : is_value ? p.value + row * p.value_stride * X::bytes
                                 : p.key + row * p.key_stride * X::bytes;
  int first[kChunks], second[kChunks], w[kChunks];
  bool there[kChunks], turns[kChunks];
  float x[kChunks][V], y[kChunks][V];
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    w[c] = (c * lanes + lane) * V;  // pairs before
    there[c] = w[c] < D / 2;
    turns[c] = !is_value && w[c] < half;
    if (is_value) {  // the halves of what is kept
      first[c] = w[c];
      second[c] = D / 2 + w[c];
    } else if (turns[c]) {
      first[c] = p.interleaved ? 2 * w[c] : w[c];
      second[c] = p.interleaved ? 2 * w[c] + V : half + w[c];
    } else {
      first[c] = p.rotary_dim + (w[c] - half);
      second[c] = first[c] + (D / 2 - half);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) x[c][e] = y[c][e] = 0.0f;
    if (there[c]) {
      load_values<X, V>(in, static_cast<int64_t>(h) * D + first[c], x[c]);
      load_values<X, V>(in, static_cast<int64_t>(h) * D + second[c], y[c]);
    }
  }
  const uint32_t length = p.batch.lengths[b];
  const bool used = i < drafted(p.batch, b);

  const HeadNorm& norm = is_query ? q.query_norm : q.key_norm;
  if (!is_value && norm.weight != nullptr) {
    float wx[kChunks][V], wy[kChunks][V];
    const int64_t at = static_cast<int64_t>(h) * norm.stride;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
#pragma unroll
      for (int e = 0; e < V; ++e) wx[c][e] = wy[c][e] = 0.0f;
      if (!there[c]) continue;
      if (norm.dtype == AFFON_ROCM_BF16) {
        load_values<BF16, V>(norm.weight, at + first[c], wx[c]);
        load_values<BF16, V>(norm.weight, at + second[c], wy[c]);
      } else {
        load_values<F32, V>(norm.weight, at + first[c], wx[c]);
        load_values<F32, V>(norm.weight, at + second[c], wy[c]);
      }
    }
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) sum = fmaf(x[c][e], x[c][e], fmaf(y[c][e], y[c][e], sum));
    for (int offset = lanes >> 1; offset > 0; offset >>= 1) sum += __shfl_xor(sum, offset);
    const float scale = 1.0f / sqrtf(sum / static_cast<float>(D) + q.epsilon);
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        x[c][e] = x[c][e] * scale * wx[c][e];
        y[c][e] = y[c][e] * scale * wy[c][e];
      }
  }

  // Where the head goes.
  uint8_t* to = p.out;
  int64_t at = (row * heads + h) * D;
  if (!is_query) {
    if (!used || length >= p.batch.capacity) return;
    const int64_t line = line_of(p.cache, p.batch, b, length + i);
    if (line < 0) return;
    to = is_value ? p.cache.values : p.cache.keys;
    at = (line + static_cast<int64_t>(h) * p.cache.page_size) * D;
  }
  const int64_t rows = static_cast<int64_t>(p.batch.sequences) * p.batch.rows;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    if (!there[c]) continue;
    if (turns[c]) {
      // The axes that these pairs have, one after the other: mostly one.
      float cosine[V], sine[V];
#pragma unroll
      for (int e = 0; e < V; ++e) cosine[e] = sine[e] = 0.0f;
      uint32_t axes = 0;  // two bits a pair, of a table of words in the arguments
      if (q.axes > 1) {
#pragma unroll
        for (int k = 0; k < kAxisWords; ++k)
          if (w[c] / 16 == k) axes = q.axis[k];
        axes >>= 2 * (w[c] % 16);
      }
      for (int axis = 0; axis < q.axes; ++axis) {
        bool any = false;
#pragma unroll
        for (int e = 0; e < V; ++e) any |= static_cast<int>(axes >> (2 * e) & 3) == axis;
        if (!any) continue;
        const uint32_t position = p.positions != nullptr ? p.positions[axis * rows + row] : length + i;
        if (position >= p.rotary_rows) continue;
        const auto* table = reinterpret_cast<const uint8_t*>(p.rotary + static_cast<int64_t>(position) * p.rotary_dim);
        float co[V], si[V];
        load_values<F32, V>(table, w[c], co);
        load_values<F32, V>(table, half + w[c], si);
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (static_cast<int>(axes >> (2 * e) & 3) == axis) {
            cosine[e] = co[e];
            sine[e] = si[e];
          }
      }
      float v[2 * V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[e] = x[c][e];
        v[V + e] = y[c][e];
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        // Interleaved: pair e is the two neighbours 2e, 2e + 1 of the 2V values.
        const float x1 = p.interleaved ? v[2 * e] : x[c][e], x2 = p.interleaved ? v[2 * e + 1] : y[c][e];
        const float y1 = x1 * cosine[e] - x2 * sine[e], y2 = x2 * cosine[e] + x1 * sine[e];
        if (p.interleaved) {
          v[2 * e] = y1;
          v[2 * e + 1] = y2;
        } else {
          v[e] = y1;
          v[V + e] = y2;
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        x[c][e] = v[e];
        y[c][e] = v[V + e];
      }
    }
    if (is_query && !used) {
#pragma unroll
      for (int e = 0; e < V; ++e) x[c][e] = y[c][e] = 0.0f;
    }
    store_values<C, V>(to, at + first[c], x[c]);
    store_values<C, V>(to, at + second[c], y[c]);
  }
}

// As the plain append: eight values at a time for many rows.
constexpr int64_t kManyRows = 64;

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
  const int v = fits(8) && rows >= kManyRows ? 8 : fits(4) ? 4 : 1;
  int lanes_log = 0;
  while (lanes_log < 6 && (v << lanes_log) < D / 2) ++lanes_log;
  const int64_t per = 256 >> lanes_log;
  const int64_t blocks = (rows * (p.heads + 2 * p.cache.kv_heads) + per - 1) / per;
  if (blocks > kMaxBlocks) return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (v == 8)
    hipLaunchKernelGGL((append_norm_kernel<X, C, 8>), grid, dim3(256), 0, stream, q, lanes_log);
  else if (v == 4)
    hipLaunchKernelGGL((append_norm_kernel<X, C, 4>), grid, dim3(256), 0, stream, q, lanes_log);
  else
    hipLaunchKernelGGL((append_norm_kernel<X, C, 1>), grid, dim3(256), 0, stream, q, lanes_log);
  return hipGetLastError();
}

}  // namespace

hipError_t append_norm_launch(const AppendNormProblem& q, hipStream_t stream) {
  const bool half = q.base.cache.dtype == AFFON_ROCM_BF16;
  if (q.base.x_dtype == AFFON_ROCM_BF16)
    return half ? launch_typed<BF16, BF16>(q, stream) : launch_typed<BF16, F32>(q, stream);
  return half ? launch_typed<F32, BF16>(q, stream) : launch_typed<F32, F32>(q, stream);
}

}  // namespace affon
