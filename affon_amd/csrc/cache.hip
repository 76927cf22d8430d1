// The paged cache's writers: keys and values of drafted tokens appended with
// the position rotation applied on the way, and the accepted ones moved up
// behind the committed ones.

#include <algorithm>
#include <type_traits>

#include "paged.h"
#include "values.h"

namespace affon {
namespace {

// Unit and row of this thread, where a row is `units` threads' work: one
// division per workgroup, and one per thread only where rows are short.
__device__ __forceinline__ void locate(uint32_t units, int64_t* row, uint32_t* unit) {
  const int64_t first = static_cast<int64_t>(blockIdx.x) * 256;
  *row = first / units;
  uint32_t u = static_cast<uint32_t>(first - *row * units) + threadIdx.x;
  if (units < 256) {
    *row += u / units;
    u %= units;
  } else if (u >= units) {
    ++*row;
    u -= units;
  }
  *unit = u;
}

// One thread rotates V pairs of a head of a token's query or key, or copies
// the 2V values of a head's kept dims, or of a value. The first and the second
// value of the pairs are V consecutive ones each; interleaved pairs are 2V
// consecutive values.
template <typename X, typename C, int V>
__global__ __launch_bounds__(256) void append_kernel(AppendProblem p) {
  const int D = p.cache.head_dim, per_head = D / (2 * V);
  const int heads = p.heads, kv = p.cache.kv_heads;
  int64_t row;
  uint32_t unit;
  locate(static_cast<uint32_t>((heads + 2 * kv) * per_head), &row, &unit);
  if (row >= static_cast<int64_t>(p.batch.sequences) * p.batch.rows) return;
  const uint32_t head = unit / per_head;
  const int w = (unit - head * per_head) * V;  // pairs before
  const int b = static_cast<int>(row / p.batch.rows);
  const uint32_t i = static_cast<uint32_t>(row - static_cast<int64_t>(b) * p.batch.rows);

  const int half = p.rotary_dim / 2;
  const bool is_value = head >= static_cast<uint32_t>(heads + kv);
  // Kept dims, and values: the halves of what they are, both copied.
  const bool turns = !is_value && w < half;
  int first, second;
  if (is_value) {
    first = w;
    second = D / 2 + w;
  } else if (turns) {
    first = p.interleaved ? 2 * w : w;
    second = p.interleaved ? 2 * w + V : half + w;
  } else {
    first = p.rotary_dim + (w - half);
    second = first + (D / 2 - half);
  }
  const bool is_query = head < static_cast<uint32_t>(heads);
  const uint32_t h = is_query ? head : is_value ? head - heads - kv : head - heads;
  const uint8_t* in = is_query ? p.query + row * p.query_stride * X::bytes
                      : is_value ? p.value + row * p.value_stride * X::bytes
                                 : p.key + row * p.key_stride * X::bytes;
  float x[V], y[V];
  load_values<X, V>(in, static_cast<int64_t>(h) * D + first, x);
  load_values<X, V>(in, static_cast<int64_t>(h) * D + second, y);

  const uint32_t length = p.batch.lengths[b];
  const bool used = i < drafted(p.batch, b);
  if (turns) {
    const uint32_t position = p.positions != nullptr ? p.positions[row] : length + i;
    float c[V], s[V];
    if (position < p.rotary_rows) {
      const auto* table = reinterpret_cast<const uint8_t*>(p.rotary + static_cast<int64_t>(position) * p.rotary_dim);
      load_values<F32, V>(table, w, c);
      load_values<F32, V>(table, half + w, s);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) c[e] = s[e] = 0.0f;
    }
    float v[2 * V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      v[e] = x[e];
      v[V + e] = y[e];
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      // Interleaved: pair e is the two neighbours 2e, 2e + 1 of the 2V values.
      const float x1 = p.interleaved ? v[2 * e] : x[e], x2 = p.interleaved ? v[2 * e + 1] : y[e];
      const float y1 = x1 * c[e] - x2 * s[e], y2 = x2 * c[e] + x1 * s[e];
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
      x[e] = v[e];
      y[e] = v[V + e];
    }
  }
  uint8_t* to;
  int64_t at;
  if (is_query) {
    to = p.out;
    at = (row * heads + h) * D;
    if (!used) {
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = y[e] = 0.0f;
    }
  } else {
    if (!used || length >= p.batch.capacity) return;
    const int64_t line = line_of(p.cache, p.batch, b, length + i);
    if (line < 0) return;
    to = is_value ? p.cache.values : p.cache.keys;
    at = (line + static_cast<int64_t>(h) * p.cache.page_size) * D;
  }
  store_values<C, V>(to, at + first, x);
  store_values<C, V>(to, at + second, y);
}

// Every thread takes one piece of 16 bytes of a token's keys or values of one
// layer through the accepted tokens in their order, eight at a time: the path
// ascends strictly, so token path[i] >= i is read before anything is written
// to its place, and no other thread touches these bytes.
constexpr int kMoves = 8;

__global__ __launch_bounds__(256) void commit_kernel(PagedCache cache, DraftBatch batch, const uint32_t* path,
                                                     int64_t path_stride, int path_columns, const uint32_t* accepted) {
  const int line_pieces = cache.head_dim * (cache.dtype == AFFON_ROCM_BF16 ? 2 : 4) / 16;
  const uint32_t units = static_cast<uint32_t>(2 * cache.kv_heads * line_pieces);
  int64_t row;
  uint32_t unit;
  locate(units, &row, &unit);
  if (row >= static_cast<int64_t>(cache.layers) * batch.sequences) return;
  const int64_t layer = row / batch.sequences;
  const int b = static_cast<int>(row - layer * batch.sequences);
  const uint32_t length = batch.lengths[b];
  if (length >= batch.capacity) return;
  const uint32_t count = min(accepted[b], static_cast<uint32_t>(path_columns));
  const uint32_t line = unit / line_pieces, piece = unit - line * line_pieces;
  const bool is_value = line >= static_cast<uint32_t>(cache.kv_heads);
  const uint32_t head = is_value ? line - cache.kv_heads : line;
  auto* data = reinterpret_cast<u32x4_t*>((is_value ? cache.values : cache.keys) + layer * cache.layer_bytes);
  const int64_t head_lines = static_cast<int64_t>(head) * cache.page_size;
  for (uint32_t i0 = 0; i0 < count; i0 += kMoves) {
    int64_t to[kMoves];
    u32x4_t v[kMoves];
#pragma unroll
    for (int j = 0; j < kMoves; ++j) {
      const uint32_t i = i0 + j;
      to[j] = -1;
      if (i >= count) continue;
      const uint32_t from = path[b * path_stride + i];
      if (from == i || from >= static_cast<uint32_t>(batch.rows)) continue;
      const int64_t source = line_of(cache, batch, b, length + from);
      if (source < 0) continue;
      to[j] = line_of(cache, batch, b, length + i);
      if (to[j] >= 0) v[j] = data[(source + head_lines) * line_pieces + piece];
    }
#pragma unroll
    for (int j = 0; j < kMoves; ++j)
      if (to[j] >= 0) data[(to[j] + head_lines) * line_pieces + piece] = v[j];
  }
}

constexpr int64_t kManyRows = 64;

template <typename X, typename C>
hipError_t append_typed(const AppendProblem& p, hipStream_t stream) {
  const int64_t rows = static_cast<int64_t>(p.batch.sequences) * p.batch.rows;
  const int half = p.rotary_dim / 2;
  // Eight or four values at a time where every row, half and table row starts
  // at a multiple of them (16-byte accesses need no more than that), else one.
  const uint64_t starts = static_cast<uint64_t>(p.query_stride | p.key_stride | p.value_stride | half |
                                                (p.cache.head_dim / 2 - half) | p.rotary_dim);
  const uintptr_t bases = reinterpret_cast<uintptr_t>(p.query) | reinterpret_cast<uintptr_t>(p.key) |
                          reinterpret_cast<uintptr_t>(p.value);
  const uintptr_t outs = reinterpret_cast<uintptr_t>(p.out);
  auto fits = [&](int v) {
    return starts % v == 0 && bases % std::min(16, v * X::bytes) == 0 && outs % std::min(16, v * C::bytes) == 0 &&
           reinterpret_cast<uintptr_t>(p.rotary) % 16 == 0 && p.cache.head_dim % (2 * v) == 0;
  };
  const int v = fits(8) && rows >= kManyRows ? 8 : fits(4) ? 4 : 1;
  const int64_t units = rows * (p.heads + 2 * p.cache.kv_heads) * (p.cache.head_dim / (2 * v));
  const int64_t blocks = (units + 255) / 256;
  if (blocks > kMaxBlocks) return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (v == 8)
    hipLaunchKernelGGL((append_kernel<X, C, 8>), grid, dim3(256), 0, stream, p);
  else if (v == 4)
    hipLaunchKernelGGL((append_kernel<X, C, 4>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((append_kernel<X, C, 1>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t append_launch(const AppendProblem& p, hipStream_t stream) {
  if (p.x_dtype == AFFON_ROCM_BF16)
    return p.cache.dtype == AFFON_ROCM_BF16 ? append_typed<BF16, BF16>(p, stream) : append_typed<BF16, F32>(p, stream);
  return p.cache.dtype == AFFON_ROCM_BF16 ? append_typed<F32, BF16>(p, stream) : append_typed<F32, F32>(p, stream);
}

hipError_t commit_launch(const PagedCache& cache, const DraftBatch& batch, const uint32_t* path, int64_t path_stride,
                         int path_columns, const uint32_t* accepted, hipStream_t stream) {
  const int line_pieces = cache.head_dim * (cache.dtype == AFFON_ROCM_BF16 ? 2 : 4) / 16;
  const int64_t units = static_cast<int64_t>(cache.layers) * batch.sequences * 2 * cache.kv_heads * line_pieces;
  const int64_t blocks = (units + 255) / 256;
  if (blocks > kMaxBlocks) return hipErrorInvalidValue;
  hipLaunchKernelGGL(commit_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, cache, batch, path,
                     path_stride, path_columns, accepted);
  return hipGetLastError();
}

}  // namespace affon
