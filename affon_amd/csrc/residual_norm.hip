// The norms before and after a block, with its gate and residual scale:
//   u = update, or update / sqrt(mean(update^2) + epsilon) * post_weight,
//   x = stream + scale * gate * u  (stored as the stream),
//   normalized = x / sqrt(mean(x^2) + epsilon) * weight,
// in f32, each result rounded once. Bound by memory: a row is read once and
// held in registers between its two sums (longer ones are read again).

#include <algorithm>
#include <type_traits>

#include "device.h"
#include "internal.h"

namespace affon {
namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
// Rows start at any element; memory takes 16-byte accesses there.
typedef u32x4_t u32x4_word_t __attribute__((aligned(4)));
typedef u32x4_t u32x4_half_t __attribute__((aligned(2)));

constexpr int kChunk = 8;  // consecutive values of a thread

// Values at .. at + 7 of a row of cols, of either type; past its end 0.
__device__ __forceinline__ void load_chunk(const void* row, bool half, int64_t at, int64_t cols, float (&v)[kChunk]) {
  const auto* base = static_cast<const uint8_t*>(row);
  if (at + kChunk <= cols) {
    if (half) {
      const u32x4_t raw = *reinterpret_cast<const u32x4_half_t*>(base + at * 2);
#pragma unroll
      for (int e = 0; e < kChunk; ++e) v[e] = __uint_as_float(e % 2 ? raw[e / 2] & 0xffff0000u : raw[e / 2] << 16);
    } else {
      const u32x4_t a = *reinterpret_cast<const u32x4_word_t*>(base + at * 4);
      const u32x4_t b = *reinterpret_cast<const u32x4_word_t*>(base + at * 4 + 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = __uint_as_float(a[e]);
        v[4 + e] = __uint_as_float(b[e]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < kChunk; ++e)
      v[e] = at + e >= cols ? 0.0f : half ? BF16::load(base, at + e) : F32::load(base, at + e);
  }
}

__device__ __forceinline__ void store_chunk(void* row, bool half, int64_t at, int64_t cols, const float (&v)[kChunk]) {
  auto* base = static_cast<uint8_t*>(row);
  if (at + kChunk <= cols) {
    if (half) {
      u32x4_t raw;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        raw[e] = f32_to_bf16_bits(v[2 * e]) | static_cast<uint32_t>(f32_to_bf16_bits(v[2 * e + 1])) << 16;
      *reinterpret_cast<u32x4_half_t*>(base + at * 2) = raw;
    } else {
      u32x4_t a, b;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = __float_as_uint(v[e]);
        b[e] = __float_as_uint(v[4 + e]);
      }
      *reinterpret_cast<u32x4_word_t*>(base + at * 4) = a;
      *reinterpret_cast<u32x4_word_t*>(base + at * 4 + 16) = b;
    }
  } else {
#pragma unroll
    for (int e = 0; e < kChunk; ++e) {
      if (at + e >= cols) continue;
      if (half)
        reinterpret_cast<uint16_t*>(base)[at + e] = f32_to_bf16_bits(v[e]);
      else
        reinterpret_cast<float*>(base)[at + e] = v[e];
    }
  }
}

// The sum over a workgroup of THREADS, in every thread; `part` is not used again before a barrier.
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* part) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) v += __shfl_xor(v, offset);
  if constexpr (THREADS > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < THREADS / 64; ++i) v += part[i];
  }
  return v;
}

// A row's pointers.
struct Row {
  const void *stream, *update, *gate;
  void *stream_out, *normalized;
};
__device__ __forceinline__ const uint8_t* at_row(const void* base, int64_t row, int64_t stride, bool half) {
  return static_cast<const uint8_t*>(base) + row * stride * (half ? 2 : 4);
}

struct NormArgs {
  affon_rocm_residual_norm_desc d;
  bool stream_half, update_half, gate_half, weight_half, normalized_half;
};

__device__ __forceinline__ Row row_of(const NormArgs& a, int64_t row) {
  Row r;
  r.stream = at_row(a.d.stream, row, a.d.stream_stride, a.stream_half);
  r.update = a.d.update == nullptr ? nullptr : at_row(a.d.update, row, a.d.update_stride, a.update_half);
  r.gate = a.d.gate == nullptr ? nullptr : at_row(a.d.gate, row, a.d.gate_stride, a.gate_half);
  r.stream_out = const_cast<uint8_t*>(at_row(a.d.stream_out, row, a.d.stream_out_stride, a.stream_half));
  r.normalized = const_cast<uint8_t*>(at_row(a.d.normalized, row, a.d.normalized_stride, a.normalized_half));
  return r;
}

// x of a chunk, from the stream's values x and the update's u: `inverse` is
// that of the update's norm.
__device__ __forceinline__ void add_update(const NormArgs& a, const Row& r, int64_t at, float inverse,
                                           const float (&u)[kChunk], float (&x)[kChunk]) {
  float f[kChunk];
#pragma unroll
  for (int e = 0; e < kChunk; ++e) f[e] = u[e];
  if (a.d.post_norm) {
#pragma unroll
    for (int e = 0; e < kChunk; ++e) f[e] *= inverse;
    if (a.d.post_weight != nullptr) {
      float w[kChunk];
      load_chunk(a.d.post_weight, a.weight_half, at, a.d.cols, w);
#pragma unroll
      for (int e = 0; e < kChunk; ++e) f[e] *= w[e];
    }
  }
  if (r.gate != nullptr) {
    float g[kChunk];
    load_chunk(r.gate, a.gate_half, at, a.d.cols, g);
#pragma unroll
    for (int e = 0; e < kChunk; ++e) f[e] *= g[e];
  }
#pragma unroll
  for (int e = 0; e < kChunk; ++e) x[e] = fmaf(a.d.scale, f[e], x[e]);
}

__device__ __forceinline__ void write_normalized(const NormArgs& a, const Row& r, int64_t at, float inverse,
                                                 float (&x)[kChunk]) {
#pragma unroll
  for (int e = 0; e < kChunk; ++e) x[e] *= inverse;
  if (a.d.weight != nullptr) {
    float w[kChunk];
    load_chunk(a.d.weight, a.weight_half, at, a.d.cols, w);
#pragma unroll
    for (int e = 0; e < kChunk; ++e) x[e] *= w[e];
  }
  store_chunk(r.normalized, a.normalized_half, at, a.d.cols, x);
}

__device__ __forceinline__ float inverse_norm(const NormArgs& a, float squares) {
  return 1.0f / sqrtf(squares / static_cast<float>(a.d.cols) + a.d.epsilon);
}

// Rows that THREADS threads hold, HELD chunks each.
template <int THREADS, int HELD>
__global__ __launch_bounds__(THREADS) void held_kernel(NormArgs a) {
  __shared__ float part[2][THREADS / 64];
  const Row r = row_of(a, blockIdx.x);
  const int64_t cols = a.d.cols;
  float x[HELD][kChunk], u[HELD][kChunk];
#pragma unroll
  for (int j = 0; j < HELD; ++j) load_chunk(r.stream, a.stream_half, (threadIdx.x + j * THREADS) * kChunk, cols, x[j]);
  if (r.update != nullptr) {
#pragma unroll
    for (int j = 0; j < HELD; ++j) load_chunk(r.update, a.update_half, (threadIdx.x + j * THREADS) * kChunk, cols, u[j]);
    float inverse = 1.0f;
    if (a.d.post_norm) {
      float squares = 0.0f;
#pragma unroll
      for (int j = 0; j < HELD; ++j)
#pragma unroll
        for (int e = 0; e < kChunk; ++e) squares = fmaf(u[j][e], u[j][e], squares);
      inverse = inverse_norm(a, block_sum<THREADS>(squares, part[0]));
    }
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      const int64_t at = (threadIdx.x + j * THREADS) * kChunk;
      add_update(a, r, at, inverse, u[j], x[j]);
      store_chunk(r.stream_out, a.stream_half, at, cols, x[j]);
    }
  } else if (a.d.stream_out != nullptr) {
#pragma unroll
    for (int j = 0; j < HELD; ++j)
      store_chunk(r.stream_out, a.stream_half, (threadIdx.x + j * THREADS) * kChunk, cols, x[j]);
  }
  float squares = 0.0f;
#pragma unroll
  for (int j = 0; j < HELD; ++j)
#pragma unroll
    for (int e = 0; e < kChunk; ++e) squares = fmaf(x[j][e], x[j][e], squares);
  const float inverse = inverse_norm(a, block_sum<THREADS>(squares, part[1]));
#pragma unroll
  for (int j = 0; j < HELD; ++j) write_normalized(a, r, (threadIdx.x + j * THREADS) * kChunk, inverse, x[j]);
}

// Longer rows: every pass reads the row again, from the caches. The stream is
// written in the last one, so that it may be the stream that is read.
constexpr int kLongThreads = 1024;
__global__ __launch_bounds__(kLongThreads) void long_kernel(NormArgs a) {
  __shared__ float part[2][kLongThreads / 64];
  const Row r = row_of(a, blockIdx.x);
  const int64_t cols = a.d.cols;
  float inverse = 1.0f;
  if (a.d.post_norm) {
    float squares = 0.0f;
    for (int64_t at = threadIdx.x * kChunk; at < cols; at += kLongThreads * kChunk) {
      float u[kChunk];
      load_chunk(r.update, a.update_half, at, cols, u);
#pragma unroll
      for (int e = 0; e < kChunk; ++e) squares = fmaf(u[e], u[e], squares);
    }
    inverse = inverse_norm(a, block_sum<kLongThreads>(squares, part[0]));
  }
  auto summed = [&](int64_t at, float (&x)[kChunk]) {
    load_chunk(r.stream, a.stream_half, at, cols, x);
    if (r.update == nullptr) return;
    float u[kChunk];
    load_chunk(r.update, a.update_half, at, cols, u);
    add_update(a, r, at, inverse, u, x);
  };
  float squares = 0.0f;
  for (int64_t at = threadIdx.x * kChunk; at < cols; at += kLongThreads * kChunk) {
    float x[kChunk];
    summed(at, x);
#pragma unroll
    for (int e = 0; e < kChunk; ++e) squares = fmaf(x[e], x[e], squares);
  }
  const float last = inverse_norm(a, block_sum<kLongThreads>(squares, part[1]));
  for (int64_t at = threadIdx.x * kChunk; at < cols; at += kLongThreads * kChunk) {
    float x[kChunk];
    summed(at, x);
    if (a.d.stream_out != nullptr) store_chunk(r.stream_out, a.stream_half, at, cols, x);
    write_normalized(a, r, at, last, x);
  }
}

template <int N>
using Int = std::integral_constant<int, N>;
constexpr int64_t kManyRows = 512;  // two workgroups to a CU

template <int THREADS, int HELD>
void launch_held(const NormArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((held_kernel<THREADS, HELD>), dim3(static_cast<unsigned>(a.d.rows)), dim3(THREADS), 0, stream, a);
}

}  // namespace

namespace {

void launch_rows(const affon_rocm_residual_norm_desc& d, hipStream_t stream) {
  const NormArgs a{d,
                   d.stream_dtype == AFFON_ROCM_BF16,
                   d.update_dtype == AFFON_ROCM_BF16,
                   d.gate_dtype == AFFON_ROCM_BF16,
                   d.weight_dtype == AFFON_ROCM_BF16,
                   d.normalized_dtype == AFFON_ROCM_BF16};
  const int64_t chunks = (d.cols + kChunk - 1) / kChunk;
  // Few rows want a thread for every chunk; many, two chunks to a thread,
  // whose loads are all in flight (2048 x 8192 f32 with a gate: 53.1 us in 512
  // threads of two, 59.3 in 1024 of one, 58.5 in 256 of four).
  const bool many = d.rows >= kManyRows;
  auto by_rows = [&](auto threads) {
    constexpr int kThreads = decltype(threads)::value;
    if (many)
      launch_held<kThreads / 2, 2>(a, stream);
    else
      launch_held<kThreads, 1>(a, stream);
  };
  if (chunks <= 64)
    launch_held<64, 1>(a, stream);
  else if (chunks <= 128)
    by_rows(Int<128>{});
  else if (chunks <= 256)
    by_rows(Int<256>{});
  else if (chunks <= 512)
    by_rows(Int<512>{});
  else if (chunks <= 1024)
    by_rows(Int<1024>{});
  else if (chunks <= 2048)
    launch_held<1024, 2>(a, stream);
  else
    hipLaunchKernelGGL(long_kernel, dim3(static_cast<unsigned>(d.rows)), dim3(kLongThreads), 0, stream, a);
}

}  // namespace

// A workgroup a row, and as many rows as a grid holds to a launch (a loop over
// rows in the kernel: 2048 x 8192 f32 with a gate 78 us against 53).
hipError_t residual_norm_launch(const affon_rocm_residual_norm_desc& d, hipStream_t stream) {
  constexpr int64_t kMaxGrid = int64_t(1) << 20;
  auto skip = [](const void* base, int64_t rows, int64_t stride, int dtype) {
    return base == nullptr ? nullptr
                           : const_cast<uint8_t*>(static_cast<const uint8_t*>(base)) +
                                 rows * stride * (dtype == AFFON_ROCM_BF16 ? 2 : 4);
  };
  for (int64_t row = 0; row < d.rows; row += kMaxGrid) {
    affon_rocm_residual_norm_desc part = d;
    part.rows = std::min(kMaxGrid, d.rows - row);
    part.stream = skip(d.stream, row, d.stream_stride, d.stream_dtype);
    part.update = skip(d.update, row, d.update_stride, d.update_dtype);
    part.gate = skip(d.gate, row, d.gate_stride, d.gate_dtype);
    part.stream_out = skip(d.stream_out, row, d.stream_out_stride, d.stream_dtype);
    part.normalized = skip(d.normalized, row, d.normalized_stride, d.normalized_dtype);
    launch_rows(part, stream);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace affon
