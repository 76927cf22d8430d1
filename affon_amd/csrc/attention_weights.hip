// The attention weights that the tokens of a cache gather: for each key head
// and token, the sum of its probabilities over the rows and query heads that
// share the key head.
//
// A row's probabilities need its largest score and the sum of its exponentials
// first, so the scores are computed twice: once for these two (stats_kernel,
// queries in registers, keys walked over), and once for the sums over the rows
// (gather_kernel, keys in registers, rows walked over). Both products are
// S^T = K Q^T on the matrix cores: lane % 16 is a row, and a lane's four results
// are keys 4 (lane / 16) .. + 3 of a tile of 16.

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "attention.h"

namespace affon {
namespace attention {
namespace {

struct WeightArgs {
  AttentionProblem p;
  int group;         // query heads per key head
  int rows;          // T * group
  int row_groups;    // workgroups of stats_kernel that share a piece's keys
  uint32_t unit;     // keys of a piece, at least
  int splits;        // pieces of a context, at most
  float log2_scale;  // |scale| * log2(e)
  float sign;        // of the scale: a factor of the queries
  float2* stats;     // (m, l) [unit][split][row]
  float2* ready;     // (m, 1 / l) [unit][row]; 1 / l = 0: the row takes no part
  float* weights;    // of the layer, [sequence][key head][capacity]
  int blocks;        // workgroups of gather_kernel along a context
};

// What a sequence holds, and where this workgroup's piece of it lies.
struct Context {
  uint32_t length, count, n;
  __device__ __forceinline__ Context(const AttentionProblem& p, int b) {
    length = committed(p.batch, b);
    count = drafted(p.batch, b);
    n = min(length + count, p.batch.capacity);
  }
};

// T: element type; KS: 64-byte pieces of a head, at most.
template <typename T, int KS>
struct Tiles {
  static constexpr bool kHalf = T::bytes == 2;

  // Rows r0 + lane % 16 of a sequence as an operand: dims past the head and
  // rows not in use are 0, and the scale's sign is theirs.
  static __device__ __forceinline__ void load_rows(const WeightArgs& a, int b, int kv, uint32_t count, int r0,
                                                   u32x4_t (&q)[KS]) {
    const AttentionProblem& p = a.p;
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int row_bytes = p.cache.head_dim * T::bytes;
    const int r = min(r0 + col, a.rows - 1), t = r / a.group;
    const uint8_t* from = p.query + ((static_cast<int64_t>(b) * p.batch.rows + t) * p.query_stride +
                                     static_cast<int64_t>(kv * a.group + r - t * a.group) * p.cache.head_dim) * T::bytes;
    const bool aligned = (reinterpret_cast<uintptr_t>(p.query) | static_cast<uintptr_t>(p.query_stride * T::bytes)) % 16 == 0;
    const uint32_t flip = a.sign < 0.0f ? (kHalf ? 0x80008000u : 0x80000000u) : 0u;
    const bool used = r0 + col < a.rows && t < static_cast<int>(count) && a.sign != 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const uint8_t* piece = from + min(s * 64 + quad * 16, row_bytes - 16);
      if (aligned) {
        q[s] = *reinterpret_cast<const u32x4_t*>(piece);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (kHalf) {
            const auto* h = reinterpret_cast<const uint16_t*>(piece) + 2 * e;
            q[s][e] = h[0] | static_cast<uint32_t>(h[1]) << 16;
          } else {
            q[s][e] = reinterpret_cast<const uint32_t*>(piece)[e];
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) q[s][e] = used && s * 64 + quad * 16 < row_bytes ? q[s][e] ^ flip : 0u;
    }
  }

  // The 16 keys at `tile` as an operand.
  static __device__ __forceinline__ void load_keys(const WeightArgs& a, const uint8_t* tile, u32x4_t (&k)[KS]) {
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int row_bytes = a.p.cache.head_dim * T::bytes;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      k[s] = *reinterpret_cast<const u32x4_t*>(tile + col * row_bytes + min(s * 64 + quad * 16, row_bytes - 16));
  }

  static __device__ __forceinline__ f32x4_t scores(const WeightArgs& a, const u32x4_t (&k)[KS], const u32x4_t (&q)[KS]) {
    const int quad = (threadIdx.x & 63) >> 4, row_bytes = a.p.cache.head_dim * T::bytes;
    f32x4_t s{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      // Past the head: zeros, as the queries hold there.
      const u32x4_t ki = i * 64 + quad * 16 < row_bytes ? k[i] : u32x4_t{0, 0, 0, 0};
      if constexpr (kHalf) {
        s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, ki), __builtin_bit_cast(bf16x8_t, q[i]), s,
                                                    0, 0, 0);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t ke = ki[e], qe = q[i][e];
          s = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(ke), __uint_as_float(qe), s, 0, 0, 0);
        }
      }
    }
    return s;
  }

  // Address of the tile that starts at token `at` of sequence b; *there: it
  // lies somewhere (else some tile's, to be loaded and not looked at).
  static __device__ __forceinline__ const uint8_t* tile_of(const WeightArgs& a, int kv, uint32_t page, uint32_t at, bool* there) {
    const PagedCache& c = a.p.cache;
    *there = page < static_cast<uint32_t>(c.pages);
    const int64_t line = (static_cast<int64_t>(*there ? page : 0) * c.kv_heads + kv) * c.page_size + at % c.page_size;
    return c.keys + line * c.head_dim * T::bytes;
  }

  // Bits of the 16 keys from `at` on that row t of the sequence sees.
  static __device__ __forceinline__ uint32_t seen(const WeightArgs& a, const Context& c, int b, int t, uint32_t at) {
    return seen_bits(a.p, static_cast<int64_t>(b) * a.p.batch.rows + t, t, static_cast<int>(at) - static_cast<int>(c.length),
                     static_cast<int>(c.n) - static_cast<int>(c.length));
  }
};

// Four waves side by side over the keys of a piece, 16 rows each.
template <typename T, int KS>
__global__ __launch_bounds__(256) void stats_kernel(WeightArgs a) {
  using Ops = Tiles<T, KS>;
  constexpr int KT = KS <= 8 ? 2 : 1;  // tiles of a step
  const AttentionProblem& p = a.p;
  __shared__ float2 parts[4][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  int id = blockIdx.x;
  const int rg = id % a.row_groups;
  id /= a.row_groups;
  const int split = id % a.splits, unit = id / a.splits;
  const int b = unit / p.cache.kv_heads, kv = unit - b * p.cache.kv_heads;
  const Context c(p, b);
  const uint32_t chunk = piece_of(c.n, a.splits, a.unit), begin = split * chunk;
  if (begin >= c.n) return;
  const uint32_t end = min(begin + chunk, c.n);
  const uint32_t sub = ((end - begin + 3) / 4 + 31) / 32 * 32;
  const uint32_t first = min(begin + wave * sub, end), last = min(first + sub, end);

  u32x4_t q[KS];
  Ops::load_rows(a, b, kv, c.count, rg * 16, q);
  const int t = min(rg * 16 + col, a.rows - 1) / a.group;
  float m = kLowest, l = 0.0f;

  uint32_t list = kNoPage;  // of 64 tiles, a lane each
  u32x4_t keys[2][KT][KS];
  bool there[2][KT];
  auto load = [&](uint32_t at, auto place) {
    constexpr int to = decltype(place)::value;
    if ((at - first) % 1024 == 0) {
      const uint32_t mine = at + lane * 16;
      list = mine < last ? page_of(p.cache, p.batch, b, mine / p.cache.page_size) : kNoPage;
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const uint32_t page = __builtin_amdgcn_readlane(static_cast<int>(list), (at - first) / 16 % 64 + kt);
      Ops::load_keys(a, Ops::tile_of(a, kv, page, at + 16 * kt, &there[to][kt]), keys[to][kt]);
    }
  };
  auto take = [&](uint32_t at, auto place) {
    constexpr int from = decltype(place)::value;
    f32x4_t s[KT];
    float top = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      s[kt] = Ops::scores(a, keys[from][kt], q);
      const uint32_t key0 = at + 16 * kt;
      if (!there[from][kt] || key0 + 16 > c.length) {
        const uint32_t seen = there[from][kt] ? Ops::seen(a, c, b, t, key0) : 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(seen >> (4 * quad + i) & 1)) s[kt][i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, s[kt][i]);
    }
    top *= a.log2_scale;
    if (__any(top > m + kSlack)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(fmaxf(top, __shfl_xor(top, 32)), m);
      l *= __builtin_amdgcn_exp2f(m - top);
      m = top;
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) l += __builtin_amdgcn_exp2f(fmaf(s[kt][i], a.log2_scale, -m));
  };
  constexpr uint32_t kStep = 16 * KT;
  if (first < last) load(first, std::integral_constant<int, 0>{});
  for (uint32_t at = first; at < last; at += 2 * kStep) {
    if (at + kStep < last) load(at + kStep, std::integral_constant<int, 1>{});
    take(at, std::integral_constant<int, 0>{});
    if (at + kStep >= last) break;
    if (at + 2 * kStep < last) load(at + 2 * kStep, std::integral_constant<int, 0>{});
    take(at + kStep, std::integral_constant<int, 1>{});
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (quad == 0) parts[wave][col] = float2{m, l};
  __syncthreads();
  const int r = rg * 16 + static_cast<int>(threadIdx.x);
  if (threadIdx.x >= 16 || r >= a.rows) return;
  float top = kLowest, sum = 0.0f;
  for (int w = 0; w < 4; ++w) top = fmaxf(top, parts[w][threadIdx.x].x);
  for (int w = 0; w < 4; ++w) sum = fmaf(parts[w][threadIdx.x].y, __builtin_amdgcn_exp2f(parts[w][threadIdx.x].x - top), sum);
  a.stats[(static_cast<int64_t>(unit) * a.splits + split) * a.rows + r] = float2{top, sum};
}

// Joins the pieces of a row: a thread each.
__global__ __launch_bounds__(256) void ready_kernel(WeightArgs a, int64_t total) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;
  const int64_t unit = i / a.rows;
  const int r = static_cast<int>(i - unit * a.rows);
  const Context c(a.p, static_cast<int>(unit / a.p.cache.kv_heads));
  const uint32_t used = c.n == 0 ? 0u : (c.n + piece_of(c.n, a.splits, a.unit) - 1) / piece_of(c.n, a.splits, a.unit);
  float m = kLowest, l = 0.0f;
  for (uint32_t s = 0; s < used; ++s) {
    const float2 st = a.stats[(unit * a.splits + s) * a.rows + r];
    const float top = fmaxf(m, st.x);
    l = fmaf(st.y, __builtin_amdgcn_exp2f(st.x - top), l * __builtin_amdgcn_exp2f(m - top));
    m = top;
  }
  const bool none = l == 0.0f || r / a.group >= static_cast<int>(c.count);
  a.ready[i] = float2{m, none ? 0.0f : 1.0f / l};
}

// Four waves side by side over the keys, KT tiles each, all rows one after the other.
template <typename T, int KS>
__global__ __launch_bounds__(256) void gather_kernel(WeightArgs a) {
  using Ops = Tiles<T, KS>;
  constexpr int KT = KS <= 4 ? 4 : KS <= 8 ? 2 : 1;
  constexpr uint32_t kKeys = 16 * KT;
  const AttentionProblem& p = a.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int unit = blockIdx.x / a.blocks, block = blockIdx.x % a.blocks;
  const int b = unit / p.cache.kv_heads, kv = unit - b * p.cache.kv_heads;
  const Context c(p, b);
  if (c.count == 0) return;
  for (uint32_t at = (block * 4 + wave) * kKeys; at < c.n; at += a.blocks * 4 * kKeys) {
    u32x4_t keys[KT][KS];
    bool there[KT], all = at + kKeys <= c.length;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const uint32_t key0 = at + 16 * kt;
      const uint32_t page = key0 < c.n ? page_of(p.cache, p.batch, b, key0 / p.cache.page_size) : kNoPage;
      Ops::load_keys(a, Ops::tile_of(a, kv, page, key0, &there[kt]), keys[kt]);
      all = all && there[kt];
    }
    f32x4_t sums[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) sums[kt] = f32x4_t{0, 0, 0, 0};
    for (int r0 = 0; r0 < a.rows; r0 += 16) {
      const int r = min(r0 + col, a.rows - 1);
      const float2 ready = a.ready[static_cast<int64_t>(unit) * a.rows + r];
      const float inverse = r0 + col < a.rows ? ready.y : 0.0f;
      u32x4_t q[KS];
      Ops::load_rows(a, b, kv, c.count, r0, q);
      f32x4_t s[KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) s[kt] = Ops::scores(a, keys[kt], q);
      const bool edge = !all || __any(inverse == 0.0f);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const uint32_t seen = !edge ? ~0u : !there[kt] || inverse == 0.0f ? 0u : Ops::seen(a, c, b, r / a.group, at + 16 * kt);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(fmaf(s[kt][i], a.log2_scale, -ready.x)) * inverse;
          sums[kt][i] += seen >> (4 * quad + i) & 1 ? e : 0.0f;
        }
      }
    }
    float* to = a.weights + static_cast<int64_t>(unit) * p.batch.capacity;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v = sums[kt][i];
#pragma unroll
        for (int offset = 1; offset < 16; offset <<= 1) v += __shfl_xor(v, offset);
        const uint32_t n = at + 16 * kt + 4 * quad + i;
        if (col == i && n < c.n) to[n] = n < c.length ? to[n] + v : v;
      }
  }
}

template <typename T, int KS>
hipError_t launch(const WeightArgs& a, int64_t units, hipStream_t stream) {
  const int64_t stats_blocks = units * a.splits * a.row_groups, total = units * a.rows;
  if (stats_blocks > kMaxBlocks || (total + 255) / 256 > kMaxBlocks || units * a.blocks > kMaxBlocks)
    return hipErrorInvalidValue;
  hipLaunchKernelGGL((stats_kernel<T, KS>), dim3(static_cast<unsigned>(stats_blocks)), dim3(256), 0, stream, a);
  hipLaunchKernelGGL(ready_kernel, dim3(static_cast<unsigned>((total + 255) / 256)), dim3(256), 0, stream, a, total);
  hipLaunchKernelGGL((gather_kernel<T, KS>), dim3(static_cast<unsigned>(units * a.blocks)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace
}  // namespace attention

hipError_t attention_weights_launch(const AttentionProblem& p, float* weights, const Launch& l) {
  using namespace attention;
  WeightArgs a{};
  a.p = p;
  a.group = p.heads / p.cache.kv_heads;
  const int64_t rows = static_cast<int64_t>(p.batch.rows) * a.group;
  if (rows > (int64_t(1) << 30)) return hipErrorInvalidValue;
  a.rows = static_cast<int>(rows);
  a.row_groups = (a.rows + 15) / 16;
  a.log2_scale = p.scale == 0.0f ? 1.0f : std::min(std::fabs(p.scale) * 1.44269504088896340736f, FLT_MAX);
  a.sign = p.scale > 0.0f ? 1.0f : p.scale < 0.0f ? -1.0f : 0.0f;
  a.weights = weights;
  const int64_t units = static_cast<int64_t>(p.batch.sequences) * p.cache.kv_heads;
  const int64_t capacity = p.batch.capacity;
  a.unit = 256;
  a.splits = static_cast<int>(std::max<int64_t>(1, std::min(1024 / (units * a.row_groups), capacity / a.unit)));
  a.blocks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(2048 / units, (capacity + 63) / 64)));
  const size_t stats = static_cast<size_t>(units) * a.splits * a.rows * sizeof(float2);
  const size_t ready = static_cast<size_t>(units) * a.rows * sizeof(float2);
  auto* scratch = static_cast<uint8_t*>(l.scratch(stats + ready));
  if (scratch == nullptr) return hipErrorOutOfMemory;
  a.stats = reinterpret_cast<float2*>(scratch);
  a.ready = reinterpret_cast<float2*>(scratch + stats);
  const int pieces = (p.cache.head_dim * (p.cache.dtype == AFFON_ROCM_BF16 ? 2 : 4) + 63) / 64;
  if (p.cache.dtype == AFFON_ROCM_BF16) {
    if (pieces <= 2) return launch<BF16, 2>(a, units, l.stream);
    if (pieces <= 3) return launch<BF16, 3>(a, units, l.stream);
    if (pieces <= 4) return launch<BF16, 4>(a, units, l.stream);
    if (pieces <= 6) return launch<BF16, 6>(a, units, l.stream);
    return launch<BF16, 8>(a, units, l.stream);
  }
  if (pieces <= 4) return launch<F32, 4>(a, units, l.stream);
  if (pieces <= 6) return launch<F32, 6>(a, units, l.stream);
  if (pieces <= 8) return launch<F32, 8>(a, units, l.stream);
  if (pieces <= 12) return launch<F32, 12>(a, units, l.stream);
  return launch<F32, 16>(a, units, l.stream);
}

}  // namespace affon
