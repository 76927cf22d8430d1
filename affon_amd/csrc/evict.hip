// Eviction: of each row (layer, sequence, key head) the `recent` last tokens
// stay, and of the others those of the largest weights, ties to the lowest
// index; they move up in their order, keys and values in their pages.
//
// One launch selects (a workgroup a row: the threshold by its digits, then the
// tokens that stay as bits, and their weights in place), another moves.

#include <algorithm>

#include "lds_pipeline.h"
#include "paged.h"

namespace affon {
namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

struct EvictArgs {
  PagedCache cache;
  DraftBatch batch;
  const float* weights;  // [layer][sequence][key head][capacity]
  float* out;
  const uint32_t* keep;
  const uint32_t* recent;
  uint64_t* kept;  // bit n % 64 of word n / 64 of a row: token n stays
  int words;       // of a row
};

// Tokens of a sequence, and how many of them stay.
struct Plan {
  uint32_t length, left, recent;
  __device__ __forceinline__ Plan(const EvictArgs& a, int b) {
    length = committed(a.batch, b);
    left = min(a.keep[b], length);
    recent = min(a.recent[b], left);
  }
};

// In the order of the weights; 0s are equal, and a NaN is below all.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kThreads = 1024, kWaves = kThreads / 64;

// A pass over a digit counts the keys that share the digits before in as many
// bins as the digit has values; the bin that the `wanted`-th largest lies in ends
// the search where all of it stays, which two of the three passes mostly find. A
// row's first 4096 weights stay in registers meanwhile. What bounds it is this
// chain of passes, each between barriers, and not memory: 2048 rows of up to
// 4096 weights 34 us, 8 rows 6.8 (with three passes always, reading the weights
// in each, and sums over lanes through LDS 53 and 9). Two or four sets of bins
// for neighbouring lanes, whose additions to one bin wait for each other, take
// as long as one.
constexpr int kDeepWindow = 4;  // tokens of a thread in a window
constexpr uint32_t kSelectWindow = kDeepWindow * kThreads;

__global__ __launch_bounds__(kThreads) void select_kernel(EvictArgs a) {
  __shared__ uint32_t bins[2048];
  __shared__ uint32_t counts[64];  // of each wave and part of a window
  __shared__ uint32_t found_bin, found_above, found_count;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = blockIdx.x;
  const int b = static_cast<int>(row / a.cache.kv_heads % a.batch.sequences);
  const float* w = a.weights + row * a.batch.capacity;
  float* out = a.out + row * a.batch.capacity;
  float first[kDeepWindow];  // of the first window, on their way beside the plan
#pragma unroll
  for (int j = 0; j < kDeepWindow; ++j) first[j] = w[min(j * kThreads + threadIdx.x, a.batch.capacity - 1)];
  const Plan plan(a, b);
  const uint32_t others = plan.length - plan.recent;  // that stay by their weight
  const uint32_t wanted = plan.left - plan.recent;

  // The `wanted`-th largest of the others, digit by digit from the highest.
  uint32_t threshold = 0, ties = 0;  // the first `ties` of those equal to it stay
  uint32_t least = 0xffffffffu;      // and all from here on
  if (plan.left < plan.length && wanted > 0) {
    uint32_t left = wanted;
    const int shifts[3] = {21, 10, 0}, widths[3] = {11, 11, 10};
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = shifts[pass];
      const uint32_t size = 1u << widths[pass], high = pass == 0 ? 0u : ~0u << shifts[pass - 1];
      for (uint32_t i = threadIdx.x; i < size; i += kThreads) bins[i] = 0;
      __syncthreads();
      auto count = [&](float weight) {
        const uint32_t key = order_of(weight);
        if ((key & high) == threshold) atomicAdd(&bins[key >> shift & (size - 1)], 1u);
      };
#pragma unroll
      for (int j = 0; j < kDeepWindow; ++j)
        if (j * kThreads + threadIdx.x < others) count(first[j]);
      for (uint32_t n = kSelectWindow + threadIdx.x; n < others; n += kThreads) count(w[n]);
      __syncthreads();
      // Sums from the highest bin down: thread i has bins 2i and 2i + 1 of the reversed order.
      const uint32_t per = size / kThreads;  // 2 or 1
      uint32_t mine[2] = {0, 0};
      for (uint32_t j = 0; j < per; ++j) mine[j] = bins[size - 1 - (threadIdx.x * per + j)];
      const uint32_t sum = scanned(mine[0] + mine[1]);
      if (lane == 63) counts[wave] = sum;
      __syncthreads();
      uint32_t above = sum - mine[0] - mine[1] + lane_of(scanned(lane < wave ? counts[lane] : 0u), 63);
      for (uint32_t j = 0; j < per; ++j) {
        if (above < left && above + mine[j] >= left) {
          found_bin = size - 1 - (threadIdx.x * per + j);
          found_above = above;
          found_count = mine[j];
        }
        above += mine[j];
      }
      __syncthreads();
      threshold |= found_bin << shift;
      left -= found_above;
      if (left == found_count) {
        least = threshold;
        left = 0;
        break;
      }
    }
    ties = left;
    if (ties > 0) least = threshold + 1;
  }

  // Windows of four parts of 1024 tokens.
  uint32_t before = 0, ties_before = 0;  // tokens that stay, and equal ones
  for (uint32_t window = 0; window < plan.length; window += kSelectWindow) {
    float v[kDeepWindow];
    uint32_t equal = 0, stays = 0;
    uint64_t ballots[kDeepWindow];
#pragma unroll
    for (int j = 0; j < kDeepWindow; ++j) {
      const uint32_t n = window + j * kThreads + threadIdx.x;
      v[j] = window == 0 ? first[j] : n < plan.length ? w[n] : 0.0f;
      const uint32_t key = order_of(v[j]);
      if (n < others && plan.left < plan.length) {
        if (key >= least) stays |= 1u << j;
        if (ties > 0 && key == threshold) equal |= 1u << j;
      } else if (n < plan.length) {
        stays |= 1u << j;
      }
      ballots[j] = __ballot(equal >> j & 1);
      if (lane == 0) counts[j * kWaves + wave] = __popcll(ballots[j]);
    }
    __syncthreads();
    // Sums over the parts and waves before, in the tokens' order.
    auto scan = [&](uint32_t* total) {
      const uint32_t own = counts[lane], sum = scanned(own);
      *total = lane_of(sum, 63);
      return sum - own;
    };
    const uint64_t below = (uint64_t(1) << lane) - 1;
    uint32_t total;
    uint32_t base = scan(&total);
#pragma unroll
    for (int j = 0; j < kDeepWindow; ++j) {
      const uint32_t rank = ties_before + lane_of(base, j * kWaves + wave) + __popcll(ballots[j] & below);
      if ((equal >> j & 1) && rank < ties) stays |= 1u << j;
    }
    ties_before += total;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kDeepWindow; ++j) {
      ballots[j] = __ballot(stays >> j & 1);
      if (lane == 0) {
        counts[j * kWaves + wave] = __popcll(ballots[j]);
        const uint32_t word = window / 64 + j * kWaves + wave;
        if (word < static_cast<uint32_t>(a.words)) a.kept[row * a.words + word] = ballots[j];
      }
    }
    __syncthreads();
    base = scan(&total);
#pragma unroll
    for (int j = 0; j < kDeepWindow; ++j) {
      // Where out is the weights themselves: this window has been read, and no token moves down.
      const uint32_t to = before + lane_of(base, j * kWaves + wave) + __popcll(ballots[j] & below);
      if (stays >> j & 1) out[to] = v[j];
    }
    before += total;
    __syncthreads();
  }
  for (uint32_t n = plan.left + threadIdx.x; n < a.batch.capacity; n += kThreads) out[n] = 0.0f;
}

// A workgroup moves 2^lanes_log pieces of 16 bytes of every line of a row, keys or
// values, as many lines at a time as its threads hold eight pieces of: all of
// them are read before one is written, and a line is written only after every
// line of its place or before has been read. Memory bounds it: 2048 rows of up to
// 4096 tokens cut to 1024 (bf16, heads of 128) 445 us, 4.8 TB/s. (Accesses that
// leave no lines in the caches took 15 us less there, but 3 more of 16 for 8 rows
// of up to 2000.) However few tokens go, all that lies behind the first of them moves: 32
// layers of 8 sequences of 4096 cut by the one of least weight 536 us (the whole
// call), by 16 of them 1118, by 256 1131.
constexpr int kMoveThreads = 256, kDeep = 8;
constexpr uint32_t kWindow = 4096;

__global__ __launch_bounds__(kMoveThreads) void move_kernel(EvictArgs a, int parts, int lanes_log, uint32_t per_page) {
  __shared__ uint16_t list[kWindow];  // sources, from the window's first token on
  __shared__ uint32_t starts[64];
  __shared__ uint32_t in_window;
  // Pages of the window's tokens and of their new places: looked up beside the
  // lines' own loads, they kept every chunk waiting (8 sequences of up to 4096
  // tokens, 32 layers: 836 us, against 482 without any lookup).
  __shared__ uint32_t pages[2][kWindow / 16 + 1];
  // Parts of a line at workgroups as far apart as there are rows: mostly on one
  // XCD, whose L2 then holds the line for them.
  const int64_t each = static_cast<int64_t>(gridDim.x) / parts, id = blockIdx.x % each;
  const int part = static_cast<int>(blockIdx.x / each);
  const bool is_value = id % 2 != 0;
  const int64_t row = id / 2;
  const int kv = static_cast<int>(row % a.cache.kv_heads);
  const int64_t above = row / a.cache.kv_heads;
  const int b = static_cast<int>(above % a.batch.sequences);
  const int64_t layer = above / a.batch.sequences;
  const Plan plan(a, b);
  if (plan.left == plan.length) return;
  const int line_pieces = a.cache.head_dim * (a.cache.dtype == AFFON_ROCM_BF16 ? 2 : 4) / 16;
  const int piece = (part << lanes_log) + (threadIdx.x & ((1 << lanes_log) - 1));
  const uint32_t lines = kMoveThreads >> lanes_log, line_of_thread = threadIdx.x >> lanes_log;
  const bool works = piece < line_pieces;
  auto* data = reinterpret_cast<u32x4_t*>((is_value ? a.cache.values : a.cache.keys) + layer * a.cache.layer_bytes);
  const int64_t head_lines = static_cast<int64_t>(kv) * a.cache.page_size;
  const uint64_t* kept = a.kept + row * a.words;
  const uint32_t size = static_cast<uint32_t>(a.cache.page_size);
  // Line of the token that lies `at` tokens after the start of the page whose number is list[0]; -1: nowhere.
  auto line_at = [&](const uint32_t* list, uint32_t at) {
    const uint32_t index = static_cast<uint32_t>(static_cast<uint64_t>(at / 16) * per_page >> 31), page = list[index];
    return page < static_cast<uint32_t>(a.cache.pages)
               ? static_cast<int64_t>(page) * a.cache.kv_heads * size + (at - index * size) : -1;
  };
  uint32_t before = 0;  // tokens that stay before the window
  for (uint32_t window = 0; window < plan.length && before < plan.left; window += kWindow) {
    // The window's tokens that stay, in their order.
    const uint32_t word = threadIdx.x / 4;
    const uint64_t bits = window / 64 + word < static_cast<uint32_t>(a.words) && window + word * 64 < plan.length
                              ? kept[window / 64 + word] : 0;
    if (threadIdx.x % 4 == 0) starts[word] = __popcll(bits);
    __syncthreads();
    if (threadIdx.x < 64) {
      const uint32_t own = starts[threadIdx.x], sum = scanned(own);
      starts[threadIdx.x] = sum - own;
      if (threadIdx.x == 63) in_window = sum;
    }
    __syncthreads();
    const uint32_t shift = threadIdx.x % 4 * 16;
    uint32_t to = starts[word] + __popcll(bits & ((uint64_t(1) << shift) - 1));
    for (uint32_t i = shift; i < shift + 16; ++i)
      if (bits >> i & 1) list[to++] = static_cast<uint16_t>(word * 64 + i);
    const uint32_t total = in_window;
    const uint32_t first_page[2] = {window / size, before / size};
    const uint32_t last_token[2] = {min(window + kWindow, plan.length) - 1, before + (total > 0 ? total - 1 : 0)};
    for (int k = 0; k < 2; ++k)
      for (uint32_t j = first_page[k] + threadIdx.x; j <= last_token[k] / size; j += kMoveThreads)
        pages[k][j - first_page[k]] = a.batch.table[b * a.batch.table_stride + j];
    __syncthreads();
    const uint32_t window_phase = window - first_page[0] * size, before_phase = before - first_page[1] * size;
    for (uint32_t i0 = 0; i0 < total; i0 += lines * kDeep) {
      u32x4_t v[kDeep];
      int64_t place[kDeep];
#pragma unroll
      for (int j = 0; j < kDeep; ++j) {
        const uint32_t i = i0 + j * lines + line_of_thread;
        place[j] = -1;
        if (!works || i >= total) continue;
        if (window + list[i] == before + i) continue;
        const int64_t from = line_at(pages[0], window_phase + list[i]), line = line_at(pages[1], before_phase + i);
        if (from < 0 || line < 0) continue;
        place[j] = (line + head_lines) * line_pieces + piece;
        v[j] = data[(from + head_lines) * line_pieces + piece];
      }
      pipeline::wait_vmcnt<0>();
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kDeep; ++j)
        if (place[j] >= 0) data[place[j]] = v[j];
    }
    before += total;
    __syncthreads();  // the list is free
  }
}

}  // namespace

hipError_t evict_launch(const PagedCache& cache, const DraftBatch& batch, const float* weights, float* out,
                        const uint32_t* keep, const uint32_t* recent, const Launch& l) {
  EvictArgs a{cache, batch, weights, out, keep, recent, nullptr, static_cast<int>((batch.capacity + 63) / 64)};
  const int64_t rows = static_cast<int64_t>(cache.layers) * batch.sequences * cache.kv_heads;
  const int line_pieces = cache.head_dim * (cache.dtype == AFFON_ROCM_BF16 ? 2 : 4) / 16;
  // Whole lines, or parts of them side by side until there are two workgroups for
  // every CU: 8 rows of up to 2000 tokens cut to 1024 (bf16, heads of 128) take 15.7 us
  // with 512 of them, 16.5 with 128, 19.5 with 64 and 25.8 with 32; 2048 rows
  // of up to 4096 by whole lines 479, quarters of them 875.
  int lanes_log = 0;
  while ((1 << lanes_log) < line_pieces && lanes_log < 6) ++lanes_log;
  while (lanes_log > 0 && rows * 2 * ((line_pieces + (1 << lanes_log) - 1) >> lanes_log) < 512) --lanes_log;
  const int parts = (line_pieces + (1 << lanes_log) - 1) >> lanes_log;
  // t * per_page >> 31 is t / (page_size / 16), for the t up to 4351 of a window and a page.
  const uint32_t unit = static_cast<uint32_t>(cache.page_size / 16), per_page = ((uint32_t(1) << 31) + unit - 1) / unit;
  if (rows * 2 * parts > kMaxBlocks / (kThreads / 256)) return hipErrorInvalidValue;
  a.kept = static_cast<uint64_t*>(l.scratch(static_cast<size_t>(rows) * a.words * sizeof(uint64_t)));
  if (a.kept == nullptr) return hipErrorOutOfMemory;
  hipLaunchKernelGGL(select_kernel, dim3(static_cast<unsigned>(rows)), dim3(kThreads), 0, l.stream, a);
  hipLaunchKernelGGL(move_kernel, dim3(static_cast<unsigned>(rows * 2 * parts)), dim3(kMoveThreads), 0, l.stream, a, parts,
                     lanes_log, per_page);
  return hipGetLastError();
}

namespace {

// The weights of accepted tokens follow them: a thread for each layer,
// sequence and key head, eight at a time as the path ascends. The other
// drafted tokens' places have gathered nothing. 8192 rows of 24 drafted tokens, 6
// of them accepted: 8 us of the commit's 20 (a launch more: 8.5 against 5.2 for 8 rows).
__global__ __launch_bounds__(256) void commit_weights_kernel(DraftBatch batch, int64_t total, int kv_heads, float* weights,
                                                             const uint32_t* path, int64_t path_stride, int path_columns,
                                                             const uint32_t* accepted) {
  constexpr int kMoves = 8;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (row >= total) return;
  const int b = static_cast<int>(row / kv_heads % batch.sequences);
  const uint32_t length = batch.lengths[b];
  if (length >= batch.capacity) return;
  float* w = weights + row * batch.capacity + length;
  const uint32_t room = min(batch.capacity - length, static_cast<uint32_t>(batch.rows));
  const uint32_t count = min(min(accepted[b], static_cast<uint32_t>(path_columns)), room);
  for (uint32_t i0 = 0; i0 < count; i0 += kMoves) {
    float v[kMoves];
#pragma unroll
    for (int j = 0; j < kMoves; ++j) {
      const uint32_t i = min(i0 + j, count - 1), from = path[b * path_stride + i];
      v[j] = from < room ? w[from] : w[i];
    }
#pragma unroll
    for (int j = 0; j < kMoves; ++j)
      if (i0 + j < count) w[i0 + j] = v[j];
  }
  for (uint32_t i = count; i < room; ++i) w[i] = 0.0f;
}

}  // namespace

hipError_t commit_weights_launch(const DraftBatch& batch, int layers, int kv_heads, float* weights, const uint32_t* path,
                                 int64_t path_stride, int path_columns, const uint32_t* accepted, hipStream_t stream) {
  const int64_t total = static_cast<int64_t>(layers) * batch.sequences * kv_heads;
  const int64_t blocks = (total + 255) / 256;
  if (blocks > kMaxBlocks) return hipErrorInvalidValue;
  hipLaunchKernelGGL(commit_weights_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, batch, total,
                     kv_heads, weights, path, path_stride, path_columns, accepted);
  return hipGetLastError();
}

namespace {

__global__ __launch_bounds__(256) void clear_weights_kernel(float* weights, int64_t count) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += static_cast<int64_t>(gridDim.x) * 256)
    weights[i] = 0.0f;
}

}  // namespace

hipError_t clear_weights_launch(float* weights, int64_t count, hipStream_t stream) {
  const int64_t blocks = std::min<int64_t>((count + 255) / 256, 4096);
  hipLaunchKernelGGL(clear_weights_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, weights, count);
  return hipGetLastError();
}

}  // namespace affon
