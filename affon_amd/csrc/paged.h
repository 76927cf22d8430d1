// Where a paged cache keeps the tokens of a sequence, as the kernels over it
// see it.
#pragma once

#include "device.h"
#include "internal.h"

namespace affon {

// Tokens of sequence b that are committed (at most what its table holds), and
// its drafted tokens in use.
__device__ __forceinline__ uint32_t committed(const DraftBatch& batch, int b) {
  return min(batch.lengths[b], batch.capacity);
}
__device__ __forceinline__ uint32_t drafted(const DraftBatch& batch, int b) {
  const uint32_t rows = static_cast<uint32_t>(batch.rows);
  return batch.counts != nullptr ? min(batch.counts[b], rows) : rows;
}

// Workgroups of up to 256 threads that a launch takes: 2^32 threads.
constexpr int64_t kMaxBlocks = (int64_t(1) << 24) - 1;

constexpr uint32_t kNoPage = 0xffffffffu;

// The page that holds page `index` of sequence b, or kNoPage.
__device__ __forceinline__ uint32_t page_of(const PagedCache& cache, const DraftBatch& batch, int b, uint32_t index) {
  const uint32_t page = batch.table[b * batch.table_stride + index];
  return page < static_cast<uint32_t>(cache.pages) ? page : kNoPage;
}

// Line of token n of sequence b among the lines [page, head, page_size] of
// head 0 of a layer, or -1 where it lies nowhere. Head h is h * page_size
// lines further.
__device__ __forceinline__ int64_t line_of(const PagedCache& cache, const DraftBatch& batch, int b, uint32_t n) {
  if (n >= batch.capacity) return -1;
  const uint32_t size = static_cast<uint32_t>(cache.page_size);
  const uint32_t index = n / size, page = page_of(cache, batch, b, index);
  if (page == kNoPage) return -1;
  return static_cast<int64_t>(page) * cache.kv_heads * size + (n - index * size);
}

}  // namespace affon
