// Attention of drafted tokens over a paged cache on the matrix cores.
//
// The query heads that share a key head, G of them, and the T drafted tokens
// of a sequence make T*G rows over the same keys and values. A wave holds 16
// or 32 of these rows and walks over keys 32 (bf16) or 16 (f32) at a time:
//   S^T = K Q^T      (MFMA, rows of the queries as columns of the result),
//   P = e^(S - m)    (one running reference m per row),
//   O^T += V^T P^T   (MFMA).
// Both products leave a query row in the column lane % 16 of a result, so a
// row's m and sum are plain per-lane values, and P^T leaves the first product
// in the lanes in which the second one takes it: lane group lane / 16 holds
// keys 4 (lane / 16) .. + 3 of each 16, and the order of the keys inside a
// product is free as long as V^T is read in the same one.
//
// What bounds it (one MI355X, head width 128, bf16): few rows, the memory (32
// sequences of one token over up to 4096: 68 us, 5.0 TB/s of keys and
// values, where a large copy reaches 5.2); many rows, the instructions around
// the products (trees of 64 of 16 sequences over up to 16384, 512 rows to a
// key head: 424 to 437 us with the join, 750 to 770 TFLOP/s; a large library
// product reaches 1272). There the matrix cores are busy a third of the time:
// without the softmax's exponentials 10% goes, without the products as much,
// without the transfers 20%, and no one of them alone is the limit. Tried
// there, us: four row tiles a wave instead of two 552 (a wave to a SIMD), one
// 516 to 582 in three or four waves, and the two tiles' products and softmax in
// turns within a wave 459, all against 447 at the time; a wave priority for
// either 434 to 443 against 437 to 442.
//
// m follows the largest score only where a score passes it by more than
// kSlack: e^(S - m) then stays below 2^kSlack, the sums and O are in f32 and
// a later m only scales them, so that most steps neither reduce across lanes
// nor touch O.
//
// Keys and values reach LDS by direct transfers, a step ahead; 16
// keys of one head and page are consecutive in memory, and every transfer
// moves whole 1 KiB pieces of them. LDS keeps their order, its 16-byte pieces
// permuted inside each row where the row is a power of two long (the banks
// would otherwise meet): the permutation is made by the source addresses.
// bf16 values are read transposed (ds_read_b64_tr_b16).
#pragma once

#include "lds_pipeline.h"
#include "paged.h"

namespace affon {
namespace attention {

using pipeline::bf16x8_t;
using pipeline::dma16;
using pipeline::f32x4_t;
using pipeline::lds_address;
using pipeline::pack_bf16;
using pipeline::u32x4_t;
using pipeline::wait_lds_reads;
using pipeline::wait_vmcnt;
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4_t* lds_s16x4;

struct Args {
  AttentionProblem p;
  int group;        // query heads per key head
  int rows;         // T * group
  int row_groups;   // workgroups that share a sequence's rows
  uint32_t chunk;   // keys of a workgroup, a multiple of kKeysAhead
  int splits;       // workgroups along the keys
  float log2_scale; // |scale| * log2(e)
  float sign;       // of the scale: a factor of the queries
  // splits > 1: sums [unit][split][row][head_dim] and (m, l) [unit][split][row],
  // unit = sequence * kv_heads + key head, row_slots rows each.
  float* sums;
  float* stats;
  int row_slots;
  // One per unit and row group, 0 between calls: the workgroup that raises it
  // to the number of splits in use joins their results. Null: a second launch does.
  uint32_t* tickets;
  // Of a call over shared prefixes (part 1 or 2): `per` sequences to a group,
  // shared[group] tokens of each in the same pages.
  const uint32_t* shared;
  int per;
  // Its prefixes cut over all groups (by the tiles' kernels): of each group the
  // number of its first piece and the pieces that each key head has, for the join.
  uint2* plan;
};

// A call over shared prefixes: the part of its own keys, and what is another one's in
// the part of the prefixes.
struct Parts : Args {
  int groups, group_rows;  // sequences and their drafted tokens there
  int prefix_rows, prefix_row_groups, prefix_splits, prefix_slots;
  uint32_t prefix_chunk;   // the least keys of a piece: both parts are cut on the device
  float *prefix_sums, *prefix_stats;
  uint2* prefix_plan;  // or null: each group is cut by itself
  unsigned prefix_blocks;  // workgroups of a launch that take prefixes, before the others
  __host__ __device__ Args prefix() const {
    Args a = *this;
    a.p.batch.sequences = groups;
    a.p.batch.rows = group_rows;
    a.p.mask = nullptr;
    a.rows = prefix_rows;
    a.row_groups = prefix_row_groups;
    a.splits = prefix_splits;
    a.row_slots = prefix_slots;
    a.chunk = prefix_chunk;
    a.sums = prefix_sums;
    a.stats = prefix_stats;
    a.plan = prefix_plan;
    return a;
  }
};

// Keys that a launch takes: all of a sequence; or, by its workgroups, the prefixes
// that the sequences of a group share, whose rows are then the rows of one
// sequence (p.batch: groups for sequences), and what each has after its prefix.
enum Keys { kAllKeys = 0, kParts = 1 };

// Tokens of a prefix that are taken once for its group: whole steps of every
// kernel, so that the own tokens start at one too. The rest is each sequence's own.
constexpr uint32_t kPrefixUnit = 64;
__device__ __forceinline__ uint32_t prefix_tokens(const Args& a, const DraftBatch& batch, int group) {
  return min(a.shared[group], batch.capacity) / kPrefixUnit * kPrefixUnit;
}
// Whether sequence b holds the prefix of its group.
__device__ __forceinline__ bool takes_prefix(const Args& a, const DraftBatch& batch, int b, int group) {
  return batch.lengths[b] >= a.shared[group] && drafted(batch, b) > 0;
}
// The first sequence of a group that does, whose pages are read for all; -1: none. For whole waves.
__device__ __forceinline__ int prefix_holder(const Args& a, int group) {
  const int lane = threadIdx.x & 63;
  DraftBatch batch = a.p.batch;  // of the sequences themselves
  batch.rows /= a.per;
  for (int i = 0; i < a.per; i += 64) {
    const int b = group * a.per + min(i + lane, a.per - 1);
    const uint64_t held = __ballot(takes_prefix(a, batch, b, group));
    if (held != 0) return group * a.per + min(i + __builtin_ctzll(held), a.per - 1);
  }
  return -1;
}
// Keys of a piece where n keys are cut into at most `splits` of them.
__device__ __forceinline__ uint32_t piece_of(uint32_t n, int splits, uint32_t unit) {
  const uint32_t each = (n + splits - 1) / splits;
  return max(unit, (each + unit - 1) / unit * unit);
}

constexpr float kSlack = 8.0f;
constexpr float kLowest = -3.0e38f;  // m before the first score
constexpr int kPageList = 256;       // pages of 16-key tiles that a workgroup holds

// A value the compiler keeps in a register instead of computing it again.
__device__ __forceinline__ int pinned(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// A wave's address in scalar registers, as the transfers take it.
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t low = __builtin_amdgcn_readfirstlane(static_cast<int>(v));
  const uint32_t high = __builtin_amdgcn_readfirstlane(static_cast<int>(v >> 32));
  return reinterpret_cast<const uint8_t*>(static_cast<uint64_t>(high) << 32 | low);
}

// A bf16 word holds an infinity or a NaN in its low or high half.
__device__ __forceinline__ bool not_finite(uint32_t w, bool half) {
  if (half) return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
  return (w & 0x7f800000u) == 0x7f800000u;
}

// Bits of a row's mask for keys base .. base + 31 of the drafted tokens (base
// may be negative: committed ones, all seen); none from count on.
__device__ __forceinline__ uint32_t seen_bits(const AttentionProblem& p, int64_t row, int t, int base, int count) {
  uint32_t bits;
  if (p.mask == nullptr) {
    const int ones = t + 1 - base;
    bits = ones >= 32 ? ~0u : ones <= 0 ? 0u : (1u << ones) - 1;
  } else {
    const uint32_t* words = p.mask + row * p.mask_stride;
    const int last = (p.batch.rows - 1) / 32;
    if (base >= 0) {
      const int w = base / 32, shift = base % 32;
      const uint32_t low = w <= last ? words[w] : 0u, high = w + 1 <= last ? words[w + 1] : 0u;
      bits = __funnelshift_r(low, high, shift);
    } else {
      bits = base <= -32 ? ~0u : words[0] << -base | ((1u << -base) - 1);
    }
  }
  const int left = count - base;
  if (left < 32) bits &= left <= 0 ? 0u : (1u << left) - 1;
  return bits;
}

// Results of one split, which a workgroup on another XCD may join: stored past
// this XCD's L2 and loaded past the reader's (relaxed accesses of agent scope),
// so that neither side has to write back or drop a whole cache: with fences
// instead, 32 sequences of one token each over up to 4160 tokens took 197 us
// in five splits, against 76 in two launches.
__device__ __forceinline__ void store_shared(float* to, float a, float b) {
  const uint64_t v = __float_as_uint(a) | static_cast<uint64_t>(__float_as_uint(b)) << 32;
  __hip_atomic_store(reinterpret_cast<uint64_t*>(to), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_shared(const float* from) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(from), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return float2{__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32))};
}

// Values at .. at + 3 of the result: sums over their probabilities' sum (0: nothing was seen).
template <typename T>
__device__ __forceinline__ void store_result(uint8_t* out, int64_t at, f32x4_t v, float sum) {
  v = sum == 0.0f ? f32x4_t{0, 0, 0, 0} : v * (1.0f / sum);
  if constexpr (T::bytes == 2) {
    const u32x2_t h{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
    if (reinterpret_cast<uintptr_t>(out) % 8 == 0) {
      *reinterpret_cast<u32x2_t*>(out + at * 2) = h;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        reinterpret_cast<uint16_t*>(out)[at + e] = static_cast<uint16_t>(e % 2 ? h[e / 2] >> 16 : h[e / 2]);
    }
  } else if (reinterpret_cast<uintptr_t>(out) % 16 == 0) {
    *reinterpret_cast<f32x4_t*>(out + at * 4) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) reinterpret_cast<float*>(out)[at + e] = v[e];
  }
}

// sum_s 2^(m_s - m) sums_s, d .. d + 3, over the splits s = first, first + step,
// .. below `used` of the row whose slot in split 0 is `slot`, with *max = m the
// largest m_s and *sum = sum_s 2^(m_s - m) l_s. kAtOnce
// splits are loaded together: their time is the memory's latency (one by one,
// the 63 splits of one sequence of 32000 tokens took 40 us).
template <bool SHARED>
__device__ __forceinline__ f32x4_t joined_sums(const Args& a, int64_t slot, int d, int D, uint32_t first, uint32_t used,
                                               uint32_t step, float* max, float* sum) {
  constexpr int kAtOnce = 8;
  float top = kLowest, l = 0.0f;
  f32x4_t v{0, 0, 0, 0};
  for (uint32_t s0 = first; s0 < used; s0 += kAtOnce * step) {
    float2 st[kAtOnce];
    f32x4_t part[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int64_t at = slot + static_cast<int64_t>(min(s0 + i * step, used - 1)) * a.row_slots;
      if constexpr (SHARED) {
        st[i] = load_shared(a.stats + 2 * at);
        const float2 low = load_shared(a.sums + at * D + d), high = load_shared(a.sums + at * D + d + 2);
        part[i] = f32x4_t{low.x, low.y, high.x, high.y};
      } else {
        st[i] = *reinterpret_cast<const float2*>(a.stats + 2 * at);
        part[i] = *reinterpret_cast<const f32x4_t*>(a.sums + at * D + d);
      }
    }
    float peak = top;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) peak = fmaxf(peak, st[i].x);
    const float keep = __builtin_amdgcn_exp2f(top - peak);
    top = peak;
    l *= keep;
    v *= keep;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (s0 + i * step >= used) break;
      const float w = __builtin_amdgcn_exp2f(st[i].x - top);
      l = fmaf(st[i].y, w, l);
      v += part[i] * w;
    }
  }
  *max = top;
  *sum = l;
  return v;
}

// T: element type; DT: 16-wide tiles of the head (an even number in bf16); EXACT: the
// head is 16 * DT wide, 64, 128 or 256, else at most that; RT: 16-row tiles
// of a wave; WR: waves side by side over the rows, sharing the keys in LDS;
// WK: waves side by side over the keys, each with its own; STAGES: steps in LDS.
template <typename T, int DT, bool EXACT, int RT, int WR, int WK, int STAGES, int KEYS>
struct Kernel {
  static constexpr bool kHalf = T::bytes == 2;
  static constexpr int kKT = kHalf ? 2 : 1;  // 16-key tiles of a step
  static constexpr int kKeys = 16 * kKT;
  static constexpr int kThreads = 64 * WR * WK;
  static constexpr int kWavesPerSimd = DT <= 8 ? 2 : 1;  // that share the registers
  static constexpr int kMaxRow = 16 * DT * T::bytes;             // bytes of a head
  static constexpr int kTile = (16 * kMaxRow + 1023) / 1024 * 1024;  // LDS bytes of 16 keys
  static constexpr int kPieces = kTile / 1024;
  static constexpr int kStage = 2 * kKT * kTile;
  static constexpr int kQSteps = kHalf ? DT / 2 : DT;  // 64-byte pieces of a head
  // Transfers of a wave and step: pieces p = wave, wave + WR, .. of the keys'
  // and the values' 2 * kPieces, each for every tile of the step.
  static constexpr int kPer = (2 * kPieces + WR - 1) / WR;
  static constexpr int kTransfers = kPer * kKT;
  static_assert(WR == 1 || WK == 1, "waves share keys or rows");
  static_assert(STAGES >= 2 && kTransfers * STAGES < 64, "transfers in flight");
  static constexpr int kRing = WK * STAGES * kStage;
  // The waves' sums, where they share rows: rows padded by 16 bytes.
  static constexpr int kJoinRow = 16 * DT + 4;
  static constexpr int kJoin = WK > 1 ? WK * RT * 16 * kJoinRow * 4 : 0;
  static constexpr int kLds = kRing > kJoin ? kRing : kJoin;

  // Offsets of a lane's reads that its permutation sets: the later ones follow
  // at whole multiples.
  static constexpr int kKeySpots = !EXACT ? 1 : kQSteps < 4 ? kQSteps : 4;
  static constexpr int kValueSpots = !EXACT ? 1 : kHalf ? (DT < 8 ? DT : 8) : 2;

  // Place of 16-byte piece c of key k's row, before the row's own offset.
  static __device__ __forceinline__ int key_swizzle(int k) { return !EXACT ? 0 : kMaxRow >= 256 ? (k & 15) : (k >> 1) & 7; }
  static __device__ __forceinline__ int value_swizzle(int k) {
    if (!EXACT) return 0;
    if (kHalf) return kMaxRow >= 256 ? 2 * (k & 7) : 2 * ((k >> 1) & 3);
    return (k >> 2 & 1) << 2;
  }

  // `block` of the launch; `shares`: it takes a prefix (KEYS = kParts).
  static __device__ void run(const Args& a, unsigned block, bool shares) {
    const AttentionProblem& p = a.p;
    const bool prefix = KEYS == kParts && shares;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kLds];
    __shared__ int64_t tile_list[kPageList];  // byte offsets of 16-key tiles in keys and values; 1: of no page
    __shared__ int missing;
    __shared__ float2 join_stats[WK > 1 ? WK * RT * 16 : 1];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int D = EXACT ? 16 * DT : p.cache.head_dim;
    const int row_bytes = D * T::bytes;

    // Workgroups b, b + 8, .. run on one XCD: those of the same keys follow
    // each other there, to find them in its L2.
    int id = block >> 3;
    const int rg = id % a.row_groups;
    id = id / a.row_groups * 8 + (block & 7);
    const int kv = id % p.cache.kv_heads;
    id /= p.cache.kv_heads;
    // The last pieces first: only the longest sequences have them, and a piece
    // that starts when the others end holds the whole call up.
    const int b = id % p.batch.sequences, split = a.splits - 1 - id / p.batch.sequences;
    if (split < 0) return;

    // The page list's first part, whose loads need not wait for the lengths.
    uint32_t start = static_cast<uint32_t>(split) * a.chunk;
    uint32_t early = kNoPage;
    if constexpr (KEYS == kAllKeys) {
      const uint32_t early_at = start + threadIdx.x * 16;
      if (early_at < p.batch.capacity) early = p.batch.table[b * p.batch.table_stride + early_at / p.cache.page_size];
    }

    uint32_t length, count, n, chunk = a.chunk;
    int table_row = b;
    if (prefix) {
      // All keys are committed, and all rows are done: those of sequences that
      // do not take the prefix are not read again.
      length = n = prefix_tokens(a, p.batch, b);
      count = static_cast<uint32_t>(p.batch.rows);
      if (n == 0) return;
      table_row = prefix_holder(a, b);
      if (table_row < 0) return;
      chunk = piece_of(n, a.splits, a.chunk);
      start = static_cast<uint32_t>(split) * chunk;
    } else {
      length = committed(p.batch, b);
      count = drafted(p.batch, b);
      n = min(length + count, p.batch.capacity);
      if constexpr (KEYS == kParts) {
        if (count == 0) return;  // zeros, without a look at its results
        const uint32_t first = takes_prefix(a, p.batch, b, b / a.per) ? prefix_tokens(a, p.batch, b / a.per) : 0u;
        chunk = piece_of(n - first, a.splits, a.chunk);
        start = first + static_cast<uint32_t>(split) * chunk;
      }
    }
    const uint32_t begin = min(start, n);
    const uint32_t end = split == a.splits - 1 ? n : min(begin + chunk, n);
    if (begin >= end && (split > 0 || prefix)) return;
    const uint32_t used = max(1u, (n + a.chunk - 1) / a.chunk);  // splits that hold keys
    const bool whole = KEYS == kAllKeys && (a.splits == 1 || used == 1);  // the result is this workgroup's

    // This wave's rows, as columns of its results.
    const int row0 = (rg * WR + (WR > 1 ? wave : 0)) * RT * 16;
    // Waves past the last row bring keys, and leave the rest out.
    const bool idle = KEYS == kParts && WR > 1 && row0 >= a.rows;
    const uint8_t* queries = p.query + static_cast<int64_t>(b) * p.batch.rows * p.query_stride * T::bytes;
    const bool aligned = (reinterpret_cast<uintptr_t>(p.query) | static_cast<uintptr_t>(p.query_stride * T::bytes)) % 16 == 0;
    u32x4_t q[RT][kQSteps];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      // Rows past the last one and dims past the head load what lies before them.
      const int r = min(row0 + rt * 16 + col, a.rows - 1), t = r / a.group;
      const uint8_t* from = queries + (t * p.query_stride + static_cast<int64_t>(kv * a.group + r - t * a.group) * D) * T::bytes;
#pragma unroll
      for (int s = 0; s < kQSteps; ++s) {
        const uint8_t* piece = from + min(s * 64 + quad * 16, row_bytes - 16);
        if (aligned) {
          q[rt][s] = *reinterpret_cast<const u32x4_t*>(piece);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (kHalf) {
              const auto* h = reinterpret_cast<const uint16_t*>(piece) + 2 * e;
              q[rt][s][e] = h[0] | static_cast<uint32_t>(h[1]) << 16;
            } else {
              q[rt][s][e] = reinterpret_cast<const uint32_t*>(piece)[e];
            }
          }
        }
      }
    }
    f32x4_t o[RT][DT];
    float m[RT], l[RT];

    // Dims past the head are 0, and the scale's sign is theirs. So are rows not
    // in use: a NaN there would leave sums that are not finite (below).
    auto place_queries = [&] {
      const uint32_t flip = a.sign < 0.0f ? (kHalf ? 0x80008000u : 0x80000000u) : 0u;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const bool used = min(row0 + rt * 16 + col, a.rows - 1) / a.group < static_cast<int>(count);
        const uint32_t keep = a.sign == 0.0f || !used ? 0u : ~0u;
#pragma unroll
        for (int s = 0; s < kQSteps; ++s)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            q[rt][s][e] = !EXACT && s * 64 + quad * 16 >= row_bytes ? 0u : (q[rt][s][e] & keep) ^ flip;
      }
    };

    // Transfers: where this lane's 16 bytes of every piece come from.
    uint32_t from[kPer];
    const int first_piece = WR > 1 ? wave : 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int piece = min(first_piece + i * WR, 2 * kPieces - 1);
      const int at = (piece % kPieces) * 1024 + lane * 16;
      if constexpr (EXACT) {
        const int k = at / kMaxRow, c = at % kMaxRow / 16;
        from[i] = k * kMaxRow + (c ^ (piece >= kPieces ? value_swizzle(k) : key_swizzle(k))) * 16;
      } else {
        from[i] = min(at, 16 * row_bytes - 16);  // rows that are shorter end before the tile does
      }
    }
    // Where this lane reads the step's keys and values, from the step's place
    // in LDS on; pinned, so that the loop adds one base to them.
    int key_at[kKeySpots], value_at[kValueSpots];
#pragma unroll
    for (int i = 0; i < kKeySpots; ++i) key_at[i] = pinned(col * row_bytes + ((i * 4 + quad) ^ key_swizzle(col)) * 16);
#pragma unroll
    for (int i = 0; i < kValueSpots; ++i) {
      if constexpr (kHalf) {
        // Lanes 4e .. 4e + 3 of 16 address key 4 * quad + e; lane j gets column j of the four.
        const int k = 4 * quad + (col >> 2);
        value_at[i] = pinned(k * row_bytes + ((2 * i + ((col & 3) >> 1)) ^ value_swizzle(k)) * 16 + (col & 1) * 8);
      } else {
        const int k = 4 * quad;
        value_at[i] = pinned(k * row_bytes + ((4 * i + (col >> 2)) ^ value_swizzle(k)) * 16 + (col & 3) * 4);
      }
    }
    const uint32_t ring = lds_address(lds) + (WK > 1 ? wave * STAGES * kStage : 0);
    const uint8_t* ring_data = lds + (WK > 1 ? wave * STAGES * kStage : 0);
    const int64_t head_bytes = static_cast<int64_t>(p.cache.page_size) * row_bytes;

    // A value that is not finite in a drafted token that some row does not see
    // would reach that row as 0 * infinity. Such values are rare, and leave
    // sums that are not finite: then, and only then, everything is done again
    // with a look at every drafted token's values (`careful`).
    bool careful = false;
  again:
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] = kLowest;
      l[rt] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4_t{0, 0, 0, 0};
    }
    for (uint32_t segment = begin; segment < end; segment += kPageList * 16) {
      const uint32_t segment_end = min(end, segment + kPageList * 16);
      __syncthreads();
      if (threadIdx.x == 0) missing = 0;
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < kPageList && segment + i * 16 < segment_end; i += kThreads) {
        const uint32_t at = segment + i * 16, index = at / p.cache.page_size;
        const uint32_t page = KEYS == kAllKeys && segment == begin && i < kThreads
                                  ? (early < static_cast<uint32_t>(p.cache.pages) ? early : kNoPage)
                                  : page_of(p.cache, p.batch, table_row, index);
        tile_list[i] = page == kNoPage ? 1
                                       : (static_cast<int64_t>(page) * p.cache.kv_heads + kv) * head_bytes +
                                             static_cast<int64_t>(at - index * p.cache.page_size) * row_bytes;
        if (page == kNoPage) missing = 1;
      }
      __syncthreads();
      if (segment == begin && !careful) place_queries();
      const bool gaps = __builtin_amdgcn_readfirstlane(missing) != 0;
      const int all = static_cast<int>((segment_end - segment + kKeys - 1) / kKeys);
      // Steps of this wave: first, first + stride, .. below all.
      const int first = WK > 1 ? wave : 0;
      const int steps = all > first ? (all - first + WK - 1) / WK : 0;

      // Byte offsets of a step's tiles. A tile past the last one repeats it:
      // the keys there are not seen.
      auto tile_offset = [&](int step, int kt) {
        const int tile = (first + step * WK) * kKT + kt, last = static_cast<int>((segment_end - segment - 1) / 16);
        return tile_list[min(tile, last)];
      };
      // Starts a step's transfers to a place in LDS.
      auto issue = [&](int place, const int64_t (&offsets)[kKT]) {
        const uint32_t to = ring + place * kStage;
#pragma unroll
        for (int kt = 0; kt < kKT; ++kt) {
          const uint32_t high = __builtin_amdgcn_readfirstlane(static_cast<int>(offsets[kt] >> 32));
          const uint32_t low = __builtin_amdgcn_readfirstlane(static_cast<int>(offsets[kt]));
          const int64_t at = static_cast<int64_t>(high) << 32 | (low & ~15u);
          const uint8_t* key_tile = uniform(p.cache.keys + at);
          const uint8_t* value_tile = uniform(p.cache.values + at);
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            const int piece = min(first_piece + i * WR, 2 * kPieces - 1);
            const bool value = kPieces % WR == 0 ? i >= kPieces / WR : piece >= kPieces;
            dma16(value ? value_tile : key_tile, from[i],
                  to + (value ? kKT * kTile : 0) + kt * kTile + (value ? piece - kPieces : piece) * 1024);
          }
        }
      };
      u32x4_t keys[kKT][kQSteps];
      auto read_keys = [&](int place) {
        const uint8_t* from_lds = ring_data + place * kStage;
#pragma unroll
        for (int kt = 0; kt < kKT; ++kt)
#pragma unroll
          for (int i = 0; i < kQSteps; ++i) {
            if constexpr (EXACT) {
              keys[kt][i] = *reinterpret_cast<const u32x4_t*>(from_lds + kt * kTile + key_at[i % kKeySpots] +
                                                              i / kKeySpots * kKeySpots * 64);
            } else {
              const int at = (i * 4 + quad) * 16;
              keys[kt][i] = *reinterpret_cast<const u32x4_t*>(from_lds + kt * kTile + col * row_bytes + min(at, row_bytes - 16));
            }
          }
      };
      f32x4_t s[RT][kKT];
      auto multiply_keys = [&] {
#pragma unroll
        for (int kt = 0; kt < kKT; ++kt)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[rt][kt] = f32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < kQSteps; ++i) {
#pragma unroll
          for (int kt = 0; kt < kKT; ++kt) {
            u32x4_t k = keys[kt][i];
            // Past the head: zeros, as the queries hold there.
            if (!EXACT && (i * 4 + quad) * 16 >= row_bytes) k = u32x4_t{0, 0, 0, 0};
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              if constexpr (kHalf) {
                s[rt][kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, k),
                                                                    __builtin_bit_cast(bf16x8_t, q[rt][i]), s[rt][kt], 0, 0, 0);
              } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint32_t ke = k[e], qe = q[rt][i][e];
                  s[rt][kt] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(ke), __uint_as_float(qe), s[rt][kt], 0, 0, 0);
                }
              }
            }
          }
        }
      };

      // A step's scores are computed at the end of the one before, so that its
      // keys come from LDS beside the values' products and both products follow
      // each other; its values come beside the softmax. A step's place in LDS
      // is free when its values are in registers.
#pragma unroll
      for (int i = 0; i < STAGES; ++i) {
        if (i >= steps) continue;
        int64_t offsets[kKT];
#pragma unroll
        for (int kt = 0; kt < kKT; ++kt) offsets[kt] = tile_offset(i, kt);
        issue(i, offsets);
      }
      if (steps >= STAGES)
        wait_vmcnt<(STAGES - 1) * kTransfers>();
      else
        wait_vmcnt<0>();
      if constexpr (WR > 1) __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (!idle) {
        read_keys(0);
        multiply_keys();
      }

      auto advance = [&](int step, auto place_of_step) {
        constexpr int place = decltype(place_of_step)::value;
        const uint8_t* values = ring_data + place * kStage + kKT * kTile;
        const uint32_t key0 = segment + static_cast<uint32_t>(first + step * WK) * kKeys;
        int64_t offsets[kKT];
#pragma unroll
        for (int kt = 0; kt < kKT; ++kt) offsets[kt] = tile_offset(step + STAGES, kt);

        // ---- steps with keys that not every row sees ----
        const bool edge = gaps || key0 + kKeys > length;
        uint32_t flagged = 0;
        uint32_t seen[RT];
        if (edge) {
          const int base = static_cast<int>(key0) - static_cast<int>(length);
          const int left = static_cast<int>(n) - static_cast<int>(length);  // drafted tokens that have a place
          uint32_t there = 0;  // bits of the step's keys that lie anywhere
#pragma unroll
          for (int kt = 0; kt < kKT; ++kt) {
            const int tile = static_cast<int>((key0 - segment) / 16) + kt;
            if (segment + tile * 16 < segment_end && __builtin_amdgcn_readfirstlane(static_cast<int>(tile_list[tile])) != 1)
              there |= 0xffffu << (16 * kt);
          }
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            const int t = min(row0 + rt * 16 + col, a.rows - 1) / a.group;
            seen[rt] = there & seen_bits(p, static_cast<int64_t>(b) * p.batch.rows + t, t, base, left);
#pragma unroll
            for (int kt = 0; kt < kKT; ++kt)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (!(seen[rt] >> (16 * kt + 4 * quad + i) & 1)) s[rt][kt][i] = -INFINITY;
          }
          // What lies in the slots of no token is cleared, as it may be
          // infinite too.
          const int past = static_cast<int>(n) - static_cast<int>(key0);
          const uint32_t exists = there & (past >= 32 ? ~0u : past <= 0 ? 0u : (1u << past) - 1);
          uint32_t clear = ~exists & (kKeys == 32 ? ~0u : 0xffffu);
          auto for_pieces = [&](auto&& f) {
#pragma unroll
            for (int kt = 0; kt < kKT; ++kt)
#pragma unroll
              for (int i = 0; i < kPieces; ++i) {
                const int at = i * 1024 + lane * 16;
                if (at < 16 * row_bytes) f(kt * 16 + at / row_bytes, const_cast<uint8_t*>(values) + kt * kTile + at);
              }
          };
          if (careful) {  // and so are values that are not finite, which are added by themselves
            const uint32_t all_see = base >= 0 ? 0u : base <= -32 ? ~0u : (1u << -base) - 1;
            uint32_t bad = 0;
            for_pieces([&](int k, uint8_t* piece) {
              const u32x4_t v = *reinterpret_cast<const u32x4_t*>(piece);
              if (not_finite(v[0], kHalf) || not_finite(v[1], kHalf) || not_finite(v[2], kHalf) || not_finite(v[3], kHalf))
                bad |= 1u << k;
            });
#pragma unroll
            for (int offset = 32; offset > 0; offset >>= 1) bad |= __shfl_xor(bad, offset);
            flagged = __builtin_amdgcn_readfirstlane(bad) & exists & ~all_see;
            clear |= flagged;
            if constexpr (WR > 1) __syncthreads();  // every wave has looked
          }
          if (clear != 0) {
            for_pieces([&](int k, uint8_t* piece) {
              if (clear >> k & 1) *reinterpret_cast<u32x4_t*>(piece) = u32x4_t{0, 0, 0, 0};
            });
            if constexpr (WR > 1)
              __syncthreads();
            else
              wait_lds_reads();
          }
        }

        if (idle) {
          wait_vmcnt<0>();
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          if (step + STAGES < steps) issue(place, offsets);
          return;
        }

        // ---- values, on the way beside the softmax ----
        using Value = typename std::conditional<kHalf, u32x4_t, f32x4_t>::type;  // eight keys, or four, of a column
        Value v[DT];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          if constexpr (kHalf) {
            const int off = value_at[dt % kValueSpots] + dt / kValueSpots * kValueSpots * 32;
            u32x2_t half[2];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
              const uint32_t address = lds_address(values + kt * kTile + (EXACT ? off : min(off, 16 * row_bytes - 8)));
              half[kt] = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                         reinterpret_cast<lds_s16x4>(static_cast<uintptr_t>(address))));
            }
            v[dt] = Value{half[0][0], half[0][1], half[1][0], half[1][1]};
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int off = value_at[dt % kValueSpots] + dt / kValueSpots * kValueSpots * 64 + i * row_bytes;
              v[dt][i] = *reinterpret_cast<const float*>(values + (EXACT ? off : min(off, 16 * row_bytes - 4)));
            }
          }
        }

        // ---- softmax ----
        u32x4_t packed[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          float top = fmaxf(fmaxf(s[rt][0][0], s[rt][0][1]), fmaxf(s[rt][0][2], s[rt][0][3]));
          if constexpr (kKT == 2)
            top = fmaxf(top, fmaxf(fmaxf(s[rt][kKT - 1][0], s[rt][kKT - 1][1]), fmaxf(s[rt][kKT - 1][2], s[rt][kKT - 1][3])));
          top *= a.log2_scale;
          if (__any(top > m[rt] + kSlack)) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(fmaxf(top, __shfl_xor(top, 32)), m[rt]);
            const float keep = __builtin_amdgcn_exp2f(m[rt] - top);
            m[rt] = top;
            l[rt] *= keep;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= keep;
          }
#pragma unroll
          for (int kt = 0; kt < kKT; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              s[rt][kt][i] = __builtin_amdgcn_exp2f(fmaf(s[rt][kt][i], a.log2_scale, -m[rt]));
              l[rt] += s[rt][kt][i];
            }
          // The matrix cores take bf16: each probability is rounded once for its
          // product, by 2^-8 at most; their sum l is of the unrounded ones, and O is
          // f32. Against 64 bits results are 1.1 to 1.4 times as far off as f32
          // throughout rounded at the end (2.2e-3 and 1.6e-3 of their norm, 32 heads
          // over 777 to 5000 tokens), a single head of one token up to 1.7 times.
          // Products with the rest as a second term take the factor to 1.0, and were
          // left out: 9.3 us against 8.8 for one token over 777, 41 and 38 for 32
          // over up to 4000 at width 80, 41.0 and 36.9 for 8 sequences of 12 tokens
          // over up to 8000.
          if constexpr (kHalf)
            packed[rt] = u32x4_t{pack_bf16(s[rt][0][0], s[rt][0][1]), pack_bf16(s[rt][0][2], s[rt][0][3]),
                                 pack_bf16(s[rt][kKT - 1][0], s[rt][kKT - 1][1]),
                                 pack_bf16(s[rt][kKT - 1][2], s[rt][kKT - 1][3])};
        }

        // ---- the next step's keys, and the step after whose place is free ----
        wait_lds_reads();
        if (step + STAGES <= steps)
          wait_vmcnt<(STAGES - 2) * kTransfers>();
        else
          wait_vmcnt<0>();
        if constexpr (WR > 1) __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (step + STAGES < steps) issue(place, offsets);
        read_keys((place + 1) % STAGES);  // after the last step: what lies there, for scores that nothing reads

        // ---- sums of values ----
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            if constexpr (kHalf) {
              o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v[dt]),
                                                                  __builtin_bit_cast(bf16x8_t, packed[rt]), o[rt][dt], 0, 0, 0);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[dt][i], s[rt][0][i], o[rt][dt], 0, 0, 0);
            }
          }

        if (flagged != 0) {  // rare: a drafted token's value that is not finite, for the rows that see it
          for (int k = 0; k < kKeys; ++k) {
            if (!(flagged >> k & 1)) continue;
            const int64_t line = line_of(p.cache, p.batch, b, key0 + k) + static_cast<int64_t>(kv) * p.cache.page_size;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              float e = 0.0f;
#pragma unroll
              for (int kt = 0; kt < kKT; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (k / 16 == kt && k % 4 == i) e = s[rt][kt][i];
              e = __shfl(e, (k % 16) / 4 * 16 + col);
              if (!(seen[rt] >> k & 1)) continue;
#pragma unroll
              for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int d = 16 * dt + 4 * quad + i;
                  if (d < D) o[rt][dt][i] = fmaf(e, T::load(p.cache.values, line * D + d), o[rt][dt][i]);
                }
            }
          }
        }
        multiply_keys();
      };
      // The places follow each other at fixed addresses.
      for (int step = 0; step < steps; step += STAGES)
        pipeline::Unroll<0, STAGES>::run([&](auto place) {
          if (step + place < steps) advance(step + place, place);
        });
      wait_lds_reads();
    }

    if (!prefix && end > length && !careful) {  // the drafted tokens are among the keys
      float odd = 0.0f;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) odd = fmaf(o[rt][dt][i], 0.0f, odd);  // 0, or NaN
      if (__syncthreads_or(odd != 0.0f || odd != odd)) {
        careful = true;
        goto again;
      }
    }

    // ---- results ----
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      l[rt] += __shfl_xor(l[rt], 16);
      l[rt] += __shfl_xor(l[rt], 32);
    }
    const int64_t unit = static_cast<int64_t>(b) * p.cache.kv_heads + kv;
    const int64_t part = (unit * a.splits + split) * a.row_slots;
    auto write_result = [&](int r, int d, f32x4_t v, float row_l) {
      const int t = r / a.group;
      const int64_t slot = (static_cast<int64_t>(b) * p.batch.rows + t) * p.heads + kv * a.group + r - t * a.group;
      store_result<T>(p.out, slot * D + d, v, t < static_cast<int>(count) ? row_l : 0.0f);
    };
    // Four values of a row, d .. d + 3: of the result, or of this split's sums.
    auto write = [&](int r, int d, f32x4_t v, float row_m, float row_l) {
      if (r >= a.rows || d >= D) return;
      if (whole) return write_result(r, d, v, row_l);
      float* to = a.sums + (part + r) * D + d;
      float* stats = a.stats + 2 * (part + r);
      if (a.tickets != nullptr) {
        store_shared(to, v[0], v[1]);
        store_shared(to + 2, v[2], v[3]);
        if (d == 0) store_shared(stats, row_m, row_l);
      } else {
        *reinterpret_cast<f32x4_t*>(to) = v;
        if (d == 0) *reinterpret_cast<float2*>(stats) = float2{row_m, row_l};
      }
    };
    if constexpr (WK == 1) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) write(row0 + rt * 16 + col, 16 * dt + 4 * quad, o[rt][dt], m[rt], l[rt]);
    } else {
      auto* joined = reinterpret_cast<float*>(lds);
      __syncthreads();  // the ring is free
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int r = wave * RT * 16 + rt * 16 + col;
        if (quad == 0) join_stats[r] = float2{m[rt], l[rt]};
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4_t*>(joined + r * kJoinRow + 16 * dt + 4 * quad) = o[rt][dt];
      }
      __syncthreads();
      const int pieces = D / 4;
      for (int i = threadIdx.x; i < RT * 16 * pieces; i += kThreads) {
        const int r = i / pieces, d = (i - r * pieces) * 4;
        if (row0 + r >= a.rows) break;
        float top = kLowest, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WK; ++w) top = fmaxf(top, join_stats[w * RT * 16 + r].x);
        f32x4_t v{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < WK; ++w) {
          const float2 st = join_stats[w * RT * 16 + r];
          const float keep = __builtin_amdgcn_exp2f(st.x - top);
          sum = fmaf(st.y, keep, sum);
          v += *reinterpret_cast<const f32x4_t*>(joined + (w * RT * 16 + r) * kJoinRow + d) * keep;
        }
        write(row0 + r, d, v, top, sum);
      }
    }
    if (whole || a.tickets == nullptr) return;

    // The last of the splits joins them, in their order whichever it is.
    __shared__ uint32_t arrived;
    wait_vmcnt<0>();  // this wave's results are past its L2
    __syncthreads();
    uint32_t* ticket = a.tickets + unit * a.row_groups + rg;
    if (threadIdx.x == 0) arrived = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (arrived + 1 != used) return;
    if (threadIdx.x == 0) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int first_row = rg * WR * RT * 16, pieces = D / 4;
    const int own_rows = min(WR * RT * 16, a.rows - first_row);
    for (int i = threadIdx.x; i < own_rows * pieces; i += kThreads) {
      const int r = i / pieces, d = (i - r * pieces) * 4;
      float top, sum;
      const f32x4_t v = joined_sums<true>(a, unit * a.splits * a.row_slots + first_row + r, d, D, 0, used, 1, &top, &sum);
      write_result(first_row + r, d, v, sum);
    }
  }
};

template <typename K>
__global__ __launch_bounds__(K::kThreads, K::kWavesPerSimd) void kernel(Args a) {
  K::run(a, blockIdx.x, false);
}
template <typename K>
__global__ __launch_bounds__(K::kThreads, K::kWavesPerSimd) void parts_kernel(Parts parts) {
  const bool shares = blockIdx.x < parts.prefix_blocks;
  const Args a = shares ? parts.prefix() : parts;
  K::run(a, shares ? blockIdx.x : blockIdx.x - parts.prefix_blocks, shares);
}

// Shape of the kernel that takes `rows` rows: 16-row tiles of a wave, waves
// over the rows (1: waves over the keys).
struct Shape {
  int tiles, waves;
  int rows() const { return 16 * tiles * waves; }
};

void launch_bf16(const Args& a, Shape shape, dim3 grid, hipStream_t stream);
void launch_f32(const Args& a, Shape shape, dim3 grid, hipStream_t stream);
void launch_parts_bf16(const Parts& parts, Shape shape, dim3 grid, hipStream_t stream);
void launch_parts_f32(const Parts& parts, Shape shape, dim3 grid, hipStream_t stream);
Shape shape_for(int rows, int head_dim);
// Heads of 64 or 128 in bf16, workgroups of 4 or 8 waves of 32 rows; of 64, 80, 96 or 128 in f32, of 8.
void launch_prefix_tiles(const Args& a, int waves, dim3 grid, hipStream_t stream);

template <typename T, int DT, bool EXACT, int RT, int WR, int KEYS, typename Launched>
void launch_shape(const Launched& a, dim3 grid, hipStream_t stream) {
  using Probe = Kernel<T, DT, EXACT, RT, WR, 1, 2, KEYS>;
  // Waves over the keys: as many as leave room in LDS for two workgroups of
  // two steps a wave; f32, which has more to compute in the same bytes, gains
  // by a third wave at widths of 65 to 96 (32 sequences of one token over up to
  // 4096, width 80: 109 us against 139), bf16 does not (48.1 and 48.0, width 96
  // 58.1 and 57.1).
  constexpr int WK = WR > 1 ? 1 : Probe::kStage <= 8192 ? 4 : Probe::kStage <= 12288 && !Probe::kHalf ? 3 : 2;
  // Two steps in LDS: three took 457 us against 446 for trees of 64 over up to 16384 tokens, four 720.
  constexpr int STAGES = 2;
  using K = Kernel<T, DT, EXACT, RT, WR, WK, STAGES, KEYS>;
  if constexpr (KEYS == kAllKeys)
    hipLaunchKernelGGL((kernel<K>), grid, dim3(K::kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((parts_kernel<K>), grid, dim3(K::kThreads), 0, stream, a);
}

template <typename T, int DT, bool EXACT, int KEYS, typename Launched>
void launch_width(const Launched& a, Shape shape, dim3 grid, hipStream_t stream) {
  if constexpr (DT <= 8) {
    if (shape.waves == 1) {
      if (shape.tiles == 1) return launch_shape<T, DT, EXACT, 1, 1, KEYS>(a, grid, stream);
      return launch_shape<T, DT, EXACT, 2, 1, KEYS>(a, grid, stream);
    }
  }
  if constexpr (DT > 8) {
    if (shape.waves == 2) return launch_shape<T, DT, EXACT, 1, 2, KEYS>(a, grid, stream);
  }
  if (shape.tiles == 1 || (!EXACT && DT > 8)) return launch_shape<T, DT, EXACT, 1, 4, KEYS>(a, grid, stream);
  if constexpr (EXACT || DT <= 8) return launch_shape<T, DT, EXACT, 2, 4, KEYS>(a, grid, stream);
}

template <typename T, int KEYS, typename Launched>
void launch_head(const Launched& a, Shape shape, dim3 grid, hipStream_t stream) {
  const int D = a.p.cache.head_dim;
  if (D == 64) return launch_width<T, 4, true, KEYS>(a, shape, grid, stream);
  if (D == 128) return launch_width<T, 8, true, KEYS>(a, shape, grid, stream);
  if (D == 256) return launch_width<T, 16, true, KEYS>(a, shape, grid, stream);
  if (D < 64) return launch_width<T, 4, false, KEYS>(a, shape, grid, stream);
  // Five tiles of 16 columns in f32, whose products cost the most.
  if constexpr (KEYS == kParts && T::bytes == 4) {
    if (D <= 80) return launch_width<T, 5, false, KEYS>(a, shape, grid, stream);
  }
  if (D <= 96) return launch_width<T, 6, false, KEYS>(a, shape, grid, stream);
  if (D < 128) return launch_width<T, 8, false, KEYS>(a, shape, grid, stream);
  // Tiles that 256 columns would waste, 32 sequences of one token over up to
  // 4096: width 192 bf16 108 us against 114, f32 322 and 477.
  if (D <= 192) return launch_width<T, 12, false, KEYS>(a, shape, grid, stream);
  launch_width<T, 16, false, KEYS>(a, shape, grid, stream);
}

}  // namespace attention
}  // namespace affon
