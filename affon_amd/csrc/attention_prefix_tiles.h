// A prefix that many rows share, on the matrix cores: bf16, heads of 64 or 128; f32 below.
//
// All its keys are committed and seen by every row, so nothing is masked: a
// workgroup of W waves holds 32 W rows and walks over a piece of the keys 32 at
// a time,
//   S^T = K Q^T,  P = e^(S - m),  O^T += V^T P^T   (32x32x16 products).
// A query row is the column lane % 32 of both results; a lane's sixteen scores
// are the keys 8 (i / 4) + 4 (lane / 32) + i % 4 of the 32, and the values are read in that order.
//
// What bounds it: per 32 rows and keys the matrix cores have 512 cycles of
// products, the vector unit about 400 of exponentials, sums and conversions,
// and LDS 128 per CU and wave. They overlap within a wave: a step's exponentials run
// between the scores of the step after it and the values' products of the one
// before it, none of which waits for them. 64 rows of 8 query heads a key head
// over 32768 tokens (8 key heads of 128): 80 us, 860 TFLOP/s, where a large library
// product reaches 1192; 0.93 us a step of 8 waves, and 14 us for the start and the
// results. Left out one at a time, on a copy (of 87 us then): the matrix products 13,
// the exponentials 6, the LDS reads 6, the transfers 4.
#pragma once

#include "attention.h"
#include "prefix_cut.h"

namespace affon {
namespace attention {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

// The keys of a workgroup: a piece of a group's prefix, of one key head; begin >=
// end: none. All groups' prefixes are cut alike, into `splits` pieces a group on
// average, so that a long one holds no workgroup longer than the others. (Four of
// up to 6000 tokens, 8 sequences each, f32: 92 us, each cut into 16 101.) In the order
// [group][key head][piece].
struct PrefixPiece {
  int row_group, kv, group;
  int64_t number;
  uint32_t begin = 0, end = 0;
  __device__ __forceinline__ explicit PrefixPiece(const Args& a) {
    const DraftBatch& batch = a.p.batch;
    const int lane = threadIdx.x & 63, groups = batch.sequences, kv_heads = a.p.cache.kv_heads;
    // Workgroups b, b + 8, .. run on one XCD: those of the same keys follow each other there.
    const int id = blockIdx.x >> 3;
    row_group = id % a.row_groups;
    number = id / a.row_groups * 8 + (blockIdx.x & 7);
    auto tokens = [&](int base) { return base + lane < groups ? prefix_tokens(a, batch, base + lane) : 0u; };
    const uint32_t mine = tokens(0);
    uint32_t chunk = max(batch.capacity, 1u);
    auto pieces_of = [&](uint32_t n) { return cut_pieces(n, chunk); };
    if (a.splits > 1) {
      uint64_t all = mine;
      for (int base = 64; base < groups; base += 64) all += tokens(base);
      all = wave_sum(all);
      const uint32_t pieces = static_cast<uint32_t>(a.splits) * groups;
      chunk = cut_chunk(all, pieces, a.chunk);
      // A few workgroups more than a round take as long as another: longer pieces, until they fit.
      if (groups <= 64)
        for (int i = 0; i < 16 && lane_of(scanned(pieces_of(mine)), 63) > pieces; ++i) chunk = cut_longer(chunk, a.chunk);
    }
    chunk = __builtin_amdgcn_readfirstlane(static_cast<int>(chunk));
    int64_t before = 0;
    for (int base = 0; base < groups; base += 64) {
      const uint32_t held = base == 0 ? mine : tokens(base), own = pieces_of(held), sum = scanned(own);
      const uint64_t past = __ballot((before + sum) * kv_heads > number);
      if (past != 0) {
        const int at = __builtin_ctzll(past);
        const uint32_t count = lane_of(own, at), rest = static_cast<uint32_t>(number - (before + lane_of(sum, at) - count) * kv_heads);
        group = base + at;
        kv = static_cast<int>(rest / count);
        const uint32_t piece = rest - static_cast<uint32_t>(kv) * count;
        if (rest == 0 && row_group == 0 && threadIdx.x == 0) a.plan[group] = uint2{static_cast<uint32_t>(number), count};
        begin = piece * chunk;
        end = min(begin + chunk, lane_of(held, at));
        return;
      }
      before += lane_of(sum, 63);
    }
  }
};

// The rows of a group that are in use, one after the other: of the sequences that
// take the prefix, their drafted tokens in use. Lane by lane, row `at` of them as a row of the
// group (-1: there are fewer), its token and its query head of the key head's; and the
// first such sequence, whose pages are read for all (-1: none).
struct UsedRow {
  int row = -1, token = 0, head, holder = -1;
  __device__ __forceinline__ UsedRow(const Args& a, int group, int at) {
    const int lane = threadIdx.x & 63, wanted = at / a.group;
    DraftBatch batch = a.p.batch;  // of the sequences themselves
    batch.rows /= a.per;
    head = at - wanted * a.group;
    int before = 0;
    for (int base = 0; base < a.per; base += 64) {
      const int i = base + lane, b = group * a.per + min(i, a.per - 1), some = min(64, a.per - base);
      const int own = i < a.per && takes_prefix(a, batch, b, group) ? static_cast<int>(drafted(batch, b)) : 0;
      const uint64_t taken = __ballot(own > 0);
      if (holder < 0 && taken != 0) holder = group * a.per + base + __builtin_ctzll(taken);
      if (__all(own == batch.rows || i >= a.per)) {  // all in use
        if (wanted >= before && wanted < before + some * batch.rows) token = base * batch.rows + wanted - before, row = 0;
        before += some * batch.rows;
      } else {
        const int sum = static_cast<int>(scanned(static_cast<uint32_t>(own)));
        int index = 0;  // sequences that end before the wanted row
        for (int k = 0; k < some; ++k) index += before + static_cast<int>(lane_of(static_cast<uint32_t>(sum), k)) <= wanted ? 1 : 0;
        const int start = before + __shfl(sum - own, min(index, 63));
        if (wanted >= before && index < some) token = (base + index) * batch.rows + wanted - start, row = 0;
        before += static_cast<int>(lane_of(static_cast<uint32_t>(sum), 63));
      }
      if (holder >= 0 && __all(row >= 0)) break;
    }
    if (row == 0) row = token * a.group + head;
  }
};

// Byte offsets of the tiles of 16 keys from `segment` on that lie somewhere, in
// their order (others hold no keys), and how many; for whole workgroups of W waves.
template <int W, int LIST>
__device__ __forceinline__ int list_tiles(const Args& a, const PrefixPiece& piece, int holder, uint32_t segment, int row_bytes,
                                          int64_t (&list)[LIST], int (&listed)[W]) {
  const AttentionProblem& p = a.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wanted = static_cast<int>(min(piece.end - segment, static_cast<uint32_t>(LIST * 16)) / 16);
  int tiles = 0;
  for (int i0 = 0; i0 < LIST && i0 < wanted; i0 += 64 * W) {
    const int i = i0 + static_cast<int>(threadIdx.x);
    int64_t offset = -1;
    if (i < wanted) {
      const uint32_t at = segment + i * 16, index = at / p.cache.page_size;
      const uint32_t page = page_of(p.cache, p.batch, holder, index);
      if (page != kNoPage)
        offset = ((static_cast<int64_t>(page) * p.cache.kv_heads + piece.kv) * p.cache.page_size +
                  (at - index * p.cache.page_size)) * row_bytes;
    }
    const uint64_t lies = __ballot(offset >= 0);
    __syncthreads();  // the list, and `listed`, are free
    if (lane == 0) listed[wave] = __popcll(lies);
    __syncthreads();
    int before = tiles;
    for (int w = 0; w < W; ++w) {
      if (w < wave) before += listed[w];
      tiles += listed[w];
    }
    if (offset >= 0) list[before + __popcll(lies & ((uint64_t(1) << lane) - 1))] = offset;
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(tiles);
}

// DT: 32-wide tiles of the head; W: waves, 32 rows each; STAGES: steps in LDS.
template <int DT, int W, int STAGES>
struct PrefixKernel {
  using Swizzle = Kernel<BF16, 2 * DT, true, 1, 1, 1, 2, kParts>;
  static constexpr int D = 32 * DT, kRowBytes = 2 * D, kThreads = 64 * W;
  static constexpr int kTile = 16 * kRowBytes, kPieces = kTile / 1024;  // of 16 keys, or values
  static constexpr int kStage = 2 * kTile;                              // keys of a step; the values' lie in a ring of their own
  static constexpr int kValues = STAGES * kStage;
  static constexpr int kPer = 4 * kPieces / W;                          // transfers of a wave and step, all of one tile
  static constexpr int kLead = STAGES - 2;                              // steps from a transfer's start to its use, and one
  static constexpr float kMostSum = 1024.0f;  // of a lane's sixteen probabilities: each is 1 at most where m is the largest score
  static constexpr int kList = 512;                                     // tiles of a segment
  static_assert(4 * kPieces % W == 0 && kPieces % kPer == 0 && kLead >= 2 && kLead * kPer < 64, "transfers in flight");
  static_assert(kValues <= 65536, "places are offsets in the instructions");
  static constexpr int kGroups = 2 * DT, kExps = 16 / kGroups;  // products of each kind in a step, exponentials beside one of each

  static __device__ void run(const Args& a) {
    const AttentionProblem& p = a.p;
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * kValues];
    __shared__ int64_t tile_list[kList];  // byte offsets of the segment's tiles that lie somewhere
    __shared__ int listed[W];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, side = lane >> 5;
    const PrefixPiece piece(a);
    if (piece.begin >= piece.end) return;
    const int kv = piece.kv, group = piece.group;
    const uint32_t begin = piece.begin, end = piece.end;

    // This wave's rows.
    const int row0 = (piece.row_group * W + wave) * 32;
    const UsedRow used(a, group, row0 + col);
    const int holder = __builtin_amdgcn_readfirstlane(used.holder);
    if (holder < 0) return;
    const bool active = __any(used.row >= 0);
    u32x4_t q[2 * DT];
    {
      const uint8_t* from = p.query + ((static_cast<int64_t>(group) * p.batch.rows + used.token) * p.query_stride +
                                       static_cast<int64_t>(kv * a.group + used.head) * D) * 2;
      const bool aligned = (reinterpret_cast<uintptr_t>(p.query) | static_cast<uintptr_t>(p.query_stride * 2)) % 16 == 0;
      const uint32_t flip = a.sign < 0.0f ? 0x80008000u : 0u, keep = a.sign == 0.0f ? 0u : ~0u;
#pragma unroll
      for (int c = 0; c < 2 * DT; ++c) {
        const uint8_t* piece = from + c * 32 + side * 16;
        if (aligned) {
          q[c] = *reinterpret_cast<const u32x4_t*>(piece);
        } else {
          const auto* h = reinterpret_cast<const uint16_t*>(piece);
#pragma unroll
          for (int e = 0; e < 4; ++e) q[c][e] = h[2 * e] | static_cast<uint32_t>(h[2 * e + 1]) << 16;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) q[c][e] = (q[c][e] & keep) ^ flip;
      }
    }

    // A wave moves pieces of one tile of a step: of the keys' first or second, or the values'.
    const int which = wave * kPer / kPieces, first_piece = wave * kPer % kPieces;
    const uint8_t* source = which >= 2 ? p.cache.values : p.cache.keys;
    // Where this lane's 16 bytes of them come from, and where it reads.
    uint32_t from[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int at = (first_piece + i) * 1024 + lane * 16, k = at / kRowBytes, c = at % kRowBytes / 16;
      from[i] = k * kRowBytes + (c ^ (which >= 2 ? Swizzle::value_swizzle(k) : Swizzle::key_swizzle(k))) * 16;
    }
    const uint32_t into = __builtin_amdgcn_readfirstlane(
        static_cast<int>(lds_address(lds) + (which >= 2 ? kValues : 0) + which % 2 * kTile + first_piece * 1024));
    int key_at[2 * DT], value_at[2][DT];
    const int key = lane & 15;
#pragma unroll
    for (int c = 0; c < 2 * DT; ++c)
      key_at[c] = pinned((col >> 4) * kTile + key * kRowBytes + ((2 * c + side) ^ Swizzle::key_swizzle(key)) * 16);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        // Lanes 4e .. 4e + 3 of 16 address key 8 h + 4 side + e; lane j gets column j of the four.
        const int k = 8 * h + 4 * side + (lane >> 2 & 3);
        value_at[h][dt] = pinned(kValues + k * kRowBytes +
                                 ((4 * dt + 2 * (lane >> 4 & 1) + (lane >> 1 & 1)) ^ Swizzle::value_swizzle(k)) * 16 + (lane & 1) * 8);
      }

    f32x16_t o[DT];
    float m = kLowest, l = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16_t{};

    for (uint32_t segment = begin; segment < end; segment += kList * 16) {
      const int tiles = list_tiles<W, kList>(a, piece, holder, segment, kRowBytes, tile_list, listed);
      if (tiles == 0) continue;
      const int steps = (tiles + 1) / 2;
      const bool odd = tiles % 2 != 0;  // the last step's second tile holds no keys

      // Transfers of a step; past the last one the last tile's again, so that their number is known.
      auto offset_of = [&](int step) { return tile_list[min(2 * step + which % 2, tiles - 1)]; };
      auto issue = [&](int place, int64_t offset) {
        const uint32_t low = __builtin_amdgcn_readfirstlane(static_cast<int>(offset));
        const uint32_t high = __builtin_amdgcn_readfirstlane(static_cast<int>(offset >> 32));
        const uint8_t* tile = uniform(source + (static_cast<int64_t>(high) << 32 | low));
#pragma unroll
        for (int i = 0; i < kPer; ++i) dma16(tile, from[i], into + place * kStage + i * 1024);
      };
      auto read_key = [&](int place, int c) { return *reinterpret_cast<const u32x4_t*>(lds + key_at[c] + place * kStage); };
      // Product g of a step's values: of 16 keys and 32 dims.
      auto read_value = [&](int place, int g) {
        u32x2_t half[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t address = lds_address(lds + value_at[h][g % DT] + place * kStage + g / DT * kTile);
          half[h] = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                    reinterpret_cast<lds_s16x4>(static_cast<uintptr_t>(address))));
        }
        return u32x4_t{half[0][0], half[0][1], half[1][0], half[1][1]};
      };
      f32x16_t s{};
      // The largest score of this lane's row, in both its lanes.
      auto largest = [&] {
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
        top *= a.log2_scale;
        return fmaxf(top, __shfl_xor(top, 32));
      };
      u32x4_t packed[2] = {u32x4_t{0, 0, 0, 0}, u32x4_t{0, 0, 0, 0}};
#pragma unroll
      for (int i = 0; i < kLead; ++i) issue(i, offset_of(i));
      int64_t coming = offset_of(kLead);
      wait_vmcnt<(kLead - 1) * kPer>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (odd && steps == 1) clear(lds + kValues + kTile);
#pragma unroll
      for (int c = 0; c < 2 * DT; ++c)
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, read_key(0, c)), __builtin_bit_cast(bf16x8_t, q[c]), s,
                                                    0, 0, 0);

      // A step, in place `place`: its exponentials between the next one's scores
      // and the last one's values. The values of step -1 are what lies there, times 0: so
      // FIRST leaves them out, as they may be infinite.
      auto advance = [&](int step, auto place_of_step, auto first_step) {
        constexpr int place = decltype(place_of_step)::value, ahead = (place + 1) % STAGES, behind = (place + STAGES - 1) % STAGES;
        constexpr bool FIRST = decltype(first_step)::value;
        wait_lds_reads();
        wait_vmcnt<(kLead - 2) * kPer>();  // step + 1 is there, and the place of step - 2 is free
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        issue((place + kLead) % STAGES, coming);
        coming = offset_of(step + kLead + 1);
        if (odd && step + 1 == steps - 1) clear(lds + kValues + ahead * kStage + kTile);
        if (!active) return;
        u32x4_t k = read_key(ahead, 0), v{};
        if constexpr (!FIRST) v = read_value(behind, 0);
        if (odd && step == steps - 1) {
          asm volatile("" ::: "memory");  // a branch, not eight selections in every step
#pragma unroll
          for (int i = 8; i < 16; ++i) s[i] = -INFINITY;
        }
        if constexpr (FIRST) {
          if (m == kLowest) m = fmaxf(m, largest());  // else the reference of the segment before
        }
        float sum = 0.0f;
        auto probabilities = [&](int i, u32x4_t (&to)[2]) {
          const float x = __builtin_amdgcn_exp2f(fmaf(s[i], a.log2_scale, -m));
          const float y = __builtin_amdgcn_exp2f(fmaf(s[i + 1], a.log2_scale, -m));
          sum += x;
          sum += y;
          // As in the other attention kernels, a probability is rounded once
          // for its product, by 2^-8 at most, and their sum is of the unrounded ones.
          to[i / 8][i % 8 / 2] = pack_bf16(x, y);
        };
        f32x16_t next{};
        u32x4_t done[2];
        pipeline::Unroll<0, kGroups>::run([&](auto group_of) {
          constexpr int g = decltype(group_of)::value;
          __builtin_amdgcn_sched_barrier(0);
          u32x4_t next_k = k, next_v = v;
          if constexpr (g + 1 < kGroups) {
            next_k = read_key(ahead, g + 1);
            if constexpr (!FIRST) next_v = read_value(behind, g + 1);
          }
          next = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, k), __builtin_bit_cast(bf16x8_t, q[g]), next, 0, 0, 0);
          if constexpr (!FIRST)
            o[g % DT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, v),
                                                                __builtin_bit_cast(bf16x8_t, packed[g / DT]), o[g % DT], 0, 0, 0);
#pragma unroll
          for (int e = 0; e < kExps; e += 2) probabilities(g * kExps + e, done);
          k = next_k;
          v = next_v;
        });
        __builtin_amdgcn_sched_barrier(0);
        // A score far past the reference shows in the sum, where no probability
        // has been multiplied yet: then, and only then, the reference moves.
        if (__any(sum > kMostSum)) {
          const float top = fmaxf(m, largest()), keep = __builtin_amdgcn_exp2f(m - top);
          m = top;
          l *= keep;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[dt] *= keep;
          sum = 0.0f;
#pragma unroll
          for (int i = 0; i < 16; i += 2) probabilities(i, done);
        }
        l += sum;
        s = next;
        packed[0] = done[0];
        packed[1] = done[1];
      };
      advance(0, std::integral_constant<int, 0>{}, std::true_type{});
      int last_place = 0;
      for (int step = 1; step < steps; step += STAGES)
        pipeline::Unroll<0, STAGES>::run([&](auto i) {
          constexpr int place = (decltype(i)::value + 1) % STAGES;
          if (step + i < steps) {
            advance(step + i, std::integral_constant<int, place>{}, std::false_type{});
            last_place = place;
          }
        });
      if (active) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
          o[g % DT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, read_value(last_place, g)),
                                                              __builtin_bit_cast(bf16x8_t, packed[g / DT]), o[g % DT], 0, 0, 0);
      }
      wait_lds_reads();
      wait_vmcnt<0>();  // transfers past the last step end before their places are used again
    }
    if (!active) return;
    l += __shfl_xor(l, 32);
    if (used.row < 0) return;
    const int64_t slot = piece.number * a.row_slots + used.row;
    float* to = a.sums + slot * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4_t*>(to + 32 * dt + 8 * j + 4 * side) =
            f32x4_t{o[dt][4 * j], o[dt][4 * j + 1], o[dt][4 * j + 2], o[dt][4 * j + 3]};
    if (side == 0) *reinterpret_cast<float2*>(a.stats + 2 * slot) = float2{m, l};
  }

  // Zeros for a tile of values that holds no keys; for whole workgroups.
  static __device__ __forceinline__ void clear(uint8_t* tile) {
    for (int i = threadIdx.x; i < kTile / 16; i += kThreads) reinterpret_cast<u32x4_t*>(tile)[i] = u32x4_t{0, 0, 0, 0};
    wait_lds_reads();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
};

// The same in f32, for heads of D = 64 to 128: S^T, and then O^T, by 32x32x2
// products, of two dims or keys at a time: the dims 8 j + 4 (lane / 32) + e and the
// keys of a lane's score, so that both operands are read in their order and P^T
// stays where it is. Bound by the matrix cores, whose f32 products take as many
// cycles for a 16th of bf16's work: D + 32 ceil(D / 32) halves of 64 cycles
// for 32 rows and keys, beside which all else is small (about 450 of exponentials and
// sums), so a step's phases follow each other and the waves of a SIMD fill each other's
// gaps. 4 prompts of up to 6000 tokens, 4 key heads of 80, 200 rows of which 140 are in
// use: 69 us (the call 92, and 110 with the general kernel, which takes them all); they
// are five tiles of 32 on four SIMDs, and the one with two holds up the others.
template <int WIDTH>
struct PrefixF32 {
  static constexpr int W = 8;
  static constexpr int D = WIDTH, kRowBytes = 4 * D, kThreads = 64 * W, DT = (D + 31) / 32;
  static constexpr int kTile = 16 * kRowBytes, kPieces = kTile / 1024;  // of 16 keys, or values
  static constexpr int kStage = 4 * kTile;                              // keys, then values, of a step
  static constexpr int kPer = (4 * kPieces + W - 1) / W;                // transfers of a wave and step
  static constexpr int kList = 512;
  static constexpr float kMostSum = 1024.0f;
  static constexpr int kSwizzle = D == 64 || D == 128 ? 15 : 0;  // of a key's pieces, where its length is a power of two
  static_assert(D % 16 == 0, "whole pieces");

  static __device__ void run(const Args& a) {
    const AttentionProblem& p = a.p;
    // Reads of dims past the last value's end stay inside it.
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * kStage + 128];
    __shared__ int64_t tile_list[kList];
    __shared__ int listed[W];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, side = lane >> 5;
    const PrefixPiece piece(a);
    if (piece.begin >= piece.end) return;
    const int row0 = (piece.row_group * W + wave) * 32;
    const UsedRow used(a, piece.group, row0 + col);
    const int holder = __builtin_amdgcn_readfirstlane(used.holder);
    if (holder < 0) return;
    const bool active = __any(used.row >= 0);
    f32x4_t q[D / 8];
    {
      const auto* from = reinterpret_cast<const float*>(p.query) +
                         (static_cast<int64_t>(piece.group) * p.batch.rows + used.token) * p.query_stride +
                         static_cast<int64_t>(piece.kv * a.group + used.head) * D;
      const bool aligned = (reinterpret_cast<uintptr_t>(p.query) | static_cast<uintptr_t>(p.query_stride * 4)) % 16 == 0;
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        const float* four = from + 8 * j + 4 * side;
        if (aligned) {
          q[j] = *reinterpret_cast<const f32x4_t*>(four);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) q[j][e] = four[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) q[j][e] = a.sign == 0.0f ? 0.0f : a.sign < 0.0f ? -q[j][e] : q[j][e];
      }
    }
    // This wave's pieces of a step's four tiles; past the last the last again.
    int which[kPer], into[kPer];
    uint32_t from[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int number = min(wave + i * W, 4 * kPieces - 1), first = number % kPieces * 1024;
      which[i] = number / kPieces;
      into[i] = which[i] * kTile + first;
      const int at = first + lane * 16, k = at / kRowBytes, c = at % kRowBytes / 16;
      from[i] = k * kRowBytes + (which[i] < 2 ? c ^ (k & kSwizzle) : c) * 16;
    }
    const uint32_t base = lds_address(lds);

    f32x16_t o[DT];
    float m = kLowest, l = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16_t{};
    for (uint32_t segment = piece.begin; segment < piece.end; segment += kList * 16) {
      const int tiles = list_tiles<W, kList>(a, piece, holder, segment, kRowBytes, tile_list, listed);
      if (tiles == 0) continue;
      const int steps = (tiles + 1) / 2;
      const bool odd = tiles % 2 != 0;  // the last step's second tile holds no keys
      auto issue = [&](int step) {
        const uint32_t place = __builtin_amdgcn_readfirstlane(static_cast<int>(base + step % 2 * kStage));
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int64_t offset = tile_list[min(2 * step + which[i] % 2, tiles - 1)];
          const uint32_t low = __builtin_amdgcn_readfirstlane(static_cast<int>(offset));
          const uint32_t high = __builtin_amdgcn_readfirstlane(static_cast<int>(offset >> 32));
          const uint8_t* source = which[i] < 2 ? p.cache.keys : p.cache.values;
          dma16(uniform(source + (static_cast<int64_t>(high) << 32 | low)), from[i], place + into[i]);
        }
      };
      issue(0);
      for (int step = 0; step < steps; ++step) {
        wait_lds_reads();
        wait_vmcnt<0>();
        __builtin_amdgcn_s_barrier();  // this step is there, and the place of the one before is free
        asm volatile("" ::: "memory");
        if (step + 1 < steps) issue(step + 1);
        const uint8_t* keys = lds + step % 2 * kStage;
        uint8_t* values = lds + step % 2 * kStage + 2 * kTile;
        const bool half = odd && step == steps - 1;
        if (half) {
          for (int i = threadIdx.x; i < kTile / 16; i += kThreads)
            reinterpret_cast<u32x4_t*>(values + kTile)[i] = u32x4_t{0, 0, 0, 0};
          wait_lds_reads();
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
        }
        if (!active) continue;
        f32x16_t s{};
        const uint8_t* row = keys + col * kRowBytes;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          const f32x4_t k = *reinterpret_cast<const f32x4_t*>(row + ((2 * j + side) ^ (col & kSwizzle)) * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e], q[j][e], s, 0, 0, 0);
        }
        if (half) {
#pragma unroll
          for (int i = 8; i < 16; ++i) s[i] = -INFINITY;
        }
        auto largest = [&] {
          float top = s[0];
#pragma unroll
          for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
          top *= a.log2_scale;
          return fmaxf(top, __shfl_xor(top, 32));
        };
        if (m == kLowest) m = fmaxf(m, largest());
        f32x16_t probability;
        float sum = 0.0f;
        auto exponentials = [&] {
          sum = 0.0f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            probability[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.log2_scale, -m));
            sum += probability[i];
          }
        };
        exponentials();
        if (__any(sum > kMostSum)) {  // a score far past the reference, which moves
          const float top = fmaxf(m, largest()), keep = __builtin_amdgcn_exp2f(m - top);
          m = top;
          l *= keep;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[dt] *= keep;
          exponentials();
        }
        l += sum;
        const uint8_t* value = values + 4 * side * kRowBytes + col * 4;
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
            o[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(
                *reinterpret_cast<const float*>(value + (8 * (i / 4) + i % 4) * kRowBytes + 128 * dt), probability[i], o[dt], 0, 0, 0);
      }
      wait_lds_reads();
    }
    if (!active) return;
    l += __shfl_xor(l, 32);
    if (used.row < 0) return;
    const int64_t slot = piece.number * a.row_slots + used.row;
    float* to = a.sums + slot * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (32 * dt + 8 * j < D)
          *reinterpret_cast<f32x4_t*>(to + 32 * dt + 8 * j + 4 * side) =
              f32x4_t{o[dt][4 * j], o[dt][4 * j + 1], o[dt][4 * j + 2], o[dt][4 * j + 3]};
    if (side == 0) *reinterpret_cast<float2*>(a.stats + 2 * slot) = float2{m, l};
  }
};

template <typename K>
__global__ __launch_bounds__(K::kThreads, 2) void prefix_kernel(Args a) {
  K::run(a);
}

}  // namespace attention
}  // namespace affon
