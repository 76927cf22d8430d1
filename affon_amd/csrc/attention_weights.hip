// The attention weights that the tokens of a cache gather: for each key head
// and token, the sum of its probabilities over the rows and query heads that
// share the key head.
//
// A row's probabilities need its largest score and the sum of its exponentials
// first (stats_kernel). For up to 16 rows of a key head the scores are then kept
// and summed over the rows by sum_kernel: the keys are read once. With more rows
// the scores would be more to write and read than the keys, and are computed
// again (gather_kernel).
//
// What bounds it, bf16 heads of 128, 8 key heads: one token of 32 sequences over
// up to 4096, memory (stats 41 us, 4.1 TB/s with the scores' writes; sum 7.3); 32
// tokens of 8 query heads a key head, four sequences over up to 16384, the
// exponentials (twice each, at a quarter of the vector rate) and what of the
// products does not run beside them (stats 36 us, gathering 35, 6 between them; the
// two sides' products are 30 us of the matrix rate); one token over 777,
// two launches and their chains of loads (11 us). Products are S^T = K Q^T on the matrix cores: lane % 16
// is a row, and a lane's four results are keys 4 (lane / 16) .. + 3 of a tile of
// 16. stats_kernel holds queries in registers and walks over the keys,
// gather_kernel holds keys and walks over the rows.

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
  int tiles;         // 16-row tiles of a wave there
  bool over_rows;    // its waves are side by side over the rows
  int pieces;        // of all contexts, for each key head: about so many, and one a sequence more at most
  int gather_pieces; // the same for gather_kernel
  float log2_scale;  // |scale| * log2(e)
  float sign;        // of the scale: a factor of the queries
  float2* stats;     // (m, l) [piece][row]
  float* ready;      // m + log2(l) [unit][row_slots]; infinite: the row takes no part
  int row_slots;     // rows, up to a whole 64
  u32x4_t* packed;   // the queries as gather_kernel's operands
  float* scores;     // [unit][row][capacity], or null: computed again
  float* weights;    // of the layer, [sequence][key head][capacity]
  int blocks;        // workgroups of sum_kernel along a context
};

// What a sequence holds.
struct Context {
  uint32_t length, count, n;
  __device__ __forceinline__ Context(const AttentionProblem& p, int b) {
    length = committed(p.batch, b);
    count = drafted(p.batch, b);
    n = min(length + count, p.batch.capacity);
  }
};

// All contexts with rows in use, cut into pieces of about the same number of keys
// by the lengths that are there: workgroups that are numbered through them have equal
// work, whatever the lengths and the table's width, and one round of them pays for its
// start (lengths, table, queries: 5 us) once. There are `pieces` of them for each key
// head at most where sequences have two on average or more (and are no more than 64),
// and never more than `pieces` + the sequences. For whole waves.
constexpr uint32_t kPieceUnit = 128;
struct Pieces {
  const DraftBatch& batch;
  uint32_t chunk;  // keys of a piece
  uint32_t mine;   // keys of the sequence of this lane, among the first 64
  __device__ __forceinline__ uint32_t keys_of(int b) const {
    const uint32_t count = drafted(batch, b);
    return count == 0 ? 0u : min(committed(batch, b) + count, batch.capacity);
  }
  __device__ __forceinline__ uint32_t keys_at(int base) const {
    const int b = base + static_cast<int>(threadIdx.x & 63);
    return base == 0 ? mine : b < batch.sequences ? keys_of(b) : 0u;
  }
  __device__ __forceinline__ uint32_t pieces_of(uint32_t keys) const { return keys == 0 ? 0u : (keys - 1) / chunk + 1; }
  __device__ __forceinline__ Pieces(const DraftBatch& batch, int pieces) : batch(batch) {
    const int lane = threadIdx.x & 63;
    mine = lane < batch.sequences ? keys_of(lane) : 0u;
    uint64_t all = mine;
    for (int b = lane + 64; b < batch.sequences; b += 64) all += keys_of(b);
    all = wave_sum(all) + (pieces - 1);
    const uint32_t by = static_cast<uint32_t>(pieces);
    const uint32_t each = all >> 32 != 0 ? static_cast<uint32_t>(min(all / by, static_cast<uint64_t>(batch.capacity)))
                                         : min(static_cast<uint32_t>(all) / by, batch.capacity);
    auto whole = [](uint32_t n) { return max(kPieceUnit, (n + kPieceUnit - 1) / kPieceUnit * kPieceUnit); };
    chunk = __builtin_amdgcn_readfirstlane(static_cast<int>(whole(each)));
    // A round of workgroups that a few more follow takes as long as two: longer pieces, until they fit.
    if (batch.sequences <= 64 && pieces >= 2 * batch.sequences)
      for (int i = 0; i < 16 && lane_of(scanned(pieces_of(mine)), 63) > by; ++i) chunk += whole(chunk / 16);
  }
  // Piece `id` of [sequence][key head][piece of the sequence]; false: there are fewer.
  __device__ __forceinline__ bool find(int64_t id, int kv_heads, int* b, int* kv, uint32_t* piece) const {
    int64_t before = 0;
    for (int base = 0; base < batch.sequences; base += 64) {
      const uint32_t own = pieces_of(keys_at(base)), sum = scanned(own);
      const uint64_t past = __ballot((before + sum) * kv_heads > id);
      if (past != 0) {
        const int at = __builtin_ctzll(past);
        const uint32_t pieces = lane_of(own, at);
        const uint32_t rest = static_cast<uint32_t>(id - (before + lane_of(sum, at) - pieces) * kv_heads);
        *b = base + at;
        *kv = static_cast<int>(rest / pieces);
        *piece = rest - static_cast<uint32_t>(*kv) * pieces;
        return true;
      }
      before += lane_of(sum, 63);
    }
    return false;
  }
  // Number of the first piece of a sequence's key head; `pieces`: of each of its key heads.
  __device__ __forceinline__ int64_t first_of(int b, int kv, int kv_heads, uint32_t pieces) const {
    uint64_t before = 0;
    for (int base = 0; base < b; base += 64)
      before += base + static_cast<int>(threadIdx.x & 63) < b ? pieces_of(keys_at(base)) : 0u;
    return static_cast<int64_t>(wave_sum(before)) * kv_heads + static_cast<int64_t>(kv) * pieces;
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

  // A tile of 16 keys is consecutive in memory and comes by whole lines, a lane
  // the 16-byte pieces lane, lane + 64, .. (`from`), through a place of the wave's
  // own in LDS, whose rows are padded against bank conflicts and hold zeros past the head.
  // (An operand's own lanes would ask for 64 bytes of 16 keys at a time.)
  static constexpr int kRow = 64 * KS + 16, kPlace = 16 * kRow + 16;  // the last 16 bytes: for pieces past the tile
  int from[KS], to[KS], at;
  __device__ __forceinline__ explicit Tiles(const WeightArgs& a) {
    const int lane = threadIdx.x & 63, row_bytes = a.p.cache.head_dim * T::bytes;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int byte = s * 1024 + lane * 16, key = byte / row_bytes;
      from[s] = min(byte, 16 * row_bytes - 16);
      to[s] = key < 16 ? key * kRow + byte - key * row_bytes : 16 * kRow;
    }
    at = (lane & 15) * kRow + (lane >> 4) * 16;
  }
  static __device__ __forceinline__ void clear(uint8_t* place, int tiles) {
    for (int i = threadIdx.x & 63; i < tiles * kPlace / 16; i += 64) reinterpret_cast<u32x4_t*>(place)[i] = u32x4_t{0, 0, 0, 0};
  }
  __device__ __forceinline__ void fetch(const uint8_t* tile, u32x4_t (&k)[KS]) const {
#pragma unroll
    for (int s = 0; s < KS; ++s) k[s] = *reinterpret_cast<const u32x4_t*>(tile + from[s]);
  }
  __device__ __forceinline__ void put(uint8_t* place, const u32x4_t (&k)[KS]) const {
#pragma unroll
    for (int s = 0; s < KS; ++s) *reinterpret_cast<u32x4_t*>(place + to[s]) = k[s];
  }
  // The tile as an operand (a wave's own LDS accesses keep their order).
  __device__ __forceinline__ void get(const uint8_t* place, u32x4_t (&k)[KS]) const {
#pragma unroll
    for (int s = 0; s < KS; ++s) k[s] = *reinterpret_cast<const u32x4_t*>(place + at + s * 64);
  }

  static __device__ __forceinline__ f32x4_t scores(const u32x4_t (&k)[KS], const u32x4_t (&q)[KS]) {
    f32x4_t s{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      if constexpr (kHalf) {
        s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, k[i]), __builtin_bit_cast(bf16x8_t, q[i]), s,
                                                    0, 0, 0);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t ke = k[i][e], qe = q[i][e];
          s = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(ke), __uint_as_float(qe), s, 0, 0, 0);
        }
      }
    }
    return s;
  }

  // Byte offset in the keys of the tile that starts at token n of sequence b; 1: it lies nowhere.
  static __device__ __forceinline__ int64_t tile_of(const WeightArgs& a, int b, int kv, uint32_t n) {
    const PagedCache& c = a.p.cache;
    const uint32_t index = n / c.page_size, page = page_of(c, a.p.batch, b, index);
    if (page == kNoPage) return 1;
    return ((static_cast<int64_t>(page) * c.kv_heads + kv) * c.page_size + (n - index * c.page_size)) * c.head_dim * T::bytes;
  }

  // Bits of the 16 keys from `at` on that row t of the sequence sees.
  static __device__ __forceinline__ uint32_t seen(const WeightArgs& a, const Context& c, int b, int t, uint32_t at) {
    return seen_bits(a.p, static_cast<int64_t>(b) * a.p.batch.rows + t, t, static_cast<int>(at) - static_cast<int>(c.length),
                     static_cast<int>(c.n) - static_cast<int>(c.length));
  }
};

// Four waves side by side over the keys of a piece, RT tiles of 16 rows each; or
// (ROWS) over the rows, which then fetch a tile of four each for all of them:
// the L2s answer some 68 requests of 128 bytes a ns, and four row groups that
// fetch the keys by themselves are bound by that.
template <typename T, int KS, int RT, bool KEEP, bool ROWS>
__global__ __launch_bounds__(256) void stats_kernel(WeightArgs a) {
  using Ops = Tiles<T, KS>;
  constexpr int KT = KS <= 4 && RT <= 2 && !ROWS ? 2 : 1;             // tiles of a step
  constexpr int kAhead = ROWS || KEEP ? 1 : RT > 2 ? 3 : KS <= 8 ? 2 : 1;  // steps on their way from memory
  constexpr int kOwn = ROWS ? 4 : 1;                                  // waves over the rows
  const AttentionProblem& p = a.p;
  __shared__ __attribute__((aligned(16))) uint8_t lds[(ROWS ? 8 : 4 * KT) * Ops::kPlace];
  __shared__ float2 parts[ROWS ? 1 : 4][16 * RT];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  // Workgroups b, b + 8, .. run on one XCD: those of the same keys follow each other there.
  int id = blockIdx.x >> 3;
  const int rg = id % a.row_groups;
  id = id / a.row_groups * 8 + (blockIdx.x & 7);
  const Pieces pieces(p.batch, a.pieces);
  const uint32_t chunk = pieces.chunk;
  int b, kv;
  uint32_t piece;
  if (!pieces.find(id, p.cache.kv_heads, &b, &kv, &piece)) return;
  const int unit = b * p.cache.kv_heads + kv;
  const Context c(p, b);
  const uint32_t begin = piece * chunk;
  const uint32_t end = min(begin + chunk, c.n);
  const uint32_t sub = ROWS ? chunk : ((end - begin + 3) / 4 + 31) / 32 * 32;
  const uint32_t first = min(begin + (ROWS ? 0 : wave * sub), end), last = min(first + sub, end);

  const int row0 = (rg * kOwn + (ROWS ? wave : 0)) * 16 * RT;
  u32x4_t q[RT][KS];
  int t[RT];
  float m[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    Ops::load_rows(a, b, kv, c.count, row0 + 16 * rt, q[rt]);
    t[rt] = min(row0 + 16 * rt + col, a.rows - 1) / a.group;
    m[rt] = kLowest;
    l[rt] = 0.0f;
  }

  // A step: its pieces come from memory (`raw`) while the step before it is
  // multiplied and the one before that goes through its exponentials.
  uint8_t* place = lds + (ROWS ? 0 : wave * KT * Ops::kPlace);
  const Ops ops(a);
  Ops::clear(ROWS ? lds + wave * 2 * Ops::kPlace : place, ROWS ? 2 : KT);
  int64_t list = 1;  // places of 64 tiles, a lane each
  u32x4_t raw[kAhead][KT][KS];
  uint32_t raw_there[kAhead];  // bit kt: tile kt lies somewhere
  auto fetch = [&](uint32_t at, auto spot) {
    constexpr int into = decltype(spot)::value;
    if ((at - first) % 1024 == 0) {
      const uint32_t mine = at + lane * 16;
      list = mine < last ? Ops::tile_of(a, b, kv, mine) : 1;
    }
    raw_there[into] = 0;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int i = static_cast<int>((at - first) / 16 % 64) + kt;
      const uint32_t low = __builtin_amdgcn_readlane(static_cast<int>(list), i);
      const uint32_t high = __builtin_amdgcn_readlane(static_cast<int>(list >> 32), i);
      ops.fetch(p.cache.keys + (static_cast<int64_t>(high) << 32 | (low & ~15u)), raw[into][kt]);
      raw_there[into] |= low & 1 ? 0u : 1u << kt;
    }
  };
  f32x4_t s[RT][KT];
  auto multiply = [&](f32x4_t (&into)[RT][KT], const uint8_t* from) {
    u32x4_t keys[KT][KS];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) ops.get(from + kt * Ops::kPlace, keys[kt]);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) into[rt][kt] = Ops::scores(keys[kt], q[rt]);
  };
  // Scores that a row does not see, the kept ones, and the reference of the exponentials.
  auto settle = [&](uint32_t at, uint32_t there) {
    if (there != (1u << KT) - 1 || at + 16 * KT > c.length) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const uint32_t seen = there >> kt & 1 ? Ops::seen(a, c, b, t[rt], at + 16 * kt) : 0u;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!(seen >> (4 * quad + i) & 1)) s[rt][kt][i] = -INFINITY;
        }
    }
    if constexpr (KEEP) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
        if (row0 + col < a.rows && at + 16 * kt < c.n)
          *reinterpret_cast<f32x4_t*>(a.scores + (static_cast<int64_t>(unit) * a.rows + row0 + col) * p.batch.capacity + at +
                                      16 * kt + 4 * quad) = s[0][kt];
    }
    float top[RT];
    bool above = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      top[rt] = fmaxf(fmaxf(s[rt][0][0], s[rt][0][1]), fmaxf(s[rt][0][2], s[rt][0][3]));
#pragma unroll
      for (int kt = 1; kt < KT; ++kt)
        top[rt] = fmaxf(top[rt], fmaxf(fmaxf(s[rt][kt][0], s[rt][kt][1]), fmaxf(s[rt][kt][2], s[rt][kt][3])));
      top[rt] *= a.log2_scale;
      above |= top[rt] > m[rt] + kSlack;
    }
    if (__any(above)) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        top[rt] = fmaxf(top[rt], __shfl_xor(top[rt], 16));
        top[rt] = fmaxf(fmaxf(top[rt], __shfl_xor(top[rt], 32)), m[rt]);
        l[rt] *= __builtin_amdgcn_exp2f(m[rt] - top[rt]);
        m[rt] = top[rt];
      }
    }
  };
  auto exponentials = [&] {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) l[rt] += __builtin_amdgcn_exp2f(fmaf(s[rt][kt][i], a.log2_scale, -m[rt]));
  };
  auto put = [&](auto spot) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) ops.put(place + kt * Ops::kPlace, raw[decltype(spot)::value][kt]);
  };
  constexpr uint32_t kStep = 16 * KT;
  if constexpr (ROWS) {
    // Four tiles at a time, one of each wave, in one half of the LDS while the other fills.
    __syncthreads();  // the halves are cleared
    f32x4_t next[RT][KT];
    auto fetch_own = [&](uint32_t four) {
      if ((four - first) % 1024 == 0) {
        const uint32_t mine = four + lane * 16;
        list = mine < last ? Ops::tile_of(a, b, kv, mine) : 1;
      }
      const int i = static_cast<int>((four - first) / 16 % 64) + wave;
      const uint32_t low = __builtin_amdgcn_readlane(static_cast<int>(list), i);
      const uint32_t high = __builtin_amdgcn_readlane(static_cast<int>(list >> 32), i);
      ops.fetch(p.cache.keys + (static_cast<int64_t>(high) << 32 | (low & ~15u)), raw[0][0]);
      uint32_t there = 0;  // bit i: tile i of the four lies somewhere
#pragma unroll
      for (int j = 0; j < 4; ++j)
        there |= __builtin_amdgcn_readlane(static_cast<int>(list), (four - first) / 16 % 64 + j) & 1 ? 0u : 1u << j;
      return there;
    };
    uint32_t coming = fetch_own(first), half = 0;
    for (uint32_t four = first; four < last; four += 64, half ^= 1) {
      uint8_t* tiles = lds + half * 4 * Ops::kPlace;
      ops.put(tiles + wave * Ops::kPlace, raw[0][0]);
      const uint32_t there = coming;
      coming = fetch_own(four + 64);  // past the last: some page's, and not looked at
      wait_lds_reads();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      multiply(s, tiles);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        settle(four + 16 * i, four + 16 * i < last ? there >> i & 1 : 0u);
        if (i < 3) multiply(next, tiles + (i + 1) * Ops::kPlace);
        exponentials();
        if (i < 3) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[rt][0] = next[rt][0];
        }
      }
    }
  } else if (first < last) {
    using First = std::integral_constant<int, 0>;
    // Steps past the last one are fetched from some page and multiplied too, and
    // not looked at: with fetches under conditions, the loads' count is not known,
    // and every step would wait for all of them.
    pipeline::Unroll<0, kAhead>::run([&](auto spot) { fetch(first + spot * kStep, spot); });
    put(First{});
    uint32_t there = raw_there[0];
    fetch(first + kAhead * kStep, First{});
    multiply(s, place);
    uint32_t at = first;
    // A step, while the next one, whose pieces are in `spot`, is multiplied; false: it was the last.
    auto advance = [&](auto spot) {
      settle(at, there);
      put(spot);
      there = raw_there[decltype(spot)::value];
      fetch(at + (kAhead + 1) * kStep, spot);
      f32x4_t next[RT][KT];
      multiply(next, place);
      exponentials();
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) s[rt][kt] = next[rt][kt];
      at += kStep;
      return at < last;
    };
    for (;;) {
      if (!advance(std::integral_constant<int, 1 % kAhead>{})) break;
      if constexpr (kAhead > 1)
        if (!advance(std::integral_constant<int, 2 % kAhead>{})) break;
      if constexpr (kAhead > 2)
        if (!advance(std::integral_constant<int, 3 % kAhead>{})) break;
    }
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l[rt] += __shfl_xor(l[rt], 16);
    l[rt] += __shfl_xor(l[rt], 32);
    const int r = row0 + 16 * rt + col;
    if constexpr (ROWS) {
      if (quad == 0 && r < a.rows) a.stats[static_cast<int64_t>(id) * a.rows + r] = float2{m[rt], l[rt]};
    } else {
      if (quad == 0) parts[wave][16 * rt + col] = float2{m[rt], l[rt]};
    }
  }
  if constexpr (ROWS) return;
  __syncthreads();
  const int own = static_cast<int>(threadIdx.x), r = row0 + own;
  if (own >= 16 * RT || r >= a.rows) return;
  float top = kLowest, sum = 0.0f;
  for (int w = 0; w < 4; ++w) top = fmaxf(top, parts[w][own].x);
  for (int w = 0; w < 4; ++w) sum = fmaf(parts[w][own].y, __builtin_amdgcn_exp2f(parts[w][own].x - top), sum);
  a.stats[static_cast<int64_t>(id) * a.rows + r] = float2{top, sum};
}

// What a row's exponents start from, m + log2(l), of its joined pieces.
__device__ __forceinline__ float ready_of(float m, float l, bool used) {
  return l == 0.0f || !used ? INFINITY : m + __builtin_amdgcn_logf(l);
}

// Joins the pieces of a row, a thread each, and lays the queries out as
// gather_kernel's operands: [unit][tile of 16 rows][piece][lane].
template <typename T, int KS>
__global__ __launch_bounds__(256) void ready_kernel(WeightArgs a, int64_t packs) {
  if (blockIdx.x < packs) {
    const int row_tiles = (a.rows + 15) / 16;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);  // a wave a tile
    const int64_t unit = i / row_tiles;
    if (unit >= static_cast<int64_t>(a.p.batch.sequences) * a.p.cache.kv_heads) return;
    const int tile = static_cast<int>(i - unit * row_tiles), b = static_cast<int>(unit / a.p.cache.kv_heads);
    u32x4_t q[KS];
    Tiles<T, KS>::load_rows(a, b, static_cast<int>(unit - static_cast<int64_t>(b) * a.p.cache.kv_heads),
                            drafted(a.p.batch, b), tile * 16, q);
#pragma unroll
    for (int s = 0; s < KS; ++s) a.packed[(i * KS + s) * 64 + (threadIdx.x & 63)] = q[s];
    return;
  }
  const int parts = (a.row_slots + 255) / 256;
  const int unit = static_cast<int>((blockIdx.x - packs) / parts);
  const int r = static_cast<int>(blockIdx.x - packs - static_cast<int64_t>(unit) * parts) * 256 + threadIdx.x;
  const int b = unit / a.p.cache.kv_heads, kv = unit - b * a.p.cache.kv_heads;
  const Context c(a.p, b);
  if (c.n == 0 || c.count == 0) return;
  const Pieces pieces(a.p.batch, a.pieces);
  const uint32_t used = pieces.pieces_of(c.n);
  const int64_t first = pieces.first_of(b, kv, a.p.cache.kv_heads, used);
  if (r >= a.row_slots) return;
  if (r >= a.rows) {
    a.ready[static_cast<int64_t>(unit) * a.row_slots + r] = INFINITY;
    return;
  }
  float m = kLowest, l = 0.0f;
  constexpr uint32_t kAtOnce = 8;  // pieces whose loads are in flight together
  for (uint32_t s0 = 0; s0 < used; s0 += kAtOnce) {
    float2 st[kAtOnce];
    float top = m;
#pragma unroll
    for (uint32_t i = 0; i < kAtOnce; ++i) st[i] = a.stats[(first + min(s0 + i, used - 1)) * a.rows + r];
#pragma unroll
    for (uint32_t i = 0; i < kAtOnce; ++i) top = fmaxf(top, st[i].x);
    l *= __builtin_amdgcn_exp2f(m - top);
    m = top;
#pragma unroll
    for (uint32_t i = 0; i < kAtOnce; ++i)
      if (s0 + i < used) l = fmaf(st[i].y, __builtin_amdgcn_exp2f(st[i].x - m), l);
  }
  a.ready[static_cast<int64_t>(unit) * a.row_slots + r] = ready_of(m, l, r / a.group < static_cast<int>(c.count));
}

// Sums of up to 16 rows' kept scores: a thread four keys, 16 lanes the pieces of a row.
__global__ __launch_bounds__(256) void sum_kernel(WeightArgs a) {
  __shared__ float ready[16];
  const AttentionProblem& p = a.p;
  const int unit = blockIdx.x / a.blocks, block = blockIdx.x % a.blocks;
  const Context c(p, unit / p.cache.kv_heads);
  if (c.count == 0 || static_cast<uint32_t>(block) * 1024 >= c.n) return;
  const Pieces pieces(p.batch, a.pieces);
  const uint32_t used = pieces.pieces_of(c.n);
  const int64_t first = pieces.first_of(unit / p.cache.kv_heads, unit % p.cache.kv_heads, p.cache.kv_heads, used);
  const int r = threadIdx.x / 16;
  float m = kLowest, l = 0.0f;
  if (r < a.rows) {
    for (uint32_t s = threadIdx.x % 16; s < used; s += 16) {
      const float2 st = a.stats[(first + s) * a.rows + r];
      const float top = fmaxf(m, st.x);
      l = fmaf(st.y, __builtin_amdgcn_exp2f(st.x - top), l * __builtin_amdgcn_exp2f(m - top));
      m = top;
    }
  }
#pragma unroll
  for (int offset = 1; offset < 16; offset <<= 1) {
    const float other_m = __shfl_xor(m, offset), other_l = __shfl_xor(l, offset), top = fmaxf(m, other_m);
    l = l * __builtin_amdgcn_exp2f(m - top) + other_l * __builtin_amdgcn_exp2f(other_m - top);
    m = top;
  }
  if (threadIdx.x % 16 == 0) ready[r] = ready_of(m, l, r < a.rows && r / a.group < static_cast<int>(c.count));
  __syncthreads();
  float* weights = a.weights + static_cast<int64_t>(unit) * p.batch.capacity;
  const float* scores = a.scores + static_cast<int64_t>(unit) * a.rows * p.batch.capacity;
  const bool aligned = reinterpret_cast<uintptr_t>(a.weights) % 16 == 0;
  for (uint32_t n = (block * 256 + threadIdx.x) * 4; n < c.n; n += a.blocks * 1024) {
    f32x4_t before{0, 0, 0, 0}, v{0, 0, 0, 0};
    const bool whole = aligned && n + 4 <= c.length;
    if (whole) before = *reinterpret_cast<const f32x4_t*>(weights + n);
    for (int row = 0; row < a.rows; ++row) {
      const float from = ready[row];
      if (from == INFINITY) continue;
      const f32x4_t s = *reinterpret_cast<const f32x4_t*>(scores + static_cast<int64_t>(row) * p.batch.capacity + n);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += __builtin_amdgcn_exp2f(fmaf(s[i], a.log2_scale, -from));
    }
    if (whole) {
      *reinterpret_cast<f32x4_t*>(weights + n) = before + v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < c.n) weights[n + i] = n + i < c.length ? weights[n + i] + v[i] : v[i];
    }
  }
}

// The sum over each 16 lanes, in all of them.
__device__ __forceinline__ float sum_of_16(float v) {
  return plus_lane<kOtherEight>(plus_lane<kOtherFour>(plus_lane<kNextPair>(plus_lane<kNextLane>(v))));
}

// Four waves side by side over the keys, KT tiles each, all rows one after the
// other, kTiles tiles of them at a time through LDS, the next ones on their way
// meanwhile, those of the next keys too. (Waited for at each step's start, with
// pages looked up and weights loaded when they were needed, 43 us instead of 35;
// four tiles of keys a wave 43: too few waves.)
template <typename T, int KS>
__global__ __launch_bounds__(256) void gather_kernel(WeightArgs a) {
  using Ops = Tiles<T, KS>;
  constexpr int KT = KS <= 4 ? 2 : 1;
  constexpr uint32_t kKeys = 16 * KT;
  constexpr int kTiles = KS <= 4 ? 4 : 2;
  constexpr int kQueries = kTiles * KS * 1024;
  const AttentionProblem& p = a.p;
  __shared__ __attribute__((aligned(16))) uint8_t lds[4 * Ops::kPlace];
  __shared__ __attribute__((aligned(16))) uint8_t queries[2][kQueries + 1024];  // and what their exponents start from
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const Pieces pieces(p.batch, a.gather_pieces);
  int b, kv;
  uint32_t piece;
  if (!pieces.find(blockIdx.x, p.cache.kv_heads, &b, &kv, &piece)) return;
  const int unit = b * p.cache.kv_heads + kv;
  const Context c(p, b);
  // Rows past the last one in use take no part.
  const int rows = min(a.rows, static_cast<int>(c.count) * a.group), tiles = (rows + 15) / 16;
  const int groups = (tiles + kTiles - 1) / kTiles;
  const auto* all_ready = reinterpret_cast<const uint8_t*>(a.ready + static_cast<int64_t>(unit) * a.row_slots);
  const u32x4_t* packed = a.packed + static_cast<int64_t>(unit) * ((a.rows + 15) / 16) * KS * 64;
  float* weights = a.weights + static_cast<int64_t>(unit) * p.batch.capacity;
  uint8_t* place = lds + wave * Ops::kPlace;
  const Ops ops(a);
  Ops::clear(place, 1);
  const uint32_t begin = piece * pieces.chunk, end = min(begin + pieces.chunk, c.n);
  auto issue = [&](int group, int turn) {
    const u32x4_t* from = packed + static_cast<int64_t>(group) * kTiles * KS * 64;
    const uint32_t into = __builtin_amdgcn_readfirstlane(static_cast<int>(lds_address(queries[turn])));
    const int pieces = min(kTiles, tiles - group * kTiles) * KS;
    for (int i = wave; i < pieces; i += 4) dma16(uniform(reinterpret_cast<const uint8_t*>(from + i * 64)), lane * 16, into + i * 1024);
    if (wave == 3) dma16(uniform(all_ready + group * kTiles * 64), min(lane, 4 * kTiles - 1) * 16, into + kQueries);
  };
  // This wave's keys of the next step, on their way while a step's rows are gone
  // through; past the last one some page's, which are not looked at.
  int64_t list = 1;  // places of 64 tiles, a lane each
  u32x4_t raw[KT][KS];
  uint32_t coming = 0;  // bit kt: tile kt lies somewhere
  auto fetch = [&](uint32_t four) {
    if ((four - begin) % 1024 == 0) {
      const uint32_t mine = four + lane * 16;
      list = mine < end ? Ops::tile_of(a, b, kv, mine) : 1;
    }
    coming = 0;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int i = static_cast<int>((four - begin) / 16 % 64) + wave * KT + kt;
      const uint32_t low = __builtin_amdgcn_readlane(static_cast<int>(list), i);
      const uint32_t high = __builtin_amdgcn_readlane(static_cast<int>(list >> 32), i);
      ops.fetch(p.cache.keys + (static_cast<int64_t>(high) << 32 | (low & ~15u)), raw[kt]);
      coming |= low & 1 ? 0u : 1u << kt;
    }
  };
  int turn = 0;
  issue(0, turn);
  fetch(begin);
  for (uint32_t four = begin; four < end; four += 4 * kKeys) {
    const uint32_t at = four + wave * kKeys, there = coming;
    const bool all = at + kKeys <= c.length && there == (1 << KT) - 1;
    u32x4_t keys[KT][KS];
    f32x4_t sums[KT];
    float before[KT];  // the weights that lanes 0 to 3 of each 16 add to
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      sums[kt] = f32x4_t{0, 0, 0, 0};
      ops.put(place, raw[kt]);
      ops.get(place, keys[kt]);
    }
    for (int group = 0; group < groups; ++group, turn ^= 1) {
      // The queries of this group were sent before the loads of the next keys and weights.
      if (group == 1)
        wait_vmcnt<KT * KS + KT>();
      else
        wait_vmcnt<0>();
      wait_lds_reads();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (group + 1 < groups)
        issue(group + 1, turn ^ 1);
      else if (four + 4 * kKeys < end)
        issue(0, turn ^ 1);
      if (group == 0) {
        fetch(four + 4 * kKeys);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) before[kt] = weights[min(at + 16 * kt + 4 * quad + min(col, 3), c.n - 1)];
      }
      const uint8_t* queries_now = queries[turn];
      auto multiply = [&](int i, f32x4_t (&s)[KT]) {
        u32x4_t q[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) q[s] = *reinterpret_cast<const u32x4_t*>(queries_now + (i * KS + s) * 1024 + lane * 16);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) s[kt] = Ops::scores(keys[kt], q);
      };
      auto add = [&](const f32x4_t (&s)[KT], float from) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sums[kt][e] += __builtin_amdgcn_exp2f(fmaf(s[kt][e], a.log2_scale, -from));
      };
      float ready[kTiles], most = 0.0f;
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        ready[i] = *reinterpret_cast<const float*>(queries_now + kQueries + (16 * i + col) * 4);
        most = fmaxf(most, ready[i]);
      }
      if (all && (group + 1) * kTiles <= tiles && !__any(most == INFINITY)) {
        // Every row sees every key: the exponentials of a tile beside the products of the next.
        f32x4_t s[KT], next[KT];
        multiply(0, s);
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          if (i + 1 < kTiles) multiply(i + 1, next);
          add(s, ready[i]);
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) s[kt] = next[kt];
        }
        continue;
      }
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        const int tile = group * kTiles + i;
        if (tile >= tiles) break;
        f32x4_t s[KT];
        multiply(i, s);
        if (!all || __any(ready[i] == INFINITY)) {
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            const uint32_t seen = !(there >> kt & 1) || ready[i] == INFINITY
                                      ? 0u : Ops::seen(a, c, b, min(16 * tile + col, a.rows - 1) / a.group, at + 16 * kt);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!(seen >> (4 * quad + e) & 1)) s[kt][e] = -INFINITY;
          }
        }
        add(s, ready[i] == INFINITY ? 0.0f : ready[i]);  // every score is -infinity there
      }
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      float v = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float sum = sum_of_16(sums[kt][i]);
        if (col == i) v = sum;
      }
      const uint32_t n = at + 16 * kt + 4 * quad + col;
      if (col < 4 && n < c.n) weights[n] = n < c.length ? before[kt] + v : v;
    }
  }
}

// Tiles of 16 rows that a wave of stats_kernel holds beside its keys, at most.
constexpr int most_tiles(int pieces) { return pieces <= 4 ? 4 : pieces <= 8 ? 2 : 1; }

template <typename T, int KS, int RT>
void launch_stats(const WeightArgs& a, dim3 grid, hipStream_t stream) {
  if constexpr (RT > 1 || most_tiles(KS) < 4) {  // more than 64 rows take two tiles or more
    if (a.over_rows) {
      hipLaunchKernelGGL((stats_kernel<T, KS, RT, false, true>), grid, dim3(256), 0, stream, a);
      return;
    }
  }
  hipLaunchKernelGGL((stats_kernel<T, KS, RT, false, false>), grid, dim3(256), 0, stream, a);
}

constexpr int64_t kMaxInt = 2147483647;
// Workgroups of a round: what of each kernel runs at once, four, two and three to
// a CU. Stats with kept scores, 32 sequences of one token over up to 4096: 512
// 55.7 us, 1024 47.6, 1280 49.5.
// More rows, 32 tokens of four sequences over up to 16384: stats and gathering
// in rounds of 512 and 768 80.8 us, 256 and 512 96.9, 1024 and 1536 93.8.
constexpr int64_t kKeepRound = 1024, kStatsRound = 512, kGatherRound = 768;

template <typename T, int KS>
hipError_t launch(const WeightArgs& a, int64_t units, hipStream_t stream) {
  const int64_t kv = a.p.cache.kv_heads, sequences = a.p.batch.sequences;
  const int64_t stats_blocks = (kv * (a.pieces + sequences) + 7) / 8 * 8 * a.row_groups;
  const int64_t gather_blocks = kv * (a.gather_pieces + sequences);
  if (stats_blocks > kMaxBlocks || gather_blocks > kMaxBlocks || units * a.blocks > kMaxBlocks) return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(stats_blocks));
  const dim3 along(static_cast<unsigned>(units * a.blocks));
  if (a.scores != nullptr) {
    hipLaunchKernelGGL((stats_kernel<T, KS, 1, true, false>), grid, dim3(256), 0, stream, a);
    hipLaunchKernelGGL(sum_kernel, along, dim3(256), 0, stream, a);
    return hipGetLastError();
  }
  if (a.tiles == 1) launch_stats<T, KS, 1>(a, grid, stream);
  if constexpr (most_tiles(KS) >= 2) {
    if (a.tiles == 2) launch_stats<T, KS, 2>(a, grid, stream);
  }
  if constexpr (most_tiles(KS) >= 4) {
    if (a.tiles == 4) launch_stats<T, KS, 4>(a, grid, stream);
  }
  const int64_t packs = (units * ((a.rows + 15) / 16) + 3) / 4, ready_blocks = packs + units * ((a.row_slots + 255) / 256);
  if (ready_blocks > kMaxBlocks) return hipErrorInvalidValue;
  hipLaunchKernelGGL((ready_kernel<T, KS>), dim3(static_cast<unsigned>(ready_blocks)), dim3(256), 0, stream, a, packs);
  hipLaunchKernelGGL((gather_kernel<T, KS>), dim3(static_cast<unsigned>(gather_blocks)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace
}  // namespace attention

hipError_t attention_weights_launch(const AttentionProblem& p, float* weights, const Launch& l) {
  using namespace attention;
  const bool half = p.cache.dtype == AFFON_ROCM_BF16;
  WeightArgs a{};
  a.p = p;
  a.group = p.heads / p.cache.kv_heads;
  const int64_t rows = static_cast<int64_t>(p.batch.rows) * a.group;
  if (rows > (int64_t(1) << 30)) return hipErrorInvalidValue;
  a.rows = static_cast<int>(rows);
  a.row_slots = (a.rows + 63) / 64 * 64;
  const int pieces = (p.cache.head_dim * (half ? 2 : 4) + 63) / 64;
  int held = half ? 2 : 4;  // pieces of the instance that takes them
  while (held < pieces) held += held % 3 == 0 ? held / 3 : held > 2 ? held / 2 : 1;
  a.tiles = 1;
  a.over_rows = a.rows > 16 * most_tiles(pieces);
  const int side = a.over_rows ? 64 : 16;  // rows of a workgroup for each tile of a wave
  while (a.tiles < most_tiles(pieces) && side * a.tiles < a.rows) a.tiles *= 2;
  a.row_groups = (a.rows + side * a.tiles - 1) / (side * a.tiles);
  a.log2_scale = p.scale == 0.0f ? 1.0f : std::min(std::fabs(p.scale) * 1.44269504088896340736f, FLT_MAX);
  a.sign = p.scale > 0.0f ? 1.0f : p.scale < 0.0f ? -1.0f : 0.0f;
  a.weights = weights;
  const int64_t units = static_cast<int64_t>(p.batch.sequences) * p.cache.kv_heads;
  const int64_t capacity = p.batch.capacity;
  // One round of workgroups, or two for every key head and sequence.
  auto pieces_for = [&](int64_t round, int64_t groups) {
    const int64_t least = 2 * static_cast<int64_t>(p.batch.sequences);
    return static_cast<int>(std::min<int64_t>(std::max(round / (p.cache.kv_heads * groups), least), kMaxInt / 2));
  };
  a.pieces = pieces_for(a.rows <= 16 ? kKeepRound : kStatsRound, a.row_groups);
  a.gather_pieces = pieces_for(kGatherRound, 1);
  const size_t stats = (static_cast<size_t>(a.pieces + p.batch.sequences) * p.cache.kv_heads * a.rows * sizeof(float2) + 255) / 256 * 256;
  // Up to 16 rows' scores are kept, where they find room: 32 sequences of up to
  // 4096 tokens 49 us with 4 rows of a key head, 52 with 8 and 59 with 16, and
  // 81 to 83 where they are computed again. More are more to write and read than
  // the keys (bf16 heads of 128: 4 bytes a row each way, against 256). The lengths
  // are on the device, so the room is for all tokens that the table could hold.
  constexpr size_t kMostScores = size_t(1) << 30;
  const size_t scores = static_cast<size_t>(units) * a.rows * capacity * sizeof(float);
  uint8_t* scratch = nullptr;
  if (a.rows <= 16 && scores <= kMostScores) scratch = static_cast<uint8_t*>(l.scratch(stats + scores));
  if (scratch != nullptr) {
    a.scores = reinterpret_cast<float*>(scratch + stats);
  } else {
    const size_t ready = (static_cast<size_t>(units) * a.row_slots * sizeof(float) + 255) / 256 * 256;
    scratch = static_cast<uint8_t*>(l.scratch(stats + ready + static_cast<size_t>(units) * ((a.rows + 15) / 16) * 1024 * held));
    if (scratch == nullptr) return hipErrorOutOfMemory;
    a.ready = reinterpret_cast<float*>(scratch + stats);
    a.packed = reinterpret_cast<u32x4_t*>(scratch + stats + ready);
  }
  a.stats = reinterpret_cast<float2*>(scratch);
  a.blocks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(2048 / units, (capacity + 1023) / 1024)));
  switch (held) {
    case 2: return launch<BF16, 2>(a, units, l.stream);
    case 3: return launch<BF16, 3>(a, units, l.stream);
    case 4: return half ? launch<BF16, 4>(a, units, l.stream) : launch<F32, 4>(a, units, l.stream);
    case 6: return half ? launch<BF16, 6>(a, units, l.stream) : launch<F32, 6>(a, units, l.stream);
    case 8: return half ? launch<BF16, 8>(a, units, l.stream) : launch<F32, 8>(a, units, l.stream);
    case 12: return launch<F32, 12>(a, units, l.stream);
    default: return launch<F32, 16>(a, units, l.stream);
  }
}

}  // namespace affon
