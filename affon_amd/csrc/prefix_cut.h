// How the prefixes of several groups are cut into pieces, for the kernels, their
// workspace and a test on the host.
#pragma once

#include <cstdint>

namespace affon {

// Whole units past n, where it is whole itself too.
constexpr uint32_t cut_past(uint32_t n, uint32_t unit) { return (n + unit) / unit * unit; }

// Tokens of a piece where `all` tokens, of all groups, go into about `pieces` of them.
constexpr uint32_t cut_chunk(uint64_t all, uint32_t pieces, uint32_t unit) {
  const uint32_t each = all >> 32 != 0 ? static_cast<uint32_t>(all / pieces) : static_cast<uint32_t>(all) / pieces;
  return each == 0 ? unit : cut_past(each - (all == static_cast<uint64_t>(each) * pieces ? 1 : 0), unit);
}
// The next longer one to try, where they are a few too many.
constexpr uint32_t cut_longer(uint32_t chunk, uint32_t unit) { return chunk + cut_past(chunk / 16, unit); }

constexpr uint32_t cut_pieces(uint32_t n, uint32_t chunk) { return n == 0 ? 0u : (n - 1) / chunk + 1; }  // (n + chunk may pass 32 bits)

// Pieces of all groups for a key head, at most, `splits` a group on average.
constexpr int64_t cut_most(int64_t groups, int splits) { return groups * splits + (splits > 1 ? groups - 1 : 0); }

}  // namespace affon
