// Prefixes of groups, cut as the kernels do: they find room in the pieces that the
// workspace has, which are no more than what some prefixes need.
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

#include "prefix_cut.h"

using namespace affon;

int64_t pieces_of(const std::vector<uint32_t>& tokens, uint32_t chunk) {
  int64_t sum = 0;
  for (uint32_t n : tokens) sum += cut_pieces(n, chunk);
  return sum;
}

int main() {
  std::mt19937_64 rng(7);
  int wrong = 0;
  for (int groups : {1, 2, 3, 5, 64, 65, 200})
    for (int splits : {1, 2, 3, 7, 32, 256}) {
      const int64_t room = cut_most(groups, splits);
      // One piece a group needs no more.
      if (splits == 1 && room != groups && ++wrong <= 5)
        std::printf("%d groups in one piece each have room for %lld\n", groups, static_cast<long long>(room));
      int64_t most = 0;
      for (int trial = 0; trial < 400; ++trial) {
        const uint32_t top = trial < 100 ? 64 : trial < 300 ? 4096 : 0x7fff0000u;
        std::vector<uint32_t> tokens(groups);
        uint64_t all = 0;
        for (uint32_t& n : tokens) all += n = static_cast<uint32_t>(rng() % (uint64_t(top) * (trial % 3 + 1) / 64 + 1)) * 64 % 0x7fffffc0u;
        const uint32_t longest = *std::max_element(tokens.begin(), tokens.end());
        const uint32_t pieces = static_cast<uint32_t>(splits) * groups;
        uint32_t chunk = splits == 1 ? std::max(longest, 1u) : cut_chunk(all, pieces, 32);
        for (int i = 0; i <= 16; ++i) {
          const int64_t have = pieces_of(tokens, chunk);
          most = std::max(most, have);
          if (have > room && ++wrong <= 5)
            std::printf("%d groups, %d splits: %lld pieces of %lld\n", groups, splits, static_cast<long long>(have),
                        static_cast<long long>(room));
          if (splits == 1) break;
          chunk = cut_longer(chunk, 32);
        }
      }
      // Short prefixes beside a long one that fills its pieces need all the room.
      if (splits > 1) {
        std::vector<uint32_t> tokens(groups, 64);
        tokens[0] = static_cast<uint32_t>(splits) * groups * 16384 - 64 * (groups - 1);
        const uint32_t chunk = cut_chunk(static_cast<uint64_t>(splits) * groups * 16384, static_cast<uint32_t>(splits) * groups, 32);
        most = std::max(most, pieces_of(tokens, chunk));
      }
      if (room > most && ++wrong <= 5)
        std::printf("%d groups, %d splits: room for %lld, %lld needed\n", groups, splits, static_cast<long long>(room),
                    static_cast<long long>(most));
    }
  return wrong != 0;
}
