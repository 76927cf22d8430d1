// rows_meet and same_rows (csrc/overlap.h) against a byte map: "seed" random
// pairs of row sets that lie beside, between and in each other.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "overlap.h"

int main(int argc, char** argv) {
  std::mt19937 rng(argc > 1 ? std::atoi(argv[1]) : 1);
  auto pick = [&](int low, int high) { return std::uniform_int_distribution<int>(low, high)(rng); };
  static char memory[4096];
  int meet = 0, apart = 0;
  for (int t = 0; t < 20000; ++t) {
    affon::Rows rows[2];
    int start[2];
    const int shared = pick(0, 30);
    for (int i = 0; i < 2; ++i) {
      const int stride = pick(0, 2) ? shared : pick(0, 30);
      start[i] = pick(0, 60);
      rows[i] = affon::rows_of(memory + start[i], pick(1, 9), pick(1, 12), stride);
    }
    std::vector<bool> mine(4096);
    for (int64_t r = 0; r < rows[0].rows; ++r)
      for (int64_t c = 0; c < rows[0].bytes; ++c) mine[start[0] + r * rows[0].stride + c] = true;
    bool want = false;
    for (int64_t r = 0; r < rows[1].rows; ++r)
      for (int64_t c = 0; c < rows[1].bytes; ++c) want = want || mine[start[1] + r * rows[1].stride + c];
    (want ? meet : apart)++;
    for (int i = 0; i < 2; ++i)
      if (affon::rows_meet(rows[i], rows[1 - i]) != want) {
        std::printf("rows at %d and %d: %lld x %lld / %lld, %lld x %lld / %lld: not %d\n", start[i], start[1 - i],
                    (long long)rows[i].rows, (long long)rows[i].bytes, (long long)rows[i].stride,
                    (long long)rows[1 - i].rows, (long long)rows[1 - i].bytes, (long long)rows[1 - i].stride, want);
        return 1;
      }
    if (!affon::same_rows(rows[0], rows[0])) return 1;
    if (affon::same_rows(rows[0], rows[1]) && !want) return 1;
  }
  const affon::Rows none = affon::rows_of(nullptr, 3, 4, 4);
  if (affon::rows_meet(none, none) || meet < 1000 || apart < 1000) return 1;
  return 0;
}
