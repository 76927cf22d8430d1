// Every width and number of shares of a join: a thread that adds shares up reads
// entries of its own row and head only, inside the workgroup's arrays.
#include <cstdio>

#include "join_thread.h"

using affon::JoinThread;
using affon::kJoinThreads;

int main() {
  int wrong = 0;
  for (int pieces = 1; pieces <= kJoinThreads; ++pieces)
    for (int shares = 1; pieces * shares <= kJoinThreads; ++shares) {
      const int per = kJoinThreads / (pieces * shares);
      int sums = 0;
      for (int t = 0; t < kJoinThreads; ++t) {
        const JoinThread thread(t, pieces, shares);
        if (thread.per != per || thread.holds() != (t < per * pieces * shares)) ++wrong;
        if (!thread.adds_up()) continue;
        ++sums;
        for (int s = 0; s < shares; ++s) {
          const int at = t + s * pieces;
          if (at >= kJoinThreads) {
            if (++wrong <= 5) std::printf("pieces %d shares %d: thread %d reads entry %d\n", pieces, shares, t, at);
            continue;
          }
          const JoinThread from(at, pieces, shares);
          if (!from.holds() || from.local != thread.local || from.piece != thread.piece || from.share != s) ++wrong;
        }
      }
      if (sums != per * pieces) ++wrong;
    }
  if (wrong) std::printf("%d wrong\n", wrong);
  return wrong != 0;
}
