// Which thread of a join holds what, for the kernels and for a test on the host.
#pragma once

namespace affon {

// A workgroup of kJoinThreads joins `per` rows and heads, each by `shares` times
// `pieces` threads side by side: a share of its partial results, four
// values of the head to a thread. The threads of share 0 then add up what the
// others left at their own index + s * pieces, s < shares.
constexpr int kJoinThreads = 256;

struct JoinThread {
  int per, local, share, piece;
  constexpr JoinThread(unsigned thread, unsigned pieces, unsigned shares)
      : per(kJoinThreads / (pieces * shares)),
        local(thread / (pieces * shares)),
        share(thread % (pieces * shares) / pieces),
        piece(thread % pieces) {}
  // Whether the thread is one of a whole row and head: threads are left over
  // where pieces * shares does not divide kJoinThreads.
  constexpr bool holds() const { return local < per; }
  constexpr bool adds_up() const { return holds() && share == 0; }
};

}  // namespace affon
