// The counters of a session's launches (Workspace::tickets) against the
// stand-in HIP runtime: launches that a graph may replay at any time get none.
#include <cstdio>

#include "memory.h"

#define CHECK(x)                                        \
  do {                                                  \
    if (!(x)) {                                         \
      std::printf("%s:%d: %s\n", __FILE__, __LINE__, #x); \
      return 1;                                         \
    }                                                   \
  } while (0)

int main() {
  {
    affon::Workspace w(0, nullptr);
    bool fresh = true;
    fake::session_capturing = true;
    CHECK(w.tickets(&fresh) == nullptr && !fresh && fake::blocks.empty());
    fake::session_capturing = false;
    uint32_t* words = w.tickets(&fresh);
    CHECK(words != nullptr && fresh && fake::blocks.at(words) == affon::Workspace::kTickets * sizeof(uint32_t));
    fake::session_capturing = true;
    CHECK(w.tickets(&fresh) == nullptr && !fresh);  // though there are some
    fake::session_capturing = false;
    CHECK(w.tickets(&fresh) == words && !fresh);
  }
  CHECK(fake::blocks.empty());
  fake::limit = 1024;
  affon::Workspace w(0, nullptr);
  bool fresh = true;
  CHECK(w.tickets(&fresh) == nullptr && !fresh);
  return 0;
}
