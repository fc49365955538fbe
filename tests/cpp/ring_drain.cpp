// What a kernel that gives up waits for: after any number of fills of a ring of N buffers, of which any subset of the newest
// ones is still under way, the wait for each buffer has to last until its own newest fill is complete, and no longer.
#include <cstdio>

#include "kernels/ring.h"

// An mbarrier whose phases complete one by one: a wait for a parity is over when the phase of that parity is the one that
// completed last (before the first completion, parity 1 counts as completed).
struct Barrier {
  int filled = 0, completed = 0;
  bool answers(unsigned int parity) const { return ((completed - 1) & 1) == static_cast<int>(parity); }
};

template <int N> int failures() {
  int bad = 0;
  for (int fills = 0; fills <= 4 * N + 1; ++fills)
    for (unsigned int open = 0; open < (1u << N); ++open) {
      Barrier b[N];
      afir::kernels::Ring<N> ring;
      for (int i = 0; i < fills; ++i, ring.next()) {
        b[ring.at].completed = b[ring.at].filled;  // a place is filled again after its last fill is complete
        ++b[ring.at].filled;
      }
      for (int s = 0; s < N; ++s) b[s].completed = b[s].filled - ((open >> s & 1u) && b[s].filled ? 1 : 0);
      for (int s = 0; s < N; ++s) {
        const unsigned int parity = afir::kernels::newestFillParity(s, ring.at, ring.phase);
        if (b[s].answers(parity) != (b[s].completed == b[s].filled)) ++bad;
        b[s].completed = b[s].filled;
        if (!b[s].answers(parity)) ++bad;
      }
    }
  return bad;
}

int main() {
  const int bad = failures<1>() + failures<2>() + failures<3>() + failures<4>() + failures<6>();
  std::printf("%d failures\n", bad);
  return bad ? 1 : 0;
}
