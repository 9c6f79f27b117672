// Runs csrc/wait_rules.h's long wait against barriers that nobody completes, on a clock of its own: two CTAs of a
// pair whose leader gives up while the follower has nothing left to load.
#include <cstdio>
#include <initializer_list>

#include "../robot-agent_b200/csrc/wait_rules.h"

static const uint64_t ONCE = 200000000ull, LIMIT = 60000000000ull;   // ns

struct Cta {
  int failed = 0;
};

int main() {
  // 1. the phase ends after some bounded waits: true, whatever their number below the limit
  for (int n : {0, 1, 7, 250}) {
    uint64_t clock = 5;
    int left = n;
    Cta c;
    const bool ok = wait_long([&] { clock += ONCE; return left-- == 0; }, [&] { return c.failed != 0; }, [&] { return clock; }, LIMIT);
    if (!ok) return printf("a phase that ends after %d waits was given up\n", n), 1;
  }
  // 2. the leader gives up at some time and tells both CTAs: the follower's wait ends at its next look
  for (uint64_t when : {ONCE / 2, 3 * ONCE, 40 * ONCE}) {
    uint64_t clock = 0;
    Cta pair[2];
    int tries = 0;
    const bool ok = wait_long(
        [&] {
          clock += ONCE;
          ++tries;
          if (clock >= when) pair[0].failed = pair[1].failed = 1;   // what pr_fail does
          return false;
        },
        [&] { return pair[1].failed != 0; }, [&] { return clock; }, LIMIT);
    if (ok || clock > when + 2 * ONCE) return printf("the follower waited on (%d tries)\n", tries), 1;
  }
  // 3. nobody tells it: the wait still ends
  uint64_t clock = 0;
  long tries = 0;
  const bool ok = wait_long([&] { clock += ONCE; return ++tries > 100000; }, [] { return false; }, [&] { return clock; }, LIMIT);
  if (ok || clock > LIMIT + 3 * ONCE) return printf("a wait without a signal did not end\n"), 1;
  printf("ok\n");
  return 0;
}
