// When a waiting role of a kernel gives up.  Plain C++ over what the kernel hands in, so that the rule also
// runs on the host.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define WAIT_FN __device__ __forceinline__
#else
#define WAIT_FN inline
#endif

// A wait that may rightly last as long as a whole tile.  `once` is one bounded wait (true: the phase is over), `failed`
// whether any role that the phase depends on has given up, `now` a clock in ns.  False when one of them
// has, or when `limit` ns have gone by since the first bounded wait ran out: it ends whatever the others do.
template <typename Once, typename Failed, typename Now>
WAIT_FN bool wait_long(Once once, Failed failed, Now now, uint64_t limit) {
  if (once()) return true;
  const uint64_t t0 = now();
  while (!failed() && now() - t0 <= limit)
    if (once()) return true;
  return false;
}
