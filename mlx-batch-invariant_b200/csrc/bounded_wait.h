// The loop of a bounded wait, free of device code so that the host's compiler takes it too.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define BI_WAIT_FN __device__ __forceinline__
#else
#define BI_WAIT_FN inline
#endif

namespace bi {

// Polls until `ready()`; gives up (false) once `*abort_flag` is set -- the flag may be null: a
// wait that no one calls off -- or `budget` ticks of `now()` after the first look at the clock.
// Flag and clock are looked at every 256th poll.
template <typename Ready, typename Now>
BI_WAIT_FN bool bounded_wait(Ready ready, Now now, const volatile int* abort_flag,
                             long long budget) {
  long long start = 0;
#pragma unroll 1
  for (uint32_t it = 0; !ready(); ++it) {
    if ((it & 255u) == 255u) {
      const long long t = now();
      if (start == 0) start = t;
      if ((abort_flag != nullptr && *abort_flag) || t - start > budget) return false;
    }
  }
  return true;
}

}  // namespace bi
