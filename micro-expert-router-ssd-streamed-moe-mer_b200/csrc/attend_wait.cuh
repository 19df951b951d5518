// Bounded waits of the attention kernels, and the way out after one that has run out: the CTA stops as a whole, and ends only when the copies that it has
// in flight have landed (or a second limit is over), so that none of them lands in the shared memory of the SM's next CTA.
#pragma once

#include <stdint.h>

#include "../../include/mer_b200.h"
#include "ptx.cuh"

namespace {

constexpr uint64_t DRAIN_NS = 100000000ull;

// For whole warps, which stay together whatever comes of it: whether the phase is complete.  If it does not come within the limit, `stop` is set, and every other
// wait of the CTA for something that has not come ends as well.
__device__ __forceinline__ bool wait_or_stop(uint64_t *bar, uint32_t parity, volatile uint32_t *stop, uint32_t *status) {
  const bool ok = mbar_wait(bar, parity, stop);
  if (!ok && !*stop) {
    *stop = 1;
    atomicOr(status, MER_DEVSTAT_TIMEOUT);
  }
  return __all_sync(0xFFFFFFFFu, ok) != 0;
}
// Copies that a barrier counts, in whatever phase it is: the wait for the other one returns at once.
__device__ __forceinline__ void drain_copies(uint64_t *bar) {
  mbar_drain(bar, 0, DRAIN_NS);
  mbar_drain(bar, 1, DRAIN_NS);
}

}  // namespace
