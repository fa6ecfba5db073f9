// Status codes of the block-FP8 operators, and the waits of their kernels, all of which end.
#pragma once
#include <cstdint>
#include "barriers.cuh"

namespace mono {
namespace lin {

enum Status : uint32_t {
  kBadExpert = 1,                            // expert id past the last expert
  kBadOffsets = 2,                           // offsets out of order or outside the rows
  kBadToken = 3,                             // row outside the rows that there are
  kBadPosition = 4,                          // position outside the partial rows
  kWaitTimeout = 5,
};

__device__ __forceinline__ void report(uint32_t* status, uint32_t code, uint32_t where) {
  if (atomicCAS(status, 0u, code) == 0u) status[1] = where;
}

// Phase `parity` of a barrier. One that does not come is reported, and from then on a wait of the CTA is one poll: every role runs
// through its loop, whatever is in memory, and the launch ends. The clock is only read once in 64 polls.
constexpr uint64_t kWaitNs = 2000000000ull;
struct Waits {
  uint32_t* stop;                            // of the CTA, in shared memory
  uint32_t* status;
  uint64_t limit = kWaitNs;
  // By whole warps.
  __device__ __forceinline__ bool stopped() const { return __any_sync(0xFFFFFFFFu, *static_cast<volatile uint32_t*>(stop) != 0u); }
  __device__ __forceinline__ bool gave_up(uint32_t polls, uint64_t& since) const {
    volatile uint32_t* s = stop;
    if (*s) return true;
    if ((polls & 63u) != 0u) return false;
    const uint64_t now = globaltimer_ns();
    if (since == 0) since = now;
    if (now - since <= limit) return false;
    report(status, kWaitTimeout, blockIdx.x);
    *s = 1u;
    return true;
  }
  // By one lane alone, or lane by lane: a phase's end may be seen by one lane and not yet by another.
  __device__ __forceinline__ void wait_lane(uint64_t* bar, uint32_t parity) const {
    uint64_t since = 0;
    for (uint32_t polls = 1; !mbar_try_wait(bar, parity) && !gave_up(polls, since); ++polls) {}
  }
  // By whole warps, which are together behind it.
  __device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity) const {
    wait_lane(bar, parity);
    __syncwarp();
  }
  // Two barriers, looked at together: each look takes some hundred cycles, ready or not. What follows a lane's own look is without
  // operations of the whole warp up to the one at the end.
  __device__ __forceinline__ void wait(uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb) const {
    const bool first = mbar_test(a, pa), second = mbar_test(b, pb);
    if (!first) wait_lane(a, pa);
    if (!second) wait_lane(b, pb);
    __syncwarp();
  }
  __device__ __forceinline__ void wait_warp(uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb) const {
    const bool first = mbar_test(a, pa), second = mbar_test(b, pb);
    if (__all_sync(0xFFFFFFFFu, first && second)) return;
    wait_warp(a, pa);
    wait_warp(b, pb);
  }
  // For what the other CTAs of the cluster send, by whole warps. They run through their roles and send it, whether they gave up or not; so a CTA that gave up
  // waits too, and does not end, its shared memory with it, before all that has come. Four limits are enough for each of them to give up.
  __device__ __forceinline__ void wait_sent(uint64_t* bar, uint32_t parity) const {
    uint64_t since = 0;
    for (uint32_t polls = 1; !mbar_try_wait(bar, parity); ++polls) {
      if ((polls & 63u) != 0u) continue;
      const uint64_t now = globaltimer_ns();
      if (since == 0) since = now;
      if (now - since <= 4 * limit) continue;
      report(status, kWaitTimeout, blockIdx.x);
      *static_cast<volatile uint32_t*>(stop) = 1u;
      break;
    }
    __syncwarp();
  }
  // With a result that the compiler sees to be the same for the whole warp: the warp that issues the products stays in uniform
  // control flow, its descriptors in uniform registers.
  __device__ __forceinline__ void wait_warp(uint64_t* bar, uint32_t parity) const {
    uint64_t since = 0;
    for (uint32_t polls = 1; !__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity)); ++polls)
      if (__any_sync(0xFFFFFFFFu, gave_up(polls, since))) break;
  }
};
// Time for what a CTA that gave up has in flight; it takes microseconds.
__device__ __forceinline__ void settle() {
  const uint64_t t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 < 200000) __nanosleep(10000);
}

}  // namespace lin
}  // namespace mono
