// Bounded waits, and what a kernel whose wait gave up does before it leaves:
// its own copies and products in flight write to shared and tensor memory that the
// next CTA gets.  Plain C++ over mbar_try_wait and globaltimer_ns (common.cuh).
#pragma once

namespace tg {

// Bounded wait for the phase with the given parity to complete.  Returns false
// (and ORs `err` into the device status) if it did not complete in time.
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, unsigned int err) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = globaltimer_ns();
  for (;;) {
    for (int i = 0; i < 64; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (globaltimer_ns() - t0 > kWaitLimitNs) {
      atomicOr(&g_device_status, err);
      return false;
    }
  }
}

// The loads of a ring of `stages` slots land: the last of the `issued` ones, one
// a slot in turn.  Each has the full limit, also after another role gave up.
__device__ __forceinline__ void ring_drain(uint64_t* full_bar, int issued, int stages, unsigned int err) {
  for (int i = issued > stages ? issued - stages : 0; i < issued; ++i)
    mbar_wait(&full_bar[i % stages], uint32_t(i / stages) & 1u, err);
}

// Waits out the limit: what this CTA has in flight after a wait gave up has landed
// by then, or never will.  For loads and products that complete on another CTA's
// barriers, or on barriers that were not told of them.
__device__ __forceinline__ void wait_out() {
  const unsigned long long t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 <= kWaitLimitNs) {
  }
}

}  // namespace tg
