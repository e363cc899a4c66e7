// The bounded waits of the tcgen05 kernels, whose roles share the SM's instruction cache: short code, no clock but the producer's.
#pragma once
#include "common.cuh"

namespace b200 {

// How long the hardware suspends a failed test is its own affair, so a count of tests is a limit but not one in time.  The time
// limit is the producer's, on the low word of the clock: it sets the abort flag, which every other wait looks at after a
// failed test.  That bounds them all: whatever hangs stops the ring that the producer waits for, and at the end the producer
// waits until every role has taken the end marker, which it does when it is through with all items.
constexpr int kT2WaitLimit = 1 << 22;
__device__ __forceinline__ bool t2_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
#pragma unroll 1
  for (int n = 0; n < kT2WaitLimit; ++n) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
  }
  *abort_flag = 1;
  return false;
}
__device__ __forceinline__ uint32_t t2_clock() {
  uint32_t c;
  asm volatile("mov.u32 %0, %%clock;" : "=r"(c));
  return c;
}
__device__ __forceinline__ bool t2_wait_timed(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  const uint32_t t0 = t2_clock();
#pragma unroll 1
  while (!mbar_try_wait(bar, parity)) {
    if (*abort_flag) return false;
    if (t2_clock() - t0 > static_cast<uint32_t>(kSpinLimitCycles)) {
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}
// On the S -> softmax -> PV chain: the second test does not come behind a look at the flag (long sequences lose 3 % to it).
__device__ __forceinline__ bool t2_wait_hot(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return mbar_try_wait(bar, parity) || t2_wait(bar, parity, abort_flag);
}

}  // namespace b200
