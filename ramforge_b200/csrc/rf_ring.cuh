// rf_ring.cuh - waits on the mbarriers of a ring in shared memory that give up after about a second
// and report through the verification error word.
#pragma once
#include "rf_tc.cuh"
#include "rf_verify.h"

namespace rf {

// Bounded wait for the phase of `bar` with `parity`; false once any wait of the CTA gave up.
static __device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t parity, volatile uint32_t* stop, unsigned* err) {
  const long long t0 = clock64();
  while (!tc_mbar_try_wait(bar, parity)) {
    if (*stop) return false;
    if (clock64() - t0 > 2000000000LL) {
      *stop = 1;
      atomicOr(err, kVerifyTimeout);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile uint32_t* stop, unsigned* err) {
  const uint32_t b = tc_smem_u32(bar);
  return tc_mbar_try_wait(b, parity) || wait_slow(b, parity, stop, err);
}
// The same by a whole warp, one answer for all of it: a phase may end between two lanes' last looks, and a warp that works as one
// afterwards (shuffles, tensor memory, tcgen05) must not part there.
__device__ __forceinline__ bool wait_bar_warp(uint64_t* bar, uint32_t parity, volatile uint32_t* stop, unsigned* err) {
  return __all_sync(0xffffffffu, wait_bar(bar, parity, stop, err));
}

}  // namespace rf
