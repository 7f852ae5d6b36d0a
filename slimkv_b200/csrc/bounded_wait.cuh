// Waits of a pipeline within one CTA that end at a limit.
//   Bars: int abort, set by the first wait that runs out (the others end with it)
//   Job:  uint64_t wait_ns, unsigned int* status
#pragma once

#include "common.cuh"

namespace slimkv {

// A try_wait keeps the thread for 4 us whatever its hint says (measured for hints
// of 1 ns to 1 ms), so limits below some of those are polled.
constexpr uint64_t kPollBelowNs = 20000;

// A wait that is over costs one test; one that is not looks for an abort of
// another warp and for its limit.
template <class Bars, class Job>
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, Bars* bs, const Job& J) {
    if (mbar_test(bar, parity)) return true;
    uint64_t start = 0;
    for (bool first = true;; first = false) {
        if (J.wait_ns < kPollBelowNs ? mbar_test(bar, parity) : mbar_try(bar, parity)) return true;
        if (first) {
            start = global_timer_ns();
        } else {
            if (*const_cast<volatile int*>(&bs->abort)) return false;
            if (global_timer_ns() - start > J.wait_ns) break;
        }
    }
    bs->abort = 1;
    report(J.status, SLIMKV_DEVICE_TIMEOUT);
    return false;
}
__device__ __forceinline__ bool all_lanes(bool x) { return __all_sync(0xffffffffu, x); }
template <class Bars, class Job>
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, Bars* bs, const Job& J) {
    return all_lanes(wait_bar(bar, parity, bs, J));
}

}  // namespace slimkv
