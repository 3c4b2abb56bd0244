// Bounded waits of the 8-bit decoder layer's kernels.
#pragma once

#include "tcgen05_common.cuh"

namespace mlel {

// tc::mbarWait without the suspension between checks.
__device__ __forceinline__ bool mbarPoll(uint64_t *bar, uint32_t parity, int code) {
    if (tc::mbarTryWait(bar, parity)) {
        return true;
    }
    const long long start = clock64();
    unsigned polls = 0;
    while (!tc::mbarTryWait(bar, parity)) {
        if ((++polls & 63u) == 0 && clock64() - start > tc::kWaitLimitCycles) {
            atomicCAS(&tc::g_tcgen05Error, 0, code);
            return false;
        }
    }
    return true;
}
// The same for a warp that goes on as a whole.
__device__ __forceinline__ bool mbarPollWarp(uint64_t *bar, uint32_t parity, int code) {
    return __all_sync(0xffffffffu, mbarPoll(bar, parity, code)) != 0;
}

} // namespace mlel
