// Which run of rows a place belongs to (attn_read.hip, attn_prompt.hpp).
#pragma once

#include "attn_internal.hpp"

namespace attn {

// The last of `runs` places of(0) <= of(1) <= ... that is at most `at`, by a whole wave, 64 of
// them at a time; `runs` where there is none.  Places that decrease give some run, never one
// out of range.
template <class F>
__device__ __forceinline__ uint32_t find_run(uint32_t runs, uint32_t at, F of) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = 0, n = runs;
    while (n > 1) {
        const uint32_t step = (n + 63) / 64, mine = lane * step;
        const uint64_t upto = __ballot(mine < n && of(lo + mine) <= at);
        if (!upto) return runs;
        const uint32_t last = 63 - (uint32_t)__clzll((long long)upto);
        lo += last * step;
        n = min(step, n - last * step);
    }
    return lo;
}

}  // namespace attn
