// The smallest key of a range at which a condition holds, for the sampling kernel and, without CUDA, for host tests of it.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define SA2_KEYS_FN __host__ __device__ __forceinline__
#else
#define SA2_KEYS_FN inline
#endif

namespace sa2 {
namespace sample {

// The smallest key of [0, best] at which `stays` holds.  It holds at `best`, and at all keys of the range above one at which it holds.  `near` is a
// guess, mostly off by a key or two: steps from it double, then halve.  At most 64 keys are looked at, wherever the answer lies: next
// to a logit of 0 it can be 2^30 keys from any guess, since (double)v - best is the same for all smaller |v|.
template <typename F> SA2_KEYS_FN uint32_t first_key(uint32_t best, uint32_t near, F stays) {
    uint32_t low = 0u, high = near < best ? near : best;         // the answer is in [low, high]
    if (stays(high)) {
        for (uint32_t step = 1u; low < high; step = step < 1u << 30 ? 2u * step : step) {
            const uint32_t x = high - (step < high ? step : high);
            if (!stays(x)) {
                low = x + 1u;
                break;
            }
            high = x;
        }
    } else {
        low = high + 1u;
        high = best;
        for (uint32_t step = 1u; low < high; step = step < 1u << 30 ? 2u * step : step) {
            const uint32_t x = step - 1u < high - low ? low + (step - 1u) : high - 1u;
            if (stays(x)) {
                high = x;
                break;
            }
            low = x + 1u;
        }
    }
    while (low < high) {
        const uint32_t x = low + (high - low) / 2u;
        if (stays(x)) high = x;
        else low = x + 1u;
    }
    return high;
}

}  // namespace sample
}  // namespace sa2
