// Division by a number known at launch (compiles without HIP).
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define JAMHIP_BOTH __host__ __device__
#else
#define JAMHIP_BOTH
#endif

namespace jamhip {

// n / d for 0 <= n < 2^31 by a multiplication: mul = ceil(2^(31 + s) / d) with 2^(s - 1) < d <= 2^s, whose excess over the
// true ratio is below 2^-31 per unit of n.
struct FastDiv {
    uint32_t mul = 0x80000000u;
    int shift = 31;
    int d = 1;
    FastDiv() = default;
    explicit FastDiv(int div) : d(div) {
        int s = 0;
        while ((int64_t(1) << s) < div) s++;
        shift = 31 + s;
        mul = (uint32_t) (((uint64_t(1) << shift) + div - 1) / div);
    }
    JAMHIP_BOTH int div(int n) const { return (int) (((uint64_t) (uint32_t) n * mul) >> shift); }
};

}  // namespace jamhip
