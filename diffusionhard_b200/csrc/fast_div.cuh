// fast_div.cuh -- division of indexes by a number that the host knows.
#pragma once

#include <stdint.h>

namespace dh {

// Division by d of any n < 2^31: with 2^s >= d and m = floor(2^32 (2^s - d) / d) + 1
// the quotient is (floor(m n / 2^32) + n) / 2^s.
struct FastDiv {
    uint32_t d = 1, m = 1, s = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t by) : d(by) {
        while ((1ull << s) < d) ++s;
        m = static_cast<uint32_t>((((1ull << s) - d) << 32) / d + 1);
    }
    __device__ __forceinline__ uint32_t of(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
    // the quotient; n becomes the remainder
    __device__ __forceinline__ uint32_t split(uint32_t& n) const {
        const uint32_t q = of(n);
        n -= q * d;
        return q;
    }
};

}  // namespace dh
