// Division by a number that is known when a kernel is launched, as a multiplication: n / d = (n m / 2^32 + n) / 2^k with k = ceil(log2 d) and
// m = 2^32 (2^k - d) / d + 1 (Granlund and Montgomery, Division by invariant integers using multiplication, 1994).
#pragma once

#include <stdint.h>

namespace splat {

struct FastDiv {               // n / d for 0 <= n < 2^31
    uint32_t mul, shift, d;
    FastDiv() = default;
    explicit FastDiv(uint32_t d_) : d(d_) {
        shift = 0;
        while ((1ull << shift) < d) ++shift;
        mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
    }
    __device__ __forceinline__ int div(int n) const { return (int)((__umulhi(mul, (uint32_t)n) + (uint32_t)n) >> shift); }
    __device__ __forceinline__ int div_floor(int n) const { return n >= 0 ? div(n) : -1 - div(-1 - n); }
};

}  // namespace splat
