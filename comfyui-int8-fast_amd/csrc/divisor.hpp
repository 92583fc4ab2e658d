// Division by a number that a launch knows.
#pragma once

#include <stdint.h>

#include <hip/hip_runtime.h>

namespace i8f {

// Division of a number below 2^31 by a fixed one: with 2^(s-1) < d <= 2^s and m = floor(2^(31+s) / d) + 1 the product is too large by less
// than a d-th.
struct Divisor {
    uint32_t m, s;
    Divisor(uint32_t d = 1) : s(d > 1 ? 32 - __builtin_clz(d - 1) : 0) { m = (uint32_t)((1ull << (31 + s)) / d + 1); }
    __device__ __forceinline__ uint32_t operator()(uint32_t x) const { return (uint32_t)(((uint64_t)x * m) >> (31 + s)); }
};

}  // namespace i8f
