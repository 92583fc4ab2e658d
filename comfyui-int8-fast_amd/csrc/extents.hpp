// What strided tensors cover in memory, for checks of arguments on the host.
#pragma once

#include <stdint.h>

#include <initializer_list>
#include <utility>

namespace i8f {

// The elements that a strided tensor reaches to from its first one, 0 for one without elements, -1 past 2^58 (so that bytes of them are numbers of 64 bits).
inline int64_t extent(std::initializer_list<std::pair<int64_t, int64_t>> dims) {
    __int128 last = 0;
    for (auto [size, stride] : dims) {
        if (size < 1) return 0;
        last += (__int128)(size - 1) * stride;
    }
    return last >= ((__int128)1 << 58) ? -1 : (int64_t)last + 1;
}

inline bool overlap(const void *a, int64_t na, const void *b, int64_t nb) {
    return na > 0 && nb > 0 && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

}  // namespace i8f
