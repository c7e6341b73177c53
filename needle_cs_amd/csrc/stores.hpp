// stores.hpp -- stores of fp32 results that no cache keeps until they are read.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace nhip {

typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));

// away: past the caches, for results of 32 MB and more (stored_away).  Where all
// a pass touches comes from memory, 4099 rows of 4096 normed and read back take
// 57.2 us so and 67.0 by ordinary stores, 8185 rows of 40 heads of 128 rotated
// 57.9 and 62.3; a residual stream that the last cache holds, normed in place
// with what comes from codes, 16.8 and 16.5 for 16.8 MB, 28.8 and 29.1 for 33.6,
// 52.2 and 51.6 for 67, 96.6 and 102 for 134.  Each instruction has to write
// whole lines: with two fours side by side a lane, by two, the rotation took 74.7.
__device__ __forceinline__ void store_f4(float* to, f4 v, bool away)
{
    if (away) {
        asm volatile("");  // (or the compiler makes one store, of the other kind, of the two)
        __builtin_nontemporal_store(v, reinterpret_cast<f4*>(to));
        asm volatile("");
    } else
        *reinterpret_cast<f4*>(to) = v;
}

inline bool stored_away(int64_t elements) { return elements >= 1 << 23; }

}  // namespace nhip
