// stores.hpp -- stores of fp32 results that no cache keeps until they are read.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace nhip {

typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));

// away: past the caches.  Each instruction has to write whole lines: with two
// fours side by side a lane, by two, the rotation took 74.7 in place of 57.9 us.
__device__ __forceinline__ void store_f4(float* to, f4 v, bool away)
{
    if (away) {
        asm volatile("");  // (or the compiler makes one store, of the other kind, of the two)
        __builtin_nontemporal_store(v, reinterpret_cast<f4*>(to));
        asm volatile("");
    } else
        *reinterpret_cast<f4*>(to) = v;
}

// Whether results go past the caches.  us of a chain with the call that reads
// them, away and by ordinary stores, at MB of results:
//   kReadAway, rotated heads and cached rows read back, which the next call reads
//   whole and finds in the last cache (256 MB) up to some 160 MB: rows of 8 to 64
//   heads of 128 filled, rotated and quantized 67.0 and 60.3 at 33.5, 122 and 107
//   at 67, 239 and 214 at 134, 271 and 266 at 151, 300 and 302 at 168, 357 and 361
//   at 201, 479 and 510 at 268 (in place the same at any size); 8 kv heads of 128
//   read back and converted 39.8 and 35.7 at 67, 60.9 and 57.7 at 134, 76.7 and
//   78.9 at 168, 136 and 147 at 268;
//   kSumsAway, the norm's sums, which a residual stream takes in place (deltas and
//   norms of two layers of 4096 columns 62.7 and 64.3 at 33.6, 102 and 104 at 67,
//   199 and 208 at 134, 450 and 449 at 268; apart 66.4 and 64.5, 110 and 105, 190
//   and 210, 445 and 453), and rows of codes read back, as a stream's deltas (16.8
//   and 16.5 at 16.8, 28.8 and 29.1 at 33.6, 52.2 and 51.6 at 67, 96.6 and 102 at
//   134; with a pass over them alone 23.0 and 21.3 at 33.6, 56.3 and 55.3 at 134,
//   87.5 and 85.5 at 201, 131 and 140 at 268).
// Where all that a pass touches comes from memory and nothing reads the results,
// ordinary stores are the slower ones from 32 MB on: 4099 rows of 4096 normed and
// read back 57.2 and 67.0, 8185 rows of 40 heads of 128 rotated 57.9 and 62.3.
constexpr int64_t kSumsAway = 32 << 20, kReadAway = 160'000'000;  // bytes
inline bool stored_away(int64_t elements, int64_t from) { return 4 * elements >= from; }

}  // namespace nhip
