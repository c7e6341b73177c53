// rotary.hpp -- what the kernels that rotate heads by position share: the
// checks of a caller's nhip_rotary, and the table as kernels see it.
#pragma once

#include "common.hpp"

namespace nhip {

constexpr int32_t kRotaryMaxDim = 512;
constexpr int32_t kRotaryMaxRows = 1 << 20;  // of a call

// Checks a caller's table; NHIP_OK or NHIP_ERR_ARG.
int32_t rotary_check(const nhip_rotary* r);

struct RotaryTable {
    const float* cos;  // [positions][dim/2]
    const float* sin;
    int32_t positions, dim, interleaved;
};
inline RotaryTable rotary_table(const nhip_rotary* r) { return {r->cos, r->sin, r->positions, r->dim, r->interleaved}; }

typedef float rotary_f4 __attribute__((ext_vector_type(4), aligned(4)));

// Elements 4l .. 4l + 3 of a head rotated by the table rows c and s, a partner
// outside them from memory (the lane beside it has just read it).
__device__ __forceinline__ rotary_f4 rotated4(const float* head, int l, rotary_f4 x, const RotaryTable& r,
                                              const float* c, const float* s)
{
    const int half = r.dim / 2;
    rotary_f4 y = x;
    if (r.interleaved) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int i = 2 * l + k;
            if (i < half) {
                y[2 * k] = x[2 * k] * c[i] - x[2 * k + 1] * s[i];
                y[2 * k + 1] = x[2 * k + 1] * c[i] + x[2 * k] * s[i];
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int i = 4 * l + e;
            if (i < half)
                y[e] = x[e] * c[i] - head[i + half] * s[i];
            else if (i < r.dim)
                y[e] = x[e] * c[i - half] + head[i - half] * s[i - half];
        }
    }
    return y;
}

}  // namespace nhip
