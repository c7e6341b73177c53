// rotary.hpp -- what the kernels that rotate heads by position share: the
// checks of a caller's nhip_rotary, the table as kernels see it, and eight
// elements of a head rotated in registers.
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
typedef float rotary_f2 __attribute__((ext_vector_type(2), aligned(4)));

// Unit u of a head: eight of its elements, a .. a + 3 and b .. b + 3, with the
// cos and sin of its pairs.  Where dim and head_dim are multiples of 8 a unit is
// four whole pairs (or elements that stay), so that it is rotated in registers,
// and its cos and sin, read once, serve every head of the row; a and b lie half
// of the rotated part (or of the rest) apart, so that neighbouring lanes' fours
// make whole lines.  Else (MIXED, a variant of its own for the registers) the
// partners and the table come from memory, element by element.
struct RotaryUnit {
    int a, b;
    enum Kind { STAYS, HALVES, NEIGHBOURS, ANY } kind;
    rotary_f4 c, s;
    const float *cos_row, *sin_row;
};

template <bool MIXED>
__device__ __forceinline__ RotaryUnit rotary_unit(const RotaryTable& r, int head_dim, int u, int pos)
{
    const size_t row = (size_t)pos * (r.dim / 2);
    RotaryUnit x = {8 * u, 8 * u + 4, RotaryUnit::STAYS, {}, {}, r.cos + row, r.sin + row};
    if (MIXED) {
        if (8 * u < r.dim) x.kind = RotaryUnit::ANY;
    } else if (8 * u >= r.dim) {
        x.a = r.dim / 2 + 4 * u;
        x.b = x.a + (head_dim - r.dim) / 2;
    } else {
        x.a = 4 * u;
        x.b = 4 * u + r.dim / 2;
        x.kind = r.interleaved ? RotaryUnit::NEIGHBOURS : RotaryUnit::HALVES;
        const int pair = r.interleaved ? 2 * u : 4 * u, other = r.interleaved ? r.dim / 4 + 2 * u : 4 * u + 2;
        const rotary_f2 c0 = *reinterpret_cast<const rotary_f2*>(x.cos_row + pair);
        const rotary_f2 c1 = *reinterpret_cast<const rotary_f2*>(x.cos_row + other);
        const rotary_f2 s0 = *reinterpret_cast<const rotary_f2*>(x.sin_row + pair);
        const rotary_f2 s1 = *reinterpret_cast<const rotary_f2*>(x.sin_row + other);
        x.c = rotary_f4{c0.x, c0.y, c1.x, c1.y};
        x.s = rotary_f4{s0.x, s0.y, s1.x, s1.y};
    }
    return x;
}

// The unit's elements xa, xb of the head at `head`, rotated.
template <bool MIXED>
__device__ __forceinline__ void rotate_unit(const RotaryTable& r, const RotaryUnit& u, const float* head, rotary_f4& xa,
                                            rotary_f4& xb)
{
    const rotary_f4 p = xa, q = xb;
    if (!MIXED && u.kind == RotaryUnit::HALVES) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            xa[e] = p[e] * u.c[e] - q[e] * u.s[e];
            xb[e] = q[e] * u.c[e] + p[e] * u.s[e];
        }
    } else if (!MIXED && u.kind == RotaryUnit::NEIGHBOURS) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            xa[2 * e] = p[2 * e] * u.c[e] - p[2 * e + 1] * u.s[e];
            xa[2 * e + 1] = p[2 * e + 1] * u.c[e] + p[2 * e] * u.s[e];
            xb[2 * e] = q[2 * e] * u.c[2 + e] - q[2 * e + 1] * u.s[2 + e];
            xb[2 * e + 1] = q[2 * e + 1] * u.c[2 + e] + q[2 * e] * u.s[2 + e];
        }
    } else if (MIXED && u.kind == RotaryUnit::ANY) {
        const int half = r.dim / 2;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int i = u.a + e;
            if (i >= r.dim) break;
            const bool second = r.interleaved ? i & 1 : i >= half;
            const int pair = r.interleaved ? i >> 1 : second ? i - half : i;
            const float own = e < 4 ? p[e & 3] : q[e & 3];
            const float other = head[r.interleaved ? i ^ 1 : second ? i - half : i + half];
            const float c = u.cos_row[pair], s = u.sin_row[pair];
            const float y = second ? own * c + other * s : own * c - other * s;
            if (e < 4)
                xa[e & 3] = y;
            else
                xb[e & 3] = y;
        }
    }
}

}  // namespace nhip
