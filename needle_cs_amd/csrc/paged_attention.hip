// paged_attention.hip -- attention over the paged int8 KV cache on gfx950.
//
// For a query (row, head) over its positions s: z_s = (q . k_s) ks_s qs /
// sqrt(qk) with the int8 dot exact, out = sum_s e^(z_s - m) vs_s v_s / sum_s
// e^(z_s - m), in one pass with a running maximum m and fp32 sums.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged.hpp"

namespace nhip {
namespace {

constexpr float kNoScore = -1e30f;  // the running maximum before any position: finite, so that a difference is never NaN

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// v, but the compiler may not pair its operation with a neighbour's (which
// keeps row_bcast from folding into it).
__device__ __forceinline__ float alone(float v)
{
    asm("" : "+v"(v));
    return v;
}

// The value that lane n of the lane's row of 16 holds.
template <int n>
__device__ __forceinline__ float row_bcast(float v)
{
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x150 + n, 0xF, 0xF, true));
}

// What one position contributes besides its codes.  With vs = frac * 2^e
// (e the scale's exponent), the weight of a position is w = 2^(z' - M) with
// z' = z log2(e) + e and M the running maximum of z' less 14, so that w frac,
// the weight of its codes, lies in [0, 2^15) whatever the scales are and is
// the sum of two fp16 numbers: 22 bits of it, or where it is small a step of
// 2^-24, which is 2^-39 of the largest weight.  The sum of the softmax takes
// w 2^-e.  A position that does not count has e = -inf, which makes w 0.
constexpr float kHeadroom = 14.0f;
constexpr float kMaxExponent = 60.0f;  // of a value scale, either way
constexpr float kLeastScale = 1.4e-45f;
struct Position {
    float ks, e, frac, inv;
};
__device__ __forceinline__ Position position(float ks, float vs, bool live)
{
    int e = (int)((__float_as_uint(vs) >> 23) & 255) - 127;
    e = min(max(e, -(int)kMaxExponent), (int)kMaxExponent);
    Position r;
    r.inv = live ? __uint_as_float((uint32_t)(127 - e) << 23) : 0.0f;
    r.frac = live ? vs * r.inv : 0.0f;
    r.ks = live ? ks : 0.0f;
    r.e = live ? (float)e : -INFINITY;
    return r;
}

__device__ __forceinline__ float scale_exponent(float vs)
{
    const int e = (int)((__float_as_uint(vs) >> 23) & 255) - 127;
    return (float)min(max(e, -(int)kMaxExponent), (int)kMaxExponent);
}

// Eight int8 codes (two words) as fp16, exactly: the byte c + 128 in the low
// bits of 1024 makes 1152 + c.
__device__ __forceinline__ f16x8 codes_f16(uint32_t lo, uint32_t hi)
{
    union {
        uint32_t u[4];
        f16x2 h[4];
        f16x8 v;
    } r;
    const uint32_t a = lo ^ 0x80808080u, b = hi ^ 0x80808080u;
    r.u[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
    r.u[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
    r.u[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
    r.u[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
    const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
#pragma unroll
    for (int k = 0; k < 4; k++) r.h[k] = r.h[k] - off;
    return r.v;
}

__device__ __forceinline__ f16x2 to_f16(float a, float b)
{
    const f32x2 v = {a, b};
    return __builtin_convertvector(v, f16x2);
}

// a and b less their fp16 parts (minus_one: -1 that the compiler does not
// know, so that each is one v_fma_mix_f32).
__device__ __forceinline__ f16x2 rest_f16(float a, float b, f16x2 part, float minus_one)
{
    return to_f16(fmaf((float)part[0], minus_one, a), fmaf((float)part[1], minus_one, b));
}

// Maximum / sum over the four lanes l, l + 16, l + 32, l + 48.
__device__ __forceinline__ float rows_max(float v)
{
    v = fmaxf(v, lane_xor<16>(v));
    return fmaxf(v, lane_xor<32>(v));
}
__device__ __forceinline__ float rows_sum(float v)
{
    v = v + lane_xor<16>(v);
    return v + lane_xor<32>(v);
}

// ---------------------------------------------------------------- decode --
//
// One workgroup of W waves per (kv head, row, part of the row's positions);
// a wave takes 64 positions at a time, in its registers from load to result:
//   scores   S^T = K Q^T by v_mfma_i32_16x16x64_i8, the group's heads (up to
//            16) as columns.  Row m of product t is position 16 (m / 4) + 4 t
//            + m % 4, so lane l, which gets rows 4 (l / 16) + i, ends with
//            positions 16 (l / 16) + 4 t + i, all of one 16-position block,
//            for head l % 16.
//   weights  in that lane; lane l also holds position l's scales, and a
//            block's 16 are the 16 lanes of its row (row_bcast).
//   values   O^T = V^T P^T by v_mfma_f32_16x16x32_f16, P split in two fp16
//            parts.  The operand slot (l / 16, j) of product u is position 16
//            (l / 16) + 8 u + j: the weights are where they have to be, and
//            the codes are the 16 bytes that the cache holds of one dimension
//            and 16 positions, one load.
// Nothing passes through LDS until the waves' parts are joined.
//
// A long call is bound by what its loads in flight bring: 32 rows of up to 32768
// positions, 8 kv heads of 128 under 32 heads (1.38 GB) take 276 us, 5.0 TB/s,
// where a reduction over 4 GiB reads 6.4.  A short one is a chain of latencies: table entry,
// keys, two exchanges of four lanes for the maximum, exponentials, values,
// join; 3 rows of up to 192 positions take 4.3 us, of which 2.5 are the launch.
// Measured and not kept: two blocks of loads in flight (360 us in the place
// of 292, for the registers); 16 waves a workgroup for dims of 64 (16 rows of up
// to 2048, 16 kv heads: 10.7 us, 10.9 with eight; but 16 rows of up to 1024, 2
// kv heads: 7.2 and 6.9).
struct DecodeParams {
    PagedLayer c;
    const int8_t* q;
    const float* q_scales;
    float* out;
    const int32_t* row_seq;
    const int32_t* row_first;
    const int32_t* row_count;
    float* parts;  // [rows][heads][max_parts][V]: a part's sums
    float* stats;  // [rows][heads][max_parts][2]: its maximum and total
    int32_t heads, group, max_count, blocks, max_parts;  // blocks: 64-position blocks of a part
    int32_t rows, rows_a_round;  // rows_a_round: of 256 workgroups, where the rows are sorted; else 0
    float scale;
};

// A row's span in 64-position blocks (none when it is out of range).
struct Span {
    int seq, first, end, block0, block1;
};
__device__ __forceinline__ Span decode_span(const DecodeParams& p, int row)
{
    Span s;
    s.seq = p.row_seq[row];
    s.first = p.row_first[row];
    int count = p.row_count[row];
    const int span = p.c.width << p.c.page_shift;
    if (s.seq < 0 || s.seq >= p.c.sequences || s.first < 0 || count < 0 || count > p.max_count ||
        s.first > span - count)
        count = s.first = 0;
    s.end = s.first + count;
    s.block0 = s.first >> 6;
    s.block1 = count > 0 ? (s.end + 63) >> 6 : s.block0;
    return s;
}

// The row of rank `place` by blocks, most first, every other round of 256
// workgroups the other way round, and its span; -1 past the last.  By one
// wave, a lane a row.
__device__ __forceinline__ int ordered_row(const DecodeParams& p, int place, Span& s)
{
    const int lane = threadIdx.x & 63, in_round = place % p.rows_a_round;
    const int rank = (place / p.rows_a_round) & 1 ? place - in_round + p.rows_a_round - 1 - in_round : place;
    if (rank >= p.rows) return -1;
    const Span own = decode_span(p, min(lane, p.rows - 1));
    const int blocks = lane < p.rows ? own.block1 - own.block0 : -1;
    int least = 0, above = p.blocks + 1;  // at most `rank` rows have `above` blocks or more, more than that have `least`
    while (above - least > 1) {
        const int middle = (least + above) / 2;
        if (__popcll(__ballot(blocks >= middle)) > rank)
            least = middle;
        else
            above = middle;
    }
    const uint64_t equal = __ballot(blocks == least);
    const int before = rank - __popcll(__ballot(blocks > least));
    const uint64_t hit = __ballot(blocks == least && __popcll(equal & (((uint64_t)1 << lane) - 1)) == before);
    const int row = __builtin_ctzll(hit);
    s.seq = __builtin_amdgcn_readlane(own.seq, row);
    s.first = __builtin_amdgcn_readlane(own.first, row);
    s.end = __builtin_amdgcn_readlane(own.end, row);
    s.block0 = __builtin_amdgcn_readlane(own.block0, row);
    s.block1 = __builtin_amdgcn_readlane(own.block1, row);
    return row;
}

// ONE: a kv head per query head, where fifteen of sixteen columns of scores
// would be spent on no head.  Then S = Q K^T with the positions as columns:
// product t has block t's positions and the head in row 4 t alone, and the
// four add up to one result in which lane l holds position l's score, so each
// is formed and weighted once.  The lanes of a row of 16 then pass their
// weights (both fp16 parts in a word) to all of them, which is the value
// product's operand (every column the same head).  16 rows of up to 2048
// positions, 16 heads of 64: 10.9 us (compared when it came: 11.3, 12.5 in the
// general form); the same over two to four heads a kv head was no faster.
//
// SORTED: calls of up to 64 whole rows and more workgroups than CUs deal the
// rows to the CUs by their length (ordered_row), so that the longest do not
// meet: 64 rows of up to 2048 positions, 8 kv heads: 18.7 us, 20.9 in the
// order of the call; 16 kv heads 27.5 and 33.0; 48 rows, 8 heads of 128 25.9
// (now 24) and 33.3; but rows of 1040 each 16.5 and 15.9.  (Its own variant: the
// registers of the choice cost the others up to 0.5 us.)
//
// Registers: the general form for dims of 128 has to stay within 168, which
// three waves a SIMD share (32 rows of up to 32768: 276 us, 289 with 169).
template <int QK, int V, int W, bool ONE, bool SORTED>
__global__ __launch_bounds__(64 * W, QK <= 64 ? 4 : ONE || SORTED ? 2 : 3) void paged_decode_kernel(DecodeParams p)
{
    constexpr int KH = (QK + 63) / 64, VT = V / 16;
    extern __shared__ __align__(16) float lds[];  // [W][group][V] sums, then [W][16] M, [W][16] total
    const PagedLayer& c = p.c;
    int row = blockIdx.x, kvh = blockIdx.y, part = blockIdx.z;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = lane & 15, g = lane >> 4;
    Span s;
    if constexpr (SORTED) {
        const int place = blockIdx.x / c.kv_heads;
        kvh = blockIdx.x - place * c.kv_heads;
        part = 0;
        row = ordered_row(p, place, s);
        if (row < 0) return;
    } else {
        s = decode_span(p, row);
    }
    const int total_blocks = s.block1 - s.block0;
    const int parts = (total_blocks + p.blocks - 1) / p.blocks;
    if (part > 0 && part >= parts) return;
    const int end_block = min(s.block1, s.block0 + (part + 1) * p.blocks);

    i32x4 q[KH];
    float qs = 0.0f;
#pragma unroll
    for (int k = 0; k < KH; k++) q[k] = i32x4{0, 0, 0, 0};
    if (ONE || h < p.group) {
        const size_t head = (size_t)row * p.heads + kvh * p.group + (ONE ? 0 : h);
#pragma unroll
        for (int k = 0; k < KH; k++)
            if (64 * k + 16 * g < QK) q[k] = *reinterpret_cast<const i32x4*>(p.q + head * QK + 64 * k + 16 * g);
        qs = p.q_scales[head] * p.scale;
    }

    const int32_t* table = c.tables + (size_t)s.seq * c.width;
    const int in_page = (1 << c.page_shift) - 1;
    // the page of position `pos` of a 64-position block: -1 where it may not be followed
    auto page_at = [&](int pos) {
        const int t = pos >> c.page_shift;
        const int page = pos < s.end ? table[min(t, c.width - 1)] : -1;
        return page >= 0 && page < c.pages ? page : -1;
    };
    i32x4 kr[4][KH], vr[VT];
    float ksr, vsr;
    bool live;
    // (a block's addresses come from its first cell in page 0 where there is none, whose bytes then meet weight 0)
    auto load_keys = [&](int block, int kpage, int vpage) {
        if constexpr (ONE) {
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const int page = max(__builtin_amdgcn_readlane(vpage, 16 * t), 0);  // block t's
                const int8_t* k = c.keys + ((((size_t)page * c.kv_heads + kvh) << c.page_shift) +
                                            ((64 * block + 16 * t) & in_page)) * QK;
#pragma unroll
                for (int half = 0; half < KH; half++)
                    kr[t][half] = *reinterpret_cast<const i32x4*>(k + (h * QK + min(64 * half + 16 * g, QK - 16)));
            }
        } else {
            const int kpos = 64 * block + 16 * (h >> 2);
            const int8_t* k = c.keys + ((((size_t)max(kpage, 0) * c.kv_heads + kvh) << c.page_shift) +
                                        (kpos & in_page) + (h & 3)) * QK;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int half = 0; half < KH; half++)
                    kr[t][half] =
                        *reinterpret_cast<const i32x4*>(k + 4 * t * QK + min(64 * half + 16 * g, QK - 16));
        }
        const int pos = 64 * block + lane;
        const size_t cell = (((size_t)max(vpage, 0) * c.kv_heads + kvh) << c.page_shift) + (pos & in_page);
        ksr = c.kscale[cell];
        vsr = c.vscale[cell];
        live = vpage >= 0 && pos >= s.first && pos < s.end;
    };
    auto load_values = [&](int block, int vpage) {
        const int pos = 64 * block + 16 * g;
        const int8_t* v = c.values + (((size_t)max(vpage, 0) * c.kv_heads + kvh) << c.page_shift) * V +
                          (size_t)((pos & in_page) >> 4) * (16 * V) + 16 * h;
#pragma unroll
        for (int t = 0; t < VT; t++) vr[t] = *reinterpret_cast<const i32x4*>(v + 256 * t);
    };

    const float minus_one = alone(-1.0f);
    float peak = kNoScore, total = 0.0f;
    f32x4 o[VT];
#pragma unroll
    for (int t = 0; t < VT; t++) o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    int block = s.block0 + part * p.blocks + wave;
    int kpage = -1, vpage = -1, vpage_now = -1;
    if (block < end_block) {
        kpage = page_at(64 * block + 16 * (h >> 2));
        vpage = page_at(64 * block + 16 * g);
        load_keys(block, kpage, vpage);
        load_values(block, vpage);
        kpage = page_at(64 * (block + W) + 16 * (h >> 2));
        vpage = page_at(64 * (block + W) + 16 * g);
    }
    for (; block < end_block; block += W) {
        i32x4 dots[ONE ? 1 : 4];
        if constexpr (ONE) {
            dots[0] = i32x4{0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int half = 0; half < KH; half++) {
                    const i32x4 none = {0, 0, 0, 0};
                    dots[0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(h == 4 * t ? q[half] : none, kr[t][half],
                                                                    dots[0], 0, 0, 0);
                }
        } else {
#pragma unroll
            for (int t = 0; t < 4; t++) {
                dots[t] = i32x4{0, 0, 0, 0};
#pragma unroll
                for (int half = 0; half < KH; half++)
                    dots[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kr[t][half], q[half], dots[t], 0, 0, 0);
            }
        }
        Position x = position(ksr, vsr, live);
        const bool more = block + W < end_block;
        if (more) load_keys(block + W, kpage, vpage);
        vpage_now = vpage;
        if (block + 2 * W < end_block) {
            kpage = page_at(64 * (block + 2 * W) + 16 * (h >> 2));
            vpage = page_at(64 * (block + 2 * W) + 16 * g);
        }
        // Values that are all 0 have scale 1 (QuantizeInt8), which says nothing of
        // their size: 0 in its place, so that the others keep their digits.
        if (__ballot(x.frac == 1.0f && x.e == 0.0f)) {
            uint32_t word = 0;  // the codes of this lane's position and three beside it, of any dimension
#pragma unroll
            for (int k = 0; k < 4; k++) {
                uint32_t any = 0;
#pragma unroll
                for (int t = 0; t < VT; t++) any |= (uint32_t)vr[t][k];
                any |= lane_xor<1>(any);
                any |= lane_xor<2>(any);
                any |= lane_xor<4>(any);
                any |= lane_xor<8>(any);
                word = ((lane >> 2) & 3) == k ? any : word;
            }
            if (x.frac == 1.0f && x.e == 0.0f && ((word >> (8 * (lane & 3))) & 255) == 0) x = position(x.ks, 0.0f, true);
        }
        float w[16];  // the weights of the 16 positions that this lane gives the value product (ONE: as words)
        if constexpr (ONE) {
            const float z = ((float)dots[0][0] * x.ks) * qs + x.e;
            const float up = fmaxf(peak, wave_max(z) - kHeadroom);
            if (up > peak) {
                const float keep = __builtin_amdgcn_exp2f(peak - up);
                peak = up;
                total *= keep;
#pragma unroll
                for (int t = 0; t < VT; t++) o[t] *= keep;
            }
            const float e = __builtin_amdgcn_exp2f(z - peak);
            total = fmaf(e, x.inv, total);
            const float y = alone(e * x.frac);  // (both conversions below have to see the rounded product)
            union {
                f16x2 h2;
                float word;
            } both;
            both.h2 = to_f16(y, fmaf((float)(_Float16)y, minus_one, y));
#define NHIP_WORD(j) w[j] = row_bcast<j>(both.word);
            NHIP_WORD(0) NHIP_WORD(1) NHIP_WORD(2) NHIP_WORD(3) NHIP_WORD(4) NHIP_WORD(5) NHIP_WORD(6) NHIP_WORD(7)
            NHIP_WORD(8) NHIP_WORD(9) NHIP_WORD(10) NHIP_WORD(11) NHIP_WORD(12) NHIP_WORD(13) NHIP_WORD(14)
            NHIP_WORD(15)
#undef NHIP_WORD
        } else {
            float z[16];
#define NHIP_SCORE(j) z[j] = ((float)dots[(j) / 4][(j) % 4] * row_bcast<j>(x.ks)) * qs + row_bcast<j>(x.e);
            NHIP_SCORE(0) NHIP_SCORE(1) NHIP_SCORE(2) NHIP_SCORE(3) NHIP_SCORE(4) NHIP_SCORE(5) NHIP_SCORE(6)
            NHIP_SCORE(7) NHIP_SCORE(8) NHIP_SCORE(9) NHIP_SCORE(10) NHIP_SCORE(11) NHIP_SCORE(12) NHIP_SCORE(13)
            NHIP_SCORE(14) NHIP_SCORE(15)
#undef NHIP_SCORE
            float up = z[0];
#pragma unroll
            for (int j = 1; j < 16; j++) up = fmaxf(up, z[j]);
            up = fmaxf(peak, rows_max(up) - kHeadroom);
            if (__ballot(up > peak)) {
                const float keep = __builtin_amdgcn_exp2f(peak - up);
                peak = up;
                total *= keep;
#pragma unroll
                for (int t = 0; t < VT; t++) o[t] *= keep;
            }
#define NHIP_WEIGHT(j)                                  \
    w[j] = __builtin_amdgcn_exp2f(z[j] - peak);         \
    total = fmaf(row_bcast<j>(x.inv), w[j], total);     \
    w[j] = alone(row_bcast<j>(x.frac) * w[j]);
            NHIP_WEIGHT(0) NHIP_WEIGHT(1) NHIP_WEIGHT(2) NHIP_WEIGHT(3) NHIP_WEIGHT(4) NHIP_WEIGHT(5)
            NHIP_WEIGHT(6) NHIP_WEIGHT(7) NHIP_WEIGHT(8) NHIP_WEIGHT(9) NHIP_WEIGHT(10) NHIP_WEIGHT(11)
            NHIP_WEIGHT(12) NHIP_WEIGHT(13) NHIP_WEIGHT(14) NHIP_WEIGHT(15)
#undef NHIP_WEIGHT
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            union {
                f16x2 h2[4];
                uint32_t u[4];
                f16x8 v;
            } hi, lo;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float a = w[8 * u + 2 * k], b = w[8 * u + 2 * k + 1];
                if constexpr (ONE) {
                    hi.u[k] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x05040100u);
                    lo.u[k] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
                } else {
                    hi.h2[k] = to_f16(a, b);
                    lo.h2[k] = rest_f16(a, b, hi.h2[k], minus_one);
                }
            }
#pragma unroll
            for (int t = 0; t < VT; t++) {
                const f16x8 v = codes_f16((uint32_t)vr[t][2 * u], (uint32_t)vr[t][2 * u + 1]);
                o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, hi.v, o[t], 0, 0, 0);
                o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, lo.v, o[t], 0, 0, 0);
            }
        }
        if (more) load_values(block + W, vpage_now);
    }
    total = rows_sum(total);
    if constexpr (ONE) {
        total += lane_xor<1>(total);
        total += lane_xor<2>(total);
        total += lane_xor<4>(total);
        total += lane_xor<8>(total);
    }

    // the waves' parts joined: every wave scales its sums to the common maximum
    float* peaks = lds + (size_t)W * p.group * V;
    float* totals = peaks + W * 16;
    if (lane < 16) {
        peaks[wave * 16 + lane] = peak;
        totals[wave * 16 + lane] = total;
    }
    __syncthreads();
    float top = kNoScore;
#pragma unroll
    for (int k = 0; k < W; k++) top = fmaxf(top, peaks[k * 16 + h]);
    const float mine = __builtin_amdgcn_exp2f(peak - top);
    if (h < p.group) {
        float* sums = lds + ((size_t)wave * p.group + h) * V + 4 * g;
#pragma unroll
        for (int t = 0; t < VT; t++) *reinterpret_cast<f32x4*>(sums + 16 * t) = o[t] * mine;
    }
    __syncthreads();
    const bool split = parts > 1;
    for (int at = threadIdx.x; at < p.group * V; at += 64 * W) {
        const int head = at / V, d = at - head * V;
        float best = kNoScore, all = 0.0f, sum = 0.0f;
#pragma unroll
        for (int k = 0; k < W; k++) best = fmaxf(best, peaks[k * 16 + head]);
#pragma unroll
        for (int k = 0; k < W; k++) {
            all = fmaf(totals[k * 16 + head], __builtin_amdgcn_exp2f(peaks[k * 16 + head] - best), all);
            sum += lds[((size_t)k * p.group + head) * V + d];
        }
        if (!split) {
            p.out[((size_t)row * p.heads + kvh * p.group + head) * V + d] = all != 0.0f ? sum / all : 0.0f;
        } else {
            const size_t at_part = ((size_t)row * p.heads + kvh * p.group + head) * p.max_parts + part;
            p.parts[at_part * V + d] = sum;
            if (d == 0) *reinterpret_cast<float2*>(p.stats + 2 * at_part) = make_float2(best, all);
        }
    }
}

constexpr int kMaxParts = 64;  // a lane each where they are joined

// Joins a row's parts, four waves per (row, head), each a quarter of the
// parts; rows of one part are done.
template <int V>
__global__ __launch_bounds__(256) void paged_join_kernel(DecodeParams p)
{
    __shared__ float factors[kMaxParts], quarters[4][V];
    const int row = blockIdx.x, head = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Span s = decode_span(p, row);
    const int parts = (s.block1 - s.block0 + p.blocks - 1) / p.blocks;
    if (parts <= 1) return;
    const size_t first = ((size_t)row * p.heads + head) * p.max_parts;
    float2 stat = make_float2(kNoScore, 0.0f);
    if (lane < parts) stat = *reinterpret_cast<const float2*>(p.stats + 2 * (first + lane));
    const float factor = __builtin_amdgcn_exp2f(stat.x - wave_max(stat.x));
    if (wave == 0) factors[lane] = factor;
    float all = factor * stat.y;
    for (int off = 32; off; off >>= 1) all += __shfl_xor(all, off);
    __syncthreads();
    constexpr int E = V / 64;
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; e++) sum[e] = 0.0f;
    const float* from = p.parts + first * V + lane;
    for (int k = wave; k < parts; k += 16) {
        float x[4][E];
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int e = 0; e < E; e++) x[u][e] = from[(size_t)min(k + 4 * u, parts - 1) * V + 64 * e];
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int e = 0; e < E; e++) sum[e] = k + 4 * u < parts ? fmaf(x[u][e], factors[k + 4 * u], sum[e]) : sum[e];
    }
#pragma unroll
    for (int e = 0; e < E; e++) quarters[wave][lane + 64 * e] = sum[e];
    __syncthreads();
    if (threadIdx.x < V) {
        const int d = threadIdx.x;
        const float t = (quarters[0][d] + quarters[1][d]) + (quarters[2][d] + quarters[3][d]);
        p.out[((size_t)row * p.heads + head) * V + d] = all != 0.0f ? t / all : 0.0f;
    }
}

// How a decode call is split: waves of a workgroup, 64-position blocks of a
// part, parts of the longest row.
struct Split {
    int waves, blocks, parts, rows_a_round;
};

// Parts cost a second launch and even out the rows.  Measured whole and in
// parts, at rows of 700, 1100, 1600 and 2400 positions (12 to 39 blocks):
//   8 or 32 workgroups, dims of 64    5.9  7.6  9.0 12.5 us   parts  8.2  8.2  8.2  8.4
//                       dims of 128   8.5 11.5 15.4 20.6             10.1 10.3 10.5 10.9
//   128 workgroups,     dims of 64    6.3  8.5 10.8 14.0              8.6 10.5 12.2 15.4
//                       dims of 128   9.5 12.6 16.7 21.8             11.9 17.3 17.2 21.3
//   256 workgroups,     dims of 64    8.2 10.4 12.8 17.4             11.3 13.9 16.8 21.3
//                       dims of 128  12.0 15.9 20.9 31.3             15.7 19.8 24.4 37.3
// So rows stay whole up to 18 blocks (for few workgroups the two meet a little
// above for dims of 64, a little below for 128), or up to 40 where the
// workgroups fill half the CUs (where 128 of them meet at 40 for dims of 128;
// rows of very different lengths gain there by parts: 16 of 32 to 2400, 8 kv
// heads of 128: 21.1 whole, 18.0 in parts).  Longer ones are cut into parts of
// at least 8 blocks such that the longest rows give 2048 workgroups (32 rows of
// up to 32768 on 8 kv heads of 128: 276 us, 294 with 1024 workgroups; 4 rows of
// up to 8000: 17.5, 49.9 whole), at most kMaxParts.  Eight waves a workgroup,
// which a row's blocks are dealt to in turn (16 rows of up to 2048, 16 kv heads:
// 10.9 us, 15.1 with four); but four where there are 512 workgroups or more (the
// 32 rows: 276 and 307), or rows of up to 10 blocks, where it makes no
// difference (16 rows of 256, 8 kv heads: 4.9 both ways).
Split decode_split(const nhip_paged_cache* c, int32_t rows, int32_t max_count)
{
    const int64_t units = (int64_t)rows * c->kv_heads;
    const int most = max_count / 64 + 2;  // blocks of a row: its ends need not be a block's
    Split s;
    if (most <= 18 || (most <= 40 && units >= 128)) {
        s.blocks = most;
    } else {
        const int64_t even = (most * units + 2047) / 2048, fewest = (most + kMaxParts - 1) / kMaxParts;
        s.blocks = (int)std::min<int64_t>(most, std::max<int64_t>({8, even, fewest}));
    }
    s.parts = (most + s.blocks - 1) / s.blocks;
    s.waves = most <= 10 || units * s.parts >= 512 ? 4 : 8;
    s.rows_a_round = s.parts == 1 && rows <= 64 && units > 256 ? std::max(1, 256 / c->kv_heads) : 0;
    return s;
}

size_t decode_workspace(const nhip_paged_cache* c, int32_t rows, int32_t heads, const Split& s)
{
    return s.parts > 1 ? (size_t)rows * heads * s.parts * (c->v_dim + 2) * sizeof(float) : 0;
}

// The factor that takes a scaled dot product to a base-2 score.
float score_scale(int32_t qk) { return (float)(1.4426950408889634 / std::sqrt((double)qk)); }

template <int QK, int V>
int32_t launch_decode(const DecodeParams& p, const Split& s, int32_t rows, hipStream_t stream)
{
    const size_t lds = (size_t)s.waves * (p.group * V + 32) * sizeof(float);
    const int rounds = s.rows_a_round ? (rows + s.rows_a_round - 1) / s.rows_a_round : 0;
    const dim3 grid = rounds ? dim3(rounds * s.rows_a_round * p.c.kv_heads) : dim3(rows, p.c.kv_heads, s.parts);
    hipError_t set = hipSuccess;
    auto launch = [&](auto kernel) {
        if (lds > 65536)  // (eight waves of 16 heads of 128)
            set = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                      hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (set == hipSuccess) hipLaunchKernelGGL(kernel, grid, dim3(64 * s.waves), lds, stream, p);
    };
    auto choose = [&](auto one, auto sorted) {
        launch(s.waves == 4 ? paged_decode_kernel<QK, V, 4, one(), sorted()>
                            : paged_decode_kernel<QK, V, 8, one(), sorted()>);
    };
    const std::true_type yes;
    const std::false_type no;
    if (p.group == 1)
        rounds ? choose(yes, yes) : choose(yes, no);
    else
        rounds ? choose(no, yes) : choose(no, no);
    NHIP_CHECK_HIP(set);
    NHIP_CHECK_HIP(hipGetLastError());
    if (s.parts > 1) {
        hipLaunchKernelGGL((paged_join_kernel<V>), dim3(rows, p.heads), dim3(256), 0, stream, p);
        NHIP_CHECK_HIP(hipGetLastError());
    }
    return NHIP_OK;
}

// ---------------------------------------------------------------- prompt --
//
// A workgroup of four waves takes 128 queries of one kv head and run; a query
// is a (row, head of the group) pair, row-major, so a tile is whole rows of
// all the group's heads whatever their number.  It walks the positions its
// rows attend 64 at a time.  The codes of a tile are staged in LDS by all
// four waves (keys as they are, values as fp16, each converted once), two
// tiles deep: the next one's loads are issued before a tile's products and
// stored after them.  Each wave keeps 32 queries as columns:
//   scores   S^T = K Q^T by v_mfma_i32_32x32x32_i8; row m = 8 b + 4 g + i of a
//            product (b = m / 8) is position 16 (b / 2) + 8 g + 4 (b % 2) + i,
//            so lane (g, query) gets in register r = 4 b + i position
//            16 (r / 8) + 8 g + r % 8 of its 32.
//   weights  in that lane.  Its row of 16 lanes holds those 16 positions'
//            scales, lane r of it register r's (row_bcast folds into the
//            multiplication), and a query's maximum and total are its lane's.
//   values   O^T = V^T P^T by v_mfma_f32_32x32x16_f16: registers 8 u .. 8 u + 7
//            are the eight weights that product u wants of this lane.
// The weights are 2^(z - M), with M such that a weight times its value scale
// stays below 2^15, which fits fp16, while the row's largest such product is at
// least 2^5: its two fp16 parts, to a step of 2^-24, keep 2^-30 of it.  M thus
// follows the maximum of z + e (e the scale's exponent), and a scale that is
// large where the weight is small does not move it.  Whether it has to move is
// asked with a bound, the tile's largest score and largest exponent; only where
// that is too large, a few times a row, is the maximum formed (in every tile
// where one position in 32 is a value of zeros the call below takes 925 us, and
// where the scales lie e^3 apart 814).
//
// Bound by the issue of instructions: a position and query costs about 10
// vector operations of 4 cycles a wave (conversion, two scalings, maximum,
// exponential, sum, two conversions and the rest between them) beside its
// share of the products, and vector and matrix instructions of a SIMD's two
// waves overlap in part only.  One run of 8192 rows, 32 heads on 8 of 128
// takes 742 us (726 to 757 from one card to the next; up to 1000 in the first
// 40 passes, until the card's clock has settled), 550 Gflop: 741 TFLOP/s.
// Its products, the values' made twice for the weights' two parts, would take
// 633 us at the rates of a large int8 and a large fp16 product (one part: 394,
// but weights of 11 bits are off by 2^-12 each).  Measured and not kept there: eight waves
// in two phases (893 us), a tile's scores ahead of the last one's values (776
// to 857, for the registers), operands read from LDS a phase ahead (788),
// 16-query waves, four a SIMD (783), set instruction orders (733 to 769), a
// raised wave priority in the products (767).
struct PromptParams {
    PagedLayer c;
    const int8_t* q;
    const float* q_scales;
    float* out;
    const int32_t* run_rows;
    const int32_t* run_seq;
    const int32_t* run_pos;
    float* parts;  // as DecodeParams'
    float* stats;
    int32_t rows, heads, group, runs, window, max_count, blocks, max_parts;
    int32_t places;  // of tiles that the grid holds
    uint32_t group_part;  // 2^31 / group, rounded up
    int32_t tiles_a_round;  // of 256 workgroups, where the tiles are sorted; else 0
    float scale;
};

constexpr int kTileQueries = 128;
constexpr float kLag = 8.0f;  // log2 of how far a product may grow before the sums are rescaled

typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Rows [row0, row1) of a run, cut to the call's.
struct RunRows {
    int row0, row1;
};
__device__ __forceinline__ RunRows run_rows(const PromptParams& p, int run)
{
    RunRows r;
    r.row0 = min(max(p.run_rows[run], 0), p.rows);
    r.row1 = max(r.row0, min(p.run_rows[run + 1], p.rows));
    return r;
}

// x / group for a query or head x < 2^24 (group <= 16, so the quotient is exact).
__device__ __forceinline__ int over_group(const PromptParams& p, int x)
{
    return (int)(((uint64_t)(uint32_t)x * p.group_part) >> 31);
}

__device__ __forceinline__ int run_tiles(const PromptParams& p, const RunRows& r)
{
    return ((r.row1 - r.row0) * p.group + kTileQueries - 1) / kTileQueries;
}

// The position that query `at` (row-major over the group's heads) of a run
// sits at, cut to the call's limit; -1 where the run has no positions.  run_pos
// belongs to the run's first row as the caller counts them, which may lie
// before row 0.
struct RunPositions {
    int64_t pos0;  // of its first row here
    int limit;
    bool known;
    __device__ __forceinline__ int at(const PromptParams& p, int query) const
    {
        const int64_t x = pos0 + over_group(p, query);
        return known ? (int)(x < limit ? x : limit - 1) : -1;
    }
};
__device__ __forceinline__ RunPositions run_positions(const PromptParams& p, int row0, int first_row, int seq, int pos)
{
    return {(int64_t)pos + row0 - first_row, min(p.c.width << p.c.page_shift, p.max_count),
            seq >= 0 && seq < p.c.sequences && pos >= 0};
}

// The 64-position tiles [begin, end) that a tile of queries at positions
// first .. last attends, and the parts that they are cut into.
struct TileSpan {
    int from, begin, end, parts;
};
__device__ __forceinline__ TileSpan tile_span(const PromptParams& p, int first, int last)
{
    TileSpan s;
    s.from = p.window > 0 ? max(first - p.window + 1, 0) : 0;
    s.begin = s.from >> 6;
    s.end = last >= 0 ? (last >> 6) + 1 : s.begin;
    s.parts = (s.end - s.begin + p.blocks - 1) / p.blocks;
    return s;
}

// The run whose tile has the place `place` in the call, the tile's number in
// the run (the last, which attends most, first) and the run's tiles, by one
// wave; -1 where the place has no tile.
//
// In the order of length: R runs a lane.  Where the workgroups are more than
// the CUs, the tiles come in the order of their last blocks, most first (a
// search for the block count that the place's rank falls into), and every
// other round of 256 workgroups the other way round: a CU takes one of each
// round, and its heavy tile meets a light one (16 runs of up to 700 rows, 16 kv
// heads: 34.2 us; in the order of the runs 37.8; sorted, but all rounds alike,
// 37.1.  40 runs of up to 900, more than are resident at once: 87, 105 and
// 86).  Fewer workgroups keep the runs' order, and so do more than 6144, which
// even out by themselves and gain by a run's tiles side by side (32 heads on 8,
// runs of up to 500: 80 of them, 5640 workgroups, 155 us sorted and 158 in the
// runs' order; 120, 8460 workgroups, 244 and 240).
constexpr int kSortedGroups = 6144;
template <int R>
__device__ __forceinline__ int find_tile_by_length(const PromptParams& p, int place, int& in_run, int& of_run)
{
    const int lane = threadIdx.x & 63;
    int rows[R], all[R], pos[R];  // a run's rows, tiles, and the position of its first row here
    int mine = 0;
#pragma unroll
    for (int k = 0; k < R; k++) {
        const int run = min(R * lane + k, p.runs - 1);
        const RunRows r = run_rows(p, run);
        rows[k] = R * lane + k < p.runs ? r.row1 - r.row0 : 0;
        all[k] = (rows[k] * p.group + kTileQueries - 1) / kTileQueries;
        const int64_t at = (int64_t)p.run_pos[run] + r.row0 - p.run_rows[run];
        pos[k] = (int)min(max(at, (int64_t)0), (int64_t)1 << 30);
        mine += all[k];
    }
    // a run's tiles that reach position 64 (blocks - 1)
    auto reach = [&](int k, int blocks) {
        const int row = min(max(64 * (blocks - 1) - pos[k], 0), rows[k]);
        return row >= rows[k] ? 0 : all[k] - row * p.group / kTileQueries;
    };
    int rank = place;
    if (p.tiles_a_round) {
        const int in_round = place % p.tiles_a_round;
        if ((place / p.tiles_a_round) & 1) rank = place - in_round + p.tiles_a_round - 1 - in_round;
    }
    if (rank >= __builtin_amdgcn_readfirstlane(wave_sum_i32(mine))) return -1;
    const int most = p.tiles_a_round ? p.max_count / 64 + 1 : 1;
    // `passed` tiles, at most the rank, have `above` blocks or more; more than the rank have `blocks`
    int blocks = 1, above = most + 1, passed = 0;
    while (above - blocks > 1) {
        const int middle = (blocks + above) / 2;
        int n = 0;
#pragma unroll
        for (int k = 0; k < R; k++) n += reach(k, middle);
        n = __builtin_amdgcn_readfirstlane(wave_sum_i32(n));
        if (n > rank) {
            blocks = middle;
        } else {
            above = middle;
            passed = n;
        }
    }
    int more[R], n[R], sum = 0;  // a run's tiles of more blocks, and of as many
#pragma unroll
    for (int k = 0; k < R; k++) {
        more[k] = above > most ? 0 : reach(k, above);
        n[k] = reach(k, blocks) - more[k];
        sum += n[k];
    }
    const int own = sum;
    for (int off = 1; off < 64; off <<= 1) {
        const int up = __shfl_up(sum, off);
        if (lane >= off) sum += up;
    }
    const uint64_t hit = __ballot(sum > rank - passed);
    if (hit == 0) return -1;
    const int l = __builtin_ctzll(hit);
    int at = rank - passed - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(own, l)), run = -1;
#pragma unroll
    for (int k = 0; k < R; k++) {
        const int here = __builtin_amdgcn_readlane(n[k], l);
        if (run < 0 && at < here) {
            run = R * l + k;
            of_run = __builtin_amdgcn_readlane(all[k], l);
            in_run = __builtin_amdgcn_readlane(more[k], l) + at;
        }
        at -= here;
    }
    return run;
}

// Up to 64 runs go by length, a lane each; up to 256 four a lane (80 of up to
// 300 rows, 8 kv heads: 34.9 us, 45.0 by the search below).  Otherwise, and for
// one run, whose tiles are in order already (4000 rows: 103 us as they come,
// 104 back and forth), run i's tiles have the places from floor(its first
// query / 128) + i on, as many as it can need however the runs before it end,
// so that 64 probes a step find the run without a sum over all (runs of 20
// rows, 2 kv heads: 1000 of them 42.7 us, 60.3 by sums of 64 at a time).
constexpr int kSortedRuns = 256;
__device__ __forceinline__ int find_tile(const PromptParams& p, int place, int& in_run, int& of_run)
{
    if (p.runs > 1 && p.runs <= 64) return find_tile_by_length<1>(p, place, in_run, of_run);
    if (p.runs > 1 && p.runs <= kSortedRuns) return find_tile_by_length<kSortedRuns / 64>(p, place, in_run, of_run);
    const int lane = threadIdx.x & 63;
    auto first_place = [&](int run) { return run_rows(p, run).row0 * p.group / kTileQueries + run; };
    int run = 0, n = p.runs;
    do {
        const int step = (n + 63) / 64;
        const uint64_t before = __ballot(lane * step < n && first_place(run + min(lane * step, n - 1)) <= place);
        if (before == 0) return -1;
        const int l = 63 - __builtin_clzll(before);
        run += l * step;
        n = min(step, n - l * step);
    } while (n > 1);
    const RunRows r = run_rows(p, run);
    of_run = run_tiles(p, r);
    in_run = place - first_place(run);
    return in_run < of_run ? run : -1;
}

// An int32 of an array that no kernel of the launch writes, by a scalar load.
__device__ __forceinline__ int32_t scalar_load(const int32_t* a, int64_t i)
{
    return ((const __attribute__((address_space(4))) int32_t*)a)[i];
}

#define NHIP_INLINE __attribute__((always_inline))

template <int QK, int V>
__global__ __launch_bounds__(256, QK <= 64 ? 3 : 2) void paged_prompt_kernel(PromptParams p)
{
    constexpr int KS = QK <= 64 ? 64 : 128;  // bytes of a key row in LDS
    constexpr int KK = KS / 32;              // products of 32 key bytes
    constexpr int DT = V / 32;               // tiles of 32 value dimensions
    constexpr int KU = KS / 64, VU = V / 64; // 16-byte units a thread stages of each
    constexpr int KCH = QK / 16;             // units of a key row
    __shared__ __align__(16) uint8_t lds_k[2][64 * KS];
    __shared__ __align__(16) uint8_t lds_v[2][V * 128];
    __shared__ float lds_ks[4][64], lds_vs[4][64];
    __shared__ __align__(8) uint16_t lds_live[4][4];
    const PagedLayer& c = p.c;
    // (a tile's kv heads side by side: with 8 of them each XCD keeps one head's positions in its L2)
    const int tile_of_call = blockIdx.x / c.kv_heads, kvh = blockIdx.x - tile_of_call * c.kv_heads;
    const int part = blockIdx.y;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 5;

    int in_run, of_run;
    const int run = __builtin_amdgcn_readfirstlane(find_tile(p, tile_of_call, in_run, of_run));
    if (run < 0) return;
    const RunRows rr = run_rows(p, run);
    const int row0 = __builtin_amdgcn_readfirstlane(rr.row0);
    const int queries = __builtin_amdgcn_readfirstlane(rr.row1 - rr.row0) * p.group;
    // the last tiles of a run attend most: they go first
    const int q0 = __builtin_amdgcn_readfirstlane((of_run - 1 - in_run) * kTileQueries);
    const int qn = min(kTileQueries, queries - q0);
    const int seq = scalar_load(p.run_seq, run);
    const RunPositions at = run_positions(p, row0, scalar_load(p.run_rows, run), seq, scalar_load(p.run_pos, run));

    // this lane's query
    const int query = q0 + 32 * wave + (lane & 31);
    const bool mine = query < q0 + qn;
    const int q_row = min(query, queries - 1) / p.group;
    const int head = kvh * p.group + min(query, queries - 1) - q_row * p.group;
    const int64_t far_pos = at.pos0 + q_row;
    const int q_pos = at.known && far_pos < at.limit ? (int)far_pos : -1;  // -1 attends nothing
    const int q_first = p.window > 0 ? max(q_pos - p.window + 1, 0) : 0;
    const size_t q_at = (size_t)(row0 + q_row) * p.heads + head;
    i32x4 q[KK];
#pragma unroll
    for (int k = 0; k < KK; k++) {
        q[k] = i32x4{0, 0, 0, 0};
        if (32 * k + 16 * g < QK) q[k] = *reinterpret_cast<const i32x4*>(p.q + q_at * QK + 32 * k + 16 * g);
    }
    float qs = p.q_scales[q_at] * p.scale;
    qs = qs == 0.0f ? 1.2e-38f : qs;  // (a score is then 0, and a position left out still -inf)

    // the wave's and the workgroup's positions (the last query's row is the furthest)
    const int wave_first = __builtin_amdgcn_readfirstlane(at.at(p, min(q0 + 32 * wave, queries - 1)));
    const int wave_last = 32 * wave < qn ? __builtin_amdgcn_readfirstlane(at.at(p, min(q0 + 32 * wave + 31, queries - 1)))
                                         : -1;
    const int first_pos = __builtin_amdgcn_readfirstlane(at.at(p, q0));
    const int last_pos = __builtin_amdgcn_readfirstlane(at.at(p, q0 + qn - 1));
    const TileSpan span = tile_span(p, first_pos, last_pos);
    const int from = span.from, parts = span.parts;
    const int from_window = p.window > 0 ? p.window - 1 : 1 << 30;  // positions before its own that a row attends
    if (part > 0 && part >= parts) return;
    const int begin = span.begin + part * p.blocks;
    const int end = min(span.end, begin + p.blocks);

    // Staging: a wave brings one 16-position block of a tile, so its page is a
    // scalar, looked up a tile ahead.  Units are spread over the banks such
    // that the 16 lanes LDS serves together find 16 different places.
    const int in_page = (1 << c.page_shift) - 1;
    const int k_pos = lane / KCH, k_ch = lane % KCH;  // (+ 8 positions for a second unit)
    const bool k_does = QK != 48 || lane < 48;
    auto key_swizzle = [](int pos) { return KS == 64 ? (pos >> 2) & 3 : (pos >> 1) & 7; };
    auto value_swizzle = [](int dim) { return (dim >> 1) & 7; };
    const int32_t* table = c.tables + (size_t)max(seq, 0) * c.width;
    auto look_up = [&](int tile) NHIP_INLINE {
        return scalar_load(table, min((64 * tile + 16 * wave) >> c.page_shift, c.width - 1));
    };
    auto cell = [&](int tile, int page) NHIP_INLINE {
        const int pg = page >= 0 && page < c.pages ? page : 0;
        return (((size_t)pg * c.kv_heads + kvh) << c.page_shift) + ((64 * tile + 16 * wave) & in_page);
    };
    i32x4 kr[KU], vr[VU];
    float scale_r;
    auto load_keys = [&](int tile, int page) NHIP_INLINE {
        const size_t at = cell(tile, page);
#pragma unroll
        for (int u = 0; u < KU; u++)
            if (k_does)
                kr[u] = *reinterpret_cast<const i32x4*>(c.keys + at * QK + ((k_pos + 8 * u) * QK + 16 * k_ch));
        scale_r = (lane & 16 ? c.vscale : c.kscale)[at + (lane & 15)];
    };
    auto load_values = [&](int tile, int page) NHIP_INLINE {
        const size_t at = cell(tile, page);
#pragma unroll
        for (int u = 0; u < VU; u++)
            vr[u] = *reinterpret_cast<const i32x4*>(c.values + at * V + 16 * (lane + 64 * u));
    };
    auto store_keys = [&](int tile, int page) NHIP_INLINE {
#pragma unroll
        for (int u = 0; u < KU; u++) {
            const int pos = 16 * wave + k_pos + 8 * u;
            if (k_does)
                *reinterpret_cast<i32x4*>(lds_k[tile & 1] + pos * KS + 16 * (k_ch ^ key_swizzle(pos))) = kr[u];
        }
        // the positions that count, [lo, hi) of the block
        const int lo = from - 64 * tile - 16 * wave, hi = last_pos + 1 - 64 * tile - 16 * wave;
        uint32_t live = page >= 0 && page < c.pages ? 0xFFFFu : 0;
        live &= lo >= 16 ? 0 : 0xFFFFu << max(lo, 0);
        live &= hi <= 0 ? 0 : 0xFFFFu >> (16 - min(hi, 16));
        // A value scale that is no finite number spoils the rows that attend
        // its position, and no others: their score becomes NaN, the scale 0.
        const uint64_t odd = __ballot((__float_as_uint(scale_r) & 0x7F800000u) == 0x7F800000u) >> 16;
        float x = (odd >> (lane & 15)) & 1 ? (lane & 16 ? 0.0f : NAN) : scale_r;
        // (a position that counts has a scale above 0: the least there is makes its products 0)
        x = (live >> (lane & 15)) & 1 ? (lane & 16 ? fmaxf(x, kLeastScale) : x) : 0.0f;
        if (lane < 32) (lane & 16 ? lds_vs : lds_ks)[tile & 3][16 * wave + (lane & 15)] = x;
        if (lane == 0) lds_live[tile & 3][wave] = (uint16_t)live;
    };
    auto store_values = [&](int tile) NHIP_INLINE {
#pragma unroll
        for (int u = 0; u < VU; u++) {
            const int dim = lane + 64 * u;
#pragma unroll
            for (int e = 0; e < 2; e++)
                *reinterpret_cast<f16x8*>(lds_v[tile & 1] + dim * 128 + 16 * ((2 * wave + e) ^ value_swizzle(dim))) =
                    codes_f16((uint32_t)vr[u][2 * e], (uint32_t)vr[u][2 * e + 1]);
        }
    };

    f32x16 o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
    // base: M; bound: an exponent that no value scale of a tile may pass (ceiling:
    // 2^(bound + 1)) and limit: base + 14 - bound, which no score may pass,
    // without M being looked at again
    float base = kNoScore, bound = 0.0f, ceiling = 0.0f, limit = kNoScore, total = 0.0f;
    const float minus_one = alone(-1.0f);
    // where this lane reads: the key row of its A row, the value rows of its dimensions
    const int m = lane & 31;
    const int key_row = 16 * (m >> 4) + 8 * ((m >> 2) & 1) + 4 * ((m >> 3) & 1) + (m & 3);
    const int key_x = g ^ key_swizzle(key_row), value_x = g ^ value_swizzle(lane & 31);
    const int slot = 16 * ((lane >> 3) & 1) + 8 * g + (lane & 7);  // the position whose scales this lane holds

    if (begin < end) {
        // (past the last tile its own is staged again, and not used)
        auto clamped = [&](int tile) NHIP_INLINE { return min(tile, end - 1); };
        int page = look_up(begin);
        load_keys(begin, page);
        load_values(begin, page);
        int page_next = look_up(clamped(begin + 1));
        store_keys(begin, page);
        store_values(begin);
        __syncthreads();
        for (int tile = begin; tile < end; tile++) {
            page = page_next;
            load_keys(clamped(tile + 1), page);
            load_values(clamped(tile + 1), page);
            page_next = look_up(clamped(tile + 2));
            if ((64 * tile <= wave_last) & (64 * tile + 63 >= wave_first - from_window)) {
                const uint8_t* kb = lds_k[tile & 1] + key_row * KS;
                i32x16 s[2];
#pragma unroll
                for (int t = 0; t < 2; t++) {
#pragma unroll
                    for (int r = 0; r < 16; r++) s[t][r] = 0;
#pragma unroll
                    for (int k = 0; k < KK; k++)
                        s[t] = __builtin_amdgcn_mfma_i32_32x32x32_i8(
                            *reinterpret_cast<const i32x4*>(kb + 32 * t * KS + 16 * (key_x ^ (2 * k))), q[k], s[t], 0,
                            0, 0);
                }
                float ks[2], vs[2];
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    ks[t] = lds_ks[tile & 3][32 * t + slot];
                    vs[t] = lds_vs[tile & 3][32 * t + slot];
                }
                const uint2 counted = *reinterpret_cast<const uint2*>(lds_live[tile & 3]);
                float z[2][16];
#pragma unroll
                for (int t = 0; t < 2; t++) {
#define NHIP_DOT(r) z[t][r] = alone(row_bcast<r>(ks[t]) * (float)s[t][r]);
                    NHIP_DOT(0) NHIP_DOT(1) NHIP_DOT(2) NHIP_DOT(3) NHIP_DOT(4) NHIP_DOT(5) NHIP_DOT(6) NHIP_DOT(7)
                    NHIP_DOT(8) NHIP_DOT(9) NHIP_DOT(10) NHIP_DOT(11) NHIP_DOT(12) NHIP_DOT(13) NHIP_DOT(14)
                    NHIP_DOT(15)
#undef NHIP_DOT
                }
                const bool whole = __builtin_amdgcn_readfirstlane(counted.x & counted.y) == ~0u;
                const float largest = fmaxf(vs[0], vs[1]);  // of the lane's two positions
                const bool masked = !whole | (64 * tile + 63 > wave_first) | (64 * tile < wave_last - from_window);
                if (masked) {
                    const int last = q_pos - 64 * tile - 8 * g, first = q_first - 64 * tile - 8 * g;
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        const uint32_t bits = (t ? counted.y : counted.x) >> (8 * g);
#pragma unroll
                        for (int r = 0; r < 16; r++) {
                            const int at = 16 * (r / 8) + r % 8;
                            const bool attends =
                                (32 * t + at <= last) & (32 * t + at >= first) & ((bits >> at) & 1);
                            z[t][r] = attends ? z[t][r] : -INFINITY;
                        }
                    }
                }
                float up = z[0][0];
#pragma unroll
                for (int r = 1; r < 32; r++) up = fmaxf(up, z[r / 16][r % 16]);
                up = fmaxf(up, lane_xor<32>(up)) * qs;
                float to = base;
                if (__ballot((up > limit) | (largest >= ceiling))) {
                    // Values that are all 0 have scale 1 (QuantizeInt8), which says nothing
                    // of their size: the least in its place, so that the others keep their digits.
                    if (__ballot((vs[0] == 1.0f) | (vs[1] == 1.0f))) {
                        uint32_t any[4] = {0, 0, 0, 0};  // of 8 positions, lanes 8 o .. 8 o + 7 those of octet o
#pragma unroll
                        for (int k = 0; k < V / 8; k++) {
                            const int dim = 8 * k + (lane & 7);
                            const uint4 x = *reinterpret_cast<const uint4*>(lds_v[tile & 1] + dim * 128 +
                                                                            16 * ((lane >> 3) ^ value_swizzle(dim)));
                            any[0] |= x.x, any[1] |= x.y, any[2] |= x.z, any[3] |= x.w;
                        }
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            any[k] |= lane_xor<1>(any[k]);
                            any[k] |= lane_xor<2>(any[k]);
                            any[k] |= lane_xor<4>(any[k]);
                        }
#pragma unroll
                        for (int t = 0; t < 2; t++) {
                            uint32_t pair = 0;  // this lane's position and its neighbour
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const uint32_t x = (uint32_t)__shfl((int)any[k], (32 * t + slot) & ~7);
                                pair = ((lane >> 1) & 3) == k ? x : pair;
                            }
                            if (vs[t] == 1.0f && ((lane & 1 ? pair >> 16 : pair) & 0xFFFF) == 0) vs[t] = kLeastScale;
                        }
                    }
                    const float e[2] = {scale_exponent(vs[0]), scale_exponent(vs[1])};
                    bound = wave_max(fmaxf(e[0], e[1]));
                    // the scales within a factor of four: one exponent stands for all
                    float most = up + bound;
                    const float least = fminf(vs[0] > 0.0f ? e[0] : bound, vs[1] > 0.0f ? e[1] : bound);
                    if (wave_max(bound - least) > 1.0f) {
                        most = -INFINITY;
#pragma unroll
                        for (int t = 0; t < 2; t++) {
#define NHIP_MOST(r) most = fmaxf(most, z[t][r] * qs + row_bcast<r>(e[t]));
                            NHIP_MOST(0) NHIP_MOST(1) NHIP_MOST(2) NHIP_MOST(3) NHIP_MOST(4) NHIP_MOST(5) NHIP_MOST(6)
                            NHIP_MOST(7) NHIP_MOST(8) NHIP_MOST(9) NHIP_MOST(10) NHIP_MOST(11) NHIP_MOST(12)
                            NHIP_MOST(13) NHIP_MOST(14) NHIP_MOST(15)
#undef NHIP_MOST
                        }
                        most = fmaxf(most, lane_xor<32>(most));
                    }
                    to = most > base + kHeadroom ? most - (kHeadroom - kLag) : base;
                    ceiling = __uint_as_float((uint32_t)(128 + (int)bound) << 23);
                    limit = to + (kHeadroom - bound);
                }
                if (__ballot(to > base)) {
                    const float keep = __builtin_amdgcn_exp2f(base - to);
                    base = to;
                    total *= keep;
#pragma unroll
                    for (int d = 0; d < DT; d++) o[d] *= keep;
                }
                float sum[2] = {0.0f, 0.0f};  // of the tile: a long row's total is a sum of tiles' sums
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    float w[16];
#define NHIP_WEIGHT(r)                                       \
    w[r] = __builtin_amdgcn_exp2f(fmaf(z[t][r], qs, -base)); \
    sum[r & 1] += w[r];                                      \
    w[r] = alone(row_bcast<r>(vs[t]) * w[r]);
                    NHIP_WEIGHT(0) NHIP_WEIGHT(1) NHIP_WEIGHT(2) NHIP_WEIGHT(3) NHIP_WEIGHT(4) NHIP_WEIGHT(5)
                    NHIP_WEIGHT(6) NHIP_WEIGHT(7) NHIP_WEIGHT(8) NHIP_WEIGHT(9) NHIP_WEIGHT(10) NHIP_WEIGHT(11)
                    NHIP_WEIGHT(12) NHIP_WEIGHT(13) NHIP_WEIGHT(14) NHIP_WEIGHT(15)
#undef NHIP_WEIGHT
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        union {
                            f16x2 h[4];
                            f16x8 v;
                        } hi, lo;
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const float a = w[8 * u + 2 * k], b = w[8 * u + 2 * k + 1];
                            hi.h[k] = to_f16(a, b);
                            lo.h[k] = rest_f16(a, b, hi.h[k], minus_one);
                        }
                        const uint8_t* vb = lds_v[tile & 1] + (lane & 31) * 128 + 16 * (value_x ^ (4 * t + 2 * u));
#pragma unroll
                        for (int d = 0; d < DT; d++) {
                            const f16x8 v = *reinterpret_cast<const f16x8*>(vb + 32 * 128 * d);
                            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, hi.v, o[d], 0, 0, 0);
                            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, lo.v, o[d], 0, 0, 0);
                        }
                    }
                }
                total += sum[0] + sum[1];
            }
            store_keys(tile + 1, page);
            store_values(tile + 1);
            __syncthreads();
        }
    }

    float all = total + lane_xor<32>(total);
    if (!mine) return;
    if (q_pos < 0) {  // a row out of range, in a tile of others
        all = 0.0f;
        base = kNoScore;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
    }
    float factor;
    float* to;
    if (parts <= 1) {
        factor = all != 0.0f ? 1.0f / all : 0.0f;
        to = p.out + q_at * V;
    } else {
        const size_t at = q_at * p.max_parts + part;
        factor = 1.0f;
        to = p.parts + at * V;
        if (g == 0) *reinterpret_cast<float2*>(p.stats + 2 * at) = make_float2(base, all);
    }
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const f32x4 x = {o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]};
            *reinterpret_cast<f32x4*>(to + 32 * d + 8 * b + 4 * g) = x * factor;
        }
}

// Joins the parts of rows that were split, a wave per (row, head); rows of no
// run have no parts.  A row's parts follow from its run, as its tile counted
// them: nothing is read of a workspace that no tile has written, also where
// the runs overlap (run_rows that do not ascend) and not every tile finds a
// place in the grid.  (Split calls have few tiles, so few runs, whose tiles
// are placed in the runs' order.)
template <int V>
__global__ __launch_bounds__(256) void paged_prompt_join_kernel(PromptParams p)
{
    const int row = blockIdx.x, lane = threadIdx.x & 63;
    const int head = (int)blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (head >= p.heads) return;
    int tiles_before = 0;
    RunRows r = {0, 0};
    RunPositions at = {};
    uint64_t hit = 0;
    for (int i0 = 0; i0 < p.runs && hit == 0; i0 += 64) {
        // (a run's four words at once: the join is a chain of latencies)
        const int i = min(i0 + lane, p.runs - 1);
        const int first_row = p.run_rows[i], seq = p.run_seq[i], pos = p.run_pos[i];
        RunRows own = run_rows(p, i);
        if (i0 + lane > i) own = {0, 0};
        hit = __ballot(row >= own.row0 && row < own.row1);
        const int l = hit ? __builtin_ctzll(hit) : 63;
        r = {__builtin_amdgcn_readlane(own.row0, l), __builtin_amdgcn_readlane(own.row1, l)};
        at = run_positions(p, r.row0, __builtin_amdgcn_readlane(first_row, l), __builtin_amdgcn_readlane(seq, l),
                           __builtin_amdgcn_readlane(pos, l));
        if (l > 0) tiles_before += wave_sum_i32(hit == 0 || lane < l ? run_tiles(p, own) : 0);
    }
    if (hit == 0) return;
    const int queries = (r.row1 - r.row0) * p.group, tiles = run_tiles(p, r);
    const int of_group = head - over_group(p, head) * p.group;
    const int tile = ((row - r.row0) * p.group + of_group) / kTileQueries;
    if (__builtin_amdgcn_readfirstlane(tiles_before) + tiles - 1 - tile >= p.places) return;
    const int q0 = tile * kTileQueries;
    const int parts = tile_span(p, at.at(p, q0), at.at(p, min(q0 + kTileQueries, queries) - 1)).parts;
    if (parts <= 1) return;
    const size_t q_at = (size_t)row * p.heads + head;
    const size_t first = q_at * p.max_parts;
    float2 stat = make_float2(kNoScore, 0.0f);
    if (lane < parts) stat = *reinterpret_cast<const float2*>(p.stats + 2 * (first + lane));
    const float factor = __builtin_amdgcn_exp2f(stat.x - wave_max(stat.x));
    float all = factor * stat.y;
    all = rows_sum(all);
    all += lane_xor<8>(all);
    all += lane_xor<4>(all);
    all += lane_xor<2>(all);
    all += lane_xor<1>(all);
    constexpr int E = V / 64;
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; e++) sum[e] = 0.0f;
    const float* from = p.parts + first * V + lane;
    for (int k = 0; k < parts; k += 4) {
        float x[4][E];
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int e = 0; e < E; e++) x[u][e] = from[(size_t)min(k + u, parts - 1) * V + 64 * e];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const float f = k + u < parts ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(factor), k + u)) : 0.0f;
#pragma unroll
            for (int e = 0; e < E; e++) sum[e] = k + u < parts ? fmaf(x[u][e], f, sum[e]) : sum[e];
        }
    }
#pragma unroll
    for (int e = 0; e < E; e++) p.out[q_at * V + lane + 64 * e] = all != 0.0f ? sum[e] / all : 0.0f;
}

int32_t check_attention(const nhip_paged_cache* c, int32_t rows, int32_t heads, int32_t max_count)
{
    int32_t rc = paged_check(c);
    if (rc) return rc;
    NHIP_REQUIRE(rows >= 0 && rows <= kPagedMaxRows, "paged attention: %d rows", rows);
    NHIP_REQUIRE(heads >= 1 && heads % c->kv_heads == 0 && heads / c->kv_heads <= 16,
                 "paged attention: %d heads on %d kv heads (a multiple, at most 16 times as many)", heads,
                 c->kv_heads);
    NHIP_REQUIRE(max_count >= 0 && max_count <= c->width * c->page_size,
                 "paged attention: max_count %d out of range (a sequence holds %d positions)", max_count,
                 c->width * c->page_size);
    return NHIP_OK;
}

int32_t check_runs(int32_t runs, int32_t window)
{
    NHIP_REQUIRE(runs >= 0 && runs <= kPagedMaxRows && window >= 0, "paged prompt: %d runs, window %d", runs, window);
    return NHIP_OK;
}

int32_t check_call(const nhip_paged_cache* c, int32_t layer, const int8_t* q, const float* q_scales, const float* out,
                   const void* ws, size_t bytes, size_t need)
{
    NHIP_REQUIRE(layer >= 0 && layer < c->layers, "paged attention: layer %d of %d", layer, c->layers);
    NHIP_REQUIRE(q && q_scales && out, "paged attention: null pointer");
    NHIP_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
                 "paged attention: q or out is not 16-byte aligned");
    NHIP_REQUIRE(need == 0 || (ws && (reinterpret_cast<uintptr_t>(ws) & 15) == 0 && bytes >= need),
                 "paged attention: the workspace (%zu bytes) is missing, misaligned or smaller than %zu bytes", bytes,
                 need);
    return NHIP_OK;
}

// How a prompt call is split: places of tiles of 128 queries, and where those
// are few, 64-position blocks of a part and parts of the longest row.
struct PromptSplit {
    int64_t tiles;
    int blocks, parts, tiles_a_round;
};

// A block takes 1 to 2.5 us of a workgroup, joining parts about 4 us.  Where
// the tiles fill the CUs, or have fewer than 6 blocks, they stay whole (16 runs of up to 700 rows, 16 kv
// heads: 34 us whole, 45 in two parts).  Up to 96 workgroups, or 256 with 32
// or more blocks each, are split until about 768 are there, in parts of two
// blocks or more (16 rows after 32,000 positions, 8 kv heads of 128: 798 us
// whole, 37 in 63 parts; 512 rows after 8,000, 16 kv heads: 182 and 56; 416
// rows from 0, 112 workgroups of up to 8 blocks: 14.8 whole, 16.7 in parts).
// A window bounds a tile's blocks; it never makes more parts, as the workspace
// is sized without it.
PromptSplit prompt_split(const nhip_paged_cache* c, int32_t rows, int32_t heads, int32_t runs, int32_t max_count,
                         int32_t window)
{
    const int group = heads / c->kv_heads;
    PromptSplit s;
    s.tiles = (int64_t)rows * group / kTileQueries + runs;
    const int64_t units = s.tiles * c->kv_heads;
    int most = max_count / 64 + 2;
    s.blocks = most;
    if (most >= 6 && (units <= 96 || (units <= 256 && most >= 32)))
        s.blocks = (int)std::min<int64_t>(
            most, std::max<int64_t>({2, (units * most + 767) / 768, (most + kMaxParts - 1) / kMaxParts}));
    s.parts = (most + s.blocks - 1) / s.blocks;
    if (window > 0 && window < max_count) {
        most = std::min<int64_t>(most, ((int64_t)window + kTileQueries / group) / 64 + 2);
        s.blocks = std::max(2, (most + s.parts - 1) / s.parts);
        s.parts = (most + s.blocks - 1) / s.blocks;
    }
    s.tiles_a_round = 0;
    const int64_t groups = s.tiles * c->kv_heads;
    if (runs > 1 && runs <= kSortedRuns && s.parts == 1 && groups > 256 && groups <= kSortedGroups) {
        s.tiles_a_round = std::max(1, 256 / c->kv_heads);
        s.tiles = (s.tiles + s.tiles_a_round - 1) / s.tiles_a_round * s.tiles_a_round;
    }
    return s;
}

size_t prompt_workspace(const nhip_paged_cache* c, int32_t rows, int32_t heads, const PromptSplit& s)
{
    return s.parts > 1 ? (size_t)rows * heads * s.parts * (c->v_dim + 2) * sizeof(float) : 0;
}

template <int QK, int V>
int32_t launch_prompt(const PromptParams& p, const PromptSplit& s, hipStream_t stream)
{
    hipLaunchKernelGGL((paged_prompt_kernel<QK, V>), dim3(s.tiles * p.c.kv_heads, s.parts), dim3(256), 0, stream, p);
    NHIP_CHECK_HIP(hipGetLastError());
    if (s.parts > 1) {
        hipLaunchKernelGGL((paged_prompt_join_kernel<V>), dim3(p.rows, (p.heads + 3) / 4), dim3(256), 0, stream, p);
        NHIP_CHECK_HIP(hipGetLastError());
    }
    return NHIP_OK;
}

}  // namespace
}  // namespace nhip

using namespace nhip;

extern "C" {

size_t nhip_paged_decode_workspace(const nhip_paged_cache* c, int32_t rows, int32_t heads, int32_t max_count)
{
    if (check_attention(c, rows, heads, max_count)) return 0;
    return decode_workspace(c, rows, heads, decode_split(c, rows, max_count));
}

int32_t nhip_paged_decode_dev(const nhip_paged_cache* c, int32_t layer, const int8_t* d_q, const float* d_q_scales,
                              int32_t rows, int32_t heads, const int32_t* d_row_seq, const int32_t* d_row_first,
                              const int32_t* d_row_count, int32_t max_count, void* d_workspace,
                              size_t workspace_bytes, float* d_out, void* stream)
{
    int32_t rc = check_attention(c, rows, heads, max_count);
    if (rc) return rc;
    if (rows == 0) return NHIP_OK;
    const Split split = decode_split(c, rows, max_count);
    rc = check_call(c, layer, d_q, d_q_scales, d_out, d_workspace, workspace_bytes,
                    decode_workspace(c, rows, heads, split));
    if (rc) return rc;
    NHIP_REQUIRE(d_row_seq && d_row_first && d_row_count, "paged decode: null pointer");
    rc = ensure_device();
    if (rc) return rc;
    DecodeParams p;
    p.c = paged_layer(c, layer);
    p.q = d_q;
    p.q_scales = d_q_scales;
    p.out = d_out;
    p.row_seq = d_row_seq;
    p.row_first = d_row_first;
    p.row_count = d_row_count;
    p.parts = static_cast<float*>(d_workspace);
    p.stats = p.parts + (size_t)rows * heads * split.parts * c->v_dim;
    p.heads = heads;
    p.group = heads / c->kv_heads;
    p.max_count = max_count;
    p.blocks = split.blocks;
    p.max_parts = split.parts;
    p.rows = rows;
    p.rows_a_round = split.rows_a_round;
    p.scale = score_scale(c->qk_dim);
    if (c->qk_dim == 48) return launch_decode<48, 64>(p, split, rows, as_stream(stream));
    if (c->qk_dim == 64) return launch_decode<64, 64>(p, split, rows, as_stream(stream));
    return launch_decode<128, 128>(p, split, rows, as_stream(stream));
}

size_t nhip_paged_prompt_workspace(const nhip_paged_cache* c, int32_t rows, int32_t heads, int32_t runs,
                                   int32_t max_count)
{
    if (check_attention(c, rows, heads, max_count) || check_runs(runs, 0)) return 0;
    return prompt_workspace(c, rows, heads, prompt_split(c, rows, heads, runs, max_count, 0));
}

int32_t nhip_paged_prompt_dev(const nhip_paged_cache* c, int32_t layer, const int8_t* d_q, const float* d_q_scales,
                              int32_t rows, int32_t heads, int32_t runs, const int32_t* d_run_rows,
                              const int32_t* d_run_seq, const int32_t* d_run_pos, int32_t window, int32_t max_count,
                              void* d_workspace, size_t workspace_bytes, float* d_out, void* stream)
{
    int32_t rc = check_attention(c, rows, heads, max_count);
    if (rc) return rc;
    rc = check_runs(runs, window);
    if (rc) return rc;
    if (rows == 0 || runs == 0) return NHIP_OK;
    const PromptSplit split = prompt_split(c, rows, heads, runs, max_count, window);
    NHIP_REQUIRE(split.tiles * c->kv_heads <= (1 << 23), "paged prompt: %d rows in %d runs of %d kv heads are too many",
                 rows, runs, c->kv_heads);
    rc = check_call(c, layer, d_q, d_q_scales, d_out, d_workspace, workspace_bytes,
                    prompt_workspace(c, rows, heads, split));
    if (rc) return rc;
    NHIP_REQUIRE(d_run_rows && d_run_seq && d_run_pos, "paged prompt: null pointer");
    rc = ensure_device();
    if (rc) return rc;
    PromptParams p;
    p.c = paged_layer(c, layer);
    p.q = d_q;
    p.q_scales = d_q_scales;
    p.out = d_out;
    p.run_rows = d_run_rows;
    p.run_seq = d_run_seq;
    p.run_pos = d_run_pos;
    p.parts = static_cast<float*>(d_workspace);
    p.stats = p.parts + (size_t)rows * heads * split.parts * c->v_dim;
    p.rows = rows;
    p.heads = heads;
    p.group = heads / c->kv_heads;
    p.runs = runs;
    p.window = window;
    p.max_count = max_count;
    p.blocks = split.blocks;
    p.max_parts = split.parts;
    p.places = (int32_t)split.tiles;
    p.group_part = (uint32_t)(((1u << 31) + p.group - 1) / p.group);
    p.tiles_a_round = split.tiles_a_round;
    p.scale = score_scale(c->qk_dim);
    if (c->qk_dim == 48) return launch_prompt<48, 64>(p, split, as_stream(stream));
    if (c->qk_dim == 64) return launch_prompt<64, 64>(p, split, as_stream(stream));
    return launch_prompt<128, 128>(p, split, as_stream(stream));
}

}  // extern "C"
