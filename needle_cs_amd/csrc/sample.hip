// sample.hip -- one id per row of logits on gfx950: temperature, top-k,
// top-p, min-p and a draw with a given number.
//
// The order of a row's ids is that of composites (key(logit), ~id), 64-bit
// whole numbers: larger comes first, and no two are equal.  Whatever a rule
// keeps is a prefix of that order, so it is "composite >= cut".  Weights are
// whole multiples of 2^-42, so that every sum of them is exact and no order of
// summation shows, those by atomics into LDS among them; a sum of 2^19 weights
// stays below 2^62.
//
// A workgroup takes a row, which it keeps in registers where it is short, and reads
// from L2 or the last cache after the first pass.  It finds the largest logit, from
// its threads' own largest a logit that what is kept will hardly fall below, and
// gathers the ids above that into LDS, where the rules and the draw are ranks of
// few ids or histograms of many.  A share of the mass is found by a histogram of
// the row, which every wave has of its own part, so that it says where the draw
// falls too.  So a row whose kept ids fit the list is read one to four times.  Rows
// that keep more than the list holds or than the guess allowed, and rows without
// rules, are walked instead, behind the passes that found that out: for each rule
// a histogram and the ids of the bin in which it ends (and where those are more
// than are ranked, a finer histogram and its ids, seven times at most), then the
// weights for the draw and the parts of the row in which it falls.
//
// One row is bound by the latency of the steps behind each pass: 32000 ids, the
// first 50 and 0.95 of the mass 12.8 us (13.3 read twice), greedy 5.2.  Rows of
// 131071 ids have a CU each however few they are; us for 1, 64 and 250 rows from
// memory (normal logits of deviation 2.5): greedy 11, 14 and 29 (131 MB, 4.5 TB/s),
// the first 50 and 0.95 of the mass 24, 27 and 51, 0.9 of the mass 77, 84 and 105,
// no rule 41, 45 and 62, the first 5000 50, 53 and 70, the first 30000, which are
// walked, 131, 158 and 193; 250 rows with a mask and settings of every kind 113 to
// 120, where the row that takes longest counts.  A pass costs about 22 by the
// reads, and 35 where it weighs: some 30 instructions an id, which all four SIMDs
// of a CU issue without a gap.
#include <algorithm>
#include <cmath>

#include "common.hpp"

namespace nhip {
namespace {

constexpr int kBins = 1024;    // of a histogram; in the first the last one holds what weighs nothing
constexpr int kSegment = 256;  // ids of a wave's step, four a lane
constexpr int kMaxIds = 1 << 19;
constexpr int kFewIds = 16384;  // at most, of a row by 256 threads
constexpr int kTerms = 10;
constexpr double kOne = 4398046511104.0;  // 2^42, the weight of the largest logit
constexpr float kLeastScore = -30.0f;     // e^-30 2^42 < 1/2: no weight

typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned long long u64;

// 2^f for |f| <= 1/2, interpolated at Chebyshev's points: within 2^-45.
constexpr double kPower[kTerms] = {1.0000000000000135,     0.6931471805599462,     0.2402265069564034,
                                   0.05550410866465167,    0.009618129193934313,   0.0013333558200794592,
                                   0.0001540343375125101,  1.5252672924850737e-05, 1.325964524488711e-06,
                                   1.0205905413765595e-07};

struct SampleParams {
    const float* logits;
    const uint32_t* mask;
    nhip_sampling s;
    int32_t* ids;
    float* logprobs;
    int32_t ldx, n, mask_ld, words;
    double power[kTerms];  // kPower, as arguments: they stay in scalar registers
    float none;            // -inf, which the compiler does not know (it would take NaN for a number)
};

// A larger key for a larger logit; +0 and -0 alike.
__device__ __forceinline__ uint32_t key_of(float l)
{
    const uint32_t u = __float_as_uint(l + 0.0f);
    return u ^ (u >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key)
{
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ u64 composite(float l, int id) { return (u64)key_of(l) << 32 | (uint32_t)~id; }
__device__ __forceinline__ float logit_in(u64 c) { return logit_of((uint32_t)(c >> 32)); }
__device__ __forceinline__ int id_in(u64 c) { return ~(int)(uint32_t)c; }

// A row's logits as they count: -inf where an id may not be drawn (by the mask,
// or a NaN); in a row with +inf that is 0 and the others -inf.
struct Row {
    const float* x;
    const uint32_t* mask;
    int n;
    float none;  // -inf
    bool infinite;
};
__device__ __forceinline__ f4 counted4(const Row& r, f4 v, uint32_t bits)
{
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = __builtin_amdgcn_fmed3f(v[e], r.none, INFINITY);  // (of a NaN the least)
    if (r.mask) {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = (bits >> e) & 1 ? v[e] : -INFINITY;
    }
    if (r.infinite) {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = v[e] == INFINITY ? 0.0f : -INFINITY;
    }
    return v;
}

// How logits become weights, by the largest of them and a temperature.
struct Scale {
    double peak, log2e;      // log2e: log2(e) / temperature
    float half_peak, bins;   // a bin is (half_peak - logit / 2) * bins, which does not overflow
    const double* power;
};
__device__ __forceinline__ Scale scale_of(float peak, float temperature, const double* power)
{
    const double inverse = 1.0 / (double)temperature;
    // (bins is never 0, so that -inf comes last under an infinite temperature too)
    const double bins = fmin(fmax(2.0 * (kBins - 1) / -kLeastScore * inverse, 1.2e-38), 3e38);
    return {(double)peak, 1.4426950408889634 * inverse, 0.5f * peak, (float)bins, power};
}

// round(2^42 e^((l - peak) / temperature)): 2^t, t = n + f with a whole n and
// |f| <= 1/2; at t = -22, which takes the place of all below it and of -inf, it is 0.
__device__ __forceinline__ u64 weight(const Scale& z, float l)
{
    const double t = fmax(fma((double)l - z.peak, z.log2e, 42.0), -22.0), n = rint(t), f = t - n;
    double y = z.power[kTerms - 1];
#pragma unroll
    for (int k = kTerms - 2; k >= 0; k--) y = fma(y, f, z.power[k]);
    // (a whole number below 2^51 plus 2^52 is itself in the low bits)
    const double x = ldexp(y, (int)n) + 4503599627370496.0;
    return (u64)__double_as_longlong(x) & 0xFFFFFFFFFFFFFull;
}

// Four of them, a chain of 20 dependent operations each, side by side.
struct Weights {
    u64 w[4];
};
__device__ __forceinline__ Weights weights4(const Scale& z, f4 l)
{
    double y[4], f[4];
    int n[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const double t = fmax(fma((double)l[e] - z.peak, z.log2e, 42.0), -22.0), whole = rint(t);
        f[e] = t - whole;
        n[e] = (int)whole;
        y[e] = z.power[kTerms - 1];
    }
#pragma unroll
    for (int k = kTerms - 2; k >= 0; k--)
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = fma(y[e], f[e], z.power[k]);
    Weights r;
#pragma unroll
    for (int e = 0; e < 4; e++)
        r.w[e] = (u64)__double_as_longlong(ldexp(y[e], n[e]) + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
    return r;
}

// The bin of the first histogram, which descends with the logit: kBins - 1 for what weighs nothing.
__device__ __forceinline__ int first_bin(const Scale& z, float l)
{
    return (int)fminf((z.half_peak - 0.5f * l) * z.bins, (float)(kBins - 1));
}

__device__ __forceinline__ uint32_t mask_bits(const Row& r, int i)
{
    return r.mask ? r.mask[i >> 5] >> (i & 31) : 15u;
}

// Four logits from id i of a segment, -inf past the row's end.
__device__ __forceinline__ f4 segment4(const Row& r, int i)
{
    f4 v;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = i + e < r.n ? r.x[i + e] : -INFINITY;
    return counted4(r, v, i < r.n ? mask_bits(r, i) : 0u);
}

// f(first id, logits) for every four ids of the segments `segment`, + step, ... below
// `end`, by one wave: a wave's 64 fours are one segment; U of its segments are at
// work and the next U's loads in flight.
template <int U, typename F>
__device__ __forceinline__ void walk(const Row& r, int segment, int end, int step, F f)
{
    const int lane = threadIdx.x & 63, whole = min(r.n / kSegment, end);
    f4 v[U], next[U];
    uint32_t bits[U], next_bits[U];
    auto load = [&](int first, f4 (&x)[U], uint32_t (&m)[U]) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = kSegment * min(first + step * u, whole - 1) + 4 * lane;
            x[u] = *reinterpret_cast<const f4*>(r.x + i);
            m[u] = mask_bits(r, i);
        }
    };
    if (segment < whole) load(segment, v, bits);
    for (; segment < whole; segment += step * U) {
        if (segment + step * U < whole) load(segment + step * U, next, next_bits);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (segment + step * u < whole) f(kSegment * (segment + step * u) + 4 * lane, counted4(r, v[u], bits[u]));
            __builtin_amdgcn_sched_barrier(0);  // (one four at a time in the registers)
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            v[u] = next[u];
            bits[u] = next_bits[u];
        }
    }
}

__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// f as above for all of the row, by the T threads of the workgroup.
template <int T, int U, typename F>
__device__ __forceinline__ void each4(const Row& r, F f)
{
    constexpr int W = T / 64;
    const int whole = r.n / kSegment;
    walk<U>(r, wave_id(), whole, W, f);
    if (whole * kSegment < r.n && wave_id() == whole % W) {
        const int i = kSegment * whole + 4 * (int)(threadIdx.x & 63);
        f(i, segment4(r, i));
    }
}

template <int S>
__device__ __forceinline__ u64 lane_xor_u64(u64 v)
{
    return (u64)lane_xor<S>((uint32_t)(v >> 32)) << 32 | lane_xor<S>((uint32_t)v);
}
template <int S>
__device__ __forceinline__ u64 add_lane_xor(u64 v)
{
    return v + lane_xor_u64<S>(v);
}
template <int S>
__device__ __forceinline__ u64 max_lane_xor(u64 v)
{
    return max(v, lane_xor_u64<S>(v));
}
// The same of a row of up to 4 G T ids, which each thread keeps, G fours of it.
template <int T>
__device__ __forceinline__ int held_id(int j)
{
    return kSegment * (wave_id() + T / 64 * j) + 4 * (int)(threadIdx.x & 63);
}
template <int T, int G>
__device__ __forceinline__ void hold(const Row& r, f4 (&v)[G])
{
    const int whole = r.n / kSegment;
    uint32_t bits[G];
#pragma unroll
    for (int j = 0; j < G; j++) {
        const int segment = wave_id() + T / 64 * j, i = held_id<T>(j);
        v[j] = f4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        bits[j] = 0;
        if (segment < whole) {
            v[j] = *reinterpret_cast<const f4*>(r.x + i);
            bits[j] = mask_bits(r, i);
        } else if (segment == whole && i < r.n) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[j][e] = i + e < r.n ? r.x[i + e] : -INFINITY;
            bits[j] = mask_bits(r, i);
        }
    }
#pragma unroll
    for (int j = 0; j < G; j++) v[j] = counted4(r, v[j], bits[j]);
}

// Sum over the wave, in every lane, and the largest.
__device__ __forceinline__ u64 wave_sum_u64(u64 v)
{
    return add_lane_xor<32>(add_lane_xor<16>(add_lane_xor<8>(add_lane_xor<4>(add_lane_xor<2>(add_lane_xor<1>(v))))));
}
__device__ __forceinline__ u64 wave_max_u64(u64 v)
{
    return max_lane_xor<32>(max_lane_xor<16>(max_lane_xor<8>(max_lane_xor<4>(max_lane_xor<2>(max_lane_xor<1>(v))))));
}
// Sum over the 2, 4 or 16 neighbours that share an id, in each of them.
__device__ __forceinline__ u64 shared_sum(u64 v, int threads)
{
    v = add_lane_xor<1>(v);
    if (threads > 2) v = add_lane_xor<2>(v);
    if (threads > 4) v = add_lane_xor<8>(add_lane_xor<4>(v));
    return v;
}
// Sum of the lanes up to this one: within rows of 16 lanes, then the last
// lane's of a row to the next one's, and lane 31's to the upper half.
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 add_lane_below(u64 v)
{
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, false);
    return v + ((u64)hi << 32 | lo);
}
__device__ __forceinline__ u64 wave_upto(u64 v)
{
    v = add_lane_below<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8
    v = add_lane_below<0x112, 0xF>(v);
    v = add_lane_below<0x114, 0xF>(v);
    v = add_lane_below<0x118, 0xF>(v);
    v = add_lane_below<0x142, 0xA>(v);  // row_bcast:15 to rows 1 and 3
    return add_lane_below<0x143, 0xC>(v);  // row_bcast:31 to rows 2 and 3
}

// A histogram of the row for every wave, of the wave's part of it.  Where ids are
// listed the list has their place, and its histograms are short.
template <int T>
struct Shared {
    static constexpr int WAVES = T / 64, LIST = kBins * WAVES / 2, OWN = LIST / WAVES;
    static constexpr int RANKED = T / 2, FEW = T / 2;  // ids that are ranked against one another
    union {
        u64 bins[WAVES * kBins];
        struct {
            u64 list[WAVES][OWN], weights[WAVES][OWN];  // each wave's own
        };
    };
    u64 counts[kBins];
    u64 few[FEW], few_weights[FEW];
    u64 waves[T / 64], parts[T / 64];
    uint32_t listed[WAVES];
    uint32_t few_listed, bin, key;
    u64 cut, before, mass, total, least, most;

    // what the sizes ask of one another
    static_assert(kBins % T == 0, "find_bin gives every thread as many bins");
    static_assert(OWN % kSegment == 0, "a row of LIST ids, its segments dealt to the waves in turn, fits their lists");
    static_assert(2 * RANKED <= T && 2 * FEW <= T, "an id that is ranked has two threads or more (shares)");
    static_assert(RANKED <= FEW, "draw_of_few's ids are copied into few");
    static_assert((T == 256 ? kFewIds : kMaxIds) / kBins <= FEW, "draw_of_many's bin of neighbours fits few");
};
static_assert(sizeof(Shared<1024>) <= 160 * 1024 && 3 * sizeof(Shared<256>) <= 160 * 1024, "LDS of a CU");

// The sum over the workgroup, in every thread.
template <int T>
__device__ __forceinline__ u64 block_sum(Shared<T>& sh, u64 v)
{
    v = wave_sum_u64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.waves[threadIdx.x >> 6] = v;
    __syncthreads();
    u64 sum = 0;
#pragma unroll
    for (int w = 0; w < T / 64; w++) sum += sh.waves[w];
    return sum;
}

// What a rule keeps, by the sum of what stands before an id: of ones (top_k) or
// of weights (top_p: those before the mass, and always the first).
struct Limit {
    u64 count;
    double mass;
    __device__ __forceinline__ bool inside(u64 before) const
    {
        return count ? before < count : (double)before < mass;
    }
};
__device__ __forceinline__ Limit mass_limit(float top_p, u64 total)
{
    return {0, fmax((double)top_p * (double)total, 0.5)};
}

// One row's settings.
struct Rules {
    int top_k;  // 0: all
    bool by_mass;
    float top_p, random;
    u64 least;  // min_p's weight, rounded up
};

// The bin of a histogram (the sum of `copies`) in which a rule ends, and
// the sum before it, in sh.bin and sh.before; kBins where it does not end.
// SHARE: the rule is the share top_p of all bins.  The sum of all bins.
template <int T, bool SHARE>
__device__ __forceinline__ u64 find_bin(Shared<T>& sh, const u64* bins, int copies, u64 before, Limit limit,
                                        float top_p)
{
    constexpr int B = kBins / T;
    u64 q[B], own = 0;
#pragma unroll
    for (int k = 0; k < B; k++) {
        const int b = B * threadIdx.x + k;
        q[k] = 0;
        for (int c = 0; c < copies; c++) q[k] += bins[c * kBins + b];
        own += q[k];
    }
    const u64 upto = wave_upto(own);
    if ((threadIdx.x & 63) == 63) sh.waves[threadIdx.x >> 6] = upto;
    if (threadIdx.x == 0) sh.bin = kBins;
    __syncthreads();
    u64 all = 0;
    before += upto - own;
#pragma unroll
    for (int w = 0; w < T / 64; w++) {
        const u64 x = sh.waves[w];
        if (w < (int)(threadIdx.x >> 6)) before += x;
        all += x;
    }
    if (SHARE) limit = mass_limit(top_p, all);
#pragma unroll
    for (int k = 0; k < B; k++) {
        if (limit.inside(before) && !limit.inside(before + q[k])) {
            sh.bin = B * threadIdx.x + k;
            sh.before = before;
        }
        before += q[k];
    }
    __syncthreads();
    return all;
}

template <int T>
__device__ __forceinline__ void clear_bins(u64* bins, int n)
{
    for (int b = threadIdx.x; b < n; b += T) bins[b] = 0;
    __syncthreads();
}

// A wave's part of a row, or of the segments [first, end) of it.
struct Part {
    int each, from, to;
};
template <int T>
__device__ __forceinline__ Part part_of(int wave, int first, int end)
{
    const int each = (end - first + T / 64 - 1) / (T / 64), from = min(first + wave * each, end);
    return {each, from, min(end, from + each)};
}
__device__ __forceinline__ int segments_of(const Row& r) { return (r.n + kSegment - 1) / kSegment; }
// f(first id, logits) for every four ids of a part.
template <typename F>
__device__ __forceinline__ void walk_part(const Row& r, const Part& p, F f)
{
    walk<2>(r, p.from, p.to, 1, f);
    if (p.from < p.to && p.to == segments_of(r) && r.n % kSegment) {
        const int i = kSegment * (p.to - 1) + 4 * (int)(threadIdx.x & 63);
        f(i, segment4(r, i));
    }
}

// The ids that the rules below are about: f(composite, logit, its weight (WEIGHTS) or 1) for each.
template <int T>
struct RowIds {  // of the row itself
    static constexpr int COPIES = Shared<T>::WAVES;
    const Row& r;
    template <bool WEIGHTS, typename F>
    __device__ __forceinline__ void each(const Shared<T>&, const Scale& z, F f) const
    {
        walk_part(r, part_of<T>(wave_id(), 0, segments_of(r)), [&](int id, f4 l) {
            Weights w = {{1, 1, 1, 1}};
            if (WEIGHTS) w = weights4(z, l);
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (l[e] > -INFINITY) f(composite(l[e], id + e), l[e], w.w[e]);
        });
    }
    __device__ __forceinline__ u64* bins(Shared<T>& sh) const { return sh.bins; }
};
template <int T>
struct ListIds {  // of sh.list, with their weights, every wave its own
    static constexpr int COPIES = 1;
    template <bool WEIGHTS, typename F>
    __device__ __forceinline__ void each(const Shared<T>& sh, const Scale&, F f) const
    {
        const int wave = wave_id(), listed = sh.listed[wave];
        for (int e = threadIdx.x & 63; e < listed; e += 64) {
            const u64 c = sh.list[wave][e];
            f(c, logit_in(c), WEIGHTS ? sh.weights[wave][e] : 1);
        }
    }
    __device__ __forceinline__ u64* bins(Shared<T>& sh) const { return sh.counts; }
};

// The wave's own list with the lanes' ids for which `taken`, `here` before and the result after,
// which is more than OWN where it has no place for them.
template <int T>
__device__ __forceinline__ int list_id(Shared<T>& sh, int here, bool taken, float l, int id)
{
    const uint64_t all = __ballot(taken);
    const int at = here + __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
    if (taken && at < Shared<T>::OWN) sh.list[wave_id()][at] = composite(l, id);
    return here + __popcll(all);
}

// The place of a thread among those that share the ids of a short list, `threads` to one.
struct Shares {
    int threads, place, step, first;
};
template <int T>
__device__ __forceinline__ Shares shares(int listed)
{
    Shares s;
    s.threads = __builtin_amdgcn_readfirstlane(listed <= T / 16 ? 16 : listed <= T / 4 ? 4 : 2);
    s.place = threadIdx.x & (s.threads - 1);
    s.step = T / s.threads;
    s.first = threadIdx.x / s.threads;
    return s;
}

// The composite of the last id that a rule keeps (masses: by weights, or by ones), where
// that is in a bin of the first histogram and `before` stands before it; cut where it is not.
// Finer histograms by composites while more ids are left than are ranked.
template <int T, typename Ids>
__device__ __forceinline__ u64 last_in_bin(Shared<T>& sh, const Scale& z, const Ids& ids, u64 cut, int bin, bool masses,
                                           const Limit& limit, u64 before)
{
    constexpr int C = Ids::COPIES;
    u64* bins = ids.bins(sh);
    u64* own_bins = bins + (C > 1 ? wave_id() * kBins : 0);
    u64 lo = 0, hi = ~(u64)0;
    auto inside = [&](u64 c, float l) { return first_bin(z, l) == bin && c >= cut && c >= lo && c <= hi; };
    int listed = 0;
    // (64 bits, ten at a time: seven rounds end it, whatever a second look at the logits says)
    for (int round = 0; round < 8; round++) {
        __syncthreads();
        if (threadIdx.x == 0) {
            sh.few_listed = 0;
            sh.least = ~(u64)0;
            sh.most = 0;
        }
        __syncthreads();
        u64 least = ~(u64)0, most = 0;
        ids.template each<false>(sh, z, [&](u64 c, float l, u64) {
            if (inside(c, l)) {
                least = min(least, c);
                most = max(most, c);
                const uint32_t at = atomicAdd(&sh.few_listed, 1u);
                if (at < (uint32_t)Shared<T>::FEW) sh.few[at] = c;
            }
        });
        if (most) {
            atomicMin(&sh.least, least);
            atomicMax(&sh.most, most);
        }
        __syncthreads();
        listed = sh.few_listed;
        if (listed <= Shared<T>::FEW) break;
        lo = sh.least;
        hi = sh.most;
        const int shift = hi > lo ? max(0, 64 - __builtin_clzll(hi - lo) - 10) : 0;
        clear_bins<T>(bins, kBins * C);
        ids.template each<true>(sh, z, [&](u64 c, float l, u64 w) {
            if (inside(c, l)) atomicAdd(&own_bins[(int)((hi - c) >> shift)], masses ? w : 1);
        });
        __syncthreads();
        find_bin<T, false>(sh, bins, C, before, limit, 0.0f);
        before = sh.before;
        hi -= (u64)min(sh.bin, (uint32_t)kBins - 1) << shift;
        lo = max(lo, hi - (((u64)1 << shift) - 1));
    }
    listed = min(listed, Shared<T>::FEW);
    if (threadIdx.x == 0) sh.cut = cut;
    if ((int)threadIdx.x < listed) sh.few_weights[threadIdx.x] = masses ? weight(z, logit_in(sh.few[threadIdx.x])) : 1;
    __syncthreads();
    const Shares s = shares<T>(listed);
    const u64 own = s.first < listed ? sh.few[s.first] : 0;
    u64 larger = 0;
    for (int i = s.place; i < listed; i += s.threads) {
        const u64 q = sh.few_weights[i];
        larger += sh.few[i] > own ? q : 0;
    }
    larger = shared_sum(larger, s.threads);
    larger += before;
    if (s.first < listed && s.place == 0 && limit.inside(larger) && !limit.inside(larger + sh.few_weights[s.first]))
        sh.cut = own;
    __syncthreads();
    return sh.cut;
}

// The composite of the last id that a rule keeps of `ids` from `cut` on: the first
// `count` (0: the share top_p of them, or with total0 the ids that weigh less than that
// share of it before them).  0 where it keeps all.  A histogram by logit, then the bin
// in which the rule ends.
template <int T, typename Ids>
__device__ __forceinline__ u64 last_kept(Shared<T>& sh, const Scale& z, const Ids& ids, u64 cut, int count, float top_p,
                                         u64 total0)
{
    const bool masses = count == 0;
    constexpr int C = Ids::COPIES;
    u64* bins = ids.bins(sh);
    u64* own_bins = bins + (C > 1 ? wave_id() * kBins : 0);
    clear_bins<T>(bins, kBins * C);
    auto add = [&](u64 c, float l, u64 q) {
        const int b = first_bin(z, l);
        if (b < kBins - 1 && c >= cut) atomicAdd(&own_bins[b], q);
    };
    if (masses)
        ids.template each<true>(sh, z, add);
    else
        ids.template each<false>(sh, z, add);
    __syncthreads();
    Limit limit = masses ? mass_limit(top_p, total0) : Limit{(u64)count, 0.0};
    if (masses && total0 == 0)
        limit = mass_limit(top_p, find_bin<T, true>(sh, bins, C, 0, limit, top_p));
    else
        find_bin<T, false>(sh, bins, C, 0, limit, 0.0f);
    const int bin = sh.bin;
    if (bin == kBins) return 0;
    return last_in_bin(sh, z, ids, cut, bin, masses, limit, sh.before);
}

__device__ __forceinline__ float log_probability(const Scale& z, float l, u64 total)
{
    return (float)(((double)l - z.peak) * z.log2e * 0.6931471805599453 - log((double)total / kOne));
}

// The t of the draw.
__device__ __forceinline__ u64 drawn(float random, u64 total)
{
    const double u = random > 0.0f ? (double)random : 0.0;
    return min((u64)fmin(u * (double)total, kOne * kMaxIds), total - 1);
}

// What a draw found: a thread that has the id has it, the others have -1; all have
// `missed` where the list did not hold enough.
struct Chosen {
    int id;
    float logprob;
    bool missed;
};

// The rules and the draw over sh.list of up to RANKED ids, by ranks.  total0: the
// weight of all ids, for top_p without top_k.
template <int T>
__device__ __forceinline__ Chosen draw_of_few(Shared<T>& sh, const Scale& z, const Rules& rules, int listed, u64 total0)
{
    const Shares s = shares<T>(listed);
    // the waves' lists one behind the other
    const int wave = wave_id(), here = sh.listed[wave];
    int at_few = threadIdx.x & 63;
#pragma unroll
    for (int w = 0; w < T / 64; w++) at_few += w < wave ? sh.listed[w] : 0;
    for (int e = threadIdx.x & 63; e < here; e += 64, at_few += 64) {
        const u64 c = sh.list[wave][e];
        sh.few[at_few] = c;
        sh.few_weights[at_few] = weight(z, logit_in(c));
    }
    if (threadIdx.x == 0) sh.mass = sh.total = 0;
    __syncthreads();
    const bool first = s.first < listed && s.place == 0;
    const u64 own = s.first < listed ? sh.few[s.first] : 0, w = s.first < listed ? sh.few_weights[s.first] : 0;
    u64 larger = 0, rank = 0;
    for (int i = s.place; i < listed; i += s.threads) {
        const u64 c = sh.few[i], x = sh.few_weights[i];
        larger += c > own ? x : 0;
        rank += c > own ? 1 : 0;
    }
    larger = shared_sum(larger, s.threads);
    rank = shared_sum(rank, s.threads);
    bool kept = first && (rules.top_k == 0 || rank < (u64)rules.top_k);
    if (rules.by_mass && kept) atomicMax(&sh.mass, larger + w);  // (the last one has all)
    __syncthreads();  // (and every thread has read the weights, of which those below are set to 0)
    if (rules.by_mass) {
        const u64 mass = sh.mass;
        const Limit limit = mass_limit(rules.top_p, rules.top_k ? mass : total0);
        kept = kept && limit.inside(larger);
    }
    kept = kept && w >= rules.least;
    if (kept) atomicMax(&sh.total, larger + w);
    if (first) sh.few_weights[s.first] = kept ? w : 0;
    __syncthreads();
    const u64 total = sh.total, at = drawn(rules.random, total);
    u64 lower = 0;  // the kept weight of lower ids
    for (int i = s.place; i < listed; i += s.threads) {
        const u64 x = sh.few_weights[i];
        lower += (uint32_t)sh.few[i] > (uint32_t)own ? x : 0;
    }
    lower = shared_sum(lower, s.threads);
    if (kept && lower <= at && at < lower + w) return {id_in(own), log_probability(z, logit_in(own), total), false};
    return {-1, 0.0f, false};
}

// The same of more ids, by histograms.
template <int T>
__device__ __forceinline__ Chosen draw_of_many(Shared<T>& sh, const Scale& z, const Rules& rules, u64 total0, int n)
{
    const int lane = threadIdx.x & 63, wave = wave_id(), listed = sh.listed[wave];
    const u64* list = sh.list[wave];
    u64* weights = sh.weights[wave];
#pragma unroll 1
    for (int e = lane; e < listed; e += 64) weights[e] = weight(z, logit_in(list[e]));
    const ListIds<T> ids;
    u64 cut = 0;
#pragma unroll 1
    for (int rule = rules.top_k ? 0 : 1; rule < (rules.by_mass ? 2 : 1); rule++)
        cut = max(cut, last_kept(sh, z, ids, cut, rule == 0 ? rules.top_k : 0, rules.top_p, rules.top_k ? 0 : total0));
    u64 sum = 0;
    for (int e = lane; e < listed; e += 64) {
        const u64 w = list[e] >= cut && weights[e] >= rules.least ? weights[e] : 0;
        weights[e] = w;
        sum += w;
    }
    const u64 total = block_sum(sh, sum), at = drawn(rules.random, total);
    // in the order of the ids: a few neighbours of them, then the id
    // (the list has an id once, so that a bin has at most 2^shift)
    const int shift = max(0, 32 - __builtin_clz(n - 1) - 10);  // (n > 1)
    clear_bins<T>(sh.counts, kBins);
    for (int e = lane; e < listed; e += 64) atomicAdd(&sh.counts[min(id_in(list[e]) >> shift, kBins - 1)], weights[e]);
    if (threadIdx.x == 0) sh.few_listed = 0;
    __syncthreads();
    find_bin<T, false>(sh, sh.counts, 1, 0, Limit{at + 1, 0.0}, 0.0f);
    const int bin = sh.bin;
    const u64 before = sh.before;
    for (int e = lane; e < listed; e += 64)
        if (id_in(list[e]) >> shift == bin && weights[e]) {
            const uint32_t to = min(atomicAdd(&sh.few_listed, 1u), (uint32_t)Shared<T>::FEW - 1);
            sh.few[to] = list[e];
            sh.few_weights[to] = weights[e];
        }
    __syncthreads();
    const int few = min(sh.few_listed, (uint32_t)Shared<T>::FEW);
    const Shares s = shares<T>(few);
    const u64 own = s.first < few ? sh.few[s.first] : 0;
    u64 lower = 0;
    for (int i = s.place; i < few; i += s.threads) {
        const u64 x = sh.few_weights[i];
        lower += (uint32_t)sh.few[i] > (uint32_t)own ? x : 0;
    }
    lower = shared_sum(lower, s.threads);
    lower += before;
    if (s.first < few && s.place == 0 && lower <= at && at < lower + sh.few_weights[s.first])
        return {id_in(own), log_probability(z, logit_in(own), total), false};
    return {-1, 0.0f, false};
}

// The draw over the row itself, of what `cut` and min_p leave: its waves' parts, then
// the parts of the one that the draw falls into, down to a segment.  known: it falls
// into the segments [first, end), whose lower neighbours weigh `before`, and all is `total`.
template <int T>
__device__ __forceinline__ Chosen draw_of_row(Shared<T>& sh, const Row& r, const Scale& z, const Rules& rules, u64 cut,
                                              bool known, int first, int end, u64 before, u64 total)
{
    constexpr int W = T / 64;
    const int lane = threadIdx.x & 63, wave = wave_id();
    const bool all = cut == 0 && rules.least == 0;
    auto kept4 = [&](int id, f4 l) {
        Weights w = weights4(z, l);
        if (!all) {
#pragma unroll
            for (int e = 0; e < 4; e++) w.w[e] = composite(l[e], id + e) >= cut && w.w[e] >= rules.least ? w.w[e] : 0;
        }
        return w;
    };
    u64 at = known ? drawn(rules.random, total) : 0;
    while (!known || end - first > 1) {
        const Part part = part_of<T>(wave, first, end);
        u64 sum = 0;
        walk_part(r, part, [&](int id, f4 l) {
            const Weights w = kept4(id, l);
            sum += (w.w[0] + w.w[1]) + (w.w[2] + w.w[3]);
        });
        sum = wave_sum_u64(sum);
        __syncthreads();
        if (lane == 0) sh.waves[wave] = sum;
        __syncthreads();
        if (!known) {
#pragma unroll
            for (int w = 0; w < W; w++) total += sh.waves[w];
            at = drawn(rules.random, total);
            known = true;
        }
        // (the last part at most, whatever a second look at the logits says: another stream may be writing them)
        int of = 0;
        for (int w = 0; w + 1 < W && first + (of + 1) * part.each < end; w++) {
            if (before + sh.waves[w] > at) break;
            before += sh.waves[w];
            of++;
        }
        end = min(end, first + (of + 1) * part.each);
        first += of * part.each;
    }
    Chosen found = {-1, 0.0f, false};
    if (threadIdx.x < 64) {
        const int id = first * kSegment + 4 * lane;
        const f4 l = segment4(r, id);
        const Weights w = kept4(id, l);
        const u64 own = (w.w[0] + w.w[1]) + (w.w[2] + w.w[3]);
        u64 from = before + wave_upto(own) - own;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (from <= at && at < from + w.w[e]) found = {id + e, log_probability(z, l[e], total), false};
            from += w.w[e];
        }
    }
    return found;
}

// top_p alone: one pass for the histograms, one that lists the ids of the bin in
// which the share ends; with those every wave knows what its part keeps.  `missed`
// where the list does not hold them.
template <int T>
__device__ __forceinline__ Chosen draw_by_mass(Shared<T>& sh, const Row& r, const Scale& z, const Rules& rules)
{
    const int lane = threadIdx.x & 63, wave = wave_id();
    const Part part = part_of<T>(wave, 0, segments_of(r));
    u64* own_bins = sh.bins + wave * kBins;
    clear_bins<T>(sh.bins, T / 64 * kBins);
    walk_part(r, part, [&](int, f4 l) {
        const Weights w = weights4(z, l);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (w.w[e]) atomicAdd(&own_bins[first_bin(z, l[e])], w.w[e]);
    });
    __syncthreads();
    const u64 all = find_bin<T, true>(sh, sh.bins, T / 64, 0, Limit{0, 0.0}, rules.top_p);
    const Limit limit = mass_limit(rules.top_p, all);
    const int bin = sh.bin;
    u64 before = sh.before, mine = 0;
    if (bin == kBins) return {-1, 0.0f, true};
    for (int b = lane; b < bin; b += 64) mine += own_bins[b];
    __syncthreads();  // (the list takes the histograms' place)
    // (a bin's logits, and a little more, by their values alone)
    const bool any_logit = z.bins < 1e-30f;  // (bins so wide that what follows might overflow)
    const float width = 2.0f / z.bins, slack = 0.02f * width + 1e-6f * fabsf((float)z.peak);
    const float above = any_logit ? INFINITY : (float)z.peak - bin * width + slack;
    const float below = any_logit ? -INFINITY : (float)z.peak - (bin + 1) * width - slack;
    int here = 0;
    walk_part(r, part, [&](int id, f4 l) {
        bool any = false;
#pragma unroll
        for (int e = 0; e < 4; e++) any = any || (l[e] <= above && l[e] >= below);
        if (__ballot(any) == 0) return;
#pragma unroll
        for (int e = 0; e < 4; e++)
            here = list_id(sh, here, l[e] > -INFINITY && first_bin(z, l[e]) == bin, l[e], id + e);
    });
    const bool missed = here > Shared<T>::OWN;
    here = min(here, Shared<T>::OWN);
    for (int e = lane; e < here; e += 64) sh.weights[wave][e] = weight(z, logit_in(sh.list[wave][e]));
    if (lane == 0) sh.listed[wave] = here;
    if (__syncthreads_or(missed)) return {-1, 0.0f, true};
    const u64 cut = last_in_bin(sh, z, ListIds<T>(), 0, bin, true, limit, before);
    for (int e = lane; e < here; e += 64) mine += sh.list[wave][e] >= cut ? sh.weights[wave][e] : 0;
    mine = wave_sum_u64(mine);
    if (lane == 0) sh.parts[wave] = mine;
    __syncthreads();
    u64 total = 0;
#pragma unroll
    for (int k = 0; k < T / 64; k++) total += sh.parts[k];
    const u64 at = drawn(rules.random, total);
    int of = 0;
    before = 0;
    while (of + 1 < T / 64 && before + sh.parts[of] <= at) before += sh.parts[of++];
    const Part there = part_of<T>(of, 0, segments_of(r));
    if (there.from >= there.to) return {-1, 0.0f, true};
    return draw_of_row(sh, r, z, rules, cut, true, there.from, there.to, before, total);
}

// A logit that at least `want` of the threads' largest are not below: of `most` each,
// or with `two` of `other` too.
template <int T>
__device__ __forceinline__ float bound_of(Shared<T>& sh, const Scale& z, float most, float other, bool two, int want)
{
    if (threadIdx.x == 0) sh.key = ~0u;
    clear_bins<T>(sh.counts, kBins);
    const int b = first_bin(z, most), b2 = two ? first_bin(z, other) : kBins - 1;
    if (b < kBins - 1) atomicAdd(&sh.counts[b], (u64)1);
    if (two && b2 < kBins - 1) atomicAdd(&sh.counts[b2], (u64)1);
    __syncthreads();
    find_bin<T, false>(sh, sh.counts, 1, 0, Limit{(u64)want, 0.0}, 0.0f);
    if (sh.bin == kBins) return -INFINITY;
    if (b == (int)sh.bin) atomicMin(&sh.key, key_of(most));
    if (two && b2 == (int)sh.bin) atomicMin(&sh.key, key_of(other));
    __syncthreads();
    return logit_of(sh.key);
}

template <int T>
__global__ __launch_bounds__(T) void sample_kernel(SampleParams p)
{
    __shared__ Shared<T> sh;
    const int row = blockIdx.x;
    Row r = {p.logits + (size_t)row * p.ldx, p.mask ? p.mask + (size_t)row * p.mask_ld : nullptr,
             p.mask ? min(p.n, 32 * min(p.words, kMaxIds / 32)) : p.n, p.none, false};
    const float t = p.s.temperature ? p.s.temperature[row] : 1.0f;
    const int top_k = p.s.top_k ? p.s.top_k[row] : 0;
    const float top_p = p.s.top_p ? p.s.top_p[row] : 1.0f;
    const float min_p = p.s.min_p ? p.s.min_p[row] : 0.0f;
    const float random = p.s.random[row];

    // the first of the thread's ids, by halves, then of the row's
    float halves[2] = {-INFINITY, -INFINITY};
    int first_id[2] = {0, 0};
    constexpr int G = 8;
    const bool held = r.n <= 4 * G * T;
    f4 own[G];
    auto largest = [&](int id, f4 l) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool more = l[e] > halves[e / 2];
            halves[e / 2] = more ? l[e] : halves[e / 2];
            first_id[e / 2] = more ? id + e : first_id[e / 2];
        }
    };
    if (held) {
        hold<T>(r, own);
#pragma unroll
        for (int j = 0; j < G; j++) largest(held_id<T>(j), own[j]);
    } else {
        each4<T, 4>(r, largest);
    }
    const bool second = halves[1] > halves[0] || (halves[1] == halves[0] && first_id[1] < first_id[0]);
    float most = second ? halves[1] : halves[0];
    u64 best = most > -INFINITY ? composite(most, second ? first_id[1] : first_id[0]) : 0;
    best = wave_max_u64(best);
    if ((threadIdx.x & 63) == 0) sh.waves[threadIdx.x >> 6] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < T / 64; w++) best = max(best, sh.waves[w]);
    __syncthreads();
    if (best == 0 || !(t > 0.0f) || top_k == 1 || top_p <= 0.0f) {
        if (threadIdx.x == 0) {
            p.ids[row] = best ? id_in(best) : -1;
            if (p.logprobs) p.logprobs[row] = best ? 0.0f : -INFINITY;
        }
        return;
    }
    r.infinite = __builtin_amdgcn_readfirstlane(logit_in(best) == INFINITY);
    if (r.infinite) {
        most = most == INFINITY ? 0.0f : -INFINITY;
#pragma unroll
        for (int k = 0; k < 2; k++) halves[k] = halves[k] == INFINITY ? 0.0f : -INFINITY;
    }
    const float peak = r.infinite ? 0.0f : logit_in(best);
    const Scale z = scale_of(peak, t, p.power);
    const Rules rules = {top_k > 0 && top_k < r.n ? top_k : 0, top_p < 1.0f, top_p, random,
                         min_p > 0.0f ? (u64)ceil((double)fminf(min_p, 1.0f) * kOne) : 0};

    // A logit that nothing that top_k keeps is below: as many of the threads' largest are not
    // below it as top_k keeps.  Where those are too few, one that most probably (open) has
    // somewhat more ids not below it: of N = 2 T shares of the row, to which ids fall by chance,
    // `want` have one where N ln(N / (N - want)) ids are spread.  Short rows are listed whole.
    float bound = -INFINITY;
    bool open = false;
    const bool sure = __builtin_amdgcn_readfirstlane(rules.top_k) <= T / 4;
    if (rules.top_k && (sure || r.n > Shared<T>::LIST)) {
        constexpr int N = 2 * T;
        const float ids = 1.12f * rules.top_k + 64.0f;
        const int want = sure ? rules.top_k : min((int)(N * (1.0f - __expf(-ids / N))), N - N / 100);
        bound = bound_of(sh, z, sure ? most : halves[0], halves[1], !sure, want);
        open = !sure && bound > -INFINITY;
    }
    // (min_p bounds it too, but the mass of top_p's ids is that of all that top_k keeps)
    if (rules.least && !(rules.top_k && rules.by_mass)) {
        // (half a unit below the least weight is what rounds to it)
        const float down = (float)((1e-12 - log(((double)rules.least - 0.5) / kOne)) * t);
        const float lowest = peak - down - 1e-5f * (fabsf(peak) + down) - 1e-30f;
        if (lowest > bound) {
            bound = lowest;
            open = false;
        }
    }

    Chosen found = {-1, 0.0f, true};
    if (rules.by_mass && !rules.top_k && !rules.least) {
        found = draw_by_mass(sh, r, z, rules);
    } else if (bound > -INFINITY || (r.n <= Shared<T>::LIST && rules.top_k)) {
        bound = fmaxf(bound, -3.4028235e38f);  // (never -inf, which is no id's)
        const bool weigh = rules.by_mass && !rules.top_k;
        const int wave = wave_id();
        int here = 0;  // ids of this wave
        u64 total = 0;
        auto gather = [&](int id, f4 l) {
            if (__ballot(fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])) >= bound) == 0) return;
#pragma unroll
            for (int e = 0; e < 4; e++) here = list_id(sh, here, l[e] >= bound, l[e], id + e);
        };
        if (weigh) {
            each4<T, 2>(r, [&](int id, f4 l) {
                const Weights w = weights4(z, l);
                total += (w.w[0] + w.w[1]) + (w.w[2] + w.w[3]);
                gather(id, l);
            });
            total = block_sum(sh, total);
        } else if (held) {
#pragma unroll
            for (int j = 0; j < G; j++) {
                if (r.infinite) {
#pragma unroll
                    for (int e = 0; e < 4; e++) own[j][e] = own[j][e] == INFINITY ? 0.0f : -INFINITY;
                }
                gather(held_id<T>(j), own[j]);
            }
        } else {
            each4<T, 4>(r, gather);
        }
        if ((threadIdx.x & 63) == 0) sh.listed[wave] = here;
        __syncthreads();
        int listed = 0, longest = 0;
#pragma unroll
        for (int w = 0; w < T / 64; w++) {
            listed += sh.listed[w];
            longest = max(longest, (int)sh.listed[w]);
        }
        if (longest <= Shared<T>::OWN && !(open && listed < rules.top_k)) {
            if (listed <= Shared<T>::RANKED)
                found = draw_of_few(sh, z, rules, listed, total);
            else
                found = draw_of_many(sh, z, rules, total, r.n);
        }
    }
    if (found.missed) {
        const RowIds<T> ids = {r};
        u64 cut = 0;
#pragma unroll 1
        for (int rule = rules.top_k ? 0 : 1; rule < (rules.by_mass ? 2 : 1); rule++) {
            __syncthreads();
            cut = max(cut, last_kept(sh, z, ids, cut, rule == 0 ? rules.top_k : 0, top_p, 0));
        }
        found = draw_of_row(sh, r, z, rules, cut, false, 0, segments_of(r), 0, 0);
    }
    if (found.id >= 0) {
        p.ids[row] = found.id;
        if (p.logprobs) p.logprobs[row] = found.logprob;
    }
}

int32_t check_sample(int32_t rows, int32_t n)
{
    NHIP_REQUIRE(rows >= 0 && rows <= 65536, "sample: %d rows", rows);
    NHIP_REQUIRE(n >= 1 && n <= kMaxIds, "sample: %d ids (at most %d)", n, kMaxIds);
    return NHIP_OK;
}

}  // namespace
}  // namespace nhip

using namespace nhip;

extern "C" {

size_t nhip_sample_workspace(int32_t rows, int32_t n)
{
    check_sample(rows, n);  // (for last_error; no call needs a workspace)
    return 0;
}

int32_t nhip_sample_dev(const float* d_logits, int32_t ldx, int32_t n, int32_t rows, const nhip_sampling* s,
                        const uint32_t* d_mask, int32_t mask_ld, int32_t words, void* d_workspace,
                        size_t workspace_bytes, int32_t* d_ids, float* d_logprobs, void* stream)
{
    int32_t rc = check_sample(rows, n);
    if (rc) return rc;
    NHIP_REQUIRE(ldx >= n, "sample: stride %d is less than %d ids", ldx, n);
    NHIP_REQUIRE(!d_mask || (words >= 0 && mask_ld >= words), "sample: a mask of %d words with stride %d", words,
                 mask_ld);
    if (rows == 0) return NHIP_OK;
    NHIP_REQUIRE(d_logits && s && s->random && d_ids, "sample: null pointer");
    rc = ensure_device();
    if (rc) return rc;
    (void)d_workspace, (void)workspace_bytes;  // (none is needed: nhip_sample_workspace)
    SampleParams p = {d_logits, d_mask, *s, d_ids, d_logprobs, ldx, n, mask_ld, words, {}, -INFINITY};
    std::copy(kPower, kPower + kTerms, p.power);
    // Rows that 256 threads hold, and somewhat longer ones, which share a CU by threes, where there are
    // more of them than CUs: us by 256 and by 1024 threads for top_k 50 with top_p 0.95, for top_p 0.9 and
    // for top_k 1000: 1 row of 4096 11.1 and 12.6, 14.0 and 15.2, 14.3 and 17.5; of 8192 12.0 and 12.9,
    // 18.1 and 17.4, 17.0 and 21.8; 300 rows of 8192 13.4 and 24.7, 23.3 and 34.3, 26.7 and 42.6; of 16384
    // 18.8 and 28.3, 34.4 and 42.7, 46.3 and 41.4; 128 rows of 32000 20.0 and 14.8, 48.4 and 30.1.
    if (n <= 8192 || (n <= kFewIds && rows > 256))
        hipLaunchKernelGGL((sample_kernel<256>), dim3(rows), dim3(256), 0, as_stream(stream), p);
    else
        hipLaunchKernelGGL((sample_kernel<1024>), dim3(rows), dim3(1024), 0, as_stream(stream), p);
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

}  // extern "C"
