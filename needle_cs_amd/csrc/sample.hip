// sample.hip -- one id per row of logits on gfx950: temperature, top-k,
// top-p, min-p and a draw with a given number.
//
// The order of a row's ids is that of composites (key(logit), ~id), 64-bit
// whole numbers: larger comes first, and no two are equal.  Whatever top-k and
// top-p keep is a prefix of that order, so it is "composite >= cut".  Weights
// are whole multiples of 2^-42, so that every sum of them is exact and no
// order of summation shows, those by atomics into LDS among them; a sum of
// 2^19 weights stays below 2^62.
#include <algorithm>
#include <cmath>

#include "common.hpp"

namespace nhip {
namespace {

constexpr int kBins = 1024;      // of a histogram; in the first the last one holds what weighs nothing
constexpr int kList = 512;       // ids that are ranked against one another
constexpr int kFew = 256;        // a top-k of no more is found without a histogram
constexpr int kSegment = 256;    // ids of a wave's step, four a lane
constexpr int kMaxIds = 1 << 19;
constexpr int kTerms = 12;
constexpr double kOne = 4398046511104.0;  // 2^42, the weight of the largest logit
constexpr double kLeastScore = -30.0;     // e^-30 2^42 < 1/2: no weight

typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned long long u64;

struct SampleParams {
    const float* logits;
    const uint32_t* mask;
    nhip_sampling s;
    int32_t* ids;
    float* logprobs;
    int32_t ldx, n, mask_ld, words;
    double taylor[kTerms];  // ln(2)^k / k!: arguments, so that they stay in scalar registers
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

struct Row {
    const float* x;
    const uint32_t* mask;
    int n;
};
struct Scale {
    float peak;
    double inverse;   // of the temperature
    double log2e;     // log2(e) times that
    float bin_scale;  // of half a difference, which does not overflow
};

// round(2^42 e^((l - peak) / temperature)): 2^t with t = n + f, |f| <= 1/2, by
// the Taylor polynomial of 2^f (the terms left out are below 2^-47 of it).
__device__ __forceinline__ u64 weight(const double (&taylor)[kTerms], Scale r, float l)
{
    const double t = ((double)l - (double)r.peak) * r.log2e;
    const double n = rint(fmax(t, -64.0)), f = t - n;
    double y = taylor[kTerms - 1];
#pragma unroll
    for (int k = kTerms - 2; k >= 0; k--) y = fma(y, f, taylor[k]);
    // (a whole number below 2^51 plus 2^52 is itself in the low bits)
    const double x = ldexp(y, (int)n + 42) + 4503599627370496.0;
    const u64 w = (u64)__double_as_longlong(x) & 0xFFFFFFFFFFFFFull;
    // (-inf, as under a peak of +inf, and NaN weigh nothing)
    return l == r.peak ? (u64)kOne : t > kLeastScore * 1.4426950408889634 ? w : 0;
}

// The bin of the first histogram, which descends with the logit: kBins - 1 for what weighs nothing.
__device__ __forceinline__ int first_bin(Scale r, float l)
{
    return l == r.peak ? 0 : (int)fminf((0.5f * r.peak - 0.5f * l) * r.bin_scale, (float)(kBins - 1));
}

// Four of the row's logits from id i on, -inf where an id may not be drawn
// (by the mask, past the end, or a NaN).
__device__ __forceinline__ f4 load4(Row r, int i)
{
    f4 v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (i + 4 <= r.n) {
        v = *reinterpret_cast<const f4*>(r.x + i);
    } else {
#pragma unroll
        for (int e = 0; e < 3; e++)
            if (i + e < r.n) v[e] = r.x[i + e];
    }
    return v;
}
__device__ __forceinline__ f4 allowed4(f4 v, uint32_t bits)
{
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = v[e] > -INFINITY && ((bits >> e) & 1) ? v[e] : -INFINITY;
    return v;
}
__device__ __forceinline__ uint32_t mask4(Row r, int i)
{
    return r.mask && i < r.n ? r.mask[i >> 5] >> (i & 31) : 15u;
}

// f(first id, logits) for every four ids of the row, by the T threads of the
// workgroup: a wave's 64 fours are one segment, U of its segments are at work
// and the next U's loads in flight.
template <int T, int U, typename F>
__device__ __forceinline__ void each4(Row r, F f)
{
    constexpr int W = T / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int whole = r.n / kSegment;
    f4 v[U], next[U];
    uint32_t bits[U], next_bits[U];
    auto load = [&](int segment, f4 (&x)[U], uint32_t (&m)[U]) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = kSegment * min(segment + W * u, whole - 1) + 4 * lane;
            x[u] = *reinterpret_cast<const f4*>(r.x + i);
            m[u] = r.mask ? r.mask[i >> 5] >> (i & 31) : 15u;
        }
    };
    if (wave < whole) load(wave, v, bits);
    for (int segment = wave; segment < whole; segment += W * U) {
        if (segment + W * U < whole) load(segment + W * U, next, next_bits);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (segment + W * u < whole) f(kSegment * (segment + W * u) + 4 * lane, allowed4(v[u], bits[u]));
            __builtin_amdgcn_sched_barrier(0);  // (one four at a time in the registers)
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            v[u] = next[u];
            bits[u] = next_bits[u];
        }
    }
    if (whole * kSegment < r.n && wave == whole % W) {
        const int i = kSegment * whole + 4 * lane;
        f(i, allowed4(load4(r, i), mask4(r, i)));
    }
}

// Sum over the wave, in every lane.
template <int S>
__device__ __forceinline__ u64 add_lane_xor(u64 v)
{
    return v + ((u64)lane_xor<S>((uint32_t)(v >> 32)) << 32 | lane_xor<S>((uint32_t)v));
}
__device__ __forceinline__ u64 wave_sum_u64(u64 v)
{
    return add_lane_xor<32>(add_lane_xor<16>(add_lane_xor<8>(add_lane_xor<4>(add_lane_xor<2>(add_lane_xor<1>(v))))));
}

// COPIES of a histogram side by side, a lane's own: lanes of a wave that meet
// in a bin would wait for one another.
template <int T>
struct Shared {
    static constexpr int COPIES = T == 1024 ? 16 : 4;
    union {
        u64 bins[kBins][COPIES];
        struct {
            u64 list[kList], weights[kList];
        };
    };
    u64 segments[T == 1024 ? kMaxIds / kSegment : kList];
    u64 waves[T / 64];
    uint32_t listed, key_lo, key_hi, bin;
    u64 cut, before;
    int id;
};

// The sum of the values of the threads before this one, and of all.
template <int T>
__device__ __forceinline__ u64 block_before(u64 v, u64* waves, u64* all)
{
    u64 upto = v;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const u64 other = __shfl_up(upto, off);
        if (lane >= off) upto += other;
    }
    __syncthreads();
    if (lane == 63) waves[threadIdx.x >> 6] = upto;
    __syncthreads();
    u64 before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < T / 64; w++) {
        if (w < (int)(threadIdx.x >> 6)) before += waves[w];
        sum += waves[w];
    }
    *all = sum;
    return before + upto - v;
}

// What a rule keeps, by the sum of what stands before an id: of ones (top_k) or
// of weights (top_p).
struct Limit {
    u64 count;
    double mass;
    __device__ __forceinline__ bool inside(u64 before) const
    {
        return count ? before < count : (double)before < mass;
    }
};

// The histogram's bin in which a rule ends, and the sum before it, in sh; kBins
// where it does not end in it.  limit_of(total): the rule.
template <int T, typename F>
__device__ __forceinline__ Limit find_bin(Shared<T>& sh, u64 before0, F limit_of)
{
    constexpr int B = kBins / T, C = Shared<T>::COPIES;
    u64 q[B], sum = 0, all;
#pragma unroll
    for (int k = 0; k < B; k++) {
        const int b = B * threadIdx.x + k;
        q[k] = 0;
#pragma unroll
        for (int c = 0; c < C; c++) q[k] += sh.bins[b][(c + b) % C];
        sum += q[k];
    }
    u64 before = before0 + block_before<T>(sum, sh.waves, &all);
    const Limit limit = limit_of(all);
    if (threadIdx.x == 0) sh.bin = kBins;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < B; k++) {
        if (limit.inside(before) && !limit.inside(before + q[k])) {
            sh.bin = B * threadIdx.x + k;
            sh.before = before;
        }
        before += q[k];
    }
    __syncthreads();
    return limit;
}

template <int T>
__device__ __forceinline__ void clear_bins(Shared<T>& sh)
{
    u64* all = &sh.bins[0][0];
    for (int b = threadIdx.x; b < kBins * Shared<T>::COPIES; b += T) all[b] = 0;
    __syncthreads();
}

// The weights of the list's ids.
template <int T>
__device__ __forceinline__ void weigh_list(Shared<T>& sh, const double (&taylor)[kTerms], Scale z, int listed)
{
    for (int e = threadIdx.x; e < listed; e += T) sh.weights[e] = weight(taylor, z, logit_of((uint32_t)(sh.list[e] >> 32)));
    __syncthreads();
}

// f(place, composite, quantity, quantity of the larger ones) for each of the
// `listed` composites of sh.list, by as many threads each as the workgroup has:
// quantities are ones (top_k) or sh.weights.
template <int T, typename F>
__device__ __forceinline__ void rank_list(Shared<T>& sh, int listed, bool ones, F f)
{
    const int most = listed <= 16 ? 16 : listed <= 64 ? 64 : listed <= 256 ? 256 : 512;
    const int threads = max(1, min(64, T / most));  // for an id, side by side in a wave
    for (int e = threadIdx.x / threads; e - (int)(threadIdx.x / threads) < listed; e += T / threads) {
        const u64 own = e < listed ? sh.list[e] : 0;
        u64 larger = 0;
        if (e < listed)
            for (int k = threadIdx.x % threads; k < listed; k += threads)
                larger += sh.list[k] > own ? (ones ? 1 : sh.weights[k]) : 0;
        for (int off = 1; off < threads; off <<= 1) larger += __shfl_xor(larger, off);
        if (e < listed && threadIdx.x % threads == 0) f(e, own, ones ? 1 : sh.weights[e], larger);
    }
}

// Moves sh.cut up to the last id that a rule keeps of those from sh.cut on:
// the first `count` of them, or (count 0) those of the share top_p.
template <int T>
__device__ __forceinline__ void keep(Shared<T>& sh, const double (&taylor)[kTerms], Row r, Scale z, int count, float top_p)
{
    const bool masses = count == 0;
    const u64 cut = sh.cut;
    const int copy = threadIdx.x % Shared<T>::COPIES;
    clear_bins(sh);
    auto add = [&](int bin, float l) { atomicAdd(&sh.bins[bin][copy], masses ? weight(taylor, z, l) : (u64)1); };
    each4<T, 2>(r, [&](int id, f4 l) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int bin = first_bin(z, l[e]);
            if (bin < kBins - 1 && composite(l[e], id + e) >= cut) add(bin, l[e]);
        }
    });
    __syncthreads();
    const Limit limit = find_bin(sh, 0, [&](u64 total) {
        return Limit{(u64)count, fmax((double)top_p * (double)total, 0.5)};
    });
    const int bin = sh.bin;
    if (bin == kBins) return;
    uint32_t lo = 0, hi = ~0u;
    u64 before = sh.before;
    auto inside = [&](float l, int id) {
        const uint32_t key = key_of(l);
        return key >= lo && key <= hi && first_bin(z, l) == bin && composite(l, id) >= cut;
    };
    int listed;
    while (true) {
        // the bin's ids, as many as the list takes, and their keys
        __syncthreads();
        if (threadIdx.x == 0) {
            sh.listed = 0;
            sh.key_lo = ~0u;
            sh.key_hi = 0;
        }
        __syncthreads();
        uint32_t least = ~0u, most = 0;
        each4<T, 4>(r, [&](int id, f4 l) {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (inside(l[e], id + e)) {
                    least = min(least, key_of(l[e]));
                    most = max(most, key_of(l[e]));
                    const uint32_t at = atomicAdd(&sh.listed, 1u);
                    if (at < kList) sh.list[at] = composite(l[e], id + e);
                }
        });
        if (most) {
            atomicMin(&sh.key_lo, least);
            atomicMax(&sh.key_hi, most);
        }
        __syncthreads();
        listed = sh.listed;
        lo = sh.key_lo;
        hi = sh.key_hi;
        __syncthreads();
        if (listed <= kList || lo == hi) break;
        // a finer histogram over the keys
        const int shift = max(0, 32 - __builtin_clz(hi - lo) - 10);
        clear_bins(sh);
        each4<T, 2>(r, [&](int id, f4 l) {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (inside(l[e], id + e)) add((hi - key_of(l[e])) >> shift, l[e]);
        });
        __syncthreads();
        find_bin(sh, before, [&](u64) { return limit; });
        before = sh.before;
        hi -= sh.bin << shift;
        lo = max(lo, hi - ((1u << shift) - 1));
    }
    if (listed > kList) {
        // more ids than that of one logit: the rule keeps the first `ties` of them by id
        const u64 w = masses ? weight(taylor, z, logit_of(lo)) : 1;
        u64 ties;
        if (limit.count) {
            ties = limit.count - before;
        } else {
            ties = (u64)fmin((limit.mass - (double)before) / (double)w, (double)listed);
            while (ties > 1 && !limit.inside(before + (ties - 1) * w)) ties--;
            while (ties < (u64)listed && limit.inside(before + ties * w)) ties++;
            ties = max(ties, (u64)1);
        }
        const int segments = (r.n + kSegment - 1) / kSegment, lane = threadIdx.x & 63;
        constexpr int S = sizeof(sh.segments) / sizeof(u64) / T > 1 ? sizeof(sh.segments) / sizeof(u64) / T : 1;
        auto equal = [&](int segment) {  // of the lane's four ids
            const int id = segment * kSegment + 4 * lane;
            const f4 l = allowed4(load4(r, id), mask4(r, id));
            uint32_t same = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) same |= (inside(l[e], id + e) ? 1u : 0u) << e;
            return same;
        };
        for (int g = threadIdx.x >> 6; g < segments; g += T / 64) {
            const int n = wave_sum_i32(__builtin_popcount(equal(g)));
            if (lane == 0) sh.segments[g] = n;
        }
        __syncthreads();
        u64 c[S], sum = 0, all;
#pragma unroll
        for (int k = 0; k < S; k++) {
            const int g = S * threadIdx.x + k;
            c[k] = g < segments ? sh.segments[g] : 0;
            sum += c[k];
        }
        u64 upto = block_before<T>(sum, sh.waves, &all);
#pragma unroll
        for (int k = 0; k < S; k++) {
            if (upto < ties && upto + c[k] >= ties) {
                sh.bin = S * threadIdx.x + k;
                sh.before = upto;
            }
            upto += c[k];
        }
        __syncthreads();
        if (threadIdx.x < 64) {
            const uint32_t same = equal(sh.bin);
            int to = __builtin_popcount(same);
            const int own = to;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int other = __shfl_up(to, off);
                if (lane >= off) to += other;
            }
            int at = (int)sh.before + to - own;
            for (int e = 0; e < 4; e++)
                if ((same >> e) & 1 && ++at == (int)ties)
                    sh.cut = (u64)lo << 32 | (uint32_t)~(int)(sh.bin * kSegment + 4 * lane + e);
        }
        __syncthreads();
        return;
    }
    if (masses) weigh_list(sh, taylor, z, listed);
    rank_list(sh, listed, !masses, [&](int, u64 own, u64 q, u64 larger) {
        if (limit.inside(before + larger) && !limit.inside(before + larger + q)) sh.cut = own;
    });
    __syncthreads();
}

__device__ __forceinline__ float log_probability(Scale r, float l, u64 total)
{
    const double z = l == r.peak ? 0.0 : ((double)l - (double)r.peak) * r.inverse;
    return (float)(z - log((double)total / kOne));
}

// The t of the draw.
__device__ __forceinline__ u64 drawn(float random, u64 total)
{
    const double u = random > 0.0f ? (double)random : 0.0;
    return min((u64)fmin(u * (double)total, kOne * kMaxIds), total - 1);
}

template <int T>
__global__ __launch_bounds__(T) void sample_kernel(SampleParams p)
{
    __shared__ Shared<T> sh;
    const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Row r = {p.logits + (size_t)row * p.ldx, p.mask ? p.mask + (size_t)row * p.mask_ld : nullptr,
                   p.mask ? min(p.n, 32 * min(p.words, kMaxIds / 32)) : p.n};
    const float t = p.s.temperature ? p.s.temperature[row] : 1.0f;
    const int top_k = p.s.top_k ? p.s.top_k[row] : 0;
    const float top_p = p.s.top_p ? p.s.top_p[row] : 1.0f;
    const float min_p = p.s.min_p ? p.s.min_p[row] : 0.0f;
    const float random = p.s.random[row];
    const double(&taylor)[kTerms] = p.taylor;

    // the thread's first id, then the row's
    float most = -INFINITY;
    int most_id = 0;
    each4<T, 4>(r, [&](int id, f4 l) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool more = l[e] > most;
            most = more ? l[e] : most;
            most_id = more ? id + e : most_id;
        }
    });
    u64 best = most > -INFINITY ? composite(most, most_id) : 0;
#pragma unroll
    for (int off = 32; off; off >>= 1) best = max(best, (u64)__shfl_xor(best, off));
    if (lane == 0) sh.waves[wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < T / 64; w++) best = max(best, sh.waves[w]);
    const bool first_only = !(t > 0.0f) || top_k == 1 || top_p <= 0.0f;
    if (best == 0 || first_only) {
        if (threadIdx.x == 0) {
            p.ids[row] = best ? ~(int)(uint32_t)best : -1;
            if (p.logprobs) p.logprobs[row] = best ? 0.0f : -INFINITY;
        }
        return;
    }
    const double inverse = 1.0 / (double)t;
    const Scale z = {logit_of((uint32_t)(best >> 32)), inverse, 1.4426950408889634 * inverse,
                     fminf((float)(2 * (kBins - 1) * inverse / -kLeastScore), 3e38f)};
    const bool by_mass = top_p < 1.0f;
    const double least = min_p > 0.0f ? (double)fminf(min_p, 1.0f) * kOne : 0.0;

    if (top_k > 0 && top_k <= kFew) {
        // At least top_k ids are as large as the top_k-th largest of the threads'
        // first ones, and not many more: all from its bin on, in a list.
        uint32_t* counts = reinterpret_cast<uint32_t*>(sh.segments);
        constexpr int B = kBins / T;
        for (int b = threadIdx.x; b < kBins; b += T) counts[b] = 0;
        if (threadIdx.x == 0) {
            sh.listed = 0;
            sh.bin = kBins - 2;
        }
        __syncthreads();
        if (most > -INFINITY) atomicAdd(&counts[first_bin(z, most)], 1u);
        __syncthreads();
        u64 sum = 0, all;
        uint32_t c[B];
#pragma unroll
        for (int k = 0; k < B; k++) {
            c[k] = B * threadIdx.x + k < kBins - 1 ? counts[B * threadIdx.x + k] : 0;
            sum += c[k];
        }
        u64 upto = block_before<T>(sum, sh.waves, &all);
#pragma unroll
        for (int k = 0; k < B; k++) {
            if (upto < (u64)top_k && upto + c[k] >= (u64)top_k) sh.bin = B * threadIdx.x + k;
            upto += c[k];
        }
        __syncthreads();
        const int bin = sh.bin;
        each4<T, 4>(r, [&](int id, f4 l) {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (first_bin(z, l[e]) <= bin) {
                    const uint32_t at = atomicAdd(&sh.listed, 1u);
                    if (at < kList) sh.list[at] = composite(l[e], id + e);
                }
        });
        __syncthreads();
        const int listed = sh.listed;
        if (listed <= kList) {
            // ranks, then what each rule keeps of them, all of the list's prefixes
            u64 first_k = 0;
            weigh_list(sh, taylor, z, listed);
            rank_list(sh, listed, true, [&](int e, u64, u64, u64 larger) { sh.segments[e] = larger; });
            __syncthreads();
            const bool mine = (int)threadIdx.x < listed, more = (int)threadIdx.x + T < listed;
            u64 before[2] = {0, 0}, w[2] = {0, 0}, kept = 0, total;
            static_assert(kList <= 2 * 256, "two ids a thread at most");
            const bool in[2] = {mine && sh.segments[threadIdx.x] < (u64)top_k,
                                more && sh.segments[threadIdx.x + T] < (u64)top_k};
            if (in[0]) w[0] = sh.weights[threadIdx.x];
            if (in[1]) w[1] = sh.weights[threadIdx.x + T];
            block_before<T>(w[0] + w[1], sh.waves, &first_k);
            if (by_mass) {
                rank_list(sh, listed, false, [&](int e, u64, u64, u64 larger) { sh.segments[e] = larger; });
                __syncthreads();
                if (in[0]) before[0] = sh.segments[threadIdx.x];
                if (in[1]) before[1] = sh.segments[threadIdx.x + T];
            }
            const double mass = (double)top_p * (double)first_k;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 2; k++) {
                if (by_mass && before[k] != 0 && !((double)before[k] < mass)) w[k] = 0;
                if ((double)w[k] < least) w[k] = 0;
                kept += w[k];
                if ((int)threadIdx.x + k * T < listed) sh.weights[threadIdx.x + k * T] = w[k];
            }
            block_before<T>(kept, sh.waves, &total);
            // the draw, in the order of the ids: composites' low halves, inverted
            const u64 at = drawn(random, total);
            for (int e = threadIdx.x; e < listed; e += T) sh.list[e] = (sh.list[e] << 32) | (sh.list[e] >> 32);
            __syncthreads();
            rank_list(sh, listed, false, [&](int, u64 own, u64 weight, u64 larger) {
                if (larger <= at && at < larger + weight) {
                    const int id = ~(int)(uint32_t)(own >> 32);
                    p.ids[row] = id;
                    if (p.logprobs) p.logprobs[row] = log_probability(z, logit_of((uint32_t)own), total);
                }
            });
            return;
        }
        __syncthreads();
    }

    if (threadIdx.x == 0) sh.cut = 0;
    __syncthreads();
    const bool by_count = top_k > 0 && top_k < r.n;
    for (int rule = by_count ? 0 : 1; rule < (by_mass ? 2 : 1); rule++) keep(sh, taylor, r, z, rule == 0 ? top_k : 0, top_p);

    // the draw, in the order of the ids
    const u64 cut = sh.cut;
    auto kept = [&](float l, int id) {
        if (!(l > -INFINITY && composite(l, id) >= cut)) return (u64)0;
        const u64 w = weight(taylor, z, l);
        return (double)w < least ? (u64)0 : w;
    };
    const int segments = (r.n + kSegment - 1) / kSegment;
    each4<T, 2>(r, [&](int id, f4 l) {
        u64 sum = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) sum += kept(l[e], id + e);
        sum = __ballot(sum != 0) ? wave_sum_u64(sum) : 0;
        if (lane == 0) sh.segments[id / kSegment] = sum;
    });
    __syncthreads();
    constexpr int S = sizeof(sh.segments) / sizeof(u64) / T > 1 ? sizeof(sh.segments) / sizeof(u64) / T : 1;
    u64 m[S], sum = 0, total;
#pragma unroll
    for (int k = 0; k < S; k++) {
        const int g = S * threadIdx.x + k;
        m[k] = g < segments ? sh.segments[g] : 0;
        sum += m[k];
    }
    u64 before = block_before<T>(sum, sh.waves, &total);
    const u64 at = drawn(random, total);
#pragma unroll
    for (int k = 0; k < S; k++) {
        if (before <= at && at < before + m[k]) {
            sh.bin = S * threadIdx.x + k;
            sh.before = before;
        }
        before += m[k];
    }
    __syncthreads();
    if (threadIdx.x >= 64) return;
    const int id = (int)sh.bin * kSegment + 4 * lane;
    const f4 l = allowed4(load4(r, id), mask4(r, id));
    u64 w[4], upto = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        w[e] = kept(l[e], id + e);
        upto += w[e];
    }
    const u64 own = upto;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const u64 other = __shfl_up(upto, off);
        if (lane >= off) upto += other;
    }
    u64 from = sh.before + upto - own;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (from <= at && at < from + w[e]) {
            p.ids[row] = id + e;
            if (p.logprobs) p.logprobs[row] = log_probability(z, l[e], total);
        }
        from += w[e];
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
    if (check_sample(rows, n)) return 0;
    return 0;
}

int32_t nhip_sample_dev(const float* d_logits, int32_t ldx, int32_t n, int32_t rows, const nhip_sampling* s,
                        const uint32_t* d_mask, int32_t mask_ld, int32_t words, void* d_workspace,
                        size_t workspace_bytes, int32_t* d_ids, float* d_logprobs, void* stream)
{
    int32_t rc = check_sample(rows, n);
    if (rc) return rc;
    NHIP_REQUIRE(ldx >= n, "sample: stride %d is less than %d ids", ldx, n);
    NHIP_REQUIRE(!d_mask || (words >= 0 && mask_ld >= words), "sample: a mask of %d words with stride %d", words, mask_ld);
    if (rows == 0) return NHIP_OK;
    NHIP_REQUIRE(d_logits && s && s->random && d_ids, "sample: null pointer");
    rc = ensure_device();
    if (rc) return rc;
    (void)d_workspace;
    (void)workspace_bytes;
    SampleParams p = {d_logits, d_mask, *s, d_ids, d_logprobs, ldx, n, mask_ld, words, {}};
    p.taylor[0] = 1.0;
    for (int k = 1; k < kTerms; k++) p.taylor[k] = p.taylor[k - 1] * 0.6931471805599453 / k;
    if (n <= 4096)
        hipLaunchKernelGGL((sample_kernel<256>), dim3(rows), dim3(256), 0, as_stream(stream), p);
    else
        hipLaunchKernelGGL((sample_kernel<1024>), dim3(rows), dim3(1024), 0, as_stream(stream), p);
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

}  // extern "C"
