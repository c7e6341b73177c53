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

constexpr int kThreads = 1024;
constexpr int kBins = 2048;      // of a histogram; in the first the last one holds what weighs nothing
constexpr int kList = 1024;      // ids that are ranked against one another
constexpr int kSegment = 256;    // ids of a wave's step, four a lane
constexpr int kMaxIds = 1 << 19;
constexpr int kSegments = kMaxIds / kSegment;
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
};

// A larger key for a larger logit; +0 and -0 alike.
__device__ __forceinline__ uint32_t key_of(float l)
{
    const uint32_t u = __float_as_uint(l + 0.0f);
    return u ^ (u >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ u64 composite(float l, int id) { return (u64)key_of(l) << 32 | (uint32_t)~id; }

struct Row {
    const float* x;
    const uint32_t* mask;
    int n;
    float peak;
    double inverse;    // of the temperature
    float bin_scale;  // of half a difference, which does not overflow
};

__device__ __forceinline__ u64 weight(const Row& r, float l)
{
    if (l == r.peak) return (u64)kOne;
    const double z = ((double)l - (double)r.peak) * r.inverse;  // -inf under a peak of +inf
    return z > kLeastScore ? (u64)rint(exp(z) * kOne) : 0;
}

// The bin of the first histogram, which descends with the logit: kBins - 1 for what weighs nothing.
__device__ __forceinline__ int first_bin(const Row& r, float l)
{
    return l == r.peak ? 0 : (int)fminf((0.5f * r.peak - 0.5f * l) * r.bin_scale, (float)(kBins - 1));
}

// f(id, logit) for every id of the row that may be drawn, by the whole workgroup.
template <typename F>
__device__ __forceinline__ void each(const Row& r, F f)
{
    for (int i = 4 * (int)threadIdx.x; i < r.n; i += 4 * kThreads) {
        float l[4];
        if (i + 4 <= r.n) {
            const f4 v = *reinterpret_cast<const f4*>(r.x + i);
            for (int e = 0; e < 4; e++) l[e] = v[e];
        } else {
            for (int e = 0; e < 4; e++) l[e] = i + e < r.n ? r.x[i + e] : -INFINITY;
        }
        const uint32_t bits = r.mask ? r.mask[i >> 5] >> (i & 31) : 15u;
        for (int e = 0; e < 4; e++)
            if (((bits >> e) & 1) && l[e] > -INFINITY) f(i + e, l[e]);
    }
}

struct Shared {
    uint32_t counts[kBins];
    u64 masses[kBins];
    u64 list[kList], list_weight[kList];
    u64 segments[kSegments];
    u64 waves[kThreads / 64];
    uint32_t listed, key_lo, key_hi;
    u64 cut, kept_mass;
    uint32_t bin, before_count;
    u64 before_mass;
};

// The sum of the values of the threads before this one, and of all.
__device__ __forceinline__ u64 block_before(u64 v, u64* waves, u64* all)
{
    u64 upto = v;
    const int lane = threadIdx.x & 63;
    for (int off = 1; off < 64; off <<= 1) {
        const u64 other = __shfl_up(upto, off);
        if (lane >= off) upto += other;
    }
    __syncthreads();
    if (lane == 63) waves[threadIdx.x >> 6] = upto;
    __syncthreads();
    u64 before = 0, sum = 0;
    for (int w = 0; w < kThreads / 64; w++) {
        if (w < (int)(threadIdx.x >> 6)) before += waves[w];
        sum += waves[w];
    }
    *all = sum;
    return before + upto - v;
}

// What a rule keeps: the first `count` ids, or (count 0) those with less than
// `mass` before them.
struct Limit {
    uint32_t count;
    double mass;
    __device__ __forceinline__ bool inside(uint32_t c, u64 m) const { return count ? c < count : (double)m < mass; }
};

// The bin of a histogram in which the rule ends, with what is before it, in
// sh; kBins where it does not end in the first `bins`.
__device__ __forceinline__ void find_bin(Shared& sh, const Limit& limit, int bins, uint32_t count0, u64 mass0)
{
    uint32_t c[2];
    u64 m[2];
    for (int k = 0; k < 2; k++) {
        const int b = 2 * threadIdx.x + k;
        c[k] = b < bins ? sh.counts[b] : 0;
        m[k] = b < bins ? sh.masses[b] : 0;
    }
    u64 all;
    uint32_t count = count0 + (uint32_t)block_before(c[0] + c[1], sh.waves, &all);
    u64 mass = mass0 + block_before(m[0] + m[1], sh.waves, &all);
    if (threadIdx.x == 0) sh.bin = kBins;
    __syncthreads();
    for (int k = 0; k < 2; k++) {
        if (limit.inside(count, mass) && !limit.inside(count + c[k], mass + m[k])) {
            sh.bin = 2 * threadIdx.x + k;
            sh.before_count = count;
            sh.before_mass = mass;
        }
        count += c[k];
        mass += m[k];
    }
    __syncthreads();
}

// Moves sh.cut up to the last id that the rule keeps of those from sh.cut on,
// and sets sh.kept_mass to their weight (MASSES) if it ends among ids that weigh
// something.
template <bool MASSES>
__device__ void keep(Shared& sh, const Row& r, const Limit& limit)
{
    const u64 cut = sh.cut;
    auto clear = [&] {
        for (int b = threadIdx.x; b < kBins; b += kThreads) {
            sh.counts[b] = 0;
            sh.masses[b] = 0;
        }
        __syncthreads();
    };
    auto add = [&](int bin, float l) {
        atomicAdd(&sh.counts[bin], 1u);
        if (MASSES) atomicAdd(&sh.masses[bin], weight(r, l));
    };
    clear();
    each(r, [&](int id, float l) {
        const int bin = first_bin(r, l);
        if (bin < kBins - 1 && composite(l, id) >= cut) add(bin, l);
    });
    __syncthreads();
    find_bin(sh, limit, kBins - 1, 0, 0);
    const int bin = sh.bin;
    if (bin == kBins) return;
    uint32_t lo = 0, hi = ~0u, count = sh.counts[bin], before_count = sh.before_count;
    u64 before_mass = sh.before_mass;
    auto inside = [&](float l, int id) {
        const uint32_t key = key_of(l);
        return key >= lo && key <= hi && first_bin(r, l) == bin && composite(l, id) >= cut;
    };
    while (count > kList) {
        // the keys of the bin's ids, and a finer histogram over them
        if (threadIdx.x == 0) {
            sh.key_lo = ~0u;
            sh.key_hi = 0;
        }
        __syncthreads();
        uint32_t least = ~0u, most = 0;
        each(r, [&](int id, float l) {
            if (inside(l, id)) {
                least = min(least, key_of(l));
                most = max(most, key_of(l));
            }
        });
        atomicMin(&sh.key_lo, least);
        atomicMax(&sh.key_hi, most);
        __syncthreads();
        lo = sh.key_lo;
        hi = sh.key_hi;
        if (lo == hi) break;
        const int shift = max(0, 32 - __builtin_clz(hi - lo) - 11);
        clear();
        each(r, [&](int id, float l) {
            if (inside(l, id)) add((hi - key_of(l)) >> shift, l);
        });
        __syncthreads();
        find_bin(sh, limit, kBins, before_count, before_mass);
        const uint32_t sub = sh.bin;
        count = sh.counts[sub];
        before_count = sh.before_count;
        before_mass = sh.before_mass;
        hi -= sub << shift;
        lo = max(lo, hi - ((1u << shift) - 1));
        __syncthreads();
    }
    if (count > kList) {
        // more ids than that of one logit: the rule keeps the first `ties` of them by id
        u64 w = 0;
        uint32_t ties;
        const uint32_t bits = lo & 0x80000000u ? lo ^ 0x80000000u : ~lo;
        if (MASSES) w = weight(r, __uint_as_float(bits));
        if (limit.count) {
            ties = limit.count - before_count;
        } else {
            ties = (uint32_t)fmin((limit.mass - (double)before_mass) / (double)w, (double)count);
            while (ties > 1 && !limit.inside(0, before_mass + (u64)(ties - 1) * w)) ties--;
            while (ties < count && limit.inside(0, before_mass + (u64)ties * w)) ties++;
            ties = max(ties, 1u);
        }
        const int segments = (r.n + kSegment - 1) / kSegment, lane = threadIdx.x & 63;
        auto equal = [&](int segment) {  // of the lane's four ids
            uint32_t same = 0;
            for (int e = 0; e < 4; e++) {
                const int id = segment * kSegment + 4 * lane + e;
                const bool in = id < r.n && (!r.mask || ((r.mask[id >> 5] >> (id & 31)) & 1));
                const float l = in ? r.x[id] : -INFINITY;
                same |= (l > -INFINITY && inside(l, id) ? 1u : 0u) << e;
            }
            return same;
        };
        for (int b = threadIdx.x; b < kSegments; b += kThreads) sh.segments[b] = 0;
        __syncthreads();
        for (int g = threadIdx.x >> 6; g < segments; g += kThreads / 64) {
            const int n = wave_sum_i32(__builtin_popcount(equal(g)));
            if (lane == 0) sh.segments[g] = n;
        }
        __syncthreads();
        u64 all;
        u64 c[2] = {sh.segments[2 * threadIdx.x], sh.segments[2 * threadIdx.x + 1]};
        u64 before = block_before(c[0] + c[1], sh.waves, &all);
        for (int k = 0; k < 2; k++) {
            if (before < ties && before + c[k] >= ties) {
                sh.bin = 2 * threadIdx.x + k;
                sh.before_count = (uint32_t)before;
            }
            before += c[k];
        }
        __syncthreads();
        if (threadIdx.x < 64) {
            const uint32_t same = equal(sh.bin);
            int upto = __builtin_popcount(same);
            const int own = upto;
            for (int off = 1; off < 64; off <<= 1) {
                const int other = __shfl_up(upto, off);
                if (lane >= off) upto += other;
            }
            int at = sh.before_count + upto - own;
            for (int e = 0; e < 4; e++)
                if ((same >> e) & 1 && ++at == (int)ties)
                    sh.cut = (u64)lo << 32 | (uint32_t)~(int)(sh.bin * kSegment + 4 * lane + e);
        }
        if (threadIdx.x == 0) sh.kept_mass = before_mass + (u64)ties * w;
        __syncthreads();
        return;
    }
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    each(r, [&](int id, float l) {
        if (inside(l, id)) {
            const uint32_t at = atomicAdd(&sh.listed, 1u);
            if (at < kList) {
                sh.list[at] = composite(l, id);
                sh.list_weight[at] = MASSES ? weight(r, l) : 0;
            }
        }
    });
    __syncthreads();
    const int listed = min(sh.listed, (uint32_t)kList);
    if ((int)threadIdx.x < listed) {
        const u64 own = sh.list[threadIdx.x];
        uint32_t rank = before_count;
        u64 mass = before_mass;
        for (int k = 0; k < listed; k++) {
            if (sh.list[k] > own) {
                rank++;
                mass += sh.list_weight[k];
            }
        }
        const u64 w = sh.list_weight[threadIdx.x];
        if (limit.inside(rank, mass) && !limit.inside(rank + 1, mass + w)) {
            sh.cut = own;
            sh.kept_mass = mass + w;
        }
    }
    __syncthreads();
}

__global__ __launch_bounds__(kThreads) void sample_kernel(SampleParams p)
{
    __shared__ Shared sh;
    const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Row r;
    r.x = p.logits + (size_t)row * p.ldx;
    r.mask = p.mask ? p.mask + (size_t)row * p.mask_ld : nullptr;
    r.n = p.mask ? min(p.n, 32 * min(p.words, kMaxIds / 32)) : p.n;
    const float t = p.s.temperature ? p.s.temperature[row] : 1.0f;
    const int top_k = p.s.top_k ? p.s.top_k[row] : 0;
    const float top_p = p.s.top_p ? p.s.top_p[row] : 1.0f;
    const float min_p = p.s.min_p ? p.s.min_p[row] : 0.0f;
    const float random = p.s.random[row];

    u64 best = 0;
    each(r, [&](int id, float l) { best = max(best, composite(l, id)); });
    for (int off = 32; off; off >>= 1) best = max(best, (u64)__shfl_xor(best, off));
    if (lane == 0) sh.waves[wave] = best;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; w++) best = max(best, sh.waves[w]);
    __syncthreads();
    const bool first_only = !(t > 0.0f) || top_k == 1 || top_p <= 0.0f;
    if (best == 0 || first_only) {
        if (threadIdx.x == 0) {
            p.ids[row] = best ? ~(int)(uint32_t)best : -1;
            if (p.logprobs) p.logprobs[row] = best ? 0.0f : -INFINITY;
        }
        return;
    }
    const uint32_t top = (uint32_t)(best >> 32);
    r.peak = __uint_as_float(top & 0x80000000u ? top ^ 0x80000000u : ~top);
    r.inverse = 1.0 / (double)t;
    r.bin_scale = fminf((float)(2 * (kBins - 1) * r.inverse / -kLeastScore), 3e38f);

    if (threadIdx.x == 0) sh.cut = 0;
    __syncthreads();
    const bool by_mass = top_p < 1.0f;
    if (top_k > 0 && top_k < r.n) {
        if (by_mass)
            keep<true>(sh, r, Limit{(uint32_t)top_k, 0.0});
        else
            keep<false>(sh, r, Limit{(uint32_t)top_k, 0.0});
    }
    if (by_mass) {
        if (sh.cut == 0) {  // (no rule before this one ended among weights)
            u64 mine = 0, all;
            each(r, [&](int, float l) { mine += weight(r, l); });
            block_before(mine, sh.waves, &all);
            if (threadIdx.x == 0) sh.kept_mass = all;
            __syncthreads();
        }
        const double mass = (double)top_p * (double)sh.kept_mass;
        __syncthreads();
        keep<true>(sh, r, Limit{0, fmax(mass, 0.5)});
    }

    // the draw, in the order of the ids
    const u64 cut = sh.cut;
    const double least = min_p > 0.0f ? (double)fminf(min_p, 1.0f) * kOne : 0.0;
    auto kept = [&](int id, u64* w) {
        const bool in = id < r.n && (!r.mask || ((r.mask[id >> 5] >> (id & 31)) & 1));
        const float l = in ? r.x[id] : -INFINITY;
        *w = l > -INFINITY && composite(l, id) >= cut ? weight(r, l) : 0;
        if ((double)*w < least) *w = 0;
        return l;
    };
    const int segments = (r.n + kSegment - 1) / kSegment;
    for (int g = threadIdx.x; g < kSegments; g += kThreads) sh.segments[g] = 0;
    __syncthreads();
    for (int g = wave; g < segments; g += kThreads / 64) {
        u64 sum = 0, w;
        for (int e = 0; e < 4; e++) {
            kept(g * kSegment + 4 * lane + e, &w);
            sum += w;
        }
        for (int off = 32; off; off >>= 1) sum += __shfl_xor(sum, off);
        if (lane == 0) sh.segments[g] = sum;
    }
    __syncthreads();
    u64 total;
    const u64 m[2] = {sh.segments[2 * threadIdx.x], sh.segments[2 * threadIdx.x + 1]};
    u64 before = block_before(m[0] + m[1], sh.waves, &total);
    const double u = random > 0.0f ? (double)random : 0.0;
    const u64 at = min((u64)fmin(u * (double)total, kOne * kMaxIds), total - 1);
    for (int k = 0; k < 2; k++) {
        if (before <= at && at < before + m[k]) {
            sh.bin = 2 * threadIdx.x + k;
            sh.before_mass = before;
        }
        before += m[k];
    }
    __syncthreads();
    if (threadIdx.x >= 64) return;
    u64 w[4], upto = 0;
    float l[4];
    const int id = (int)sh.bin * kSegment + 4 * lane;
    for (int e = 0; e < 4; e++) {
        l[e] = kept(id + e, &w[e]);
        upto += w[e];
    }
    const u64 own = upto;
    for (int off = 1; off < 64; off <<= 1) {
        const u64 other = __shfl_up(upto, off);
        if (lane >= off) upto += other;
    }
    u64 from = sh.before_mass + upto - own;
    for (int e = 0; e < 4; e++) {
        if (from <= at && at < from + w[e]) {
            p.ids[row] = id + e;
            const double z = l[e] == r.peak ? 0.0 : ((double)l[e] - (double)r.peak) * r.inverse;
            if (p.logprobs) p.logprobs[row] = (float)(z - log((double)total / kOne));
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
    const SampleParams p = {d_logits, d_mask, *s, d_ids, d_logprobs, ldx, n, mask_ld, words};
    hipLaunchKernelGGL(sample_kernel, dim3(rows), dim3(kThreads), 0, as_stream(stream), p);
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

}  // extern "C"
