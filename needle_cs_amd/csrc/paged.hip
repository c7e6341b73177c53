// paged.hip -- the paged int8 KV cache on gfx950: writing new positions and
// moving, sharing, taking and giving up pages (attention over it is in
// paged_attention.hip).
//
// append quantizes fp32 keys and values per (row, kv head) (QuantizeInt8,
// src/Needle/Scalar.cs:67-74, bit for bit) into their pages.
//
// The bookkeeping (tables, lengths, refs) lives in device memory and is
// changed by kernels, so that a server's step can branch, grow and free its
// sequences inside a captured graph, without the host waiting for a count.
// Every choice is a function of the call's inputs alone: free pages are
// taken lowest first in entry order, found by ordered prefix sums; the only
// atomics are integer additions to refs, whose order does not show.
#include <algorithm>

#include "paged.hpp"

namespace nhip {

int32_t paged_check(const nhip_paged_cache* c)
{
    NHIP_REQUIRE(c, "paged cache: NULL");
    NHIP_REQUIRE(c->keys && c->key_scales && c->values && c->value_scales && c->tables && c->lengths && c->refs,
                 "paged cache: null array");
    NHIP_REQUIRE(c->page_size >= 16 && c->page_size <= 256 && (c->page_size & (c->page_size - 1)) == 0,
                 "paged cache: page size %d is not 16, 32, 64, 128 or 256", c->page_size);
    NHIP_REQUIRE((c->qk_dim == 48 && c->v_dim == 64) || (c->qk_dim == 64 && c->v_dim == 64) ||
                     (c->qk_dim == 128 && c->v_dim == 128),
                 "paged cache: head dims %d / %d are not 48 / 64, 64 / 64 or 128 / 128", c->qk_dim, c->v_dim);
    NHIP_REQUIRE(c->layers >= 1 && c->layers <= 4096 && c->pages >= 1 && c->pages <= (1 << 20) && c->kv_heads >= 1 &&
                     c->kv_heads <= 256 && c->sequences >= 1 && c->sequences <= 65536,
                 "paged cache: %d layers, %d pages, %d kv heads, %d sequences out of range", c->layers, c->pages,
                 c->kv_heads, c->sequences);
    NHIP_REQUIRE(c->width >= 1 && (int64_t)c->width * c->page_size <= (1 << 30),
                 "paged cache: %d pages a sequence out of range", c->width);
    NHIP_REQUIRE(((reinterpret_cast<uintptr_t>(c->keys) | reinterpret_cast<uintptr_t>(c->key_scales) |
                   reinterpret_cast<uintptr_t>(c->values) | reinterpret_cast<uintptr_t>(c->value_scales)) &
                  15) == 0,
                 "paged cache: a pool is not 16-byte aligned");
    NHIP_REQUIRE(((reinterpret_cast<uintptr_t>(c->tables) | reinterpret_cast<uintptr_t>(c->lengths) |
                   reinterpret_cast<uintptr_t>(c->refs)) &
                  3) == 0,
                 "paged cache: an int32 array is not 4-byte aligned");
    return NHIP_OK;
}

namespace {

constexpr int kMaxEntries = 1024;

// ---------------------------------------------------------------- append --

struct AppendParams {
    PagedLayer c;
    const float* k;
    const float* v;
    const int32_t* row_seq;
    const int32_t* row_pos;
    int32_t ldk, ldv, rows;
};

// A workgroup takes 16 rows of one kv head; L lanes share a row's key (or
// value) head, four elements each, so a head's peak is a few DPP steps and 16
// rows of keys leave as whole dwords.  Values change places through LDS: the
// cache holds 16 positions of a dimension together, and where the 16 rows are
// consecutive positions of one sequence (a prompt) a lane writes four of them
// at once; else each goes by itself.  Bound by the bytes read and written:
// 8185 rows of 8 kv heads of 128 (84 MB) take APPEND_US us, APPEND_TBS TB/s.
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));

template <int L>
__device__ __forceinline__ float group_max(float v)
{
    v = fmaxf(v, lane_xor<1>(v));
    v = fmaxf(v, lane_xor<2>(v));
    v = fmaxf(v, lane_xor<4>(v));
    v = fmaxf(v, lane_xor<8>(v));
    return L == 32 ? fmaxf(v, lane_xor<16>(v)) : v;
}

template <int QK, int V>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendParams p)
{
    constexpr int L = V <= 64 ? 16 : 32, PASSES = L / 16, ROWS = 256 / L;  // rows of a pass
    __shared__ size_t cells[16];
    __shared__ int places[16], positions[16], sequences[16];
    __shared__ __align__(16) uint8_t turned[V][20];  // value codes by dimension, then row
    const PagedLayer& c = p.c;
    const int kvh = blockIdx.y, row0 = (int)blockIdx.x * 16, n = min(16, p.rows - row0);
    const int l = threadIdx.x & (L - 1), row_of_pass = threadIdx.x / L;
    f4 x[PASSES][2];
#pragma unroll
    for (int k = 0; k < PASSES; k++) {
        const size_t r = row0 + min(row_of_pass + k * ROWS, n - 1);
        x[k][0] = x[k][1] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        if (4 * l < QK) x[k][0] = *reinterpret_cast<const f4*>(p.k + r * p.ldk + kvh * QK + 4 * l);
        if (4 * l < V) x[k][1] = *reinterpret_cast<const f4*>(p.v + r * p.ldv + kvh * V + 4 * l);
    }
    // where each row's position lives: its page's first cell (of this kv head) and its place in the page, -1 if nowhere
    if (threadIdx.x < 16) {
        const int i = threadIdx.x, r = row0 + min(i, n - 1);
        const int seq = p.row_seq[r], pos = p.row_pos[r];
        int page = -1;
        if (seq >= 0 && seq < c.sequences && pos >= 0 && (pos >> c.page_shift) < c.width)
            page = c.tables[(size_t)seq * c.width + (pos >> c.page_shift)];
        const bool ok = i < n && page >= 0 && page < c.pages;
        cells[i] = ok ? ((size_t)page * c.kv_heads + kvh) << c.page_shift : 0;
        places[i] = ok ? pos & ((1 << c.page_shift) - 1) : -1;
        positions[i] = pos;
        sequences[i] = seq;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PASSES; k++) {
        const int i = row_of_pass + k * ROWS;
        const int at = places[i];
        const size_t cell = cells[i];
#pragma unroll
        for (int part = 0; part < 2; part++) {
            const f4 y = x[k][part];
            const float peak =
                group_max<L>(fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3]))));
            const float scale = peak > 0.0f ? peak / 127.0f : 1.0f;
            const uint32_t codes = ref_quantize4(make_float4(y[0], y[1], y[2], y[3]), 1.0f / scale);
            if (part == 1 && 4 * l < V) {
#pragma unroll
                for (int e = 0; e < 4; e++) turned[4 * l + e][i] = (uint8_t)(codes >> (8 * e));
            }
            if (at < 0) continue;
            if (part == 0 && 4 * l < QK) *reinterpret_cast<uint32_t*>(c.keys + (cell + at) * QK + 4 * l) = codes;
            if (l == 0) (part ? c.vscale : c.kscale)[cell + at] = scale;
        }
    }
    __syncthreads();
    bool consecutive = true;
    for (int i = 0; i < n; i++)
        consecutive &= places[i] >= 0 && positions[i] == positions[0] + i && sequences[i] == sequences[0];
    if (consecutive) {
        // five quads of positions cover 16 rows whatever place the first has in its quad
        const int lead = positions[0] & 3;
        for (int item = threadIdx.x; item < 5 * V; item += 256) {
            const int d = item & (V - 1), first = 4 * (item / V) - lead;  // the quad's first row
            if (first >= n) continue;
            const int some = max(first, 0), at = places[some] & ~3;
            uint8_t* to = reinterpret_cast<uint8_t*>(c.values) + cells[some] * V + (size_t)(at >> 4) * (16 * V) +
                          d * 16 + (at & 15);
            if (first >= 0 && first + 4 <= n) {
                uint32_t word = 0;
#pragma unroll
                for (int e = 0; e < 4; e++) word |= (uint32_t)turned[d][first + e] << (8 * e);
                *reinterpret_cast<uint32_t*>(to) = word;
            } else {
                for (int e = 0; e < 4; e++)
                    if (first + e >= 0 && first + e < n) to[e] = turned[d][first + e];
            }
        }
    } else {
        for (int item = threadIdx.x; item < n * V; item += 256) {
            const int d = item & (V - 1), i = item / V, at = places[i];
            if (at >= 0)
                c.values[cells[i] * V + (size_t)(at >> 4) * (16 * V) + d * 16 + (at & 15)] = (int8_t)turned[d][i];
        }
    }
}

// ----------------------------------------------------------------- pages --

struct Pages {
    nhip_paged_cache c;
    int32_t page_shift;
    size_t key_units, scale_units, value_units;  // 16-byte units of a page in one layer
};

Pages pages_of(const nhip_paged_cache* c)
{
    const size_t cells = (size_t)c->kv_heads * c->page_size;
    return {*c, __builtin_ctz((unsigned)c->page_size), cells * c->qk_dim / 16, cells * 4 / 16,
            cells * c->v_dim / 16};
}

__device__ __forceinline__ bool is_page(const Pages& p, int page) { return page >= 0 && page < p.c.pages; }

// A sequence's length, and the pages that hold it, whatever the array says.
__device__ __forceinline__ int held_length(const Pages& p, int seq)
{
    return min(max(p.c.lengths[seq], 0), p.c.width << p.page_shift);
}
__device__ __forceinline__ int page_count(const Pages& p, int length)
{
    return (length + (1 << p.page_shift) - 1) >> p.page_shift;
}

__device__ __forceinline__ void copy_units(uint8_t* pool, size_t units, size_t layer_page, size_t from, size_t to)
{
    const uint4* s = reinterpret_cast<const uint4*>(pool) + (layer_page + from) * units;
    uint4* d = reinterpret_cast<uint4*>(pool) + (layer_page + to) * units;
    for (size_t u = threadIdx.x; u < units; u += blockDim.x) d[u] = s[u];
}

// One layer of page `from` to page `to`, by a workgroup.
__device__ __forceinline__ void copy_page_layer(const Pages& p, int layer, int from, int to)
{
    const size_t base = (size_t)layer * p.c.pages;
    copy_units((uint8_t*)p.c.keys, p.key_units, base, from, to);
    copy_units((uint8_t*)p.c.values, p.value_units, base, from, to);
    copy_units((uint8_t*)p.c.key_scales, p.scale_units, base, from, to);
    copy_units((uint8_t*)p.c.value_scales, p.scale_units, base, from, to);
}

// Pairs of pages; entries out of range (a page that is not to be copied) are
// skipped.  `total` (may be NULL) holds the number of pairs on the device.
__global__ __launch_bounds__(256) void paged_copy_kernel(Pages p, const int32_t* src, const int32_t* dst,
                                                         const int32_t* total, int32_t count)
{
    const size_t n = (size_t)(total ? *total : count) * p.c.layers;
    for (size_t i = blockIdx.x; i < n; i += gridDim.x) {
        const size_t pair = i / p.c.layers;
        const int from = src[pair], to = dst[pair];
        if (is_page(p, from) && is_page(p, to) && from != to) copy_page_layer(p, (int)(i - pair * p.c.layers), from, to);
    }
}

__global__ __launch_bounds__(256) void paged_reset_kernel(Pages p)
{
    const size_t tid = (size_t)blockIdx.x * 256 + threadIdx.x, stride = (size_t)gridDim.x * 256;
    const size_t entries = (size_t)p.c.sequences * p.c.width;
    for (size_t i = tid; i < entries; i += stride) p.c.tables[i] = -1;
    for (size_t i = tid; i < (size_t)p.c.sequences; i += stride) p.c.lengths[i] = 0;
    for (size_t i = tid; i < (size_t)p.c.pages; i += stride) p.c.refs[i] = 0;
}

// Whether an entry before i names the same sequence (the whole workgroup asks).
__device__ __forceinline__ bool named_before(const int32_t* seq, int i)
{
    const int s = seq[i];
    bool found = false;
    for (int j = threadIdx.x; j < i; j += blockDim.x) found |= seq[j] == s;
    return __syncthreads_or(found) != 0;
}

// fork, first half: entry i's new row and length into the workspace, and the
// holds that it takes.  A second launch gives up the old holds and writes the
// rows, so that every source is read as it was before the call.
__global__ __launch_bounds__(256) void paged_fork_stage_kernel(Pages p, const int32_t* dst, const int32_t* src,
                                                               const int32_t* length, int32_t* staged_length,
                                                               int32_t* staged)
{
    const int i = blockIdx.x;
    const int d = dst[i], s = src[i];
    const bool ok = d >= 0 && d < p.c.sequences && s >= 0 && s < p.c.sequences;
    if (named_before(dst, i) || !ok) {
        if (threadIdx.x == 0) staged_length[i] = -1;
        return;
    }
    const int has = held_length(p, s);
    const int keep = length ? min(max(length[i], 0), has) : has;
    const int n = page_count(p, keep);
    for (int t = threadIdx.x; t < n; t += 256) {
        const int page = p.c.tables[(size_t)s * p.c.width + t];
        staged[(size_t)i * p.c.width + t] = page;
        if (is_page(p, page)) atomicAdd(&p.c.refs[page], 1);
    }
    if (threadIdx.x == 0) staged_length[i] = keep;
}

__global__ __launch_bounds__(256) void paged_fork_write_kernel(Pages p, const int32_t* dst,
                                                               const int32_t* staged_length, const int32_t* staged)
{
    const int i = blockIdx.x;
    const int keep = staged_length[i];
    if (keep < 0) return;
    const int d = dst[i];
    const int old = page_count(p, held_length(p, d)), n = page_count(p, keep);
    int32_t* row = p.c.tables + (size_t)d * p.c.width;
    for (int t = threadIdx.x; t < max(old, n); t += 256) {
        const int page = row[t];
        if (t < old && is_page(p, page)) atomicAdd(&p.c.refs[page], -1);
        row[t] = t < n ? staged[(size_t)i * p.c.width + t] : -1;
    }
    __syncthreads();
    if (threadIdx.x == 0) p.c.lengths[d] = keep;
}

// Exclusive prefix sum over the 1024 threads of a workgroup; *total is the
// sum.  `waves` is 16 ints of LDS, free again after the call.
__device__ __forceinline__ int block_scan(int v, int* waves, int* total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int sum = v;
    for (int off = 1; off < 64; off <<= 1) {
        const int up = __shfl_up(sum, off);
        if (lane >= off) sum += up;
    }
    if (lane == 63) waves[wave] = sum;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < 16; w++) {
        before += w < wave ? waves[w] : 0;
        all += waves[w];
    }
    __syncthreads();
    *total = all;
    return before + sum - v;
}

constexpr int kPlan = 1024;      // threads of the planning kernels
constexpr int kPlanPages = 4;    // pages a thread looks at per round
typedef int32_t i4 __attribute__((ext_vector_type(4), aligned(4)));

// The refs of pages [base + 4 tid, base + 4 tid + 4), -1 past the last page.
__device__ __forceinline__ i4 plan_refs(const Pages& p, int base)
{
    const int at = base + kPlanPages * (int)threadIdx.x;
    if (at + 4 <= p.c.pages) return *reinterpret_cast<const i4*>(p.c.refs + at);
    i4 r = {-1, -1, -1, -1};
    for (int k = 0; k < 4; k++)
        if (at + k < p.c.pages) r[k] = p.c.refs[at + k];
    return r;
}

// resize: one workgroup, a thread per entry.  Every decision first (what an
// entry gives up, copies and takes), then the free pages it all needs, in
// order; only when they suffice is anything changed.  pair_src / pair_dst
// [count] receive the pages to copy (-1: none), which a second launch copies.
__global__ __launch_bounds__(kPlan) void paged_resize_kernel(Pages p, const int32_t* seq, const int32_t* length,
                                                             int32_t count, int32_t* status, int32_t* pair_src,
                                                             int32_t* pair_dst, int32_t* free_list)
{
    __shared__ int waves[16];
    __shared__ int entry_seq[kMaxEntries], entry_tail[kMaxEntries], entry_has[kMaxEntries], entry_want[kMaxEntries],
        entry_start[kMaxEntries];
    __shared__ uint8_t entry_copies[kMaxEntries];
    const int i = threadIdx.x;
    const int s = i < count ? seq[i] : -1;
    const int want_length = i < count && length ? length[i] : 0;
    entry_seq[i] = s;
    __syncthreads();
    bool ok = i < count && s >= 0 && s < p.c.sequences;
    const bool refused = i < count && (!ok || want_length < 0 || want_length > (p.c.width << p.page_shift));
    ok = ok && !refused;
    if (ok)
        for (int j = 0; j < i; j++) ok &= entry_seq[j] != s;
    int has = 0, want = 0, tail = -1;
    if (ok) {
        const int old = held_length(p, s);
        has = page_count(p, old);
        want = page_count(p, want_length);
        if (want_length > old && (old & ((1 << p.page_shift) - 1)) != 0) {
            const int page = p.c.tables[(size_t)s * p.c.width + has - 1];
            if (is_page(p, page)) tail = page;
        }
    }
    entry_tail[i] = tail;
    entry_has[i] = has;
    entry_want[i] = want;
    __syncthreads();
    bool copies = false;
    if (tail >= 0) {
        int earlier = 0;
        for (int j = 0; j < i; j++) earlier += entry_tail[j] == tail;
        copies = earlier < p.c.refs[tail] - 1;
    }
    entry_copies[i] = copies;
    int total, refusals;
    // (more than the pool holds counts as one page more than that, so the sum stays an int)
    const int start = block_scan(copies + min(max(want - has, 0), p.c.pages + 1), waves, &total);
    entry_start[i] = start;
    block_scan(refused, waves, &refusals);
    // the `total` lowest free pages
    int found = 0;
    for (int base = 0; base < p.c.pages && found < total; base += kPlan * kPlanPages) {
        const i4 r = plan_refs(p, base);
        int here, mine = 0;
        for (int k = 0; k < 4; k++) mine += r[k] == 0;
        int at = found + block_scan(mine, waves, &here);
        for (int k = 0; k < 4; k++)
            if (r[k] == 0) {
                if (at < total) free_list[at] = base + kPlanPages * i + k;
                at++;
            }
        found += here;
    }
    const int missing = max(total - found, 0);
    if (i == 0 && status) {
        status[0] = missing;
        status[1] = refusals;
    }
    if (i < count) pair_src[i] = pair_dst[i] = -1;
    if (missing) return;
    __syncthreads();  // free_list; and every refs read is done
    if (copies) {
        const int page = free_list[start];
        pair_src[i] = tail;
        pair_dst[i] = page;
        atomicAdd(&p.c.refs[tail], -1);
        atomicAdd(&p.c.refs[page], 1);
        p.c.tables[(size_t)s * p.c.width + has - 1] = page;
    }
    if (ok) p.c.lengths[s] = want_length;
    // the pages given up and taken, a wave per entry
    for (int e = i >> 6; e < count; e += kPlan / 64) {
        const int a = entry_has[e], b = entry_want[e];
        if (a == b) continue;
        int32_t* row = p.c.tables + (size_t)entry_seq[e] * p.c.width;
        for (int t = b + (i & 63); t < a; t += 64) {
            if (is_page(p, row[t])) atomicAdd(&p.c.refs[row[t]], -1);
            row[t] = -1;
        }
        for (int t = a + (i & 63); t < b; t += 64) {
            const int page = free_list[entry_start[e] + entry_copies[e] + t - a];
            row[t] = page;
            atomicAdd(&p.c.refs[page], 1);
        }
    }
}

// compact: one workgroup counts the held pages n, then pairs the free pages
// below n with the held ones from n on, both in order.
__global__ __launch_bounds__(kPlan) void paged_compact_plan_kernel(Pages p, int32_t* status, int32_t* total,
                                                                   int32_t* src, int32_t* dst)
{
    __shared__ int waves[16];
    int held = 0;
    for (int base = 0; base < p.c.pages; base += kPlan * kPlanPages) {
        const i4 r = plan_refs(p, base);
        for (int k = 0; k < 4; k++) held += r[k] > 0;
    }
    int n;
    block_scan(held, waves, &n);
    int holes = 0, movers = 0;
    for (int base = 0; base < p.c.pages; base += kPlan * kPlanPages) {
        const i4 r = plan_refs(p, base);
        const int at = base + kPlanPages * (int)threadIdx.x;
        int hole = 0, mover = 0, sum;
        for (int k = 0; k < 4; k++) {
            hole += r[k] == 0 && at + k < n;
            mover += r[k] > 0 && at + k >= n;
        }
        int h = holes + block_scan(hole, waves, &sum);
        holes += sum;
        int m = movers + block_scan(mover, waves, &sum);
        movers += sum;
        for (int k = 0; k < 4; k++) {
            if (r[k] == 0 && at + k < n) dst[h++] = at + k;
            if (r[k] > 0 && at + k >= n) src[m++] = at + k;
        }
    }
    if (threadIdx.x == 0) {
        *total = min(movers, holes);
        if (status) *status = n;
    }
}

// The new page of each moved one, over `remap` [pages] (written only where
// something moves), and the refs that move with them.
__global__ __launch_bounds__(256) void paged_compact_remap_kernel(Pages p, const int32_t* total, const int32_t* src,
                                                                  const int32_t* dst, int32_t* remap)
{
    const int n = *total;
    for (int i = (int)blockIdx.x * 256 + (int)threadIdx.x; i < n; i += (int)gridDim.x * 256) {
        remap[src[i]] = dst[i];
        p.c.refs[dst[i]] = p.c.refs[src[i]];
    }
}

__global__ __launch_bounds__(256) void paged_compact_tables_kernel(Pages p, const int32_t* total, const int32_t* src,
                                                                   const int32_t* remap)
{
    const int n = *total;
    if (n == 0) return;
    const size_t tid = (size_t)blockIdx.x * 256 + threadIdx.x, stride = (size_t)gridDim.x * 256;
    for (size_t i = tid; i < (size_t)n; i += stride) p.c.refs[src[i]] = 0;
    // the movers are the held pages from the first one's index on
    const int first = src[0];
    for (int s = blockIdx.x; s < p.c.sequences; s += gridDim.x) {
        const int held = page_count(p, held_length(p, s));
        int32_t* row = p.c.tables + (size_t)s * p.c.width;
        for (int t = threadIdx.x; t < held; t += 256)
            if (row[t] >= first && row[t] < p.c.pages) row[t] = remap[row[t]];
    }
}

int32_t check_entries(const nhip_paged_cache* c, int32_t count)
{
    int32_t rc = paged_check(c);
    if (rc) return rc;
    NHIP_REQUIRE(count >= 0 && count <= kMaxEntries, "%d entries (at most %d)", count, kMaxEntries);
    return NHIP_OK;
}

// Workspace words: fork count * (1 + width); resize 2 count + count *
// (width + 1) free pages; compact 1 + 2 * pages + pages.
size_t pages_workspace_words(const nhip_paged_cache* c, int32_t count)
{
    return 16 + std::max((size_t)count * ((size_t)c->width + 4), (size_t)3 * c->pages);
}

int32_t check_workspace(const nhip_paged_cache* c, int32_t count, const void* ws, size_t bytes)
{
    NHIP_REQUIRE(ws && (reinterpret_cast<uintptr_t>(ws) & 3) == 0 && bytes >= 4 * pages_workspace_words(c, count),
                 "paged cache: the workspace (%zu bytes) is missing, misaligned or smaller than %zu bytes", bytes,
                 4 * pages_workspace_words(c, count));
    return NHIP_OK;
}

void launch_copy(const Pages& p, const int32_t* src, const int32_t* dst, const int32_t* total, int32_t most,
                 hipStream_t stream)
{
    const size_t items = (size_t)most * p.c.layers;
    hipLaunchKernelGGL(paged_copy_kernel, dim3((unsigned)std::min<size_t>(items, 4096)), dim3(256), 0, stream, p, src,
                       dst, total, most);
}

int32_t resize(const nhip_paged_cache* c, int32_t count, const int32_t* d_seq, const int32_t* d_length, bool grows,
               int32_t* d_status, void* ws, size_t bytes, void* stream)
{
    int32_t rc = check_entries(c, count);
    if (rc) return rc;
    NHIP_REQUIRE(count == 0 || (d_seq && (d_length || !grows)), "paged resize: null pointer");
    if (count == 0 && !d_status) return NHIP_OK;
    rc = check_workspace(c, count, ws, bytes);
    if (rc) return rc;
    rc = ensure_device();
    if (rc) return rc;
    const Pages p = pages_of(c);
    int32_t* w = static_cast<int32_t*>(ws);
    hipLaunchKernelGGL(paged_resize_kernel, dim3(1), dim3(kPlan), 0, as_stream(stream), p, d_seq, d_length, count,
                       d_status, w, w + count, w + 2 * count);
    NHIP_CHECK_HIP(hipGetLastError());
    if (grows && count) launch_copy(p, w, w + count, nullptr, count, as_stream(stream));
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

}  // namespace
}  // namespace nhip

using namespace nhip;

extern "C" {

int32_t nhip_paged_reset_dev(const nhip_paged_cache* c, void* stream)
{
    int32_t rc = paged_check(c);
    if (rc) return rc;
    rc = ensure_device();
    if (rc) return rc;
    const size_t most = std::max((size_t)c->sequences * c->width, (size_t)c->pages);
    hipLaunchKernelGGL(paged_reset_kernel, dim3((unsigned)std::min<size_t>((most + 255) / 256, 2048)), dim3(256), 0,
                       as_stream(stream), pages_of(c));
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

int32_t nhip_paged_append_dev(const nhip_paged_cache* c, int32_t layer, const float* d_k, int32_t ldk,
                              const float* d_v, int32_t ldv, const int32_t* d_row_seq, const int32_t* d_row_pos,
                              int32_t rows, void* stream)
{
    int32_t rc = paged_check(c);
    if (rc) return rc;
    NHIP_REQUIRE(layer >= 0 && layer < c->layers, "paged append: layer %d of %d", layer, c->layers);
    NHIP_REQUIRE(rows >= 0 && rows <= kPagedMaxRows, "paged append: %d rows", rows);
    if (rows == 0) return NHIP_OK;
    NHIP_REQUIRE(d_k && d_v && d_row_seq && d_row_pos, "paged append: null pointer");
    NHIP_REQUIRE(ldk >= c->kv_heads * c->qk_dim && ldv >= c->kv_heads * c->v_dim,
                 "paged append: row strides %d, %d below a row's columns", ldk, ldv);
    rc = ensure_device();
    if (rc) return rc;
    const AppendParams p{paged_layer(c, layer), d_k, d_v, d_row_seq, d_row_pos, ldk, ldv, rows};
    const dim3 grid((unsigned)(rows + 15) / 16, (unsigned)c->kv_heads);
    if (c->qk_dim == 48)
        hipLaunchKernelGGL((paged_append_kernel<48, 64>), grid, dim3(256), 0, as_stream(stream), p);
    else if (c->qk_dim == 64)
        hipLaunchKernelGGL((paged_append_kernel<64, 64>), grid, dim3(256), 0, as_stream(stream), p);
    else
        hipLaunchKernelGGL((paged_append_kernel<128, 128>), grid, dim3(256), 0, as_stream(stream), p);
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

size_t nhip_paged_pages_workspace(const nhip_paged_cache* c, int32_t count)
{
    return check_entries(c, count) ? 0 : 4 * pages_workspace_words(c, count);
}

int32_t nhip_paged_copy_dev(const nhip_paged_cache* c, int32_t count, const int32_t* d_src, const int32_t* d_dst,
                            void* stream)
{
    int32_t rc = check_entries(c, count);
    if (rc) return rc;
    if (count == 0) return NHIP_OK;
    NHIP_REQUIRE(d_src && d_dst, "paged copy: null pointer");
    rc = ensure_device();
    if (rc) return rc;
    launch_copy(pages_of(c), d_src, d_dst, nullptr, count, as_stream(stream));
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

int32_t nhip_paged_fork_dev(const nhip_paged_cache* c, int32_t count, const int32_t* d_dst, const int32_t* d_src,
                            const int32_t* d_length, void* d_workspace, size_t workspace_bytes, void* stream)
{
    int32_t rc = check_entries(c, count);
    if (rc) return rc;
    if (count == 0) return NHIP_OK;
    NHIP_REQUIRE(d_dst && d_src, "paged fork: null pointer");
    rc = check_workspace(c, count, d_workspace, workspace_bytes);
    if (rc) return rc;
    rc = ensure_device();
    if (rc) return rc;
    const Pages p = pages_of(c);
    int32_t* w = static_cast<int32_t*>(d_workspace);
    hipLaunchKernelGGL(paged_fork_stage_kernel, dim3(count), dim3(256), 0, as_stream(stream), p, d_dst, d_src,
                       d_length, w, w + count);
    NHIP_CHECK_HIP(hipGetLastError());
    hipLaunchKernelGGL(paged_fork_write_kernel, dim3(count), dim3(256), 0, as_stream(stream), p, d_dst, w, w + count);
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

int32_t nhip_paged_resize_dev(const nhip_paged_cache* c, int32_t count, const int32_t* d_seq,
                              const int32_t* d_length, int32_t* d_status, void* d_workspace, size_t workspace_bytes,
                              void* stream)
{
    return resize(c, count, d_seq, d_length, true, d_status, d_workspace, workspace_bytes, stream);
}

int32_t nhip_paged_free_dev(const nhip_paged_cache* c, int32_t count, const int32_t* d_seq, void* d_workspace,
                            size_t workspace_bytes, void* stream)
{
    return resize(c, count, d_seq, nullptr, false, nullptr, d_workspace, workspace_bytes, stream);
}

int32_t nhip_paged_compact_dev(const nhip_paged_cache* c, int32_t* d_status, void* d_workspace,
                               size_t workspace_bytes, void* stream)
{
    int32_t rc = paged_check(c);
    if (rc) return rc;
    rc = check_workspace(c, 0, d_workspace, workspace_bytes);
    if (rc) return rc;
    rc = ensure_device();
    if (rc) return rc;
    const Pages p = pages_of(c);
    int32_t* w = static_cast<int32_t*>(d_workspace);
    int32_t *total = w, *src = w + 16, *dst = src + c->pages, *remap = dst + c->pages;
    hipStream_t s = as_stream(stream);
    hipLaunchKernelGGL(paged_compact_plan_kernel, dim3(1), dim3(kPlan), 0, s, p, d_status, total, src, dst);
    NHIP_CHECK_HIP(hipGetLastError());
    const unsigned grid = (unsigned)std::min((c->pages + 255) / 256, 1024);
    hipLaunchKernelGGL(paged_compact_remap_kernel, dim3(grid), dim3(256), 0, s, p, total, src, dst, remap);
    NHIP_CHECK_HIP(hipGetLastError());
    launch_copy(p, src, dst, total, (c->pages + 1) / 2, s);
    NHIP_CHECK_HIP(hipGetLastError());
    hipLaunchKernelGGL(paged_compact_tables_kernel, dim3((unsigned)std::min(c->sequences, 1024)), dim3(256), 0, s, p,
                       total, src, remap);
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

}  // extern "C"
