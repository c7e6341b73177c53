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
// atomics are integer additions to refs, whose order does not show.  Of these
// calls only the copies move many bytes; the rest are chains of latencies in
// one workgroup: a fork of 3 rows 2.6 us, a resize 5 to 10 (entries, tables,
// refs, then the free pages by prefix sums), a compaction's plan 6.
#include <algorithm>
#include <type_traits>

#include "paged.hpp"
#include "rotary.hpp"
#include "stores.hpp"

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
    const int32_t* refs;
    int32_t ldk, ldv, rows;
};

// The same with the rows' queries and keys rotated by position first.
struct RotaryAppendParams : AppendParams {
    RotaryTable r;
    const float* q;
    int8_t* codes;
    float* q_scales;
    int32_t ldq, heads;
};

// A row whose page other sequences hold too writes nothing: a resize that found
// too few pages has not made the row's copy of it, and only the device knows.
//
// A workgroup takes 16 rows of one kv head; L lanes share a row's key (or
// value) head, four elements each, so a head's peak is a few DPP steps and 16
// rows of keys leave as whole dwords.  Values change places through LDS: the
// cache holds 16 positions of a dimension together, and where the rows are
// consecutive positions of one sequence (a prompt) a lane writes as many of
// them at once as lie in a block; else each goes by itself.  Bound by the
// bytes: 8185 rows of 8 kv heads of 128 (84 MB) take 18.2 us, 4.6 TB/s (with
// the groups dealt to the XCDs one by one 26 MB were written for 17, 1.2 us
// more; with 64 rows a workgroup, fewer of which are in flight, 3.7 us more).
// One step's 16 rows take 4.5 us: a launch (2.5) and the chain sequence, page,
// holders, store, which the codes are formed beside.
constexpr int kAppendRows = 16;

template <int L>
__device__ __forceinline__ float group_max(float v)
{
    v = fmaxf(v, lane_xor<1>(v));
    v = fmaxf(v, lane_xor<2>(v));
    v = fmaxf(v, lane_xor<4>(v));
    v = fmaxf(v, lane_xor<8>(v));
    return L == 32 ? fmaxf(v, lane_xor<16>(v)) : v;
}

// A position's page and its place there, for a row to be written: page -1 where
// it may not be.
struct Place {
    int page, at;
};
// Heads and rows that one workgroup rotates.
constexpr int kRotatedHeads = 4;
template <int QK>
__host__ __device__ constexpr int rotated_rows()
{
    return 256 / (QK <= 64 ? 8 : 16) / kRotatedHeads;
}
__device__ __forceinline__ Place place_of(const PagedLayer& c, const int32_t* refs, int seq, int pos)
{
    int page = -1;
    if (seq >= 0 && seq < c.sequences && pos >= 0 && (pos >> c.page_shift) < c.width)
        page = c.tables[(size_t)seq * c.width + (pos >> c.page_shift)];
    if (page < 0 || page >= c.pages || refs[page] > 1) page = -1;
    return {page, pos & ((1 << c.page_shift) - 1)};
}

// Query and key heads rotated and quantized: four neighbouring heads of each row,
// L lanes a head, a unit of eight elements each.  Heads from p.heads on are the
// keys'.  A lane's eight elements are two 16-byte loads and two 4-byte stores of
// codes; the peak is the maximum over L lanes.  Bytes bound it: 8185 rows of
// 32 + 8 heads of 128 and their values, 205 MB read and 52 written, take 46 us,
// 5.6 TB/s, behind passes that store past the caches, and 56 to 61 behind others,
// as all that follows here: 84 where the XCDs' shares of these workgroups and the
// values' were uneven; 58 to 68 with a row's heads far apart in the grid, for the
// table came from memory again for each; 62 to 65 with 16 rows of one head, whose
// reads are 512 bytes apart from one another.  Two or four heads a lane, for which
// the table is read once, take 39.2 and 41.0 us in place of 40.0 from the last
// cache, for 512 rows 5.3 and 6.3 in place of 5.1; eight neighbouring heads in
// place of four the same.  MIXED, for dimensions that are no multiple of 8, is bound
// by the element-wise reads of partners and table: the same rows with 60 rotated 97
// (halves) and 107 (neighbours), 54.5 with 64; 16 rows 5.2 and 4.0.
template <int QK, bool MIXED>
__device__ __forceinline__ void append_rotated(const RotaryAppendParams& p, int first_head, int row0)
{
    constexpr int L = QK <= 64 ? 8 : 16;
    const PagedLayer& c = p.c;
    const int l = threadIdx.x % L, slot = threadIdx.x / L;
    const int row = row0 + slot / kRotatedHeads, at = min(row, p.rows - 1);
    const int heads = p.heads + c.kv_heads, head = min(first_head + slot % kRotatedHeads, heads - 1);
    const int pos = p.row_pos[at];
    const bool known = pos >= 0 && pos < p.r.positions, mine = 8 * l < QK;
    const RotaryUnit unit = rotary_unit<MIXED>(p.r, QK, mine ? l : 0, known ? pos : 0);
    const float* from = head < p.heads ? p.q + ((size_t)at * p.ldq + head * QK)
                                       : p.k + ((size_t)at * p.ldk + (head - p.heads) * QK);
    f4 a = *reinterpret_cast<const f4*>(from + unit.a), b = *reinterpret_cast<const f4*>(from + unit.b);
    Place place = {-1, 0};
    if (head >= p.heads && known) place = place_of(c, p.refs, p.row_seq[at], pos);
    rotate_unit<MIXED>(p.r, unit, from, a, b);
    if (!known || !mine) a = b = f4{0.0f, 0.0f, 0.0f, 0.0f};
    float peak = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; e++) peak = fmaxf(peak, fmaxf(fabsf(a[e]), fabsf(b[e])));
    peak = fmaxf(peak, lane_xor<1>(peak));
    peak = fmaxf(peak, lane_xor<2>(peak));
    peak = fmaxf(peak, lane_xor<4>(peak));
    if (L == 16) peak = fmaxf(peak, lane_xor<8>(peak));
    const float scale = peak > 0.0f ? peak / 127.0f : 1.0f, inverse = 1.0f / scale;
    if (row >= p.rows || first_head + slot % kRotatedHeads >= heads) return;
    auto put = [&](int8_t* codes, float* scales, size_t to) {
        codes += to * QK;
        if (mine) {
            *reinterpret_cast<uint32_t*>(codes + unit.a) = ref_quantize4(make_float4(a[0], a[1], a[2], a[3]), inverse);
            *reinterpret_cast<uint32_t*>(codes + unit.b) = ref_quantize4(make_float4(b[0], b[1], b[2], b[3]), inverse);
        }
        if (l == 0) scales[to] = scale;
    };
    if (head < p.heads)
        put(p.codes, p.q_scales, (size_t)row * p.heads + head);
    else if (place.page >= 0)
        put(c.keys, c.kscale, (((size_t)place.page * c.kv_heads + head - p.heads) << c.page_shift) + place.at);
}

// ROTARY: the keys go with the queries, in workgroups of their own.
template <int QK, int V, bool MIXED, typename Params>
__global__ __launch_bounds__(256) void paged_append_kernel(Params p)
{
    constexpr bool ROTARY = std::is_same<Params, RotaryAppendParams>::value;
    constexpr int N = kAppendRows, L = V <= 64 ? 16 : 32, ROWS = 256 / L, PASSES = N / ROWS;  // rows of a pass
    __shared__ size_t cells[N];
    __shared__ int places[N], first_position;
    // value codes by dimension, then row from 16 on: a block's 16 rows may begin before the first and end behind the last
    __shared__ __align__(16) uint8_t turned[V][N + 36];
    __shared__ bool consecutive;
    const PagedLayer& c = p.c;
    // an XCD takes neighbouring groups of rows, so that the pieces of a block that two workgroups write meet in its L2
    // (and, where keys go apart, as much of either kind of workgroup as the others)
    const uint32_t id = blockIdx.y * gridDim.x + blockIdx.x;
    const uint32_t groups = (p.rows + N - 1) / N, all = groups * c.kv_heads;
    const uint32_t share = ROTARY ? (all + 7) / 8 : gridDim.x * gridDim.y / 8;
    if constexpr (ROTARY) {
        if (id / 8 >= share) {
            constexpr int R = rotated_rows<QK>();
            const uint32_t sides = (p.heads + c.kv_heads + kRotatedHeads - 1) / kRotatedHeads;
            const uint32_t rotated = (p.rows + R - 1) / R * sides;
            const uint32_t part = (id & 7) * ((rotated + 7) / 8) + id / 8 - share, group = part / sides;
            if (id / 8 - share < (rotated + 7) / 8 && part < rotated)
                append_rotated<QK, MIXED>(p, (part - group * sides) * kRotatedHeads, (int)group * R);
            return;
        }
    }
    const uint32_t group = (id & 7) * share + id / 8;
    if (group >= all) return;
    const int kvh = group / groups, row0 = (int)(group - kvh * groups) * N, n = min(N, p.rows - row0);
    const int l = threadIdx.x & (L - 1), row_of_pass = threadIdx.x / L;
    f4 x[PASSES][2];
#pragma unroll
    for (int k = 0; k < PASSES; k++) {
        const size_t r = row0 + min(row_of_pass + k * ROWS, n - 1);
        x[k][0] = x[k][1] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        if (!ROTARY && 4 * l < QK) x[k][0] = *reinterpret_cast<const f4*>(p.k + r * p.ldk + kvh * QK + 4 * l);
        if (4 * l < V) x[k][1] = *reinterpret_cast<const f4*>(p.v + r * p.ldv + kvh * V + 4 * l);
    }
    // where each row's position lives: its page's first cell (of this kv head) and its place in the page, -1 if nowhere
    int seq = -1, pos = 0, page = -1;
    if (threadIdx.x < N) {
        const int r = row0 + min((int)threadIdx.x, n - 1);
        seq = p.row_seq[r], pos = p.row_pos[r];
        bool known = pos >= 0;
        if constexpr (ROTARY) known = known && pos < p.r.positions;
        if (seq >= 0 && seq < c.sequences && known && (pos >> c.page_shift) < c.width)
            page = c.tables[(size_t)seq * c.width + (pos >> c.page_shift)];
    }
    float scales[PASSES][2];
    uint32_t codes[PASSES][2];
#pragma unroll
    for (int k = 0; k < PASSES; k++) {
        const int i = row_of_pass + k * ROWS;
#pragma unroll
        for (int part = ROTARY ? 1 : 0; part < 2; part++) {
            const f4 y = x[k][part];
            const float peak =
                group_max<L>(fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3]))));
            scales[k][part] = peak > 0.0f ? peak / 127.0f : 1.0f;
            codes[k][part] = ref_quantize4(make_float4(y[0], y[1], y[2], y[3]), 1.0f / scales[k][part]);
            if (part == 1 && 4 * l < V) {
#pragma unroll
                for (int e = 0; e < 4; e++) turned[4 * l + e][16 + i] = (uint8_t)(codes[k][part] >> (8 * e));
            }
        }
    }
    if (threadIdx.x < N) {
        const int i = threadIdx.x;
        const bool ok = i < n && page >= 0 && page < c.pages && p.refs[page] <= 1;
        cells[i] = ok ? ((size_t)page * c.kv_heads + kvh) << c.page_shift : 0;
        places[i] = ok ? pos & ((1 << c.page_shift) - 1) : -1;
        // (the first wave's: whether the rows are consecutive positions of one sequence)
        const int seq0 = __builtin_amdgcn_readfirstlane(seq), pos0 = __builtin_amdgcn_readfirstlane(pos);
        const uint64_t odd = __ballot(i < n && (!ok || seq != seq0 || pos != pos0 + i));
        if (i == 0) {
            consecutive = odd == 0;
            first_position = pos;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PASSES; k++) {
        const int at = places[row_of_pass + k * ROWS];
        const size_t cell = cells[row_of_pass + k * ROWS];
        if (at < 0) continue;
        if (!ROTARY && 4 * l < QK) *reinterpret_cast<uint32_t*>(c.keys + (cell + at) * QK + 4 * l) = codes[k][0];
        if (l == 0) {
            if (!ROTARY) c.kscale[cell + at] = scales[k][0];
            c.vscale[cell + at] = scales[k][1];
        }
    }
    if (consecutive) {
        // blocks of 16 positions, whole ones as one store a dimension, the ends in quads where they have them
        const int lead = first_position & 15;
        for (int item = threadIdx.x; item < (N / 16 + 1) * V; item += 256) {
            const int d = item & (V - 1), first = 16 * (item / V) - lead;  // the block's first row
            if (first >= n) continue;
            const int some = max(first, 0), at = places[some] & ~15;
            uint8_t* to = reinterpret_cast<uint8_t*>(c.values) + cells[some] * V + (size_t)(at >> 4) * (16 * V) + d * 16;
            const uint32_t* from = reinterpret_cast<const uint32_t*>(turned[d] + ((16 + first) & ~3));
            uint32_t words[5];
#pragma unroll
            for (int k = 0; k < 5; k++) words[k] = from[k];
#pragma unroll
            for (int k = 0; k < 4; k++) words[k] = __builtin_amdgcn_alignbyte(words[k + 1], words[k], first & 3);
            if (first >= 0 && first + 16 <= n) {
                *reinterpret_cast<uint4*>(to) = make_uint4(words[0], words[1], words[2], words[3]);
                continue;
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int row = first + 4 * k;
                if (row >= 0 && row + 4 <= n) {
                    *reinterpret_cast<uint32_t*>(to + 4 * k) = words[k];
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (row + e >= 0 && row + e < n) to[4 * k + e] = (uint8_t)(words[k] >> (8 * e));
                }
            }
        }
    } else {
        for (int item = threadIdx.x; item < n * V; item += 256) {
            const int d = item & (V - 1), i = item / V, at = places[i];
            if (at >= 0)
                c.values[cells[i] * V + (size_t)(at >> 4) * (16 * V) + d * 16 + (at & 15)] = (int8_t)turned[d][16 + i];
        }
    }
}

template <int QK, int V, bool MIXED, typename Params>
void launch_append(const Params& p, unsigned groups, hipStream_t stream)
{
    const unsigned x = std::min((groups + 7) / 8 * 8, 1u << 20);  // (a multiple of 8)
    hipLaunchKernelGGL((paged_append_kernel<QK, V, MIXED, Params>), dim3(x, (groups + x - 1) / x), dim3(256), 0, stream,
                       p);
}
unsigned row_groups(int rows) { return (unsigned)(rows + kAppendRows - 1) / kAppendRows; }
template <int QK, int V>
void launch_append(const AppendParams& p, hipStream_t stream)
{
    launch_append<QK, V, false>(p, row_groups(p.rows) * p.c.kv_heads, stream);
}
template <int QK, int V>
void launch_append(const RotaryAppendParams& p, hipStream_t stream)
{
    constexpr unsigned R = rotated_rows<QK>();
    const unsigned sides = (p.heads + p.c.kv_heads + kRotatedHeads - 1) / kRotatedHeads;
    // (each XCD's share of either kind of workgroup, rounded up)
    const unsigned all = (row_groups(p.rows) * p.c.kv_heads + 7) / 8 * 8 + ((p.rows + R - 1) / R * sides + 7) / 8 * 8;
    if (p.r.dim % 8)
        launch_append<QK, V, true>(p, all, stream);
    else
        launch_append<QK, V, false>(p, all, stream);
}

template <typename Params>
int32_t launch_append(const nhip_paged_cache* c, const Params& p, hipStream_t stream)
{
    if (c->qk_dim == 48)
        launch_append<48, 64>(p, stream);
    else if (c->qk_dim == 64)
        launch_append<64, 64>(p, stream);
    else
        launch_append<128, 128>(p, stream);
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

int32_t check_append(const nhip_paged_cache* c, const char* what, int32_t layer, int32_t rows)
{
    int32_t rc = paged_check(c);
    if (rc) return rc;
    NHIP_REQUIRE(layer >= 0 && layer < c->layers, "paged %s: layer %d of %d", what, layer, c->layers);
    NHIP_REQUIRE(rows >= 0 && rows <= kPagedMaxRows, "paged %s: %d rows", what, rows);
    return NHIP_OK;
}

// ------------------------------------------------------------------ read --

struct ReadParams {
    PagedLayer c;
    const int32_t* row_seq;
    const int32_t* row_pos;
    float* k;
    float* v;
    int32_t ldk, ldv, rows;
    bool away;
};

// 4 L threads take the keys or the values (blockIdx.y) of 16 rows of one kv
// head, L lanes a row.  Where the rows are consecutive positions of one sequence
// a thread reads, for each block of 16 positions, the four bytes that four
// positions have in each of four dimensions, and has four rows' values; else a
// value is a byte by itself, and a line of the cache is read 16 times (from L2).
// Bytes bound it, four out for one in: 8185 rows of 8 kv heads of 128, 17 MB
// read and 67 written, 16.4 to 20.4 us, 4.1 to 5.1 TB/s (up to 2 less past the
// caches, which the call that reads them pays for: stores.hpp); in no order, where a
// value is a byte by itself, 26.4.
template <int QK, int V>
__global__ __launch_bounds__(256) void paged_read_kernel(ReadParams p)
{
    constexpr int N = kAppendRows, L = V <= 64 ? 16 : 32, UNITS = 256 / (4 * L);
    __shared__ size_t cells[UNITS][N];
    __shared__ bool consecutive[UNITS];
    const PagedLayer& c = p.c;
    const int l = threadIdx.x & (L - 1), sub = (threadIdx.x / L) & 3, u = threadIdx.x / (4 * L);
    const uint32_t unit = blockIdx.x * UNITS + u, group = unit / c.kv_heads;
    const int kvh = unit - group * c.kv_heads, row0 = (int)group * N, n = min(N, p.rows - row0);
    if (threadIdx.x % (4 * L) < N && n > 0) {
        const int i = threadIdx.x % (4 * L), row = row0 + min(i, n - 1), seq = p.row_seq[row], pos = p.row_pos[row];
        int page = -1;
        if (seq >= 0 && seq < c.sequences && pos >= 0 && (pos >> c.page_shift) < c.width)
            page = c.tables[(size_t)seq * c.width + (pos >> c.page_shift)];
        if (page >= c.pages) page = -1;
        cells[u][i] = page < 0 ? (size_t)-1
                               : (((size_t)page * c.kv_heads + kvh) << c.page_shift) + (pos & ((1 << c.page_shift) - 1));
        const int lane0 = (threadIdx.x & 63) & ~15;
        const int seq0 = __shfl(seq, lane0), pos0 = __shfl(pos, lane0);
        const uint64_t odd = __ballot(page < 0 || seq != seq0 || (int64_t)pos != (int64_t)pos0 + min(i, n - 1));
        if (i == 0) consecutive[u] = ((odd >> lane0) & 0xFFFF) == 0;
    }
    __syncthreads();
    if (n <= 0) return;
    const f4 none = {0.0f, 0.0f, 0.0f, 0.0f};
    if (blockIdx.y == (p.k ? 0 : 2)) {
        if (4 * l >= QK) return;
        uint32_t codes[4];
        float scale[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const size_t cell = cells[u][min(sub + 4 * k, n - 1)], at = cell == (size_t)-1 ? 0 : cell;
            codes[k] = *reinterpret_cast<const uint32_t*>(c.keys + at * QK + 4 * l);
            scale[k] = c.kscale[at];
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = sub + 4 * k;
            if (i >= n) break;
            f4 y;
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = (float)(int8_t)(codes[k] >> (8 * e)) * scale[k];
            store_f4(p.k + (size_t)(row0 + i) * p.ldk + kvh * QK + 4 * l, cells[u][i] == (size_t)-1 ? none : y, p.away);
        }
        return;
    }
    float* to = p.v + (size_t)row0 * p.ldv + kvh * V + 4 * l;
    if (consecutive[u]) {
        const int lead = (int)(cells[u][0] & 15);
#pragma unroll
        for (int block = 0; block < 2; block++) {
            const int first = 16 * block + 4 * sub - lead;  // row of the thread's first position
            if (first + 3 < 0 || first >= n) continue;
            // (its positions lie in one quad, so in one page)
            const size_t cell = (cells[u][max(first, 0)] & ~(size_t)15) + 4 * sub;
            uint32_t codes[4];
#pragma unroll
            for (int e = 0; e < 4; e++)
                codes[e] = *reinterpret_cast<const uint32_t*>(c.values + (cell - 4 * sub) * V + 16 * (4 * l + e) + 4 * sub);
            const f4 scale = *reinterpret_cast<const f4*>(c.vscale + cell);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (first + k < 0 || first + k >= n) continue;
                f4 y;
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = (float)(int8_t)(codes[e] >> (8 * k)) * scale[k];
                store_f4(to + (size_t)(first + k) * p.ldv, y, p.away);
            }
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int i = sub + 4 * k;
        if (i >= n) break;
        const size_t cell = cells[u][i], at = cell == (size_t)-1 ? 0 : cell;
        const int8_t* from = c.values + (at & ~(size_t)15) * V + 64 * l + (at & 15);
        const float scale = c.vscale[at];
        f4 y;
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = (float)from[16 * e] * scale;
        store_f4(to + (size_t)i * p.ldv, cell == (size_t)-1 ? none : y, p.away);
    }
}

// ----------------------------------------------------------------- pages --

struct Pages {
    nhip_paged_cache c;
    int32_t page_shift;
    uint32_t key_units, scale_units, value_units;  // 16-byte units of a page in one layer
};

Pages pages_of(const nhip_paged_cache* c)
{
    const uint32_t cells = (uint32_t)c->kv_heads * c->page_size;
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

// A page of one layer is copied in slices of kSliceUnits 16-byte units, a
// workgroup each: eight loads a lane, then eight stores, past the caches (a
// compaction of 650 MB takes 140 us, 151 through them).
constexpr int kSliceUnits = 2048;

__host__ __device__ inline uint32_t page_units(const Pages& p)
{
    return p.key_units + p.value_units + 2 * p.scale_units;
}
__host__ __device__ inline uint32_t page_slices(const Pages& p)
{
    return (page_units(p) + kSliceUnits - 1) / kSliceUnits;
}

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// Where unit u of a page's layer lies in the pools, u counting keys, values,
// key scales, value scales; `cell` is layer * pages + page.
__device__ __forceinline__ u4* page_unit(const Pages& p, size_t cell, uint32_t u)
{
    const uint32_t k = p.key_units, v = p.value_units, s = p.scale_units;
    const bool keys = u < k, values = u < k + v, key_scales = u < k + v + s;
    u4* pool = reinterpret_cast<u4*>(keys ? (void*)p.c.keys
                                     : values ? (void*)p.c.values
                                     : key_scales ? (void*)p.c.key_scales : (void*)p.c.value_scales);
    const uint32_t units = keys ? k : values ? v : s;
    const uint32_t at = keys ? u : values ? u - k : key_scales ? u - k - v : u - k - v - s;
    return pool + cell * units + at;
}

__device__ __forceinline__ void copy_slice(const Pages& p, int layer, int from, int to, uint32_t slice)
{
    const size_t base = (size_t)layer * p.c.pages;
    const uint32_t first = slice * kSliceUnits + threadIdx.x, last = page_units(p) - 1;
    u4 x[8];
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] = __builtin_nontemporal_load(page_unit(p, base + from, min(first + 256 * k, last)));
#pragma unroll
    for (int k = 0; k < 8; k++)
        if (first + 256 * k <= last) __builtin_nontemporal_store(x[k], page_unit(p, base + to, first + 256 * k));
}

// The slices of `n` pairs of pages in every layer, spread over `workers`
// workgroups; a pair out of range (a page that is not to be copied) is skipped.
__device__ __forceinline__ void copy_pairs(const Pages& p, const int32_t* src, const int32_t* dst, int n, int worker,
                                           int workers)
{
    // (a page's layer is at least 1920 bytes, so a pool that fits the device has fewer than 2^32 slices)
    const uint32_t slices = page_slices(p), layers = p.c.layers;
    const uint32_t items = (uint32_t)n * layers * slices;
    for (uint32_t i = worker; i < items; i += workers) {
        const uint32_t rest = i / slices, pair = rest / layers;
        const int from = src[pair], to = dst[pair];
        if (is_page(p, from) && is_page(p, to) && from != to)
            copy_slice(p, (int)(rest - pair * layers), from, to, i - rest * slices);
    }
}

__global__ __launch_bounds__(256) void paged_copy_kernel(Pages p, const int32_t* src, const int32_t* dst,
                                                         int32_t count)
{
    copy_pairs(p, src, dst, count, blockIdx.x, gridDim.x);
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

// How many of the first n entries of an LDS list equal v (n need not be a
// multiple of 4; the list is padded to one).
__device__ __forceinline__ int count_equal(const int* list, int n, int v)
{
    int found = 0;
    const int4* l4 = reinterpret_cast<const int4*>(list);
#pragma unroll 8
    for (int j = 0; j < n / 4; j++) {
        const int4 x = l4[j];
        found += (x.x == v) + (x.y == v) + (x.z == v) + (x.w == v);
    }
    const int4 x = l4[n / 4];
    const int rest = n & 3;
    found += (rest > 0 && x.x == v) + (rest > 1 && x.y == v) + (rest > 2 && x.z == v);
    return found;
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

// fork of a few short rows in one launch: one workgroup, the halves on either
// side of a barrier, a wave per entry.
constexpr int kForkThreads = 1024;
__global__ __launch_bounds__(kForkThreads) void paged_fork_kernel(Pages p, const int32_t* dst, const int32_t* src,
                                                                  const int32_t* length, int32_t count,
                                                                  int32_t* staged)
{
    __shared__ __align__(16) int entry_dst[kMaxEntries];
    __shared__ int entry_keep[kMaxEntries];
    const int i = threadIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int d = i < count ? dst[i] : -1, s = i < count ? src[i] : -1;
    entry_dst[i] = d;
    __syncthreads();
    int keep = -1;
    if (d >= 0 && d < p.c.sequences && s >= 0 && s < p.c.sequences && count_equal(entry_dst, i, d) == 0) {
        const int has = held_length(p, s);
        keep = length ? min(max(length[i], 0), has) : has;
    }
    entry_keep[i] = keep;
    __syncthreads();
    for (int e = wave; e < count; e += kForkThreads / 64) {
        const int n = page_count(p, max(entry_keep[e], 0));
        const int32_t* row = p.c.tables + (size_t)(n ? src[e] : 0) * p.c.width;
        for (int t = lane; t < n; t += 64) {
            const int page = row[t];
            staged[(size_t)e * p.c.width + t] = page;
            if (is_page(p, page)) atomicAdd(&p.c.refs[page], 1);
        }
    }
    __syncthreads();
    for (int e = wave; e < count; e += kForkThreads / 64) {
        if (entry_keep[e] < 0) continue;
        const int to = entry_dst[e];
        const int n = page_count(p, entry_keep[e]), old = page_count(p, held_length(p, to));
        int32_t* row = p.c.tables + (size_t)to * p.c.width;
        for (int t = lane; t < max(old, n); t += 64) {
            const int page = row[t];
            if (t < old && is_page(p, page)) atomicAdd(&p.c.refs[page], -1);
            row[t] = t < n ? staged[(size_t)e * p.c.width + t] : -1;
        }
        if (lane == 0) p.c.lengths[to] = entry_keep[e];
    }
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

constexpr int kPlan = 1024;     // threads of the planning kernels
constexpr int kPlanPages = 16;  // pages a thread looks at per round
typedef int32_t i4 __attribute__((ext_vector_type(4), aligned(4)));

// The refs of this thread's kPlanPages pages of a round from `base`, -1 past the last page.
struct PlanRefs {
    int32_t r[kPlanPages];
};
__device__ __forceinline__ PlanRefs plan_refs(const Pages& p, int base)
{
    PlanRefs x;
    const int at = base + kPlanPages * (int)threadIdx.x;
#pragma unroll
    for (int k = 0; k < kPlanPages; k += 4) {
        if (at + k + 4 <= p.c.pages) {
            const i4 v = *reinterpret_cast<const i4*>(p.c.refs + at + k);
#pragma unroll
            for (int e = 0; e < 4; e++) x.r[k + e] = v[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) x.r[k + e] = at + k + e < p.c.pages ? p.c.refs[at + k + e] : -1;
        }
    }
    return x;
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
    __shared__ __align__(16) int entry_seq[kMaxEntries], entry_tail[kMaxEntries];
    __shared__ int entry_has[kMaxEntries], entry_want[kMaxEntries], entry_start[kMaxEntries];
    __shared__ uint8_t entry_copies[kMaxEntries];
    const int i = threadIdx.x;
    const PlanRefs round0 = plan_refs(p, 0);  // (ahead of the loads that depend on one another)
    const int s = i < count ? seq[i] : -1;
    const int want_length = i < count && length ? length[i] : 0;
    entry_seq[i] = s;
    __syncthreads();
    bool ok = i < count && s >= 0 && s < p.c.sequences;
    const bool refused = i < count && (!ok || want_length < 0 || want_length > (p.c.width << p.page_shift));
    ok = ok && !refused;
    ok = ok && count_equal(entry_seq, i, s) == 0;
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
        const int holders = p.c.refs[tail];
        copies = holders > 1 && count_equal(entry_tail, i, tail) < holders - 1;
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
        const PlanRefs x = base == 0 ? round0 : plan_refs(p, base);
        int here, mine = 0;
#pragma unroll
        for (int k = 0; k < kPlanPages; k++) mine += x.r[k] == 0;
        int at = found + block_scan(mine, waves, &here);
#pragma unroll
        for (int k = 0; k < kPlanPages; k++)
            if (x.r[k] == 0) {
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

// compact, first launch: one workgroup counts the held pages n, pairs the
// free pages below n with the held ones from n on, both in order, and moves
// their refs.  remap [pages] (written only where something moves) receives the
// moved pages' new places.
__global__ __launch_bounds__(kPlan) void paged_compact_plan_kernel(Pages p, int32_t* status, int32_t* total,
                                                                   int32_t* src, int32_t* dst, int32_t* remap)
{
    __shared__ int waves[16];
    int held = 0;
    for (int base = 0; base < p.c.pages; base += kPlan * kPlanPages) {
        const PlanRefs x = plan_refs(p, base);
#pragma unroll
        for (int k = 0; k < kPlanPages; k++) held += x.r[k] > 0;
    }
    int n;
    block_scan(held, waves, &n);
    int holes = 0, movers = 0;
    for (int base = 0; base < p.c.pages; base += kPlan * kPlanPages) {
        const PlanRefs x = plan_refs(p, base);
        const int at = base + kPlanPages * (int)threadIdx.x;
        int both = 0, sum;  // holes in the low half, movers in the high (a round has 2^14 pages)
#pragma unroll
        for (int k = 0; k < kPlanPages; k++)
            both += (x.r[k] == 0 && at + k < n ? 1 : 0) + (x.r[k] > 0 && at + k >= n ? 1 << 16 : 0);
        const int before = block_scan(both, waves, &sum);
        int h = holes + (before & 0xFFFF), m = movers + (before >> 16);
        holes += sum & 0xFFFF;
        movers += sum >> 16;
#pragma unroll
        for (int k = 0; k < kPlanPages; k++) {
            if (x.r[k] == 0 && at + k < n) dst[h++] = at + k;
            if (x.r[k] > 0 && at + k >= n) src[m++] = at + k;
        }
    }
    __syncthreads();
    const int pairs = min(movers, holes);
    for (int i = threadIdx.x; i < pairs; i += kPlan) {
        const int from = src[i], to = dst[i];
        remap[from] = to;
        p.c.refs[to] = p.c.refs[from];
        p.c.refs[from] = 0;
    }
    if (threadIdx.x == 0) {
        *total = pairs;
        if (status) *status = n;
    }
}

// Second launch: the first `table_blocks` workgroups rewrite the tables, the
// others copy the pages.
__global__ __launch_bounds__(256) void paged_compact_move_kernel(Pages p, const int32_t* total, const int32_t* src,
                                                                 const int32_t* dst, const int32_t* remap,
                                                                 int table_blocks)
{
    const int n = *total;
    if (n == 0) return;
    if ((int)blockIdx.x >= table_blocks) {
        copy_pairs(p, src, dst, n, (int)blockIdx.x - table_blocks, (int)gridDim.x - table_blocks);
        return;
    }
    const int first = src[0];  // every held page from the first moved one on has moved
    for (int s = blockIdx.x; s < p.c.sequences; s += table_blocks) {
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

// Workgroups that copy up to `pairs` pages (the pairs in use may be fewer:
// each worker walks on by the number of workers).
unsigned copy_workers(const Pages& p, int64_t pairs)
{
    return (unsigned)std::min<int64_t>(std::max<int64_t>(pairs * p.c.layers * page_slices(p), 1), 8192);
}

void launch_copy(const Pages& p, const int32_t* src, const int32_t* dst, int32_t count, hipStream_t stream)
{
    hipLaunchKernelGGL(paged_copy_kernel, dim3(copy_workers(p, count)), dim3(256), 0, stream, p, src, dst, count);
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
    if (grows && count) launch_copy(p, w, w + count, count, as_stream(stream));
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
    int32_t rc = check_append(c, "append", layer, rows);
    if (rc) return rc;
    if (rows == 0) return NHIP_OK;
    NHIP_REQUIRE(d_k && d_v && d_row_seq && d_row_pos, "paged append: null pointer");
    NHIP_REQUIRE(ldk >= c->kv_heads * c->qk_dim && ldv >= c->kv_heads * c->v_dim,
                 "paged append: row strides %d, %d below a row's columns", ldk, ldv);
    rc = ensure_device();
    if (rc) return rc;
    const AppendParams p{paged_layer(c, layer), d_k, d_v, d_row_seq, d_row_pos, c->refs, ldk, ldv, rows};
    return launch_append(c, p, as_stream(stream));
}

int32_t nhip_paged_rotary_append_dev(const nhip_paged_cache* c, int32_t layer, const nhip_rotary* r, const float* d_q,
                                     int32_t ldq, int32_t heads, const float* d_k, int32_t ldk, const float* d_v,
                                     int32_t ldv, const int32_t* d_row_seq, const int32_t* d_row_pos, int32_t rows,
                                     int8_t* d_codes, float* d_q_scales, void* stream)
{
    int32_t rc = check_append(c, "rotary append", layer, rows);
    if (rc) return rc;
    rc = rotary_check(r);
    if (rc) return rc;
    NHIP_REQUIRE(r->dim <= c->qk_dim, "paged rotary append: %d of %d dimensions rotated", r->dim, c->qk_dim);
    NHIP_REQUIRE(heads >= 1 && heads <= 4096 && heads % c->kv_heads == 0,
                 "paged rotary append: %d heads on %d kv heads (a multiple, at most 4096)", heads, c->kv_heads);
    NHIP_REQUIRE(ldq >= heads * c->qk_dim && ldk >= c->kv_heads * c->qk_dim && ldv >= c->kv_heads * c->v_dim,
                 "paged rotary append: row strides %d, %d, %d below a row's columns", ldq, ldk, ldv);
    if (rows == 0) return NHIP_OK;
    NHIP_REQUIRE(d_q && d_k && d_v && d_row_seq && d_row_pos && d_codes && d_q_scales,
                 "paged rotary append: null pointer");
    NHIP_REQUIRE((reinterpret_cast<uintptr_t>(d_codes) & 3) == 0, "paged rotary append: the codes are not 4-byte aligned");
    rc = ensure_device();
    if (rc) return rc;
    const RotaryAppendParams p{{paged_layer(c, layer), d_k, d_v, d_row_seq, d_row_pos, c->refs, ldk, ldv, rows},
                               rotary_table(r), d_q, d_codes, d_q_scales, ldq, heads};
    return launch_append(c, p, as_stream(stream));
}

int32_t nhip_paged_read_dev(const nhip_paged_cache* c, int32_t layer, const int32_t* d_row_seq,
                            const int32_t* d_row_pos, int32_t rows, float* d_k, int32_t ldk, float* d_v, int32_t ldv,
                            void* stream)
{
    int32_t rc = check_append(c, "read", layer, rows);
    if (rc) return rc;
    if (rows == 0) return NHIP_OK;
    NHIP_REQUIRE(d_row_seq && d_row_pos && (d_k || d_v), "paged read: null pointer");
    NHIP_REQUIRE((!d_k || ldk >= c->kv_heads * c->qk_dim) && (!d_v || ldv >= c->kv_heads * c->v_dim),
                 "paged read: row strides %d, %d below a row's columns", ldk, ldv);
    rc = ensure_device();
    if (rc) return rc;
    const int64_t elements = (int64_t)rows * c->kv_heads * ((d_k ? c->qk_dim : 0) + (d_v ? c->v_dim : 0));
    const ReadParams p{paged_layer(c, layer), d_row_seq, d_row_pos, d_k, d_v, ldk, ldv, rows,
                       stored_away(elements, kReadAway)};
    const unsigned units = row_groups(rows) * c->kv_heads, of_one = c->v_dim <= 64 ? 4 : 2;
    const dim3 grid((units + of_one - 1) / of_one, d_k && d_v ? 2 : 1);
    if (c->qk_dim == 48)
        hipLaunchKernelGGL((paged_read_kernel<48, 64>), grid, dim3(256), 0, as_stream(stream), p);
    else if (c->qk_dim == 64)
        hipLaunchKernelGGL((paged_read_kernel<64, 64>), grid, dim3(256), 0, as_stream(stream), p);
    else
        hipLaunchKernelGGL((paged_read_kernel<128, 128>), grid, dim3(256), 0, as_stream(stream), p);
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
    launch_copy(pages_of(c), d_src, d_dst, count, as_stream(stream));
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
    // 3 rows of 12 pages take 4.1 us in one launch and 6.7 in two, 16 of 63 4.2 and 6.6, but 64 of 19 10.6 and 6.6, 8 of
    // 1875 31.8 and 11.5: one launch where a wave has one row and few rounds of it.
    if (count <= kForkThreads / 64 && c->width <= 128) {
        hipLaunchKernelGGL(paged_fork_kernel, dim3(1), dim3(kForkThreads), 0, as_stream(stream), p, d_dst, d_src,
                           d_length, count, w);
        NHIP_CHECK_HIP(hipGetLastError());
        return NHIP_OK;
    }
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
    hipLaunchKernelGGL(paged_compact_plan_kernel, dim3(1), dim3(kPlan), 0, s, p, d_status, total, src, dst, remap);
    NHIP_CHECK_HIP(hipGetLastError());
    const unsigned table_blocks = (unsigned)std::min(c->sequences, 1024);
    hipLaunchKernelGGL(paged_compact_move_kernel, dim3(table_blocks + copy_workers(p, c->pages / 2)), dim3(256), 0, s, p,
                       total, src, dst, remap, (int)table_blocks);
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

}  // extern "C"
