// paged_attention.hip -- attention over the paged int8 KV cache on gfx950.
//
// For a query (row, head) over its positions s: z_s = (q . k_s) ks_s qs /
// sqrt(qk) with the int8 dot exact, out = sum_s e^(z_s - m) vs_s v_s / sum_s
// e^(z_s - m), in one pass with a running maximum m and fp32 sums.
#include <algorithm>
#include <cmath>

#include "paged.hpp"

namespace nhip {
namespace {

constexpr float kNoScore = -1e30f;  // the running maximum before any position: finite, so that a difference is never NaN

struct PagedAttn {
    PagedLayer c;
    const int8_t* q;
    const float* q_scales;
    float* out;
    const int32_t* row_seq;
    const int32_t* row_first;
    const int32_t* row_count;
    const int32_t* run_rows;
    const int32_t* run_seq;
    const int32_t* run_pos;
    int32_t rows, heads, group, runs, window, max_count;
    float scale;  // 1 / sqrt(qk)
};

// The run that holds row r, or -1.
__device__ int run_of(const PagedAttn& p, int r)
{
    for (int i = 0; i < p.runs; i++)
        if (r >= p.run_rows[i] && r < p.run_rows[i + 1]) return i;
    return -1;
}

// One wave per (row, head): 64 positions at a time, a lane per position for
// the scores, a lane per value dimension for the sums.
template <bool PROMPT>
__global__ __launch_bounds__(64) void paged_attention_kernel(PagedAttn p)
{
    const PagedLayer& c = p.c;
    const int r = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const int kvh = h / p.group;
    const int span = c.width << c.page_shift;
    int seq, first, count;
    if constexpr (PROMPT) {
        const int run = run_of(p, r);
        if (run < 0) return;
        seq = p.run_seq[run];
        const int64_t at = (int64_t)p.run_pos[run] + (r - p.run_rows[run]);
        const bool ok = p.run_pos[run] >= 0 && at < min(span, p.max_count);
        first = ok && p.window > 0 ? max(0, (int)at - p.window + 1) : 0;
        count = ok ? (int)at + 1 - first : 0;
    } else {
        seq = p.row_seq[r];
        first = p.row_first[r];
        count = p.row_count[r];
        if (first < 0 || count < 0 || count > p.max_count || first > span - count) count = 0;
    }
    if (seq < 0 || seq >= c.sequences) count = 0;
    const int8_t* q = p.q + ((size_t)r * p.heads + h) * c.qk;
    const float qs = p.q_scales[(size_t)r * p.heads + h] * p.scale;
    float peak = kNoScore, total = 0.0f, o[2] = {0.0f, 0.0f};
    for (int base = 0; base < count; base += 64) {
        const int s = base + lane, pos = first + s;
        int page = -1;
        if (s < count) page = c.tables[(size_t)seq * c.width + (pos >> c.page_shift)];
        const bool live = page >= 0 && page < c.pages;
        const int at = pos & ((1 << c.page_shift) - 1);
        const size_t cell = live ? ((size_t)page * c.kv_heads + kvh) << c.page_shift : 0;
        float z = -INFINITY, vs = 0.0f;
        if (live) {
            int dot = 0;
            for (int d = 0; d < c.qk; d += 4)
                dot = __builtin_amdgcn_sdot4(*(const int*)(q + d), *(const int*)(c.keys + (cell + at) * c.qk + d), dot,
                                             false);
            z = (float)dot * c.kscale[cell + at] * qs;
            vs = c.vscale[cell + at];
        }
        const float up = fmaxf(peak, wave_max(z));
        const float keep = expf(peak - up);
        const float e = live ? expf(z - up) : 0.0f;
        peak = up;
        float sum = e;
        for (int off = 32; off; off >>= 1) sum += __shfl_xor(sum, off);
        total = total * keep + sum;
        o[0] *= keep;
        o[1] *= keep;
        const float w = live ? e * vs : 0.0f;
        for (int j = 0; j < 64; j++) {
            if (!__shfl((int)live, j)) continue;
            const float wj = __shfl(w, j);
            const size_t first_cell = ((size_t)(uint32_t)__shfl((int)(cell >> 32), j) << 32) | (uint32_t)__shfl((int)cell, j);
            const int aj = __shfl(at, j);
            const int8_t* v = c.values + first_cell * c.v + (size_t)(aj >> 4) * 16 * c.v + (aj & 15);
            for (int e2 = 0; e2 < 2; e2++)
                if (lane + 64 * e2 < c.v) o[e2] = fmaf(wj, (float)v[16 * (lane + 64 * e2)], o[e2]);
        }
    }
    for (int e = 0; e < 2; e++)
        if (lane + 64 * e < c.v)
            p.out[((size_t)r * p.heads + h) * c.v + lane + 64 * e] = total != 0.0f ? o[e] / total : 0.0f;
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

PagedAttn attn_params(const nhip_paged_cache* c, int32_t layer, const int8_t* q, const float* q_scales, int32_t rows,
                      int32_t heads, int32_t max_count, float* out)
{
    PagedAttn p{};
    p.c = paged_layer(c, layer);
    p.q = q;
    p.q_scales = q_scales;
    p.out = out;
    p.rows = rows;
    p.heads = heads;
    p.group = heads / c->kv_heads;
    p.max_count = max_count;
    p.scale = 1.0f / std::sqrt((float)c->qk_dim);
    return p;
}

}  // namespace
}  // namespace nhip

using namespace nhip;

extern "C" {

size_t nhip_paged_decode_workspace(const nhip_paged_cache* c, int32_t rows, int32_t heads, int32_t max_count)
{
    if (check_attention(c, rows, heads, max_count)) return 0;
    return 0;
}

int32_t nhip_paged_decode_dev(const nhip_paged_cache* c, int32_t layer, const int8_t* d_q, const float* d_q_scales,
                              int32_t rows, int32_t heads, const int32_t* d_row_seq, const int32_t* d_row_first,
                              const int32_t* d_row_count, int32_t max_count, void* d_workspace,
                              size_t workspace_bytes, float* d_out, void* stream)
{
    int32_t rc = check_attention(c, rows, heads, max_count);
    if (rc) return rc;
    if (rows == 0) return NHIP_OK;
    rc = check_call(c, layer, d_q, d_q_scales, d_out, d_workspace, workspace_bytes, 0);
    if (rc) return rc;
    NHIP_REQUIRE(d_row_seq && d_row_first && d_row_count, "paged decode: null pointer");
    rc = ensure_device();
    if (rc) return rc;
    PagedAttn p = attn_params(c, layer, d_q, d_q_scales, rows, heads, max_count, d_out);
    p.row_seq = d_row_seq;
    p.row_first = d_row_first;
    p.row_count = d_row_count;
    hipLaunchKernelGGL((paged_attention_kernel<false>), dim3(rows, heads), dim3(64), 0, as_stream(stream), p);
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

size_t nhip_paged_prompt_workspace(const nhip_paged_cache* c, int32_t rows, int32_t heads, int32_t runs,
                                   int32_t max_count)
{
    (void)runs;
    if (check_attention(c, rows, heads, max_count)) return 0;
    return 0;
}

int32_t nhip_paged_prompt_dev(const nhip_paged_cache* c, int32_t layer, const int8_t* d_q, const float* d_q_scales,
                              int32_t rows, int32_t heads, int32_t runs, const int32_t* d_run_rows,
                              const int32_t* d_run_seq, const int32_t* d_run_pos, int32_t window, int32_t max_count,
                              void* d_workspace, size_t workspace_bytes, float* d_out, void* stream)
{
    int32_t rc = check_attention(c, rows, heads, max_count);
    if (rc) return rc;
    NHIP_REQUIRE(runs >= 0 && runs <= kPagedMaxRows && window >= 0, "paged prompt: %d runs, window %d", runs, window);
    if (rows == 0 || runs == 0) return NHIP_OK;
    rc = check_call(c, layer, d_q, d_q_scales, d_out, d_workspace, workspace_bytes, 0);
    if (rc) return rc;
    NHIP_REQUIRE(d_run_rows && d_run_seq && d_run_pos, "paged prompt: null pointer");
    rc = ensure_device();
    if (rc) return rc;
    PagedAttn p = attn_params(c, layer, d_q, d_q_scales, rows, heads, max_count, d_out);
    p.run_rows = d_run_rows;
    p.run_seq = d_run_seq;
    p.run_pos = d_run_pos;
    p.runs = runs;
    p.window = window;
    hipLaunchKernelGGL((paged_attention_kernel<true>), dim3(rows, heads), dim3(64), 0, as_stream(stream), p);
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

}  // extern "C"
