// rotary.hip -- rotary positions on gfx950: tables of cos and sin, and heads
// rotated by them (with the cache's append in paged.hip).
#include <algorithm>
#include <cmath>

#include "rotary.hpp"

namespace nhip {

int32_t rotary_check(const nhip_rotary* r)
{
    NHIP_REQUIRE(r, "rotary: NULL");
    NHIP_REQUIRE(r->dim >= 2 && r->dim <= kRotaryMaxDim && r->dim % 2 == 0,
                 "rotary: %d dimensions are not an even number up to %d", r->dim, kRotaryMaxDim);
    NHIP_REQUIRE(r->positions >= 1 && r->positions <= (1 << 30), "rotary: %d positions out of range", r->positions);
    NHIP_REQUIRE(r->interleaved == 0 || r->interleaved == 1, "rotary: interleaved %d", r->interleaved);
    NHIP_REQUIRE(r->cos && r->sin, "rotary: null table");
    return NHIP_OK;
}

namespace {

// ----------------------------------------------------------------- table --

struct TableParams {
    float* cos;
    float* sin;
    int32_t first, count, half;
    double magnitude;
    double f[kRotaryMaxDim / 2];
};

__global__ __launch_bounds__(256) void rotary_table_kernel(TableParams p)
{
    const size_t n = (size_t)p.count * p.half;
    for (size_t at = (size_t)blockIdx.x * 256 + threadIdx.x; at < n; at += (size_t)gridDim.x * 256) {
        const size_t row = at / p.half;
        double s, c;
        sincos((double)(p.first + (int)row) * p.f[at - row * p.half], &s, &c);
        p.cos[at] = (float)(c * p.magnitude);
        p.sin[at] = (float)(s * p.magnitude);
    }
}

void frequencies(const nhip_rotary_scaling& s, int dim, double* f)
{
    const double tau = 6.283185307179586;
    const double theta = s.kind == NHIP_ROTARY_BASE ? s.theta * std::pow(s.factor, dim / (dim - 2.0)) : s.theta;
    auto place = [&](double turns) { return dim * std::log(s.original / (tau * turns)) / (2.0 * std::log(s.theta)); };
    double lo = 0.0, hi = 0.0;
    if (s.kind == NHIP_ROTARY_PARTS) {
        lo = std::max(std::floor(place(s.high)), 0.0);
        hi = std::min(std::ceil(place(s.low)), dim - 1.0);
        if (hi == lo) hi = lo + 0.001;
    }
    for (int i = 0; i < dim / 2; i++) {
        const double plain = std::pow(theta, -2.0 * i / dim);
        f[i] = plain;
        if (s.kind == NHIP_ROTARY_LINEAR) f[i] = plain / s.factor;
        if (s.kind == NHIP_ROTARY_PARTS) {
            const double r = std::min(std::max((i - lo) / (hi - lo), 0.0), 1.0);
            f[i] = plain / s.factor * r + plain * (1.0 - r);
        }
        if (s.kind == NHIP_ROTARY_BANDS) {
            const double r = std::min(std::max((s.original * plain / tau - s.low) / (s.high - s.low), 0.0), 1.0);
            f[i] = plain / s.factor * (1.0 - r) + plain * r;
        }
    }
}

int32_t check_scaling(const nhip_rotary_scaling* s, int32_t dim)
{
    NHIP_REQUIRE(s, "rotary table: NULL scaling");
    NHIP_REQUIRE(s->kind >= NHIP_ROTARY_PLAIN && s->kind <= NHIP_ROTARY_BANDS, "rotary table: scaling kind %d", s->kind);
    NHIP_REQUIRE(s->theta > 1.0 && s->theta <= 1e12, "rotary table: theta %g is not in (1, 1e12]", s->theta);
    NHIP_REQUIRE(s->magnitude > 0.0 && s->magnitude <= 1e6, "rotary table: magnitude %g is not in (0, 1e6]",
                 s->magnitude);
    NHIP_REQUIRE(s->kind == NHIP_ROTARY_PLAIN || (s->factor >= 1.0 && s->factor <= 1e6),
                 "rotary table: factor %g is not in [1, 1e6]", s->factor);
    NHIP_REQUIRE(s->kind != NHIP_ROTARY_BASE || dim > 2, "rotary table: a scaled base needs more than 2 dimensions");
    NHIP_REQUIRE(s->kind < NHIP_ROTARY_PARTS || (s->low > 0.0 && s->high > s->low && s->high <= 1e9 &&
                                                 s->original > 0.0 && s->original <= 1e9),
                 "rotary table: low %g, high %g, original %g (0 < low < high, original > 0)", s->low, s->high,
                 s->original);
    return NHIP_OK;
}

// ---------------------------------------------------------------- rotate --

struct RotateParams {
    RotaryTable r;
    const float* x;
    const int32_t* row_pos;
    float* y;
    int32_t ldx, ldy, heads, head_dim, rows;
};

// A thread takes a pair or, behind them, an element that stays.
__global__ __launch_bounds__(256) void rotate_kernel(RotateParams p)
{
    const int half = p.r.dim / 2, units = half + p.head_dim - p.r.dim;
    const int n = p.heads * units;
    for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const int pos = p.row_pos[row];
        if (pos < 0 || pos >= p.r.positions) continue;
        const float* c = p.r.cos + (size_t)pos * half;
        const float* s = p.r.sin + (size_t)pos * half;
        for (int at = threadIdx.x; at < n; at += 256) {
            const int head = at / units, u = at - head * units;
            const float* from = p.x + (size_t)row * p.ldx + head * p.head_dim;
            float* to = p.y + (size_t)row * p.ldy + head * p.head_dim;
            if (u >= half) {
                to[u + half] = from[u + half];
            } else {
                const int a = p.r.interleaved ? 2 * u : u, b = p.r.interleaved ? 2 * u + 1 : u + half;
                const float x0 = from[a], x1 = from[b];
                to[a] = x0 * c[u] - x1 * s[u];
                to[b] = x1 * c[u] + x0 * s[u];
            }
        }
    }
}

}  // namespace
}  // namespace nhip

using namespace nhip;

extern "C" {

int32_t nhip_rotary_table_dev(float* d_cos, float* d_sin, int32_t first, int32_t count, int32_t dim,
                              const nhip_rotary_scaling* scaling, void* stream)
{
    NHIP_REQUIRE(dim >= 2 && dim <= kRotaryMaxDim && dim % 2 == 0,
                 "rotary table: %d dimensions are not an even number up to %d", dim, kRotaryMaxDim);
    NHIP_REQUIRE(first >= 0 && count >= 0 && (int64_t)first + count <= (1 << 30),
                 "rotary table: positions %d to %d + %d out of range", first, first, count);
    int32_t rc = check_scaling(scaling, dim);
    if (rc) return rc;
    if (count == 0) return NHIP_OK;
    NHIP_REQUIRE(d_cos && d_sin, "rotary table: null pointer");
    rc = ensure_device();
    if (rc) return rc;
    TableParams p;
    p.cos = d_cos;
    p.sin = d_sin;
    p.first = first;
    p.count = count;
    p.half = dim / 2;
    p.magnitude = scaling->magnitude;
    frequencies(*scaling, dim, p.f);
    const size_t n = (size_t)count * p.half;
    hipLaunchKernelGGL(rotary_table_kernel, dim3((unsigned)std::min<size_t>((n + 255) / 256, 1 << 20)), dim3(256), 0,
                       as_stream(stream), p);
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

int32_t nhip_rotary_dev(const nhip_rotary* r, const float* d_x, int32_t ldx, int32_t heads, int32_t head_dim,
                        const int32_t* d_row_pos, int32_t rows, float* d_y, int32_t ldy, void* stream)
{
    int32_t rc = rotary_check(r);
    if (rc) return rc;
    NHIP_REQUIRE(rows >= 0 && rows <= kRotaryMaxRows, "rotary: %d rows", rows);
    NHIP_REQUIRE(head_dim >= r->dim && head_dim <= 4096, "rotary: heads of %d dimensions, %d of them rotated", head_dim,
                 r->dim);
    NHIP_REQUIRE(heads >= 1 && (int64_t)heads * head_dim <= (1 << 24), "rotary: %d heads of %d", heads, head_dim);
    NHIP_REQUIRE(ldx >= heads * head_dim && ldy >= heads * head_dim, "rotary: strides %d, %d are less than %d columns",
                 ldx, ldy, heads * head_dim);
    if (rows == 0) return NHIP_OK;
    NHIP_REQUIRE(d_x && d_row_pos && d_y, "rotary: null pointer");
    NHIP_REQUIRE(d_y != d_x || ldy == ldx, "rotary: heads rotated in place have their rows' stride");
    rc = ensure_device();
    if (rc) return rc;
    const RotateParams p = {rotary_table(r), d_x, d_row_pos, d_y, ldx, ldy, heads, head_dim, rows};
    hipLaunchKernelGGL(rotate_kernel, dim3(rows), dim3(256), 0, as_stream(stream), p);
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

}  // extern "C"
