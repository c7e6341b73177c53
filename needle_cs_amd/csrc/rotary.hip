// rotary.hip -- rotary positions on gfx950: tables of cos and sin, and heads
// rotated by them (with the cache's append in paged.hip).
#include <algorithm>
#include <cmath>

#include "rotary.hpp"
#include "stores.hpp"

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

// A workgroup takes kSpan positions and 32 frequencies.  The cos and sin of
// first + 16 a + b are one complex product of those of first + 16 a and b, all
// in 64 bits: 24 of either for 128 positions instead of 128, and an error of
// three roundings of 2^-53 more.  131,072 positions of 64 pairs, 67 MB to be written:
// 14.0 us, 4.8 TB/s; 32.2 with a cos and sin for each.
constexpr int kCoarse = 8, kFine = 16, kSpan = kCoarse * kFine;
__global__ __launch_bounds__(256) void rotary_table_kernel(TableParams p)
{
    __shared__ double2 steps[kCoarse + kFine][32];  // cos, sin
    const int lane = threadIdx.x & 31, i = blockIdx.y * 32 + lane;
    const int64_t base = (int64_t)blockIdx.x * kSpan;
    const double f = p.f[min(i, p.half - 1)];
    for (int k = threadIdx.x / 32; k < kCoarse + kFine; k += 8) {
        const bool coarse = k < kCoarse;
        double s, c;
        sincos((coarse ? (double)(p.first + base + kFine * k) : (double)(k - kCoarse)) * f, &s, &c);
        const double scale = coarse ? p.magnitude : 1.0;
        steps[k][lane] = make_double2(c * scale, s * scale);
    }
    __syncthreads();
    if (i >= p.half) return;
    for (int k = threadIdx.x / 32; k < kSpan && base + k < p.count; k += 8) {
        const double2 x = steps[k / kFine][lane], y = steps[kCoarse + k % kFine][lane];
        const size_t at = (size_t)(base + k) * p.half + i;
        p.cos[at] = (float)fma(x.x, y.x, -(x.y * y.y));
        p.sin[at] = (float)fma(x.y, y.x, x.x * y.y);
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
    bool away;
};

// L threads a head, a unit each, and further heads of the row in turn, so that
// a unit's cos and sin are read once a row.  Bytes bound it: 8185 rows of 40 heads
// of 128 with 64 dimensions rotated, 337 MB read and written, take 57.6 us, 5.9
// TB/s (113 with a pair a thread, whose accesses are 4 bytes wide; 63.6 with two
// neighbouring fours a lane for neighbouring pairs, by ordinary stores 62.3); 3 rows of 12
// heads 2 us beside a launch.
constexpr int kHeadsAhead = 4;  // loads in flight
template <int L>
__global__ __launch_bounds__(256) void rotate_kernel(RotateParams p)
{
    const int units = p.head_dim / 8, slot = threadIdx.x / L;
    for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const int pos = p.row_pos[row];
        if (pos < 0 || pos >= p.r.positions) continue;
        const float* from = p.x + (size_t)row * p.ldx;
        float* to = p.y + (size_t)row * p.ldy;
        for (int u = threadIdx.x % L; u < units; u += L) {
            const RotaryUnit unit = rotary_unit<false>(p.r, p.head_dim, u, pos);
            for (int h0 = slot; h0 < p.heads; h0 += kHeadsAhead * (256 / L)) {
                rotary_f4 a[kHeadsAhead], b[kHeadsAhead];
#pragma unroll
                for (int k = 0; k < kHeadsAhead; k++) {
                    const float* head = from + min(h0 + k * (256 / L), p.heads - 1) * p.head_dim;
                    a[k] = *reinterpret_cast<const rotary_f4*>(head + unit.a);
                    b[k] = *reinterpret_cast<const rotary_f4*>(head + unit.b);
                }
#pragma unroll
                for (int k = 0; k < kHeadsAhead; k++) {
                    const int h = h0 + k * (256 / L);
                    if (h >= p.heads) break;
                    rotate_unit<false>(p.r, unit, nullptr, a[k], b[k]);
                    store_f4(to + h * p.head_dim + unit.a, a[k], p.away);
                    store_f4(to + h * p.head_dim + unit.b, b[k], p.away);
                }
            }
        }
    }
}

// Dimensions that are no multiple of 8, where a unit of four pairs would pass
// them: a thread takes a pair or, behind them, an element that stays, by accesses
// of 4 bytes, which bound it: 8000 rows of 40 heads of 80 with 20 rotated 85 us, 2.4
// TB/s (41 by the other kernel with 24 rotated), of 64 heads of 50 67.
__global__ __launch_bounds__(256) void rotate_pairs_kernel(RotateParams p)
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

template <int L>
void launch_rotate(const RotateParams& p, hipStream_t stream)
{
    hipLaunchKernelGGL((rotate_kernel<L>), dim3(p.rows), dim3(256), 0, stream, p);
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
    hipLaunchKernelGGL(rotary_table_kernel, dim3((count + kSpan - 1) / kSpan, (p.half + 31) / 32), dim3(256), 0,
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
    const RotateParams p = {rotary_table(r), d_x, d_row_pos, d_y, ldx, ldy, heads, head_dim, rows,
                            stored_away((int64_t)rows * heads * head_dim, kReadAway)};
    hipStream_t st = as_stream(stream);
    if (r->dim % 8 || head_dim % 8)
        hipLaunchKernelGGL(rotate_pairs_kernel, dim3(rows), dim3(256), 0, st, p);
    else if (head_dim <= 64)
        launch_rotate<8>(p, st);
    else if (head_dim <= 128)
        launch_rotate<16>(p, st);
    else
        launch_rotate<32>(p, st);
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

}  // extern "C"
