// rows.hip -- row operations between a layer's int8 products on gfx950: the
// residual's addition with the root-mean-square norm and QuantizeInt8, and
// rows of codes back to numbers.
#include <algorithm>

#include "common.hpp"
#include "stores.hpp"

namespace nhip {
namespace {

constexpr int32_t kMaxRows = 1 << 26, kMaxCols = 1 << 20;
constexpr int kMaxGroups = 1 << 20;  // workgroups of a launch; they take the further rows in turn

typedef uint32_t u32_bytes __attribute__((aligned(1)));

// Elements i .. i + 3 of a row of n, 0 past its end.
__device__ __forceinline__ float4 load4(const float* row, int i, int n)
{
    if (i + 4 <= n) {
        const f4 v = *reinterpret_cast<const f4*>(row + i);
        return make_float4(v[0], v[1], v[2], v[3]);
    }
    return make_float4(i < n ? row[i] : 0.0f, i + 1 < n ? row[i + 1] : 0.0f, i + 2 < n ? row[i + 2] : 0.0f, 0.0f);
}
__device__ __forceinline__ void store4(float* row, int i, int n, float4 v, bool away)
{
    if (i + 4 <= n) {
        store_f4(row + i, f4{v.x, v.y, v.z, v.w}, away);
        return;
    }
    if (i < n) row[i] = v.x;
    if (i + 1 < n) row[i + 1] = v.y;
    if (i + 2 < n) row[i + 2] = v.z;
}
__device__ __forceinline__ void store_codes4(int8_t* row, int i, int n, uint32_t codes)
{
    if (i + 4 <= n) {
        *reinterpret_cast<u32_bytes*>(row + i) = codes;
        return;
    }
    for (int e = 0; e < 3 && i + e < n; e++) row[i + e] = (int8_t)(codes >> (8 * e));
}

struct NormParams {
    const float* x;
    const float* delta;
    const float* gain;
    float* sum;
    int8_t* q;
    float* scales;
    int32_t ldx, ldd, lds, rows, cols, zero_centered;
    float eps;
    double inverse_cols;
    bool away;
};

__device__ __forceinline__ float4 gain4(const NormParams& p, int i)
{
    if (!p.gain) return make_float4(1.0f, 1.0f, 1.0f, 1.0f);
    float4 g = load4(p.gain, i, p.cols);
    if (p.zero_centered) g = make_float4(1.0f + g.x, 1.0f + g.y, 1.0f + g.z, 1.0f + g.w);
    return g;
}

__device__ __forceinline__ float4 sum4(const NormParams& p, size_t row, int i)
{
    float4 v = load4(p.x + row * p.ldx, i, p.cols);
    if (p.delta) {
        const float4 d = load4(p.delta + row * p.ldd, i, p.cols);
        v = make_float4(v.x + d.x, v.y + d.y, v.z + d.z, v.w + d.w);
    }
    return v;
}

__device__ __forceinline__ double squares4(float4 v, double s)
{
    s = fma((double)v.x, (double)v.x, s);
    s = fma((double)v.y, (double)v.y, s);
    s = fma((double)v.z, (double)v.z, s);
    return fma((double)v.w, (double)v.w, s);
}

__device__ __forceinline__ float4 normed4(float4 v, float r, float4 g)
{
    return make_float4((v.x * r) * g.x, (v.y * r) * g.y, (v.z * r) * g.z, (v.w * r) * g.w);
}

__device__ __forceinline__ float peak4(float m, float4 v)
{
    return fmaxf(fmaxf(m, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
}

template <int S>
__device__ __forceinline__ double add_lane_xor(double v)
{
    return v + __hiloint2double((int)lane_xor<S>((uint32_t)__double2hiint(v)),
                                (int)lane_xor<S>((uint32_t)__double2loint(v)));
}

// The sum and the maximum over the T threads of a row, in every thread.  (A
// row's two uses alternate, each behind a barrier of its own.)
template <int T>
__device__ __forceinline__ double row_sum(double v, double* lds)
{
    if constexpr (T > 32) v = add_lane_xor<32>(v);
    if constexpr (T > 16) v = add_lane_xor<16>(v);
    v = add_lane_xor<1>(add_lane_xor<2>(add_lane_xor<4>(add_lane_xor<8>(v))));
    if constexpr (T > 64) {
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0;
        for (int w = 0; w < T / 64; w++) v += lds[w];
    }
    return v;
}
template <int T>
__device__ __forceinline__ float row_max(float v, float* lds)
{
    if constexpr (T > 32) v = fmaxf(v, lane_xor<32>(v));
    if constexpr (T > 16) v = fmaxf(v, lane_xor<16>(v));
    v = fmaxf(v, lane_xor<8>(v));
    v = fmaxf(v, lane_xor<4>(v));
    v = fmaxf(v, lane_xor<2>(v));
    v = fmaxf(v, lane_xor<1>(v));
    if constexpr (T > 64) {
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = lds[0];
        for (int w = 1; w < T / 64; w++) v = fmaxf(v, lds[w]);
    }
    return v;
}

__device__ __forceinline__ float inverse_rms(const NormParams& p, double squares)
{
    return (float)rsqrt(squares * p.inverse_cols + (double)p.eps);
}

__device__ __forceinline__ float scale_of(float peak) { return peak > 0.0f ? peak / 127.0f : 1.0f; }

// T threads a row, which they hold in registers, G groups of four elements
// each: it is read once and written once (13 bytes an element with the addition
// and the sums; 4099 rows of 4096, 218 MB, take 34 us, 6.4 TB/s, where the last
// cache has a part of them, and 57.2 with 84 MB that read the codes back behind
// them, 5.3 TB/s of 302 MB, where it has none).  What a group's
// code costs shows where there are few rows, also where no element is left for
// it: 3 rows of 512 with a wave take 4.1 us by G = 4, 3.4 by 2.
template <int T, int G>
__global__ __launch_bounds__(T < 256 ? 256 : T) void add_rms_quantize_kernel(NormParams p)
{
    constexpr int WG = T < 256 ? 256 : T;
    __shared__ double sums[WG / 64];
    __shared__ float peaks[WG / 64];
    const int t = threadIdx.x % T;
    for (size_t row = (size_t)blockIdx.x * (WG / T) + threadIdx.x / T; row < (size_t)p.rows;
         row += (size_t)gridDim.x * (WG / T)) {
        float4 v[G], g[G];
        double squares = 0.0;
#pragma unroll
        for (int j = 0; j < G; j++) v[j] = sum4(p, row, 4 * (t + T * j));
#pragma unroll
        for (int j = 0; j < G; j++) g[j] = gain4(p, 4 * (t + T * j));
#pragma unroll
        for (int j = 0; j < G; j++) squares = squares4(v[j], squares);
        if (p.sum) {
#pragma unroll
            for (int j = 0; j < G; j++) store4(p.sum + row * p.lds, 4 * (t + T * j), p.cols, v[j], p.away);
        }
        const float r = inverse_rms(p, row_sum<T>(squares, sums));
        float peak = 0.0f;
#pragma unroll
        for (int j = 0; j < G; j++) {
            v[j] = normed4(v[j], r, g[j]);
            peak = peak4(peak, v[j]);
        }
        const float scale = scale_of(row_max<T>(peak, peaks)), inverse = 1.0f / scale;
#pragma unroll
        for (int j = 0; j < G; j++)
            store_codes4(p.q + row * p.cols, 4 * (t + T * j), p.cols, ref_quantize4(v[j], inverse));
        if (t == 0) p.scales[row] = scale;
    }
}

// Rows of any length, by T threads, read for each of the three passes: from the
// sums, where they are kept (x may be the same memory).  The second and third come
// from the caches in part: 1024 rows of 20001 columns with the sums 80 us, 3.3 TB/s
// of what has to move (of 16384 columns, held in registers, 47, 4.7 TB/s), 256 rows
// of 65536 67, 3 of 20001 10.3.
template <int T>
__global__ __launch_bounds__(T) void add_rms_quantize_long_kernel(NormParams p)
{
    __shared__ double sums[T / 64];
    __shared__ float peaks[T / 64];
    const int first = 4 * threadIdx.x;
    for (size_t row = blockIdx.x; row < (size_t)p.rows; row += gridDim.x) {
        double squares = 0.0;
        for (int i = first; i < p.cols; i += 4 * T) {
            const float4 v = sum4(p, row, i);
            squares = squares4(v, squares);
            if (p.sum) store4(p.sum + row * p.lds, i, p.cols, v, p.away);
        }
        const float r = inverse_rms(p, row_sum<T>(squares, sums));
        auto again = [&](int i) {
            return normed4(p.sum ? load4(p.sum + row * p.lds, i, p.cols) : sum4(p, row, i), r, gain4(p, i));
        };
        float peak = 0.0f;
        for (int i = first; i < p.cols; i += 4 * T) peak = peak4(peak, again(i));
        const float scale = scale_of(row_max<T>(peak, peaks)), inverse = 1.0f / scale;
        for (int i = first; i < p.cols; i += 4 * T)
            store_codes4(p.q + row * p.cols, i, p.cols, ref_quantize4(again(i), inverse));
        if (threadIdx.x == 0) p.scales[row] = scale;
    }
}

// The fewest groups that hold a row, by as many threads as have four elements
// each; more rows than there are CUs keep more elements a thread.  us, 3 rows
// and 8192 rows: 512 columns <256, 1> 3.1 and 15.8, <64, 2> 3.4 and 11.3 (equal
// for 512 rows); 1024 columns <256, 1> 3.2 and 21.9, <64, 4> 4.2 and 19.6 (equal
// for 2048 rows); 4096 columns <1024, 1> 4.3 and 91, <256, 4> 4.7 and 87 (5.3
// and 5.6 for 256 rows, 7.0 and 6.8 for 512).  200,000 rows of 48 columns:
// 25 us by 16 threads, 72 by 64.
template <int T, int G>
void launch_norm(const NormParams& p, hipStream_t stream)
{
    constexpr int WG = T < 256 ? 256 : T, ROWS = WG / T;
    hipLaunchKernelGGL((add_rms_quantize_kernel<T, G>), dim3(std::min((p.rows + ROWS - 1) / ROWS, kMaxGroups)), dim3(WG),
                       0, stream, p);
}

// L lanes a row, of four elements each: as few as the row has for rows of up to
// 64 columns (200,000 of 48: 9.8 us with 16 lanes, 13.8 with 32), then few enough
// (8192 rows of 256: 3.9 with 32, 5.4 with 256; of 512: 5.4 with 64, 6.2 with 256;
// of 1024: 8.5 with 64, 8.3 with 256).  Bytes bound it: 262,000 rows of 128
// columns, 34 MB read and 134 written, 24.6 us, 6.8 TB/s.
template <int L>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(const int8_t* q, const float* scales, int rows, int cols,
                                                             float* x, int ldx, bool away)
{
    const int l = threadIdx.x % L;
    for (size_t row = (size_t)blockIdx.x * (256 / L) + threadIdx.x / L; row < (size_t)rows;
         row += (size_t)gridDim.x * (256 / L)) {
        const float scale = scales[row];
        const int8_t* from = q + row * cols;
        for (int i = 4 * l; i < cols; i += 4 * L) {
            uint32_t c = 0;
            if (i + 4 <= cols)
                c = *reinterpret_cast<const u32_bytes*>(from + i);
            else
                for (int e = 0; i + e < cols; e++) c |= (uint32_t)(uint8_t)from[i + e] << (8 * e);
            store4(x + row * ldx, i, cols,
                   make_float4((float)(int8_t)c * scale, (float)(int8_t)(c >> 8) * scale,
                               (float)(int8_t)(c >> 16) * scale, (float)(int8_t)(c >> 24) * scale),
                   away);
        }
    }
}

template <int L>
void launch_dequantize(const int8_t* q, const float* scales, int rows, int cols, float* x, int ldx, hipStream_t stream)
{
    hipLaunchKernelGGL((dequantize_rows_kernel<L>), dim3(std::min((rows + 256 / L - 1) / (256 / L), kMaxGroups)),
                       dim3(256), 0, stream, q, scales, rows, cols, x, ldx,
                       stored_away((int64_t)rows * cols, kSumsAway));
}

int32_t check_rows(const char* what, int32_t rows, int32_t cols)
{
    NHIP_REQUIRE(rows >= 0 && rows <= kMaxRows && cols >= 1 && cols <= kMaxCols, "%s: %d rows of %d out of range", what,
                 rows, cols);
    return NHIP_OK;
}

}  // namespace
}  // namespace nhip

using namespace nhip;

extern "C" {

int32_t nhip_add_rms_quantize_dev(const float* d_x, int32_t ldx, const float* d_delta, int32_t ldd,
                                  const float* d_gain, int32_t zero_centered, float eps, int32_t rows, int32_t cols,
                                  float* d_sum, int32_t ld_sum, int8_t* d_q, float* d_scales, void* stream)
{
    int32_t rc = check_rows("add_rms_quantize", rows, cols);
    if (rc) return rc;
    NHIP_REQUIRE(ldx >= cols && (!d_delta || ldd >= cols) && (!d_sum || ld_sum >= cols),
                 "add_rms_quantize: strides %d, %d, %d are less than %d columns", ldx, ldd, ld_sum, cols);
    NHIP_REQUIRE(eps > 0.0f && eps <= 1.0f, "add_rms_quantize: eps %g is not in (0, 1]", (double)eps);
    NHIP_REQUIRE(zero_centered == 0 || zero_centered == 1, "add_rms_quantize: zero_centered %d", zero_centered);
    if (rows == 0) return NHIP_OK;
    NHIP_REQUIRE(d_x && d_q && d_scales, "add_rms_quantize: null pointer");
    NHIP_REQUIRE((d_sum != d_x || ld_sum == ldx) && (!d_sum || d_sum != d_delta || ld_sum == ldd),
                 "add_rms_quantize: sums in place have their rows' stride");
    rc = ensure_device();
    if (rc) return rc;
    const NormParams p = {d_x,      d_delta, d_gain, d_sum, d_q,  d_scales, ldx,
                          ldd, ld_sum,  rows,   cols,  zero_centered, eps, 1.0 / cols,
                          stored_away((int64_t)rows * cols, kSumsAway)};
    hipStream_t s = as_stream(stream);
    if (cols <= 64)
        launch_norm<16, 1>(p, s);
    else if (cols <= 128)
        launch_norm<32, 1>(p, s);
    else if (cols <= 256)
        launch_norm<64, 1>(p, s);
    else if (cols <= 1024 && rows <= 512)
        launch_norm<256, 1>(p, s);
    else if (cols <= 512)
        launch_norm<64, 2>(p, s);
    else if (cols <= 1024)
        launch_norm<64, 4>(p, s);
    else if (cols <= 2048)
        launch_norm<256, 2>(p, s);
    else if (cols <= 4096 && rows <= 256)
        launch_norm<1024, 1>(p, s);
    else if (cols <= 4096)
        launch_norm<256, 4>(p, s);
    else if (cols <= 8192)
        launch_norm<1024, 2>(p, s);
    else if (cols <= 16384)
        launch_norm<1024, 4>(p, s);
    else
        hipLaunchKernelGGL((add_rms_quantize_long_kernel<1024>), dim3(std::min(rows, kMaxGroups)), dim3(1024), 0, s, p);
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

int32_t nhip_dequantize_rows_dev(const int8_t* d_q, const float* d_scales, int32_t rows, int32_t cols, float* d_x,
                                 int32_t ldx, void* stream)
{
    int32_t rc = check_rows("dequantize_rows", rows, cols);
    if (rc) return rc;
    NHIP_REQUIRE(ldx >= cols, "dequantize_rows: stride %d is less than %d columns", ldx, cols);
    if (rows == 0) return NHIP_OK;
    NHIP_REQUIRE(d_q && d_scales && d_x, "dequantize_rows: null pointer");
    rc = ensure_device();
    if (rc) return rc;
    hipStream_t s = as_stream(stream);
    if (cols <= 64)
        launch_dequantize<16>(d_q, d_scales, rows, cols, d_x, ldx, s);
    else if (cols <= 128)
        launch_dequantize<32>(d_q, d_scales, rows, cols, d_x, ldx, s);
    else if (cols <= 512)
        launch_dequantize<64>(d_q, d_scales, rows, cols, d_x, ldx, s);
    else
        launch_dequantize<256>(d_q, d_scales, rows, cols, d_x, ldx, s);
    NHIP_CHECK_HIP(hipGetLastError());
    return NHIP_OK;
}

}  // extern "C"
