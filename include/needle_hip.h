/*
 * needle_hip.h -- C ABI of libneedle_hip.so, the MI355X (gfx950) quantized
 * decode hot path of needle-cs.
 *
 * Two groups of entry points:
 *
 *  1. Kernel-table entries.  Same signatures and semantics as the reference's
 *     cdecl KernelTable slots (src/Needle/Kernels/KernelTable.cs:6-47, filled
 *     by src/Needle/Kernels/Net10KernelExports.cs:118-150): host pointers,
 *     synchronous, void (the reference has no error channel), rows outside
 *     [rowStart,rowEnd) untouched, tokens == 0 or an empty range a no-op.
 *     Weights are resolved to device-resident copies through a host-pointer ->
 *     device-pointer cache filled on first use, so a model's weights cross
 *     PCIe once.  A failure leaves the outputs untouched and sets
 *     nhip_last_error().
 *
 *  2. Device-resident API (the performance path).  Weights are uploaded once
 *     and stay in HBM; activations, outputs and KV caches are device pointers;
 *     every call is asynchronous on the given stream (NULL = the library's
 *     default stream) and returns 0 on success or a negative nhip_status.
 *
 * Every struct below matches the reference's C# sequential layout on x86-64
 * (natural alignment, 8-byte pointers).
 */
#ifndef NEEDLE_HIP_H
#define NEEDLE_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------ status ---- */

typedef enum nhip_status {
    NHIP_OK = 0,
    NHIP_ERR_ARG = -1,      /* invalid argument (shape, range, null pointer) */
    NHIP_ERR_HIP = -2,      /* a HIP runtime call failed */
    NHIP_ERR_NODEV = -3,    /* no usable gfx950 device */
    NHIP_ERR_FORMAT = -4,   /* malformed .cact archive */
    NHIP_ERR_CAPACITY = -5, /* KV capacity or slot count exceeded */
    NHIP_ERR_UNSUPPORTED = -6
} nhip_status;

/* Text of the last error on the calling thread ("" if none). */
const char* nhip_last_error(void);
/* Library and device description, e.g. "needle_hip 0.1 gfx950 (256 CUs)". */
const char* nhip_describe(void);

/* --------------------------------------------- reference struct layouts */

/* src/Needle/Model.cs:36-42 (Codebook: 100 bytes) */
typedef struct nhip_codebook {
    float levels[16];
    uint8_t bytes[32];
    float byte_scale;
} nhip_codebook;

/* src/Needle/Model.cs:8-34 (Cq: codebook-quantized weight view, 40 bytes).
 * indices: rows x (cols*bits/8) bytes; norms: fp16 [rows][cols/128]. */
typedef struct nhip_cq {
    const uint8_t* indices;
    const uint16_t* norms;
    const nhip_codebook* book;
    int32_t rows, cols, bits;
} nhip_cq;

/* src/Needle/Quant.cs:11-28 (Activations, 40 bytes).  values: int8
 * [tokens][cols] in planes order; scales/offsets: fp32 [tokens][stride],
 * stride = roundup8(cols/128). */
typedef struct nhip_activations {
    int8_t* values;
    float* scales;
    float* offsets;
    int32_t cols, groups, stride;
} nhip_activations;

/* src/Needle/Blocks.cs:11-27 (AttentionTile, 128 bytes) */
typedef struct nhip_attn_tile {
    const int8_t* queries;
    const float* query_scales;
    int32_t heads;
    const int8_t* keys;
    const float* key_scales;
    const int8_t* values;
    const float* value_scales;
    int32_t key_stride, value_stride, scale_stride, first, count;
    float* scores;
    float* output;
    float* probabilities;
    int32_t probability_stride;
    float* peaks;
    float* sums;
} nhip_attn_tile;

/* ------------------------------------------------- kernel-table entries */

/* Replaces slot 0, Quant.MatMulRows (src/Needle/Quant.cs:615-633; scalar
 * semantics src/Needle/Scalar.cs:146-192).  Results are bit-identical to the
 * reference's scalar kernel. */
void nhip_matmul_rows(const nhip_cq* w, const nhip_activations* a, int32_t tokens, float* y,
                      int32_t ldy, int32_t row_start, int32_t row_end);

/* Replaces slot 1, Quant.Prepare (src/Needle/Quant.cs:439-502; scalar branch
 * Quant.cs:473-488): per 128-group Walsh-Hadamard, int8 quantization,
 * planes permutation and offsets 63*sum(q). */
void nhip_prepare(float* x, int32_t tokens, int32_t cols, int32_t bits, const nhip_activations* a);

/* Replaces slot 3, Attention.Run (src/Needle/Blocks.cs:65-84; scalar
 * src/Needle/Scalar.cs:290-321).  With peaks/sums set, writes the
 * un-normalised partial (output, peak, sum per head) as the position-split
 * path expects (Blocks.cs:188-199, 950-958). */
void nhip_attention_tile(const nhip_attn_tile* tile);

/* Replaces slot 4, Attention.MergePartials (src/Needle/Blocks.cs:750-817). */
void nhip_merge_partials(const float* partials, int32_t count, int32_t heads, float* output);

/* Replaces slot 22, Quant.QuantizeInt8 (src/Needle/Quant.cs:103-132;
 * scalar src/Needle/Scalar.cs:67-74).  Returns the scale. */
float nhip_quantize_int8(const float* x, int32_t n, int8_t* destination);

/* The kernel-table entries above return void, as the reference's do: a
 * failure (no device, a HIP error, an argument the reference's caller would
 * have rejected) leaves the outputs untouched and sets nhip_last_error(), so
 * a host installs the table only after a probe call leaves nhip_last_error()
 * empty.  Weights are looked up in a cache by their view's host pointers and
 * shape; nhip_table_release drops every cached device copy whose index
 * pointer lies in [base, base + bytes) (all of them when base is NULL) and
 * frees its HBM -- call it when the host disposes of the model that owns
 * those bytes (Model.Dispose), with no entry running on its weights, so that
 * a later model mapped at the same addresses is uploaded afresh.
 * nhip_table_cached reports the cached entries and their HBM bytes. */
int32_t nhip_table_release(const void* base, size_t bytes, int32_t* released);
int32_t nhip_table_cached(int32_t* entries, size_t* device_bytes);

/* Mirror of Net10KernelExports.Fill (src/Needle/Kernels/Net10KernelExports.cs:118-150):
 * writes this library's entries into a 27-slot KernelTable (slots 0, 1, 3, 4,
 * 22; every other slot is set to NULL so the reference falls back to its own
 * kernels).  Returns NHIP_ERR_ARG if count < 27 or table is NULL. */
int32_t nhip_fill_kernel_table(void** table, int32_t count);

/* ------------------------------------------------ runtime plumbing ------ */

int32_t nhip_init(int32_t device);
int32_t nhip_device_count(int32_t* count);
int32_t nhip_malloc(void** ptr, size_t bytes);
int32_t nhip_free(void* ptr);
int32_t nhip_memcpy_htod(void* dst, const void* src, size_t bytes);
int32_t nhip_memcpy_dtoh(void* dst, const void* src, size_t bytes);
int32_t nhip_memcpy_dtod(void* dst, const void* src, size_t bytes, void* stream);
/* Device-to-device copy by a kernel on `stream` (NULL = the library stream);
 * asynchronous and capturable in a graph.  Used for KV-slot copies. */
int32_t nhip_copy_dev(void* dst, const void* src, size_t bytes, void* stream);
int32_t nhip_memset(void* dst, int32_t value, size_t bytes);
int32_t nhip_stream_create(void** stream);
int32_t nhip_stream_destroy(void* stream);
int32_t nhip_stream_sync(void* stream);
int32_t nhip_device_sync(void);
int32_t nhip_event_create(void** event);
int32_t nhip_event_destroy(void* event);
int32_t nhip_event_record(void* event, void* stream);
int32_t nhip_event_elapsed_ms(void* start, void* stop, float* ms);

/* HIP graphs: capture the device-resident calls issued on `stream` between
 * begin and end into an executable graph, then replay it with one launch.
 * The library records no memset nodes into captured work. */
int32_t nhip_graph_begin(void* stream);
int32_t nhip_graph_end(void* stream, void** graph_exec);
int32_t nhip_graph_launch(void* graph_exec, void* stream);
int32_t nhip_graph_destroy(void* graph_exec);

/* --------------------------------------------- device-resident weights */

typedef struct nhip_weights nhip_weights;

/* Literal int8 format: int8 weights [rows][cols] row-major, one fp16 scale
 * per 32 consecutive elements [rows][cols/32].  cols must be a multiple of
 * 32.  Uploaded once and re-tiled in HBM for 1 KB coalesced loads. */
int32_t nhip_weights_i8_create(const int8_t* w, const uint16_t* scales, int32_t rows,
                               int32_t cols, nhip_weights** out);
/* Same from device buffers (no host copy; the inputs may be freed after). */
int32_t nhip_weights_i8_create_dev(const int8_t* d_w, const uint16_t* d_scales, int32_t rows,
                                   int32_t cols, nhip_weights** out);
/* Codebook format of .cact (Model.cs:257-267): indices + fp16 norms +
 * codebook, host pointers, 2- or 4-bit, cols a multiple of 128. */
int32_t nhip_weights_cq_create(const nhip_cq* w, nhip_weights** out);
int32_t nhip_weights_destroy(nhip_weights* w);
/* rows, cols, bits (8 for the literal format), HBM bytes held. */
int32_t nhip_weights_info(const nhip_weights* w, int32_t* rows, int32_t* cols, int32_t* bits,
                          size_t* device_bytes);

/* ------------------------------------------------ device-resident ops -- */

/* Per-row dynamic quantization (Scalar.QuantizeInt8 on each row):
 * x fp32 [tokens][cols] -> q int8 [tokens][cols], scales fp32 [tokens]. */
int32_t nhip_quantize_rows_dev(const float* d_x, int32_t tokens, int32_t cols, int8_t* d_q,
                               float* d_scales, void* stream);

/* x fp32 rows of codes back to numbers, the inverse of nhip_quantize_rows_dev:
 * d_x[r*ldx + i] = d_q[r*cols + i] * d_scales[r].  rows <= 2^26, cols <= 2^20,
 * ldx >= cols. */
int32_t nhip_dequantize_rows_dev(const int8_t* d_q, const float* d_scales, int32_t rows, int32_t cols, float* d_x,
                                 int32_t ldx, void* stream);

/* A layer's residual addition, root-mean-square norm and quantization, the
 * rows of the next int8 product in one launch (no counterpart in the
 * reference, whose engine runs them one after the other).  For row r:
 *   s = x + delta                    (d_delta NULL: s = x), to d_sum if given
 *   h = (s * (1 / sqrt(mean(s^2) + eps))) * g
 *   d_q[r][..], d_scales[r] = QuantizeInt8(h), as nhip_quantize_rows_dev's
 * with g = d_gain[i] (d_gain NULL: 1), or 1 + d_gain[i] with zero_centered
 * (Ops.ZeroCenteredRms's gains).  The mean and the square root are formed in
 * 64 bits and the inverse rounded to fp32 once; every other operation is one
 * fp32 operation, so that the result does not depend on how a row is summed
 * (but for one rounding of the inverse in some 10^8 rows).  d_x, d_delta and
 * d_sum have row strides ldx, ldd and ld_sum >= cols (columns of wider
 * matrices); d_sum may be d_x or d_delta (with its stride), and overlaps
 * nothing else.  A row with a NaN or an infinity has codes of no meaning, and
 * no effect on the others.  0 < eps <= 1, rows <= 2^26, cols <= 2^20. */
int32_t nhip_add_rms_quantize_dev(const float* d_x, int32_t ldx, const float* d_delta, int32_t ldd,
                                  const float* d_gain, int32_t zero_centered, float eps, int32_t rows, int32_t cols,
                                  float* d_sum, int32_t ld_sum, int8_t* d_q, float* d_scales, void* stream);

/* Quant.Prepare on device (Quant.cs:473-488): x fp32 [tokens][cols] ->
 * values int8 [tokens][cols] (planes order), scales/offsets fp32
 * [tokens][stride]. */
int32_t nhip_prepare_dev(const float* d_x, int32_t tokens, int32_t cols, int32_t bits,
                         int8_t* d_values, float* d_scales, float* d_offsets, int32_t stride,
                         void* stream);

/* y[t*ldy+n] = sum_g (h(scale[n][g]) * qscale[t]) * dot_g(w[n], q[t]) for
 * n in [row_start,row_end), t < tokens, in Scalar.MatMulRows' order
 * (Scalar.cs:160-189).  Literal int8 weights.  Past 16 tokens a
 * 16-byte aligned d_q takes a faster kernel. */
int32_t nhip_matmul_i8_dev(const nhip_weights* w, const int8_t* d_q, const float* d_qscale,
                           int32_t tokens, float* d_y, int32_t ldy, int32_t row_start,
                           int32_t row_end, void* stream);

/* Bandwidth calibration, no reference counterpart: reads `bytes` (a multiple
 * of 16) from d_src with the decode GEMV's access pattern (16-byte
 * non-temporal loads, 1 KB per wave instruction, 32 KB per 256-thread
 * workgroup) and writes each workgroup's XOR of the words it read to
 * d_sink[ceil(bytes / 32768)].  The time of one launch is the read ceiling
 * of a GEMV over the same bytes. */
int32_t nhip_read_stream_dev(const void* d_src, size_t bytes, uint32_t* d_sink, void* stream);

/* Prefill form of nhip_matmul_i8_dev with a fused epilogue: the same exact
 * int32 group sums D_g, accumulated as acc = fma(h(scale[n][g]), D_g, acc)
 * and scaled once, y = acc * qscale[t] -- two VALU operations per (token,
 * row, group) instead of the reference's four, so the fp32 outputs agree with
 * Scalar.MatMulRows to 1e-4 of RMS(y), not bit for bit.  For prefill
 * throughput; nhip_matmul_i8_dev stays bit-exact for every token count, and
 * runs in its place where d_q is not 16-byte aligned. */
int32_t nhip_matmul_i8_fused_dev(const nhip_weights* w, const int8_t* d_q, const float* d_qscale,
                                 int32_t tokens, float* d_y, int32_t ldy, int32_t row_start,
                                 int32_t row_end, void* stream);

/* Scalar.MatMulRows on device for codebook weights (Scalar.cs:146-192):
 * activations as produced by nhip_prepare_dev (d_values' alignment as
 * nhip_matmul_i8_dev's d_q). */
int32_t nhip_matmul_cq_dev(const nhip_weights* w, const int8_t* d_values, const float* d_scales,
                           const float* d_offsets, int32_t stride, int32_t tokens, float* d_y,
                           int32_t ldy, int32_t row_start, int32_t row_end, void* stream);

/* Quant.MatMulBatch (src/Needle/Quant.cs:679-816): `count` (1..4) weight
 * matrices of one format and one K that share the activations (Needle 3's
 * Q, K, V and Gate projections), each job j computing all of its rows into
 * d_y[j] with row stride ldy[j] (>= its rows), as nhip_matmul_i8_dev
 * (literal: d_scales [tokens], d_offsets and stride unused) or
 * nhip_matmul_cq_dev (codebook) would.  Literal batches of up to 16 tokens
 * and codebook batches of any count run as one launch over every job's row
 * tiles; literal ones past 16 run the jobs in turn.  Bit-identical with the
 * single-matrix calls.  w and d_y / ldy are host arrays of `count` entries. */
int32_t nhip_matmul_batch_dev(const nhip_weights* const* w, int32_t count, const int8_t* d_q,
                              const float* d_scales, const float* d_offsets, int32_t stride,
                              int32_t tokens, float* const* d_y, const int32_t* ldy, void* stream);

/* The int32 group sums D[t][n-row_start][g] (Scalar.cs:162-184) that the
 * matmuls accumulate, for checking them bit-exactly.  Literal / codebook. */
int32_t nhip_group_dots_i8_dev(const nhip_weights* w, const int8_t* d_q, int32_t tokens,
                               int32_t row_start, int32_t row_end, int32_t* d_dots,
                               void* stream);
int32_t nhip_group_dots_cq_dev(const nhip_weights* w, const int8_t* d_values, int32_t tokens,
                               int32_t row_start, int32_t row_end, int32_t* d_dots,
                               void* stream);

/* ------------------------------------------ decode attention (KV cache) -- */

/* Ragged decode attention over a pooled int8 KV cache (one launch for a
 * batch of rows from independent slots).  Replaces the per-row
 * AttentionBatch.Run / ExecuteChunk + MergePartials path
 * (src/Needle/Blocks.cs:849-966, 750-817) that EngineCore.RunAttentionBatch
 * drives (src/Needle/Engine.cs:2480-2596).  Layout per layer, as the
 * reference's KV cache (src/Needle/Engine.cs:127-136, 184-187) with one
 * region per slot:
 *   keys   int8 [slots][capacity][kv_heads*qk_dim], key_scales   fp32 [slots][capacity][kv_heads]
 *   values int8 [slots][capacity][kv_heads*64],     value_scales fp32 [slots][capacity][kv_heads]
 *   q int8 [rows][heads][qk_dim] with q_scales [rows][heads] (QuantizeInt8
 *   per head), out fp32 [rows][heads][64].
 * Row r attends positions row_first[r] .. row_first[r]+row_count[r]-1 of
 * slot row_slot[r] (device arrays, so a captured graph can be replayed with
 * new spans); query head h reads kv head h / (heads/kv_heads).  Each (row,
 * head) is split into at most max_chunks chunks by the reference's plan
 * (8 reproduces the reference; 64 fills the GPU), each chunk is the
 * reference tile in partial form and the chunks are merged in
 * MergePartials' order, with the polynomial Ops.Exp.  Rows whose slot or
 * span is out of range produce zeros.  qk_dim is 48 or 64, v dim 64,
 * heads/kv_heads <= 16; q, keys, values and out 16-byte aligned.
 * The workspace (nhip_attention_decode_workspace bytes) holds the chunk
 * partials; it needs no initialisation (nhip_attention_decode_workspace_init
 * zeroes it, for callers that want defined contents).  Calls that share a
 * workspace must not overlap. */
size_t nhip_attention_decode_workspace(int32_t rows, int32_t heads, int32_t max_chunks);
int32_t nhip_attention_decode_workspace_init(void* d_workspace, size_t bytes, void* stream);
int32_t nhip_attention_decode_dev(const int8_t* d_q, const float* d_q_scales, int32_t rows,
                                  int32_t heads, int32_t kv_heads, int32_t qk_dim,
                                  const int8_t* d_keys, const float* d_key_scales,
                                  const int8_t* d_values, const float* d_value_scales,
                                  int32_t slots, int32_t capacity, const int32_t* d_row_slot,
                                  const int32_t* d_row_first, const int32_t* d_row_count,
                                  int32_t max_chunks, void* d_workspace, size_t workspace_bytes,
                                  float* d_out, void* stream);

/* No counterpart in the reference: nhip_attention_decode_dev for callers
 * that cannot allocate (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc).  Same arguments, semantics and results,
 * without the workspace: the chunk partials go to a fixed 8 MiB device
 * scratch array that the library holds on each GPU until the process ends
 * (its address is looked up at nhip_init, which must have been called).
 * Calls whose partials (nhip_attention_decode_workspace(rows, heads,
 * max_chunks) bytes) exceed 8 MiB fail with NHIP_ERR_ARG.  No allocation
 * happens in the call.  Every call on a GPU shares that GPU's scratch:
 * calls that overlap on one GPU (other streams or threads) race, so
 * serialise them. */
int32_t nhip_attention_decode_noalloc_dev(const int8_t* d_q, const float* d_q_scales, int32_t rows,
                                          int32_t heads, int32_t kv_heads, int32_t qk_dim,
                                          const int8_t* d_keys, const float* d_key_scales,
                                          const int8_t* d_values, const float* d_value_scales,
                                          int32_t slots, int32_t capacity, const int32_t* d_row_slot,
                                          const int32_t* d_row_first, const int32_t* d_row_count,
                                          int32_t max_chunks, float* d_out, void* stream);

/* --------------------------------------------------- rotary positions ---- */

/* Rotation of query and key heads by position.  A head's first `dim`
 * dimensions are pairs (x0, x1): dimensions i and i + dim/2 (Scalar.Rope,
 * src/Needle/Scalar.cs:233-248), or with `interleaved` dimensions 2i and
 * 2i + 1, i < dim/2.  At position p
 *   x0' = x0 * cos[p][i] - x1 * sin[p][i],  x1' = x1 * cos[p][i] + x0 * sin[p][i]
 * (every operation rounded to fp32, as the decoder engine rotates); the head's
 * other dimensions stay as they are.  cos and sin are device tables
 * [positions][dim/2], made by nhip_rotary_table_dev or by the caller.  dim is
 * even and at most 512.  The struct is read during the call. */
typedef struct nhip_rotary {
    const float* cos;
    const float* sin;
    int32_t positions, dim, interleaved;
} nhip_rotary;

/* How a table's frequencies follow from theta, f_i = theta^(-2i/dim), for
 * contexts longer than a model was made for (factor >= 1):
 *   NHIP_ROTARY_PLAIN   f_i
 *   NHIP_ROTARY_LINEAR  f_i / factor (positions packed closer)
 *   NHIP_ROTARY_BASE    theta times factor^(dim/(dim-2)): the slowest pair is
 *                       slowed by factor, the fastest not (dim > 2)
 *   NHIP_ROTARY_PARTS   a ramp over the pairs: those that turn more than `high`
 *                       times over `original` positions keep f_i, those of less
 *                       than `low` turns take f_i / factor.  With b(t) = dim *
 *                       ln(original / (2 pi t)) / (2 ln theta), lo =
 *                       max(floor(b(high)), 0), hi = min(ceil(b(low)), dim - 1) (lo +
 *                       0.001 where they are equal): r = clamp((i - lo) / (hi -
 *                       lo), 0, 1), f_i / factor * r + f_i * (1 - r)
 *   NHIP_ROTARY_BANDS   the same by the turns themselves: r = clamp((original *
 *                       f_i / (2 pi) - low) / (high - low), 0, 1),
 *                       f_i / factor * (1 - r) + f_i * r
 * (PARTS is its formula where that leaves the words: with a hi below 0 every
 * pair keeps f_i, with a lo above hi every one takes f_i / factor.)  cos and sin
 * are multiplied by magnitude (1 for none).  theta in (1, 10^12], factor in [1,
 * 10^6] (but for PLAIN, which has none), magnitude in (0, 10^6]; low, high and
 * original are used by the last two (0 < low < high <= 10^9, 0 < original <= 10^9). */
enum {
    NHIP_ROTARY_PLAIN = 0,
    NHIP_ROTARY_LINEAR = 1,
    NHIP_ROTARY_BASE = 2,
    NHIP_ROTARY_PARTS = 3,
    NHIP_ROTARY_BANDS = 4
};
typedef struct nhip_rotary_scaling {
    double theta, factor, low, high, original, magnitude;
    int32_t kind;
} nhip_rotary_scaling;

/* cos and sin of positions first .. first+count-1 (0 <= first, first + count <=
 * 2^30) into d_cos, d_sin [count][dim/2]: angles and their cos and sin in 64
 * bits, rounded to fp32 at the end.  A table grows by calls on its next rows. */
int32_t nhip_rotary_table_dev(float* d_cos, float* d_sin, int32_t first, int32_t count, int32_t dim,
                              const nhip_rotary_scaling* scaling, void* stream);
/* The heads of every row, d_x[r*ldx + h*head_dim ..], rotated by position
 * d_row_pos[r] into d_y[r*ldy + h*head_dim ..].  d_y may be d_x (with ldy =
 * ldx), and overlaps it in no other way.  Rows whose position is outside
 * [0, positions) write nothing.  rows <= 2^20, head_dim >= dim, head_dim <=
 * 4096, heads * head_dim <= ldx, ldy and 2^24. */
int32_t nhip_rotary_dev(const nhip_rotary* r, const float* d_x, int32_t ldx, int32_t heads, int32_t head_dim,
                        const int32_t* d_row_pos, int32_t rows, float* d_y, int32_t ldy, void* stream);

/* --------------------------------------------- paged KV cache (serving) -- */

/* No counterpart in the reference: an int8 KV cache in pages, for servers
 * whose sequences grow, branch and end at different times.  The pooled cache
 * above gives every slot its whole capacity and copies a slot position by
 * position; here a sequence holds pages of `page_size` positions named by its
 * row of `tables`, sequences share pages, and a page is copied only when one
 * of its holders writes past a shared part.
 *
 * The caller owns every array (device memory; the four pools 16-byte aligned):
 *   keys         int8 [layers][pages][kv_heads][page_size][qk_dim]
 *   key_scales   fp32 [layers][pages][kv_heads][page_size]
 *   values       int8 [layers][pages][kv_heads][page_size/16][v_dim][16]
 *   value_scales fp32 [layers][pages][kv_heads][page_size]
 *   tables       int32 [sequences][width]: the page of positions
 *                [t*page_size, (t+1)*page_size), -1 past the sequence's pages
 *   lengths      int32 [sequences]: positions held; a sequence holds the
 *                ceil(length / page_size) pages that its row begins with
 *   refs         int32 [pages]: how many sequences hold a page (0: free)
 * A page holds a kv head's positions together, and 16 positions of a value
 * dimension together, so that both products of attention read matrix
 * operands straight from the cache.
 * page_size 16, 32, 64, 128 or 256; (qk_dim, v_dim) (48, 64), (64, 64) or
 * (128, 128); kv_heads <= 256; layers <= 4096; pages <= 2^20; sequences <=
 * 65536; width * page_size <= 2^30; a call takes up to 2^20 rows.
 *
 * Scales, the queries' among them, are not negative (QuantizeInt8's are
 * positive).  A scale that is no finite number may spoil the rows that attend
 * its position, and only those; so may a value scale of more than 2^60, and
 * outputs under 2^-60 lose digits.
 *
 * The calls below take this struct by pointer (read during the call), are
 * asynchronous on `stream` and may be captured in a graph; calls that write
 * a cache must be ordered with the other calls on it.  A table entry outside
 * [0, pages) is never followed. */
typedef struct nhip_paged_cache {
    int8_t* keys;
    float* key_scales;
    int8_t* values;
    float* value_scales;
    int32_t* tables;
    int32_t* lengths;
    int32_t* refs;
    int32_t layers, pages, page_size, kv_heads, qk_dim, v_dim, sequences, width;
} nhip_paged_cache;

/* An empty cache: tables -1, lengths and refs 0 (the pools need no clearing). */
int32_t nhip_paged_reset_dev(const nhip_paged_cache* c, void* stream);

/* Row r's new key and value, QuantizeInt8 (src/Needle/Scalar.cs:67-74) per kv
 * head, into layer `layer` at position row_pos[r] of sequence row_seq[r]:
 * keys d_k[r*ldk + kvh*qk_dim ..], values d_v[r*ldv + kvh*v_dim ..] (fp32;
 * columns of a wider matrix; ldk >= kv_heads*qk_dim, ldv >= kv_heads*v_dim).
 * They are cached as they are: what a model does to its keys before attention
 * (rotation by position, normalization) is done before this call.  The position's page must
 * be held already (nhip_paged_resize_dev) and by this sequence alone: rows
 * whose sequence, position or page is out of range write nothing, nor do rows
 * whose page has more than one holder (refs), so that after a resize that
 * found too few pages no other sequence's positions are written.  Two rows of
 * a call at one position leave it unspecified.  lengths are not read. */
int32_t nhip_paged_append_dev(const nhip_paged_cache* c, int32_t layer, const float* d_k, int32_t ldk,
                              const float* d_v, int32_t ldv, const int32_t* d_row_seq, const int32_t* d_row_pos,
                              int32_t rows, void* stream);

/* nhip_rotary_dev on the rows' query and key heads, nhip_quantize_rows_dev on
 * the queries and nhip_paged_append_dev, in one launch and with their bits:
 * row r's query heads d_q[r*ldq + h*qk_dim ..] and keys d_k[r*ldk + ..] rotated
 * by row_pos[r], the queries' codes and scales to d_codes int8
 * [rows][heads][qk_dim] and d_q_scales [rows][heads], ready for the attention
 * calls, keys and values to position row_pos[r] of sequence row_seq[r].  Rows
 * that nhip_paged_append_dev would not write write nothing to the cache; rows
 * whose position is outside the table write nothing to it either, and have
 * queries of codes 0 and scale 1.  r->dim <= qk_dim; heads <= 4096 (a multiple
 * of kv_heads); d_codes 4-byte aligned. */
int32_t nhip_paged_rotary_append_dev(const nhip_paged_cache* c, int32_t layer, const nhip_rotary* r, const float* d_q,
                                     int32_t ldq, int32_t heads, const float* d_k, int32_t ldk, const float* d_v,
                                     int32_t ldv, const int32_t* d_row_seq, const int32_t* d_row_pos, int32_t rows,
                                     int8_t* d_codes, float* d_q_scales, void* stream);

/* Cached positions back to numbers: the keys and values that layer `layer`
 * holds at position row_pos[r] of sequence row_seq[r], code * scale, to
 * d_k[r*ldk + kvh*qk_dim ..] and d_v[r*ldv + kvh*v_dim ..] (fp32; either may be
 * NULL; strides as nhip_paged_append_dev's).  Rows whose sequence, position or
 * page is out of range give zeros.  lengths are not read. */
int32_t nhip_paged_read_dev(const nhip_paged_cache* c, int32_t layer, const int32_t* d_row_seq,
                            const int32_t* d_row_pos, int32_t rows, float* d_k, int32_t ldk, float* d_v, int32_t ldv,
                            void* stream);

/* Attention of one new token per row: row r's query heads (q int8
 * [rows][heads][qk_dim] with q_scales [rows][heads], QuantizeInt8 per head)
 * attend positions row_first[r] .. row_first[r]+row_count[r]-1 of sequence
 * row_seq[r]; query head h reads kv head h / (heads/kv_heads) and scores are
 * scaled by 1/sqrt(qk_dim), as in nhip_attention_decode_dev.  out fp32
 * [rows][heads][v_dim].  Scores, softmax statistics and sums are fp32 and the
 * result is within 1e-5 of RMS(out) of exact arithmetic, or within 1e-7 of it
 * times the row's largest |score| where that is above 100 (up to 1e6: a score
 * is rounded to 2^-24 of itself); it is the same for the same call, but not
 * the bits of the reference's order.  max_count bounds every
 * row_count (it decides how the work is split).  Rows of count 0, and rows
 * whose sequence or span is out of range or whose count exceeds max_count,
 * give zeros; positions on pages outside [0, pages) are left out.
 * heads/kv_heads <= 16; q and out 16-byte aligned.  The workspace needs no
 * initialisation; calls that may overlap need one each. */
size_t nhip_paged_decode_workspace(const nhip_paged_cache* c, int32_t rows, int32_t heads, int32_t max_count);
int32_t nhip_paged_decode_dev(const nhip_paged_cache* c, int32_t layer, const int8_t* d_q, const float* d_q_scales,
                              int32_t rows, int32_t heads, const int32_t* d_row_seq, const int32_t* d_row_first,
                              const int32_t* d_row_count, int32_t max_count, void* d_workspace,
                              size_t workspace_bytes, float* d_out, void* stream);

/* Causal attention of whole prompts, or of their next parts, packed one
 * behind the other: run i is the rows run_rows[i] .. run_rows[i+1]-1 (device
 * array [runs+1], ascending), which sit at positions run_pos[i], run_pos[i]+1,
 * ... of sequence run_seq[i].  Their keys and values are in the cache already
 * (nhip_paged_append_dev), as are those of the positions before them.  The row
 * at position p attends [0, p], or with window > 0 [max(0, p-window+1), p].
 * Everything else as nhip_paged_decode_dev; a position's weight times its value
 * scale is kept to 2^-30 of the row's largest such product (values whose codes
 * are all 0, with QuantizeInt8's scale of 1, count as none).  max_count bounds every position + 1 (rows
 * beyond give zeros), and rows behind the last run are left as they are.
 * (rows * heads / kv_heads / 128 + runs) * kv_heads <= 2^23. */
size_t nhip_paged_prompt_workspace(const nhip_paged_cache* c, int32_t rows, int32_t heads, int32_t runs,
                                   int32_t max_count);
int32_t nhip_paged_prompt_dev(const nhip_paged_cache* c, int32_t layer, const int8_t* d_q, const float* d_q_scales,
                              int32_t rows, int32_t heads, int32_t runs, const int32_t* d_run_rows,
                              const int32_t* d_run_seq, const int32_t* d_run_pos, int32_t window, int32_t max_count,
                              void* d_workspace, size_t workspace_bytes, float* d_out, void* stream);

/* Attention over a window and a sequence's first positions ("sinks"), which
 * stay visible however far the window has moved.  decode: row r attends the
 * first min(sinks, row_first[r]) positions of its sequence beside [row_first[r],
 * row_first[r] + row_count[r]) (a row of count 0 attends nothing); prompt: the
 * row at position p attends the positions up to p that lie in [max(0, p-window+1), p]
 * or in [0, sinks).  Everything else as the calls without sinks, which these are for sinks =
 * 0 (and for window = 0); positions between sinks and window are not read, and
 * their pages' table entries may be anything.  sinks >= 0. */
size_t nhip_paged_decode_sinks_workspace(const nhip_paged_cache* c, int32_t rows, int32_t heads, int32_t sinks,
                                         int32_t max_count);
int32_t nhip_paged_decode_sinks_dev(const nhip_paged_cache* c, int32_t layer, const int8_t* d_q,
                                    const float* d_q_scales, int32_t rows, int32_t heads, const int32_t* d_row_seq,
                                    const int32_t* d_row_first, const int32_t* d_row_count, int32_t sinks,
                                    int32_t max_count, void* d_workspace, size_t workspace_bytes, float* d_out,
                                    void* stream);
size_t nhip_paged_prompt_sinks_workspace(const nhip_paged_cache* c, int32_t rows, int32_t heads, int32_t runs,
                                         int32_t sinks, int32_t max_count);
int32_t nhip_paged_prompt_sinks_dev(const nhip_paged_cache* c, int32_t layer, const int8_t* d_q,
                                    const float* d_q_scales, int32_t rows, int32_t heads, int32_t runs,
                                    const int32_t* d_run_rows, const int32_t* d_run_seq, const int32_t* d_run_pos,
                                    int32_t window, int32_t sinks, int32_t max_count, void* d_workspace,
                                    size_t workspace_bytes, float* d_out, void* stream);

/* Pages.  All of a call's entries act together (as if every entry read the
 * cache as it was before the call); of entries that name the same sequence
 * only the first counts, and entries out of range do nothing.  count <= 1024.
 * The workspace holds nhip_paged_pages_workspace bytes, needs no
 * initialisation, and one call's is free for the next call of the stream.
 *
 * copy     page src[i]'s contents (all layers) to page dst[i]; tables and refs
 *          stay.  A page may be the source of several entries, but must not be
 *          the destination of one and named by another.
 * fork     sequence dst[i] gives up its pages and becomes a copy of the first
 *          length[i] positions of sequence src[i] (d_length NULL, or a longer
 *          length: all of it), sharing its pages (refs).  A beam step's
 *          reorder is one call with dst 0..n-1 and src the beams' parents.
 * resize   sequence seq[i] takes length[i].  Shorter: pages past it are given
 *          up.  Longer: if its last page is partly filled and held by others
 *          too, it gets a copy of that page; then it takes the pages it lacks.
 *          (Of several entries of one call that grow into the same page, as
 *          many of the first copy it as leave one holder.)  Pages are taken in
 *          entry order, the lowest free page first; pages given up in the
 *          call are free from the next call on.  If the free pages do not
 *          suffice nothing changes at all.  d_status (may be NULL) int32 [2]:
 *          the pages missing (0: done; an entry that lacks more than the pool
 *          has counts as pages + 1), the entries refused (out of range).
 *          A refused entry keeps its sequence as it is.
 * free     resize to 0.
 * compact  moves pages to the front of the pool: with n pages held, the k-th
 *          free page below n takes the contents and holders of the k-th held
 *          page from n on.  d_status (may be NULL) int32 [1]: n. */
size_t nhip_paged_pages_workspace(const nhip_paged_cache* c, int32_t count);
int32_t nhip_paged_copy_dev(const nhip_paged_cache* c, int32_t count, const int32_t* d_src, const int32_t* d_dst,
                            void* stream);
int32_t nhip_paged_fork_dev(const nhip_paged_cache* c, int32_t count, const int32_t* d_dst, const int32_t* d_src,
                            const int32_t* d_length, void* d_workspace, size_t workspace_bytes, void* stream);
int32_t nhip_paged_resize_dev(const nhip_paged_cache* c, int32_t count, const int32_t* d_seq,
                              const int32_t* d_length, int32_t* d_status, void* d_workspace, size_t workspace_bytes,
                              void* stream);
int32_t nhip_paged_free_dev(const nhip_paged_cache* c, int32_t count, const int32_t* d_seq, void* d_workspace,
                            size_t workspace_bytes, void* stream);
int32_t nhip_paged_compact_dev(const nhip_paged_cache* c, int32_t* d_status, void* d_workspace,
                               size_t workspace_bytes, void* stream);

/* ------------------------------------ Needle 3 attention inputs (rows) -- */

/* Needle 3's step from a row's raw Q/K/V projections to its int8 query heads
 * and KV-cache row (EngineCore.TapsAndAttentionHeadsSingle,
 * src/Needle/Engine.cs:1302-1387, and Scalar.Taps3's multi-frame form,
 * src/Needle/Scalar.cs:285-288): for every query, key and value head the
 * three-tap convolution over time with the slot's two previous frames
 * (taps [3][width] per part: current, previous, two back), then for queries
 * and keys ZeroCenteredRms (q_norm / k_norm [qk_dim], shared by the heads),
 * Rope at the row's position (cos / sin tables [capacity][qk_dim/2]) and
 * QuantizeInt8 per head; values QuantizeInt8 per head.  Queries go to
 * d_q [rows][heads*qk_dim] / d_q_scales [rows][heads]; keys and values to the
 * cache at (slot, position): keys [slots][capacity][kv_heads*qk_dim],
 * values [slots][capacity][kv_heads*v_dim], scales [slots][capacity][kv_heads].
 * d_raw: [rows][qw + kw + vw] (qw = heads*qk_dim, kw = kv_heads*qk_dim,
 * vw = kv_heads*v_dim); d_history: [slots] x ([2][qw], [2][kw], [2][vw]),
 * frame 1 the latest, moved on to each slot's last two frames.  The rows of a
 * slot must be one contiguous run of consecutive positions (a row takes its
 * previous frames from the rows before it in the run); rows with an
 * out-of-range slot or position get q = 0, scale 1 and touch nothing.
 * qk_dim even and <= 64, v_dim <= 64.  Bit-identical with the reference's
 * scalar row-by-row step on the same tables. */
int32_t nhip_needle3_attention_inputs_dev(const float* d_raw, int32_t rows, int32_t heads, int32_t kv_heads,
                                          int32_t qk_dim, int32_t v_dim, const float* d_q_taps,
                                          const float* d_k_taps, const float* d_v_taps, const float* d_q_norm,
                                          const float* d_k_norm, const float* d_rope_cos,
                                          const float* d_rope_sin, float* d_history,
                                          const int32_t* d_row_slot, const int32_t* d_row_pos, int32_t slots,
                                          int32_t capacity, int8_t* d_q, float* d_q_scales, int8_t* d_keys,
                                          float* d_key_scales, int8_t* d_values, float* d_value_scales,
                                          void* stream);

/* ---------------------------------------------- decode loop (engine) -- */

/* The beam/ragged-batched decode step of a pre-norm int8 decoder (RMSNorm,
 * fused QKV, rotary positions, int8 KV cache per slot, SwiGLU FFN, LM head)
 * with every linear in the literal int8 format.  One forward packs `rows`
 * rows from independent cache slots, as EngineCore.ForwardBatch does
 * (src/Needle/Engine.cs:2303-2350, 2480-2596); beam search drives it as
 * Whistle.BeamSearch does (src/Needle/Whistle.Decode.cs:226-350) but with
 * the beams batched into one forward per step, which is the step API of the
 * performance path (nhip_step / slot copy).  Element-wise operations follow
 * the canonical order the CPU restatement shares, so logits and token streams
 * are bit-identical with it. */
typedef struct nhip_decoder nhip_decoder;

typedef struct nhip_decoder_dims {
    int32_t layers, d, heads, kv_heads, head_dim, ffn, vocab;
    int32_t capacity;   /* positions per cache slot */
    int32_t slots;      /* cache slots (beams, sequences) */
    int32_t max_rows;   /* rows per forward (prompt length for prefill) */
    int32_t max_chunks; /* attention position-split cap (64 fills the GPU) */
    double theta;       /* RoPE base */
    float eps;          /* RMSNorm epsilon */
} nhip_decoder_dims;

typedef struct nhip_decode_stats {
    double prefill_seconds, decode_seconds;
    int64_t fed_rows; /* rows fed after the prompt (row-tokens) */
    int32_t steps;
} nhip_decode_stats;

int32_t nhip_decoder_create(const nhip_decoder_dims* dims, nhip_decoder** out);
/* Host weights of one layer, uploaded and re-tiled: wqkv [(heads+2kv)*64][d],
 * wo [d][heads*64], wgu [2*ffn][d] (gate rows then up rows), wd [d][ffn],
 * each int8 with fp16 group-32 scales; RMSNorm gains [d]. */
int32_t nhip_decoder_set_layer(nhip_decoder* m, int32_t layer, const int8_t* wqkv, const uint16_t* sqkv,
                               const int8_t* wo, const uint16_t* so, const int8_t* wgu, const uint16_t* sgu,
                               const int8_t* wd, const uint16_t* sd, const float* attn_norm,
                               const float* ffn_norm);
/* Embedding fp32 [vocab][d], final RMSNorm gain [d], LM head [vocab][d]. */
int32_t nhip_decoder_set_head(nhip_decoder* m, const float* embedding, const float* final_norm,
                              const int8_t* wlm, const uint16_t* slm);
/* One synchronous forward of `rows` rows (host token/slot/position arrays):
 * writes each layer's K/V at the row's position in its slot, returns logits
 * [rows][vocab] if non-NULL and the top-k ids / log-probabilities
 * (TopKLogSoftmax, ids 0,2,3 masked) if k > 0 (k <= 8). */
int32_t nhip_decoder_forward(nhip_decoder* m, const int32_t* tokens, const int32_t* slots,
                             const int32_t* positions, int32_t rows, float* logits, int32_t k,
                             int32_t* topk_idx, float* topk_lp);
/* Grammar-constrained greedy step: one forward whose LM head computes only
 * the 16-row vocab tiles that hold an id allowed by some row's mask
 * (Engine.LogitsForRows' sparse head, src/Needle/Engine.cs:2191-2195,
 * 2683-2700), then Ops.ArgMaxMasked per row (src/Needle/Ops.cs:1223-1266):
 * best[r] = the lowest allowed id holding row r's largest allowed logit
 * above -inf, or -1.  masks: host [rows][words] bitsets, bit id%32 of word
 * id/32 (ids from vocab on are ignored); best_logit optional.  rows <= 16.
 * The allowed logits are bit-identical with the dense head's. */
int32_t nhip_decoder_forward_masked(nhip_decoder* m, const int32_t* tokens, const int32_t* slots,
                                    const int32_t* positions, int32_t rows, const uint32_t* masks,
                                    int32_t words, int32_t* best, float* best_logit);
/* Ops.ArgMaxMasked (src/Needle/Ops.cs:1223-1266; kernel-table slot 25's
 * operation) over `rows` device rows: row r reads d_x + r*ldx and the mask
 * d_mask + r*mask_ld ([words] bitsets, ids >= length ignored) and writes the
 * chosen id (or -1) to d_index[r] and, if d_value is non-NULL, its value
 * (-inf for -1).  Asynchronous on `stream`. */
int32_t nhip_argmax_masked_dev(const float* d_x, int32_t ldx, const uint32_t* d_mask, int32_t mask_ld,
                               int32_t words, int32_t length, int32_t rows, int32_t* d_index, float* d_value,
                               void* stream);
/* Ops.TopKLogSoftmax (src/Needle/Ops.cs:1092-1221) as the decoder's head
 * runs it, over `rows` device rows of n logits (row r at d_logits + r*n):
 * the k (1..8) best ids by value, ties to the lower id, ids 0, 2 and 3
 * excluded, and their log-probabilities v - (peak + log S), with S summed
 * over blocks of 2048 ids in the canonical order.  d_idx / d_lp: [rows][k].
 * n <= 524288.  The workspace (nhip_topk_lse_workspace bytes) holds the
 * per-block partial lists; nothing needs clearing.  Asynchronous on
 * `stream`. */
size_t nhip_topk_lse_workspace(int32_t rows, int32_t n);
int32_t nhip_topk_lse_dev(const float* d_logits, int32_t rows, int32_t n, int32_t k, void* d_workspace,
                          size_t workspace_bytes, int32_t* d_idx, float* d_lp, void* stream);
/* Ops.ArgMax (src/Needle/Ops.cs:1052-1090; Engine.Greedy, Engine.cs:103)
 * over `rows` device rows of n values (row r at d_x + r*ldx): d_index[r] =
 * the lowest id holding the row's largest non-NaN value, 0 when x[0] is NaN
 * (the scalar loop's `x[i] > x[best]` from best = 0: +0 and -0 are equal, an
 * all -inf row gives 0; the AVX path gives the same ids on NaN-free rows);
 * d_value[r] (optional) = that value.  Asynchronous on `stream`. */
int32_t nhip_argmax_dev(const float* d_x, int32_t ldx, int32_t n, int32_t rows, int32_t* d_index, float* d_value,
                        void* stream);
/* One id per row of logits, drawn with a given number (no counterpart in the
 * reference, which takes the largest).  Row r's ids are those with a finite or +inf
 * logit d_logits[r*ldx + i], i < n, and a set bit in the row's mask
 * (as nhip_argmax_masked_dev's; d_mask NULL: every id; ids past `words` * 32
 * have none), in the order of their logits, the largest first, ties to the lower
 * id.  Weights are e^((logit - largest) / temperature), as whole multiples of
 * 2^-42 (of the largest logit's weight, 1).  Kept are, one rule behind the other,
 *   top_k  the first top_k ids (<= 0: all);
 *   top_p  of those, an id as long as the ones before it weigh less than top_p
 *          times all of them; always the first (>= 1 or NaN: all);
 *   min_p  of those, ids of weight >= min_p (at most 1; NaN: all).
 * With t = floor(random * total weight of the kept ids), d_ids[r] is the lowest
 * kept id for which the weights of the kept ids up to it exceed t.  (Sums are
 * exact; the products random * and top_p * total are rounded to 64-bit floats.)  A
 * temperature <= 0 or NaN takes the first id; where the largest logit is +inf,
 * the ids that have it weigh 1 and the others 0.  random counts as
 * clamped to [0, 1) (NaN: 0).  d_logprobs (may be NULL) is ln(weight / total
 * weight of the kept ids).  A row without ids gives -1 and -inf.
 * Every sum is one of whole numbers: the same call gives the same ids.
 * The parameters are device arrays of `rows` entries each; NULL for
 * temperature (1), top_k, top_p, min_p (all ids).  n <= 2^19, rows <= 2^16. */
typedef struct nhip_sampling {
    const float* random;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
} nhip_sampling;
/* (None is needed at present: 0, as for sizes that are refused, and d_workspace
 * may be NULL.  One that is needs no initialisation, and calls that may overlap
 * need one each.) */
size_t nhip_sample_workspace(int32_t rows, int32_t n);
int32_t nhip_sample_dev(const float* d_logits, int32_t ldx, int32_t n, int32_t rows, const nhip_sampling* s,
                        const uint32_t* d_mask, int32_t mask_ld, int32_t words, void* d_workspace,
                        size_t workspace_bytes, int32_t* d_ids, float* d_logprobs, void* stream);
/* Engine.CopyFrom (src/Needle/Engine.cs:367-379): positions [0, length) of
 * slot src into slot dst, whose length (for nhip_decoder_step) becomes
 * `length`. */
int32_t nhip_decoder_copy_slot(nhip_decoder* m, int32_t dst, int32_t src, int32_t length);
/* The step API of the batched engine: BatchedEngine.ForwardBatch /
 * EngineCore.ForwardBatch (src/Needle/BatchEngine.cs:38-39,
 * src/Needle/Engine.cs:2303-2350).  Rows carry tokens[r] into slot
 * row_slots[r]; the rows of a slot form one contiguous run and sit at the
 * slot's length + their offset in the run (Engine.cs:2655-2661), and every
 * slot's length grows by its run (NHIP_ERR_ARG past the capacity, before any
 * device work).  The LM head runs only over head_rows[0..heads) (rows of
 * this call): row i of the outputs is row head_rows[i] -- logits [heads][vocab]
 * (BatchLogitsRow), the top-k ids / log-probabilities [heads][k] if k > 0,
 * Ops.ArgMax of each head row into argmax[heads] if non-NULL.  rows <= 16
 * replay a graph captured per (rows, heads, k, argmax).  Synchronous.
 * nhip_decoder_forward (explicit positions) leaves the lengths alone. */
int32_t nhip_decoder_step(nhip_decoder* m, const int32_t* tokens, const int32_t* row_slots, int32_t rows,
                          const int32_t* head_rows, int32_t heads, float* logits, int32_t k, int32_t* topk_idx,
                          float* topk_lp, int32_t* argmax);
/* BatchedEngine.ResetSlot / MarkSlot / RewindSlot / SlotLength
 * (src/Needle/BatchEngine.cs:25-30): reset sets a slot's length (and mark) to
 * 0, mark records its length, rewind returns to the mark; the next step
 * overwrites the cache from there. */
int32_t nhip_decoder_slot_reset(nhip_decoder* m, int32_t slot);
int32_t nhip_decoder_slot_mark(nhip_decoder* m, int32_t slot);
int32_t nhip_decoder_slot_rewind(nhip_decoder* m, int32_t slot);
int32_t nhip_decoder_slot_length(const nhip_decoder* m, int32_t slot, int32_t* length);
/* Greedy decoding, ToolCaller.Complete's loop (src/Needle/ToolCaller.cs:
 * 59-77) on slot 0: reset it, feed the prompt (chunks of max_rows rows, the
 * head on the last row only), then up to max_new times take Ops.ArgMax of
 * the last logits on the device, stop before a token equal to `stop` (-1:
 * none), otherwise record it and feed it.  Writes the tokens (without the
 * prompt) and their count. */
int32_t nhip_decoder_greedy(nhip_decoder* m, const int32_t* prompt, int32_t prompt_len, int32_t max_new,
                            int32_t stop, int32_t* out_tokens, int32_t* out_len, nhip_decode_stats* stats);
/* Prefill `prompt` into slot 0, then beam search of `width` beams for up to
 * max_new tokens (length penalty 1, EOS `eos`); writes the winner's tokens
 * (without the prompt), its length and normalised score. */
int32_t nhip_decoder_beam_search(nhip_decoder* m, const int32_t* prompt, int32_t prompt_len, int32_t width,
                                 int32_t max_new, int32_t eos, int32_t* out_tokens, int32_t* out_len,
                                 float* out_score, nhip_decode_stats* stats);
int32_t nhip_decoder_destroy(nhip_decoder* m);

/* ------------------------------------------------- .cact archives (Model) -- */

/* Model.Open / Model.FromMemory (src/Needle/Model.cs:307-389, 400-411): the
 * archive is parsed in place and every tensor is uploaded to HBM once.  The
 * layout is the reference's (Model.cs:190-276 Record / Reader;
 * ModelInfo.cs:7-8 magic 0x05E12A84 and the 196-byte header): 48 uint32
 * header words + the RoPE theta float, header[2] codebook floats, header[1]
 * packed 44-byte records, then the data.  Malformed archives (Model.cs:372-389's
 * checks, plus each record's data inside the archive) give NHIP_ERR_FORMAT
 * before any device work.  Codebook-quantized records become weights for
 * nhip_matmul_cq_dev (2-bit book = Codebook.Fill(levels 0..3), 4-bit =
 * Codebook.Fill(levels 12..27)); fp16 / fp32 records become fp32 device
 * arrays (fp16 by Scalar.HalfToSingle); raw records (the tokenizer blob)
 * stay in the caller's bytes at record.offset.  The model holds no pointer
 * into the archive after nhip_open returns. */
enum { NHIP_CACT_FP16 = 1, NHIP_CACT_FP32 = 2, NHIP_CACT_CQ = 3, NHIP_CACT_RAW = 4 };

typedef struct nhip_record_info {
    int32_t dtype, ndim;
    uint32_t shape[4];
    uint64_t offset, bytes; /* in the archive */
    uint32_t group, bits;   /* codebook-quantized records: 128, 2 or 4 */
} nhip_record_info;

typedef struct nhip_model nhip_model;

int32_t nhip_open(const uint8_t* cact, size_t length, nhip_model** out);
/* header words [48] (geometry: Model.cs:65-105), RoPE theta, record count;
 * any output may be NULL */
int32_t nhip_model_info(const nhip_model* m, uint32_t* header48, float* rope_theta, int32_t* records);
int32_t nhip_model_record(const nhip_model* m, int32_t index, nhip_record_info* info);
/* the device weights of a codebook-quantized record, else NULL */
nhip_weights* nhip_model_weights(const nhip_model* m, int32_t index);
/* the fp32 device array of an fp16 / fp32 record, else NULL */
const float* nhip_model_dense(const nhip_model* m, int32_t index);
/* the record's bytes (indices, then fp16 norms) on the device, for row
 * gathers (Quant.GatherRow, src/Needle/Quant.cs:566-575), of a
 * codebook-quantized record, else NULL */
const uint8_t* nhip_model_raw(const nhip_model* m, int32_t index);
/* the archive's 2-bit and 4-bit codebooks (Model.cs:318-321); either may be NULL */
int32_t nhip_model_codebooks(const nhip_model* m, nhip_codebook* book2, nhip_codebook* book4);
int32_t nhip_model_close(nhip_model* m);

/* ----------------------------------- Needle 3 batched engine (step API) -- */

/* BatchedEngine over an opened Needle 3 archive (src/Needle/BatchEngine.cs:5-50,
 * EngineCore.ForwardBatch, src/Needle/Engine.cs:2285-2350): `slots` (1..16)
 * independent sequences of up to `capacity` positions each, steps of up to
 * `chunk` rows (0: the reference's default 64).  Attention splits a row's
 * span into at most `max_chunks` chunks by the reference's plan (0: 8, the
 * reference's MaxChunks, Blocks.cs:832).  Scratch is held for nhip_slot_feed's
 * long steps too, min(512, capacity) rows whatever the chunk (about 55 MB at
 * Needle 3's geometry).  The model must stay open while the
 * context lives.  One context is single-threaded; it owns a HIP stream and
 * its device state (KV cache, convolution and engram histories, snapshots). */
typedef struct nhip_ctx nhip_ctx;

int32_t nhip_ctx_create(const nhip_model* model, int32_t capacity, int32_t slots, int32_t chunk,
                        int32_t max_chunks, nhip_ctx** out);
int32_t nhip_ctx_destroy(nhip_ctx* c);
/* any output may be NULL */
int32_t nhip_ctx_info(const nhip_ctx* c, int32_t* vocab, int32_t* slots, int32_t* capacity, int32_t* chunk);
/* ForwardBatch (Engine.cs:2303-2350): row r feeds tokens[r] to slot
 * row_slots[r]; a slot's rows form one contiguous run at the slot's length +
 * their offset in it, and every slot's length grows by its run (NHIP_ERR_ARG
 * past the capacity, before any device work).  The LM head runs only over
 * head_rows[0..heads): output row i is row head_rows[i] -- logits
 * [heads][vocab] if non-NULL (BatchLogitsRow), the top-k ids and
 * log-probabilities [heads][k] if k > 0 (Ops.TopKLogSoftmax as
 * nhip_topk_lse_dev), Ops.ArgMax of each head row into argmax[heads] if
 * non-NULL.  Synchronous.  After a failed step the slots it named must be
 * reset. */
int32_t nhip_step(nhip_ctx* c, const int32_t* tokens, const int32_t* row_slots, int32_t rows,
                  const int32_t* head_rows, int32_t heads, float* logits, int32_t k, int32_t* topk_idx,
                  float* topk_lp, int32_t* argmax);
/* FeedSlot (Engine.cs:2285-2301): `count` tokens into one slot, logits [vocab]
 * of the last token if non-NULL.  Prompts longer than `chunk` go in equal steps
 * of up to 512 rows (fewer for a smaller context or very many attention
 * chunks), with the results of any other cut; if a token is out of range,
 * those before its chunk of `chunk` tokens are fed. */
int32_t nhip_slot_feed(nhip_ctx* c, int32_t slot, const int32_t* tokens, int32_t count, float* logits);
/* ResetSlot / MarkSlot / RewindSlot / SlotLength (BatchEngine.cs:24-29,
 * Engine.cs:2224-2283): reset clears the slot's histories and sets its length
 * and mark to 0; mark snapshots the histories and records the length; rewind
 * restores the snapshot and the length. */
int32_t nhip_slot_reset(nhip_ctx* c, int32_t slot);
int32_t nhip_slot_mark(nhip_ctx* c, int32_t slot);
int32_t nhip_slot_rewind(nhip_ctx* c, int32_t slot);
int32_t nhip_slot_length(const nhip_ctx* c, int32_t slot, int32_t* length);
/* Engine.CopyFrom (Engine.cs:367-379) between two slots of one context (a
 * beam reorder): dst becomes a clone of src -- KV positions [0, length of
 * src), histories, snapshot, previous tokens, length and mark. */
int32_t nhip_slot_copy(nhip_ctx* c, int32_t dst, int32_t src);

/* ------------------------------------------ synthetic workload inputs -- */

/* Deterministic host-side generators for the benchmark workloads: one
 * XorShift64 stream (tests/Needle.Tests/Conformance/Conformance.cs:10-38),
 * 53-bit uniforms, N(0,1) by Box-Muller, fp16 by round-to-nearest-even.
 * The state is updated in place. */
void nhip_synth_normal(uint64_t* state, float* x, size_t n);
void nhip_synth_uniform(uint64_t* state, float* x, size_t n, float lo, float hi);
void nhip_synth_int8(uint64_t* state, int8_t* x, size_t n);
void nhip_synth_half_uniform(uint64_t* state, uint16_t* x, size_t n, float lo, float hi);

#ifdef __cplusplus
}
#endif
#endif
