/*
 * emmyrt_ops -- operators of a served decoder layer for sm_100a, launched through a C ABI.
 *
 * They stand beside the modules that the compiler emits: a problem's IR covers RMSNorm, a
 * rotation by given cosines, attention over 16-bit keys or a per-tensor FP8 product; these
 * entry points cover the forms of the same operators that serving a decoder layer needs
 * (residual norms in one pass, rotary positions from their angles, a paged 4-bit cache and
 * the attention over it, FP8 products with a scale for each block of 128).
 *
 * Conventions (those of emmyrt.h)
 *   - every entry point returns 0, a cudaError_t value (> 0) of the failing call, or a
 *     negative EMMY_RT_E* code; emmy_ops_last_error() then has the text (per thread);
 *   - rows of an operand do not overlap, but those of an input may all be one (a stride of 0);
 *   - arguments are checked before anything is enqueued, as far as the host can see them;
 *     device pointers are 64-bit handles, strides are in elements, element types are
 *     EMMY_OPS_* codes;
 *   - work is enqueued on `stream` (0 = the legacy default stream) of `device`, which is made
 *     current for the call; nothing is allocated, nothing waits for the device, so every
 *     call can be captured into a CUDA graph;
 *   - workspaces belong to the caller; calls that share one must not overlap on the GPU.
 */
#ifndef EMMYRT_OPS_H
#define EMMYRT_OPS_H

#include <stdint.h>

#include "emmyrt.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
#define EMMY_OPS_F32  0
#define EMMY_OPS_F16  1
#define EMMY_OPS_BF16 2

const char *emmy_ops_last_error(void);

/* The ordinal of the calling thread's current device. */
int emmy_ops_current_device(int *device);

/* ---- norms after and before a block, with its gate and residual scale ------------------ */

#define EMMY_OPS_NORM_RMS   0
#define EMMY_OPS_NORM_LAYER 1

#define EMMY_OPS_NORM_MAX_DIM 16384

/* y = x + scale * gate * N(block; post),  h = N(y; pre)   (y in h's norm is not yet rounded)
 *
 *   N(v; w, b) = v / sqrt(mean(v^2) + eps) * w + b             EMMY_OPS_NORM_RMS
 *   N(v; w, b) = (v - mean v) / sqrt(var v + eps) * w + b       EMMY_OPS_NORM_LAYER
 *
 * post_norm 0: N(block) is block itself.  gate: row r / rows_per_gate of [gates, dim], 0 for
 * none.  Weights and biases: [dim] each or 0 (1 and 0).  h 0: only y.  y may be x and h may be
 * block, element for element; other overlaps are the caller's error. */
typedef struct {
    uint64_t x, block, y, h;
    int64_t x_stride, block_stride, y_stride, h_stride;   /* elements from row to row */
    uint64_t post_weight, post_bias, gate, pre_weight, pre_bias;
    int64_t gate_stride, rows_per_gate, rows, dim;
    int32_t dtype;                                        /* of x, block, y, h */
    int32_t post_weight_dtype, post_bias_dtype, gate_dtype, pre_weight_dtype, pre_bias_dtype;
    int32_t kind, post_norm;
    float eps, scale;
} emmy_ops_norm_args;

int emmy_ops_residual_norm(const emmy_ops_norm_args *a, int device, uint64_t stream);

/* ---- rotary positions -------------------------------------------------------------------- */

#define EMMY_OPS_ROTARY_HALF        0   /* pair i: elements i and i + rotary / 2  */
#define EMMY_OPS_ROTARY_INTERLEAVED 1   /* pair i: elements 2 i and 2 i + 1        */

/* Turns pair i of every head of token t by positions[t] * turns[i] / 2^64 of a full turn and
 * multiplies it by magnitude; elements from `rotary` on are copied.  transpose != 0 turns the
 * other way, which is the gradient's map.  Cosines and sines are f32 of the turn's upper 24 bits (off by up to
 * 2^-25 of half a turn, whatever the position).  x[1] (tokens, heads[1], dim) is optional (0 heads).
 * out may be x; other overlaps are the caller's error. */
typedef struct {
    uint64_t x[2], out[2];
    int64_t x_token[2], x_head[2], out_token[2], out_head[2];   /* strides in elements */
    int32_t heads[2];
    uint64_t positions, turns;          /* int32 or int64 [tokens]; uint64 [rotary / 2] */
    int64_t tokens;
    int32_t positions_64, dtype, dim, rotary, layout, transpose;
    float magnitude;
} emmy_ops_rotary_args;

int emmy_ops_rotary(const emmy_ops_rotary_args *a, int device, uint64_t stream);

/* ---- FP8 (e4m3) products with a scale for each block of 128 --------------------------------- */

/* q = e4m3(x / s), s = amax / 448 (1 where that is 0), over 128 columns of a row (square 0:
 * s is [blocks of columns][rows]) or over 128 x 128 (square 1: s is [blocks of rows][blocks of
 * columns]).  Rows of q are a multiple of 16 bytes apart; without square, columns up to the
 * next multiple of 16 become zero, those of the last row too.  A single row whose q_stride is less
 * than that has no such columns. */
typedef struct {
    uint64_t x, q, s;
    int64_t x_stride, q_stride, s_stride, rows, cols;
    int32_t dtype, square;                    /* dtype of x */
} emmy_ops_blockfp8_quantize_args;

int emmy_ops_blockfp8_quantize(const emmy_ops_blockfp8_quantize_args *a, int device, uint64_t stream);

/* y[m, n] = sum over blocks b of xs[b, m] ws[n / 128, b] sum over k in b of xq[m, k] wq[n, k], in
 * f32, as quantised above (xq without square, its padding zero, rows of xs a multiple of 4 apart; wq
 * with).  *status (a word of
 * device memory, zeroed by the caller once) gets a bit when a wait inside the kernel gave
 * up after 2 s; y is then not valid.  parts (0: none, else on 16 bytes) is memory for the parts of a
 * product that is cut along k where y alone has too few tiles for the GPU: 16 times m rows of f32, n
 * rounded up to a multiple of 4, serve every cut; a cut that they do not hold is not made. */
typedef struct {
    uint64_t xq, xs, wq, ws, y, status, parts, parts_bytes;
    int64_t xq_stride, xs_stride, wq_stride, ws_stride, y_stride, m, n, k;
    int32_t dtype, reserved;                  /* dtype of y */
} emmy_ops_blockfp8_args;

int emmy_ops_blockfp8_product(const emmy_ops_blockfp8_args *a, int device, uint64_t stream);

/* Both in a row: x (m x k, of x_dtype) quantised into product.xq and product.xs, then the product. */
typedef struct {
    emmy_ops_blockfp8_args product;
    uint64_t x;
    int64_t x_stride;
    int32_t x_dtype, reserved;
} emmy_ops_blockfp8_linear_args;

int emmy_ops_blockfp8_linear(const emmy_ops_blockfp8_linear_args *a, int device, uint64_t stream);

/* ---- a paged key / value cache in 4 bits -------------------------------------------------- */

/* Levels [pages, heads, page, dim / 2] bytes (element 2 i in the low half of byte i) and
 * [pages, heads, page, 2] f16 pairs (step, least): an element stands for level * step + least.
 * dim is 64 or 128. */
typedef struct {
    uint64_t k, v, k_meta, v_meta;
    int64_t pages;
    int32_t heads, page, dim;
} emmy_ops_cache4;

/* Quantises n tokens' keys and values into the cache's slots (page * page_size + row).  A
 * token whose slot is negative or past the cache is left out.  Two tokens of one call must
 * not have the same slot.  k_stored / v_stored (0: not wanted, else contiguous
 * [n, heads, dim] of dtype) receive what the cache then stands for. */
typedef struct {
    emmy_ops_cache4 cache;
    uint64_t k, v, slots, k_stored, v_stored;   /* slots: int32 or int64 [tokens] */
    int64_t k_token, k_head, v_token, v_head, tokens;
    int32_t slots_64, dtype;
} emmy_ops_cache4_append_args;

int emmy_ops_cache4_append(const emmy_ops_cache4_append_args *a, int device, uint64_t stream);

/* Attention of `tokens` queries a sequence over its cached positions: query i of sequence b
 * stands at position lengths[b] - tokens + i and sees the positions up to its own; one that
 * sees nothing gives zeros.  q and out are (batch, tokens, q_heads, dim), the last one
 * contiguous; q_heads / cache.heads query heads share a head of the cache.  Sequence b's
 * positions lie in the pages table[b * table_stride ..] (max_pages of them); lengths beyond
 * them are cut there, and nothing is seen of a page that is no page of the cache.  The workspace is emmy_ops_cache4_attend_workspace bytes; nothing in it is kept
 * from call to call. */
typedef struct {
    emmy_ops_cache4 cache;
    uint64_t q, out, table, lengths, workspace, workspace_bytes;   /* table, lengths: int32 */
    int64_t q_batch, q_token, q_head, out_batch, out_token, out_head, table_stride;
    int32_t batch, tokens, q_heads, max_pages, dtype;
    float scale;
} emmy_ops_cache4_attend_args;

int emmy_ops_cache4_attend_workspace(int dim, int device, uint64_t *bytes);
int emmy_ops_cache4_attend(const emmy_ops_cache4_attend_args *a, int device, uint64_t stream);

#ifdef __cplusplus
}
#endif

#endif /* EMMYRT_OPS_H */
