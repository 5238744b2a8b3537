/*
 * litemind_fp8.h -- C ABI of the 8-bit floating point (FP8) products of the
 * feed-forward path on one MI355X (gfx950): rows and weights in blocks that
 * share a scale, their matrix products, the products grouped by expert, and
 * the layers' path through them at one byte a weight.
 *
 * LiteMind computes in BF16 and fp32; nothing here has a counterpart in it.
 * Conventions are those of include/litemind_moe.h: int status, lm_last_error,
 * *_dev device pointers, work on the context stream, one host thread at a time
 * per context.
 *
 * Format.  Codes are OCP e4m3 (1 sign, 4 exponent, 3 mantissa bits, largest
 * 448, no infinity; uint8_t here, row-major, rows of `features` bytes).  A
 * block is 128 codes of a row, or 128 rows of 128; the last block of a row or
 * column may be smaller.  With the largest magnitude m of a block's finite
 * values its scale is s = max(m / 448, 2^-126) and the code of x the e4m3 nearest
 * to 448 x / m (to x 2^126 where s is 2^-126), ties to even, the quotient exact; a
 * code stands for code * s.  NaN and infinity become the NaN code 0x7f, and so reach
 * every product of theirs.  Scales are fp32, [row blocks][ceil(features / 128)].
 * Where two blocks meet in a product, their scales are multiplied in fp32 first:
 * past its range (blocks of 1e20 times others of 1e20) the output is infinite or
 * NaN, under it (1e-17 times 1e-17) bits are lost.
 *
 * lm_fp8_quantize, lm_fp8_gemm, lm_fp8_grouped_gemm and lm_fp8_grouped_swiglu
 * may be captured into a HIP graph on the context's stream; the products after
 * the context's first call of one of them (before it LM_EINVAL).  Replays share
 * the context's scratch: they run on the context's stream, or on another one
 * that waits for it and that it waits for.
 */
#ifndef LITEMIND_FP8_H
#define LITEMIND_FP8_H

#include "litemind_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define LM_FP8_BLOCK 128

/* x [rows][width] of `dtype` (LM_DT_F32, LM_DT_F16 or LM_DT_BF16), rows
 * row_stride elements apart (at least width), into q_dev [rows][width] codes and
 * scale_dev [ceil(rows / block_rows)][ceil(width / 128)].  block_rows is 1 (a
 * product's rows) or 128 (its weights).  rows under 2^31, of a matrix at most 2^23 -
 * 128 (more in several calls, from a multiple of 128 on); width at most 2^24,
 * row_stride 2^28; q_dev 16-byte aligned; the outputs overlap nothing.  Asynchronous. */
int lm_fp8_quantize(lm_context* ctx, const void* x_dev, int32_t dtype, int64_t rows, int64_t width, int64_t row_stride,
                    int32_t block_rows, uint8_t* q_dev, float* scale_dev);

/* out[r][n] = sum over blocks b of a_scale[r][b] * w_scale[n / 128][b] *
 *             sum over k in b of a[r][k] * w[n][k]
 *   a_dev [rows][in_features], a_scale_dev [rows][ceil(in_features / 128)]
 *   w_dev [out_features][in_features],
 *   w_scale_dev [ceil(out_features / 128)][ceil(in_features / 128)]
 *   out_dev [rows][out_features] of out_dtype (LM_DT_F32, LM_DT_F16, LM_DT_BF16)
 * Products are exact.  An fp32 output's sums are fp32; fp16 and BF16 outputs' are
 * so for few rows, and else (lm_fp8_plan_gemm's fp32_sums) those of the FP8 matrix
 * cores, off by 1.4e-5 to 4e-5 of their norm and at most 2^-10 of the sum of
 * magnitudes, rounded once at the end: one that is far smaller than its products
 * keeps less than its type's bits; where those count, the output is fp32.
 * in_features a multiple of 16 up to 2^20, out_features at most 2^24; rows, rows *
 * in_features and out_features * in_features under 2^31, 2^32 and 2^32.  A launch
 * has room for 2^22 tiles, of 128 rows by 256 features at most (16-bit outputs 256
 * by 256; every group begins one): LM_EINVAL past it.  a_dev, w_dev and out_dev
 * 16-byte aligned; out_dev overlaps no input.  Asynchronous. */
int lm_fp8_gemm(lm_context* ctx, const uint8_t* a_dev, const float* a_scale_dev, int64_t rows, const uint8_t* w_dev,
                const float* w_scale_dev, int64_t out_features, int64_t in_features, void* out_dev, int32_t out_dtype);

/* The rows of each expert, as lm_permute leaves them: group g has rows
 * offsets[g] .. offsets[g + 1] - 1, none of them where the two are equal.  All
 * arrays are device memory of the caller. */
typedef struct lm_fp8_groups {
    int32_t groups;         /* 1 .. 512 */
    int32_t divisor;        /* with source: at least 1; without: 0 */
    int64_t rows;           /* rows that the arrays hold: at least offsets[groups] */
    const int32_t* offsets; /* [groups + 1], 0 at first, rising */
    const int32_t* source;  /* NULL: row i reads row i of a.  Or [rows]: row source[i] / divisor
                               (lm_permute's perm and top_k: the token of each assignment) */
    const int32_t* target;  /* NULL: row i of the output.  Or [rows]: row target[i], each at most
                               once (lm_permute's perm: assignment order) */
} lm_fp8_groups;

/* lm_fp8_gemm with a matrix for each group: w_dev [groups][out_features]
 * [in_features] and w_scale_dev [groups][ceil(out_features / 128)]
 * [ceil(in_features / 128)].  a_dev has a_rows rows, out_dev out_rows; the sizes'
 * limits hold for a_rows and for each group's matrix.  Output rows that no row is
 * written to stay as they were.  Rows past `rows` and indexes outside a or out are
 * not followed: what they would read is taken as row 0, what they would write is
 * left out, and the next lm_synchronize or lm_copy_d2h returns LM_EKERNEL; so it
 * does for offsets that fall.  Asynchronous. */
int lm_fp8_grouped_gemm(lm_context* ctx, const lm_fp8_groups* groups, const uint8_t* a_dev, const float* a_scale_dev,
                        int64_t a_rows, const uint8_t* w_dev, const float* w_scale_dev, int64_t out_features,
                        int64_t in_features, void* out_dev, int64_t out_rows, int32_t out_dtype);

/* The gate and up products of each group's expert, SwiGLU, and the down
 * product's input blocks: w_dev [groups][2][inter][in_features] (gate, then up)
 * and w_scale_dev [groups][2][ceil(inter / 128)][ceil(in_features / 128)]; with
 * gate_i, up_i the two products of row i, both fp32,
 *     act_i = gate_i / (1 + exp(-gate_i)) * up_i
 * goes to row i of q_dev [rows][inter] and scale_dev [rows][ceil(inter / 128)] in
 * blocks of 1 x 128, by fp32's quotients: the code of a value within 2^-22 of the
 * middle between two may be the other.  The exponential is off by 2^-23 (2 +
 * |gate_i|) of itself, and 1 / (1 + exp(-gate_i)) under 2^-126 may be 0.  target must be NULL.  inter a multiple of 16 up to 2^20,
 * rows * inter and 2 * inter * in_features under 2^32; tiles of 128 rows by 128
 * channels at most; the rest as above.  Asynchronous. */
int lm_fp8_grouped_swiglu(lm_context* ctx, const lm_fp8_groups* groups, const uint8_t* a_dev, const float* a_scale_dev,
                          int64_t a_rows, const uint8_t* w_dev, const float* w_scale_dev, int64_t inter,
                          int64_t in_features, uint8_t* q_dev, float* scale_dev);

/* ---- which kernel ----
 * What lm_fp8_gemm (groups = 0), lm_fp8_grouped_gemm and lm_fp8_grouped_swiglu
 * launch for given sizes (rows: what the groups' arrays hold); host only, no context
 * or GPU.  Sizes that they refuse are LM_EINVAL. */
typedef struct lm_fp8_plan {
    int32_t tile_rows;     /* of a workgroup's tile */
    int32_t tile_features; /* 16 x 16: the kernel of few rows */
    int32_t shares;        /* workgroups that share a tile's reduced axis; more than 1: a second launch adds them up */
    int32_t fp32_sums;     /* 1: fp32 sums, 0: the FP8 matrix cores' */
    int32_t kernel;        /* which of the kernels of its kind, -1: that of few rows */
    int32_t reserved;
    int64_t tiles;         /* that the launch has room for, at most 2^22 */
} lm_fp8_plan;
int lm_fp8_plan_gemm(int32_t groups, int64_t rows, int64_t out_features, int64_t in_features, int32_t out_dtype,
                     lm_fp8_plan* out);
int lm_fp8_plan_swiglu(int32_t groups, int64_t rows, int64_t inter, int64_t in_features, lm_fp8_plan* out);

/* ---- the layers' FFNs at one byte a weight ----
 * After lm_finalize_layer: the layer's experts and shared experts, or its dense
 * FFN, in FP8 blocks of 128 x 128, from the BF16 weights.  LM_PATH_FP8 then runs
 * the layer in lm_moe_forward, lm_grouped_swiglu, lm_dense_forward,
 * lm_stack_forward and its graphs, lm_decoder_forward and
 * lm_paged_decoder_forward: router and weights of the experts as on the other
 * paths, the FFN's input and activations in blocks of 1 x 128, outputs fp32, the
 * sums of large batches those of the FP8 matrix cores.  The quantization is what
 * results differ by: a layer's outputs are off by 6.4e-2 of their norm.  A call
 * takes fewer tokens than 2^32 over the widest of H, a token's routed activations
 * (experts per token * moe_intermediate_size), the shared experts' and the dense
 * FFN's.
 *
 * only = 1 frees the layer's BF16 and fp16 weights (4 bytes a weight beside FP8's
 * 1: DeepSeek-V2's 236 GB fit one MI355X); the other paths are LM_ENOTRES then.
 * An upload into the layer ends its FP8 weights until the next lm_fp8_layer;
 * after only = 1 all its FFN weights are uploaded again.  H and the FFNs' widths
 * in multiples of 16 up to 2^20, gate and up together under 2^32 weights.
 * LM_EINVAL while the context's stream is being captured, and with only = 1 while
 * stack graphs are alive. */
int lm_fp8_layer(lm_context* ctx, int32_t layer, int32_t only);

/* What LM_PATH_FP8 launches for `tokens` tokens of a MoE layer (dense = 0) or of
 * a dense FFN; host only. */
typedef struct lm_fp8_layer_plan {
    lm_fp8_plan gate_up, down;             /* the routed experts' */
    lm_fp8_plan other_gate_up, other_down; /* the shared experts' or the dense FFN's, where they have launches of their own */
    int32_t beside;                        /* 1: the shared experts' tiles lie in the routed experts' launches */
    int32_t reserved;
} lm_fp8_layer_plan;
int lm_fp8_plan_layer(const lm_moe_config* config, int32_t dense, int64_t tokens, lm_fp8_layer_plan* out);

#ifdef __cplusplus
}
#endif
#endif
