/*
 * snipper_fp8.h -- C ABI of the 8-bit block-scaled products and of the layer norm of rows of any width.
 *
 * The 8-bit operators stand beside the bf16 products of snipper_dense.h: the Linears of the transformer
 * (models/deformable_transformer.py:194-198, models/ops/modules/ms_deform_attn.py:60-66) with both operands in 8 bits.
 * The layer norm stands beside snipper_add_dropout_layernorm_*: any width up to 16384, float16 too, strided rows.
 *
 * THE FORMAT ("blocks").  A matrix [R][C] is held as
 *   data   [R][P]  bytes, P = 128 * ceil(C / 128), zeros behind the last column;
 *   scale  [R][Q]  bytes, Q = 4 * ceil(C / 512): byte b of a row is the biased exponent e + 127 of the scale 2^e of the row's
 *                  elements 128 b .. 128 b + 127; 127 (2^0) behind the last block.  255 stands for NaN.
 * Element (r, c) is data[r][c] * 2^e.  fmt 0 = e4m3 (largest value 448), 1 = e5m2 (57344, infinities).
 * The quantizers choose the smallest e >= -127 with (largest finite magnitude of the block) / 2^e <= the type's largest value, so
 * nothing saturates; a block of zeros has e = 0; elements are rounded to nearest, ties to even.  A NaN stays a NaN, an infinity
 * becomes an infinity (e5m2) or a NaN (e4m3): neither has a say in the scale.
 *
 * Conventions of snipper_msda.h: device pointers, `stream` = hipStream_t as void*, 0 = success, negative SNIPPER_E_* for rejected
 * arguments, positive hipError_t otherwise; nothing is allocated, nothing synchronises, calls can be captured into a graph.
 * Element types: 0 = float32, 1 = bfloat16, 3 = float16.  Sums are held in float32.
 */
#ifndef SNIPPER_FP8_H_
#define SNIPPER_FP8_H_

#include <stddef.h>
#include <stdint.h>
#include "snipper_msda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* x [rows][cols] (row stride ldx elements) into blocks.  tile_rows = 1: a scale for each 128 elements of a row (data / scale) and,
 * if data_t is given, for each 128 elements of a column (data_t / scale_t: the blocks of the transposed matrix [cols][rows]).
 * tile_rows = 128: one scale for each 128 x 128 tile, the same in both forms.  Either form may be NULL, not both.
 * mean / rstd [rows] float32 (or both NULL): x is normalised first, (x - mean) * rstd * gamma + beta, gamma / beta [cols] of type
 * p_dtype or NULL (1 / 0); with tile_rows = 1 only.
 * Data pointers 16-byte, scale pointers 4-byte aligned.
 * colsum [cols] of type colsum_dtype or NULL: the sums of x over the rows, of the unrounded elements, in float32 and a fixed order;
 * needs snipper_fp8_quantize_workspace_bytes of workspace (0 without it), 4-byte aligned.  rows, cols <= 2^23. */
size_t snipper_fp8_quantize_workspace_bytes(int rows, int cols, int with_colsum);
int snipper_fp8_quantize(void *stream, const void *x, int x_dtype, long long ldx, int rows, int cols, int tile_rows, int fmt,
                         const float *mean, const float *rstd, const void *gamma, const void *beta, int p_dtype,
                         uint8_t *data, uint8_t *scale, uint8_t *data_t, uint8_t *scale_t, void *colsum, int colsum_dtype,
                         void *workspace, size_t workspace_bytes);

/* out [M][N] = act(A [M][K] . B [N][K]^T + bias [N]) of two matrices in blocks; act = ReLU if relu, bias of type bias_dtype or NULL.
 * A, B and out 16-byte, scale pointers 4-byte aligned.  out [M][N] contiguous, of type out_dtype.
 * A bfloat16 / float16 result comes from the 8-bit matrix instructions.  They add the products of eight neighbours of a row after
 * aligning them to the largest of the eight, and cut each off at 2^-13 of it; all further sums are float32.  So an element is off by
 * less than 7 * 2^-13 (8.5e-4) of the sum of the groups' largest magnitudes, hence of sum |a b|, before it is rounded (half a step of
 * bfloat16 is 2^-8, of float16 2^-11); 1.5e-5 of the result's norm on random data, whatever K.
 * A float32 result comes from the bfloat16 instructions on exactly converted operands (1e-7), at a quarter of the rate; so does a 16-bit
 * one of up to 16 rows, or with out_dtype | SNIPPER_FP8_FULL_SUMS.
 * Both hold for scales from end to end of their range: what counts is the size of the products.  M, N, K <= 2^23, M N < 2^40. */
#define SNIPPER_FP8_FULL_SUMS 16
size_t snipper_fp8_matmul_workspace_bytes(int M, int N, int K, int out_dtype);
int snipper_fp8_matmul(void *stream, const uint8_t *A, const uint8_t *a_scale, int a_fmt, const uint8_t *B, const uint8_t *b_scale,
                       int b_fmt, int M, int N, int K, const void *bias, int bias_dtype, int relu, void *out, int out_dtype,
                       void *workspace, size_t workspace_bytes);

/* y = (x - mean) * rstd * gamma + beta over rows of `cols` elements, rstd = 1 / sqrt(variance + eps).  x, y of type x_dtype, x rows
 * ldx apart, y contiguous; gamma / beta of type p_dtype, each may be NULL (1 / 0).  mean / rstd [rows] float32 or both NULL.
 * data / scale (or both NULL): the result as blocks (fmt), from the unrounded values.  y may be NULL where one of the other
 * outputs is wanted.  rows <= 2^31 - 1, cols <= 16384. */
int snipper_layernorm_forward(void *stream, const void *x, int x_dtype, long long ldx, const void *gamma, const void *beta,
                              int p_dtype, int rows, int cols, float eps, void *y, float *mean, float *rstd, uint8_t *data,
                              uint8_t *scale, int fmt);

/* The adjoint: dx (type x_dtype, contiguous) or NULL, dgamma / dbeta [cols] of type p_dtype or both NULL (fully written, also for
 * rows = 0; fixed order of summation).  g of type x_dtype, contiguous. */
size_t snipper_layernorm_backward_workspace_bytes(int rows, int cols);
int snipper_layernorm_backward(void *stream, const void *g, const void *x, int x_dtype, long long ldx, const float *mean,
                               const float *rstd, const void *gamma, int p_dtype, int rows, int cols, void *dx, void *dgamma,
                               void *dbeta, void *workspace, size_t workspace_bytes);

#ifdef __cplusplus
}
#endif
#endif
