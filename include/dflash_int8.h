/*
 * dflash_int8.h — projections in 8-bit integers: weights quantised once per
 * output channel, rows per token, the product exact in 32-bit integers.
 * Conventions (return codes, streams, no allocation, no synchronisation) are
 * those of dflash_gdn.h.
 *
 * Quantisation of a row x of K values (an output channel of a weight, or a
 * token's features): a = max(max |x|, 2^-100), scale = a / 127 (fp32), code =
 * rint(127 x / a), ties to even, as real arithmetic gives it: never a code off
 * for inputs of bf16 or fp16.  A row that holds a NaN or an infinity has scale
 * NaN and codes 0.
 *
 * Product: out[m][n] = (sum_k x[m][k] w[n][k]) * w_scale[n] * x_scale[m], the sum
 * exact, the factors in fp32 in this order (rows near the type's largest value stay
 * finite), rounded once to the output's type.
 * gated (the MLP's gate and up projections stacked, N even): out[m][j] =
 * silu(g) * u with g and u the products of channels j and N / 2 + j, in fp32.
 *
 * A packed weight holds the codes as the matrix unit's fragments, [K / 64 steps]
 * [channel tiles of 16][64 lanes][16 bytes]: lane l of a fragment is channel
 * l % 16, k = 16 (l / 16) .. + 15 of the step; K padded with zeros to a multiple
 * of 128.  Channel tiles are in order, the last one padded with zeros; of a gated
 * weight tile 2 j holds channels 16 j .. + 15 of the gate and tile 2 j + 1 those
 * of up, each half padded for itself.  scales: fp32, 16 a tile, padded with zeros.
 */
#ifndef DFLASH_INT8_H
#define DFLASH_INT8_H

#include "dflash_gdn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Largest K: |sum| < 2^31, for any codes below it, and at it if no code of the weight is -128
 * (quantised ones are -127 to 127). */
#define DFLASH_I8_MAX_K 131072
/* Largest N: offsets of channel scales fit 32 bits. */
#define DFLASH_I8_MAX_N 268435456

/* Bytes of a packed weight's codes, and the count of its scales; 0: a size is out of
 * range (1 <= N <= DFLASH_I8_MAX_N, 1 <= K <= DFLASH_I8_MAX_K, N even if gated). */
size_t dflash_weight_i8_bytes(int N, int K, int gated);
size_t dflash_weight_i8_scales(int N, int gated);

/* Pack int8 codes [N, K] (rows row_stride bytes apart) and scales [N]. */
int dflash_weight_pack_i8(const void* codes, int64_t row_stride, const float* scale, void* packed_codes,
                          float* packed_scale, int N, int K, int gated, void* stream);

/* Codes [M, K] (codes_row_stride bytes apart, a multiple of 16 and at least K rounded
 * up to 16; the bytes from K up to there are written as 0) and scales [M] of rows x (bf16
 * or fp16, x_row_stride elements apart). */
int dflash_quantize_rows_i8(const void* x, int x_dtype, int64_t x_row_stride, void* codes,
                            int64_t codes_row_stride, float* scale, int M, int K, void* stream);

/* The product of codes x [M, K] (16-byte aligned, rows x_row_stride bytes apart, a multiple
 * of 16 and at most 2^23; rows are read up to K rounded up to 16, whatever is there) with a packed
 * weight.  out: bf16, fp16 or fp32, out_row_stride elements apart, at least N
 * (gated: N / 2) and at most 2^26.
 * workspace: dflash_gemm_i8_workspace_bytes(M, N, K, gated) bytes (for the current device; may be
 * 0), 16-byte aligned. */
size_t dflash_gemm_i8_workspace_bytes(int M, int N, int K, int gated);
int dflash_gemm_i8(const void* x, int64_t x_row_stride, const float* x_scale, const void* packed_codes,
                   const float* packed_scale, void* out, int out_dtype, int64_t out_row_stride, int M, int N,
                   int K, int gated, void* workspace, size_t workspace_bytes, void* stream);

/* The residual add and RMSNorm before a projection, with the rows quantised for it
 * (custom_qwen35_model.py:824-827, 841-845): h_out = bf16(h + r), row by row x = bf16(h_out *
 * rsqrt(mean(h_out^2) + eps) * weight), codes and scales of x as dflash_quantize_rows_i8 gives
 * them.  All of [M, H] bf16, contiguous; h_out may be h; r null: no add.  capture: null, or h_out
 * again, capture_stride elements a row (a multiple of 8).  H a multiple of 16, at most 32768;
 * every pointer 16-byte aligned. */
int dflash_add_rmsnorm_i8(const void* h, const void* r, const void* weight, void* h_out, void* capture,
                          int64_t capture_stride, void* codes, int64_t codes_row_stride, float* scale, int M,
                          int H, float eps, void* stream);

/* Both in one call: rows x (bf16 or fp16) quantised and multiplied, the same bits.  workspace:
 * dflash_linear_i8_workspace_bytes(M, N, K, gated) bytes (for the current device), 16-byte
 * aligned.  out lies apart from x (and from the codes, in the call above): a row may be read
 * while outputs are stored. */
size_t dflash_linear_i8_workspace_bytes(int M, int N, int K, int gated);
int dflash_linear_i8(const void* x, int x_dtype, int64_t x_row_stride, const void* packed_codes,
                     const float* packed_scale, void* out, int out_dtype, int64_t out_row_stride, int M, int N,
                     int K, int gated, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
