/*
 * ridge_int8.h -- C ABI of the MI355X (gfx950) 8-bit operators: rows held in 8 bits
 * with one scale each, the operators that make them, and their matrix product.
 *
 * An 8-bit row stands for the values q[j] * scale: q is a whole number in -127 .. 127
 * and scale the row's largest magnitude over 127 (the smallest normal float, where it
 * would be less). The rows that are rounded are f32, and halves round to even: q is the
 * whole number next to 127 value / largest, not to the quotient by the scale's f32, which
 * is off by its own rounding (half of the largest value, 63.5, is 64 in every row):
 *   quantize:  the rows as they are;
 *   silu_mul:  g / (1 + exp(-g)) * u of a row that holds g and then u;
 *   rms_norm:  s / sqrt(mean(s^2) + eps) * weight of s = x + residual.
 * A row that holds a NaN or an infinity has a scale that is one: nothing of it comes
 * back finite. So does a norm's row whose sum of squares passes the range of f32.
 *
 * The product of rows A [M, K] and rows B [N, K] (a weight's output channels) is
 *   C[m, n] = (sum over k of A[m, k] B[n, k]) scaleA[m] scaleB[n] + bias[n],
 * the sum exact in 32-bit integers, the rest in f32, rounded once to C's type.
 *
 * Conventions, those of ridge_gemm.h: the caller allocates everything on the device; a
 * call neither allocates nor synchronises and is asynchronous on `stream` (NULL: the
 * default stream); errors come back as hipError_t values, and a refused call
 * (hipErrorInvalidValue, 1) enqueues nothing. Types are RIDGE_F16, RIDGE_BF16 or
 * RIDGE_F32. A stride (ld*) is the distance of rows in elements, at least the row's
 * length; strides and pointers of 16- and 32-bit matrices need the alignment of their
 * type only. 8-bit rows start at multiples of 16 bytes (pointer and stride), and their
 * last 16 bytes are readable: what they hold behind the row's length does not matter.
 * What a call writes shares no byte with anything else of the call, residualOut excepted
 * where its comment says so: workgroups run in any order, and this is not checked here.
 * No rows is a call that does nothing; a row of no columns is refused.
 *
 * No HIP header is needed to use this file: streams are passed as void*.
 */
#ifndef RIDGE_INT8_H
#define RIDGE_INT8_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { RIDGE_F16 = 0, RIDGE_BF16 = 1, RIDGE_F32 = 2 };

/* Largest K of a product, whose sum of K products of 8 bits still fits 32. */
enum { RIDGE_INT8_MAX_K = 131071 };

/* A stride for 8-bit rows of cols columns, at which the product reads them fastest:
 * multiples of 128 bytes for rows of more than 512, whose pieces then lie in whole cache
 * lines (212 x 6684 x 12772 44.1 us, in rows 12784 bytes apart 62.4), of 16 for shorter
 * ones, which would grow too much. */
int64_t ridge_int8_row_stride(int64_t cols);

/* q, scale <- x [rows, cols] of `type`. */
int ridge_int8_quantize(const void* x, int64_t ldx, int type, int8_t* q, int64_t ldq, float* scale, int64_t rows,
                        int64_t cols, void* stream);

/* q [rows, cols], scale <- x [rows, 2 cols] of `type`: g its first cols columns, u the others. */
int ridge_int8_silu_mul(const void* x, int64_t ldx, int type, int8_t* q, int64_t ldq, float* scale, int64_t rows,
                        int64_t cols, void* stream);

/* q, scale <- the norm of x + residual, times weight [cols] (of `type` or RIDGE_F32); and
 * residualOut <- x + residual, rounded to `type`. residual and residualOut are both null
 * for a norm of x alone. residualOut may be x or residual itself, at the same stride. */
int ridge_int8_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ldResidual, const void* weight,
                        int weightType, float eps, int type, void* residualOut, int64_t ldResidualOut, int8_t* q,
                        int64_t ldq, float* scale, int64_t rows, int64_t cols, void* stream);

/* out [rows, cols] of `type` <- q * scale, in f32, rounded once. */
int ridge_int8_dequantize(const int8_t* q, int64_t ldq, const float* scale, void* out, int64_t ldOut, int type,
                          int64_t rows, int64_t cols, void* stream);

/* C [M, N] of `type` <- the product above; bias [N] of `type`, or null. K is at most
 * RIDGE_INT8_MAX_K, an 8-bit stride below 2^23, and C at most 2^23 - 1024 tiles of 256 x
 * 256. */
int ridge_int8_gemm(const int8_t* A, int64_t lda, const float* scaleA, const int8_t* B, int64_t ldb,
                    const float* scaleB, const void* bias, void* C, int64_t ldc, int type, int64_t M, int64_t N,
                    int64_t K, void* stream);

/* Which of its forms a product of contiguous rows runs in: 0 .. 5 tiles of 256x256,
 * 256x128, 128x128, 128x128 (two on a CU), 64x128 and 64x64; 6 .. 8 tiles of 16x16, 32x16
 * and 32x32 whose K a workgroup's waves share. -1 for sizes that ridge_int8_gemm refuses or
 * that hold no element. No device is touched. */
int ridge_int8_gemm_form(int64_t M, int64_t N, int64_t K);

#ifdef __cplusplus
}
#endif

#endif /* RIDGE_INT8_H */
