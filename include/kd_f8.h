/*
 * kd_f8.h - C ABI of the gfx950 linear layers in 8-bit floating point, and
 * of what makes their operands: rows held as e4m3 codes with one
 * power-of-two scale for each block of 128 consecutive values.  Exported by
 * libkd_fa.so next to kd_mm.h, whose product they stand beside: the same
 * Linear node (ops::linear, src/core/ops.hpp:27-43) at half the weight bytes
 * of BF16 and twice the matrix rate.  Three operators:
 *
 *   kd_f8_quantize   rows of F32, BF16 or F16 -> codes and scales (a weight
 *                    once, at model load; an activation ahead of a layer)
 *   kd_f8_norm_run   residual addition and RMS norm (RMSNorm,
 *                    src/core/module.hpp:163-180) with codes and scales out
 *   kd_f8_mm_run     the product of two operands in that form, plus bias
 *
 * The format.  A row of K values (K % 16 == 0) has ceil(K / 128) blocks, the
 * last one K % 128 long where that is not 0.  value = code * scale with
 *   code   e4m3 (OCP: 4 exponent bits, 3 of mantissa, largest 448, no
 *          infinities)
 *   scale  E8M0: byte b stands for 2^(b - 127), 255 for NaN
 * A block y of finite values gets the scale 2^e with e the smallest integer
 * >= -127 for which max|y| <= 448 * 2^e, and the codes y * 2^-e rounded to
 * the nearest e4m3 value (ties to even).  A block that holds an infinity or
 * a NaN gets the scale NaN and NaN codes throughout.  Since codes are
 * floating point, a power of two as scale costs them no precision above the
 * smallest exponent, and the matrix cores multiply by it at no cost.
 *
 * Tensor views are kd_fa_tensor (ggml's type / ne / nb / data); ggml has no
 * type ids for the two 8-bit types, so theirs lie outside its range.  Rows
 * [.., M, M2, M3] are flattened as kd_mm.h's (nb[2] = nb[1] * ne[1], nb[3] =
 * nb[2] * ne[2]).  The scales of a row are bytes in block order, each row at
 * a multiple of 4 bytes; the product reads them in aligned words, so up to 3
 * bytes behind a row's last scale, in the same word, are read (not used).
 *
 * All device pointers belong to the caller; nothing is allocated, freed,
 * synchronised or retained, and each call is one kernel on the given HIP
 * stream, so calls may be captured into a graph and may run side by side.
 * Outputs must not overlap inputs, but for kd_f8_norm_run's sum, which may
 * be its x or its residual (the same view).  Equal calls give equal bits.
 * Calls with no rows (or no outputs) do nothing.  Inference only: there is
 * no gradient.  Status codes are the KD_FA_* codes of kd_fa.h.
 */
#ifndef KD_F8_H
#define KD_F8_H

#include "kd_fa.h"

#ifdef __cplusplus
extern "C" {
#endif

enum {
    KD_F8_TYPE_F32  = 0,
    KD_F8_TYPE_F16  = 1,
    KD_F8_TYPE_BF16 = 30,
    KD_F8_TYPE_E4M3 = 4096,
    KD_F8_TYPE_E8M0 = 4097
};

/* values of one scale */
#define KD_F8_BLOCK 128

/* Rows in 8 bits. */
typedef struct kd_f8_rows {
    kd_fa_tensor codes;    /* E4M3 [K, M, M2, M3], rows 16-byte aligned               */
    kd_fa_tensor scales;   /* E8M0 [ceil(K / 128), M, M2, M3], rows 4-byte aligned     */
} kd_f8_rows;

/* kd_f8_quantize: out = x in 8 bits. */
typedef struct kd_f8_quantize_desc {
    kd_fa_tensor x;        /* F32, BF16 or F16 [K, M, M2, M3], rows 16-byte aligned    */
    kd_f8_rows   out;
} kd_f8_quantize_desc;

/*
 * kd_f8_norm_run: for each row
 *   s = x + residual in F32, rounded to sum's type (x itself without one)
 *   y = s / sqrt(mean(s^2) + eps) * weight, the mean summed in double and y
 *       rounded to F32 (within 2^-23 of it)
 * sum = s, out = y in 8 bits.  residual and sum come together: both given or
 * neither (data == NULL).
 */
typedef struct kd_f8_norm_desc {
    kd_fa_tensor x;        /* F32 or BF16 [K, M, M2, M3], rows 16-byte aligned         */
    kd_fa_tensor residual; /* F32 or BF16, as x; or data == NULL                       */
    kd_fa_tensor weight;   /* F32 [K], 16-byte aligned                                 */
    kd_fa_tensor sum;      /* residual's type, as x; or data == NULL                   */
    kd_f8_rows   out;
    float        eps;      /* finite, >= 0                                             */
} kd_f8_norm_desc;

/*
 * kd_f8_mm_run: dst[m][n] = sum_k w[n][k] * x[m][k] (+ bias[n]), rounded to
 * BF16.  The products and their sums are the matrix cores': within 16
 * consecutive k of a block the products are added with 13 bits below the
 * largest of them (what lies lower is cut off), and everything else in F32.
 * That leaves sums of normally distributed values 1.6e-5 off (relative, in
 * norm), a hundredth of dst's own rounding; it is why dst is not offered in
 * 32 bits.  The order of a row's sum depends on M, N and K, as kd_mm_run's.
 */
typedef struct kd_f8_mm_desc {
    kd_f8_rows   w;        /* [K, N]                                                   */
    kd_f8_rows   x;        /* [K, M, M2, M3]                                           */
    kd_fa_tensor bias;     /* F32 [N], 16-byte aligned; or data == NULL                */
    kd_fa_tensor dst;      /* BF16 [N, M, M2, M3], N % 4 == 0, rows 8-byte aligned     */
} kd_f8_mm_desc;

/*
 * Each *_supports returns 1 when its operator can execute the descriptor,
 * else 0 with the first failed condition's KD_FA_ERR_* code in *reason (when
 * reason != NULL).  Host-only.  K is at most 32768 for kd_f8_norm_run, whose
 * rows stay in registers.
 */
int kd_f8_quantize_supports(const kd_f8_quantize_desc *desc, int *reason);
int kd_f8_norm_supports(const kd_f8_norm_desc *desc, int *reason);
int kd_f8_mm_supports(const kd_f8_mm_desc *desc, int *reason);

/*
 * Enqueue the operator on `stream` (a hipStream_t).  Each returns KD_FA_OK
 * or a negative KD_FA_ERR_* code, in which case nothing is enqueued.
 */
int kd_f8_quantize(const kd_f8_quantize_desc *desc, void *stream);
int kd_f8_norm_run(const kd_f8_norm_desc *desc, void *stream);
int kd_f8_mm_run(const kd_f8_mm_desc *desc, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* KD_F8_H */
