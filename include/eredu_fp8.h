/*
 * eredu_fp8.h -- C ABI of the linears in 8-bit floating point with block scales
 * (gfx950), in the same library and under the same conventions as eredu_hip.h:
 * borrowed device pointers, kernels enqueued on `stream` without synchronising,
 * 0 or an error with eq_last_error()'s message, arguments checked before
 * anything is launched.
 */
#ifndef EREDU_FP8_H
#define EREDU_FP8_H

#include "eredu_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * A value is an e4m3 code (one sign, four exponent and three mantissa bits,
 * largest 448, no infinities, 0x7f and 0xff NaN) times an f32 scale.  Weights
 * [n, k] have a scale for each block of 128 x 128, scales [ceil(n / 128),
 * ceil(k / 128)], as checkpoints of block-scaled projections store them (the
 * reference's block-FP8 linears, eredu/src/backend/mlx/nn/fp8.rs).  Activations
 * [rows, k] have one for each 128 columns of a row; they are stored block by
 * block, all rows of a block side by side: the scale of row r and block b is
 * scales[b * scale_stride + r], scale_stride >= rows.  The last block of an
 * axis may be smaller.
 *
 * A group of values v is quantized to the scale max|v| / 448, at least 2^-126,
 * and the codes 448 v / max|v| rounded to the nearest, ties to even: once where v has 16 bits; of f32
 * values the quotient is off by up to 3 * 2^-24 of itself before.  Where a value of the
 * group is not finite, its scale is NaN and its codes are 0.
 *
 * dtypes: f32, f16 or bf16 (EQ_DTYPE_*).  Row lengths (cols, dim, k) are
 * multiples of 16 below 2^22, pointers to rows 16-byte aligned, row strides (in
 * elements, below 2^23) multiples of 16 bytes; a call has fewer than 2^26 groups of 128
 * columns of rows, eq_fp8_quantize_weight fewer than 2^22 blocks of 128 x 128.  EQ_DTYPE_F8E4M3
 * names codes as the type of x.
 */
#define EQ_DTYPE_F8E4M3 4

/* codes [rows, cols] and scales of x (row r at element r * x_stride). */
int eq_fp8_quantize(void* codes, float* scales, int64_t scale_stride, const void* x, int64_t x_stride, int64_t rows,
                    int64_t cols, int dtype, eq_stream_t stream);

/* codes [count, rows, cols] and scales [count, ceil(rows / 128), ceil(cols / 128)]
 * of `count` weights w [rows, cols]. */
int eq_fp8_quantize_weight(void* codes, float* scales, const void* w, int64_t count, int64_t rows, int64_t cols,
                           int dtype, eq_stream_t stream);

/* hidden += residual (rounded to dtype; NULL: none), then codes and scales of
 * hidden / sqrt(mean(hidden^2) + eps) * weight over its rows [rows, dim]:
 * eq_rms_norm with its result in codes, which are rounded once, from f32.  The sum of
 * squares is held in f32 too: rows whose sum passes its range become zeros. */
int eq_fp8_rms_norm(void* codes, float* scales, int64_t scale_stride, void* hidden, const void* residual,
                    const void* weight, int64_t rows, int64_t dim, float eps, int dtype, eq_stream_t stream);

/* codes and scales of silu(gate) * up = gate / (1 + e^-gate) * up, held in f32
 * until it is rounded to the codes.  gate and up have strides of their own (they
 * may be slices of one projection). */
int eq_fp8_silu_mul(void* codes, float* scales, int64_t scale_stride, const void* gate, int64_t gate_stride,
                    const void* up, int64_t up_stride, int64_t rows, int64_t cols, int dtype, eq_stream_t stream);

/* y [m, n] = x . w^T, held in f32 and rounded once to y_dtype (f32, f16 or
 * bf16).  x [m, k]: codes (x_dtype EQ_DTYPE_F8E4M3) with x_scales, or values
 * of x_dtype, which the call quantizes (x_scales NULL).  Where y is f16 or bf16 the
 * matrix cores cut each of 8 neighbouring products of codes off at 2^-13 of the
 * largest one's power of two, towards zero, before they are summed in f32: of random codes about 2e-5 of
 * a row's result, where it is rounded by 2e-4 or 2e-3; at the worst, 8 products of one size, 7 * 2^-13 = 8.5e-4
 * of that size, which is more than f16's rounding.  Where y is f32 the products are exact and take twice the time.
 *
 * The scales of a block, one of x and one of w, are multiplied in f32: where their product passes
 * f32's range the results are not finite, and where it is below 2^-126 they lose bits.
 *
 * m and n are below 2^30, and the result has at most 2^23 - 4096 tiles (of 16 columns where m is at most
 * 16, and for each of 64 routes or fewer; else of 128 columns by 32 rows or more).
 *
 * scratch: scratch_bytes of device memory (256-byte aligned) that the call may
 * use until it has run, at least what the query below returns; NULL: the
 * library's workspace of `stream`, which cannot grow while `stream` is
 * capturing and which graphs captured on one stream share, so such graphs must
 * not run at the same time.  (Calls of several host threads on one stream may
 * share it: a call keeps its launches together.) */
int eq_fp8_matmul(void* y, const void* x, int64_t x_stride, const float* x_scales, int64_t scale_stride, const void* w,
                  const float* w_scales, int64_t m, int64_t n, int64_t k, int x_dtype, int y_dtype, void* scratch,
                  int64_t scratch_bytes, eq_stream_t stream);
/* Scratch bytes of eq_fp8_matmul with these sizes (0: none), -1 for sizes it refuses. */
int64_t eq_fp8_matmul_scratch(int64_t m, int64_t n, int64_t k, int x_dtype, int y_dtype);

/* Routed experts: y [routes, n], y[r] = x[rows[r]] . w[ids[r]]^T with a bank of
 * `experts` (at most 4095) weights w [experts, n, k], scales one after the other
 * too; ids and rows are device int32 (rows NULL: row r, x_rows = routes), in any
 * order.  A route whose expert or row is out of range gives zeros; x has a row at
 * least.  x_rows * x_stride of codes, or x_rows * k of values, is below 3 * 2^30.  scratch as
 * in eq_fp8_matmul. */
int eq_fp8_grouped_matmul(void* y, const void* x, int64_t x_stride, const float* x_scales, int64_t scale_stride,
                          int64_t x_rows, const void* w, const float* w_scales, int64_t experts, const int32_t* ids,
                          const int32_t* rows, int64_t routes, int64_t n, int64_t k, int x_dtype, int y_dtype,
                          void* scratch, int64_t scratch_bytes, eq_stream_t stream);
/* Scratch bytes of eq_fp8_grouped_matmul with these sizes, -1 for sizes it refuses. */
int64_t eq_fp8_grouped_matmul_scratch(int64_t x_rows, int64_t experts, int64_t routes, int64_t n, int64_t k, int x_dtype,
                                      int y_dtype);

#ifdef __cplusplus
}
#endif

#endif /* EREDU_FP8_H */
