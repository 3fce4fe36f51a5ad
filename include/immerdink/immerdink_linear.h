/* C ABI of the quantised linear layer: libimmerdink_linear.so (sm_100a).
 *
 * Where immerdink.h scales FP64 rows, quantises them to 8 bits and multiplies them exactly, these
 * entry points do the same for the 8-bit and 4-bit operands of a language model's linear layers:
 *
 *   imd_norm_quantize   h = x + residual;  y = h * rsqrt(mean(h^2) + eps) * weight;
 *                       scale[t] = max_j |y[t,j]| / Q;  q[t,j] = round(y[t,j] / scale[t])
 *   imd_scaled_linear   out[t,n] = x_scale[t] * w_scale[n] * sum_k x[t,k] * w[n,k]     (8-bit x, w)
 *   imd_linear_w4       out[t,n] = sum_k x[t,k] * w_scale[n,k/group] * (w[n,k] - zeros[n,k/group])
 *
 * Contract shared by every entry point: status codes only (nothing throws); the caller owns every
 * buffer and the stream; a call only enqueues kernels on `stream` (no allocation, no
 * synchronisation, no workspace), so it can be captured in a CUDA graph, and any number of calls
 * may be in flight. The current device must be the one that holds the buffers. A call that fails
 * its checks touches nothing. Results do not depend on the run: no atomics, sums in a fixed order.
 *
 * Matrices are row-major with unit stride inside a row; `*_stride` is the distance between rows in
 * ELEMENTS of the matrix (bytes for packed 4-bit weights), not looked at for a single row. Inputs may
 * repeat rows (stride 0); an output's rows must not overlap. Every buffer is aligned to its element size; any alignment
 * above that is optional (16-byte aligned rows take the wide loads).
 *
 * Checks, in order: types and sizes out of range -> INVALID_VALUE (a combination that exists in no
 * kernel -> NOT_SUPPORTED); an empty output -> SUCCESS; null pointers, strides -> INVALID_VALUE;
 * an output that overlaps another buffer -> ALIASING; element alignment -> MISALIGNED. Columns of one
 * buffer (rows at the same distance in bytes) do not overlap where they share no byte; matrices that
 * interleave at different distances count as overlapping. */
#ifndef IMMERDINK_B200_LINEAR_H
#define IMMERDINK_B200_LINEAR_H

#include <stddef.h>
#include <stdint.h>

#include <cuda_runtime_api.h>

#include "immerdink/immerdink_host.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. E4M3: 4 exponent and 3 mantissa bits, no infinities, largest value 448. */
enum { IMD_TYPE_F32 = 0, IMD_TYPE_BF16 = 1, IMD_TYPE_F16 = 2, IMD_TYPE_I8 = 3, IMD_TYPE_E4M3 = 4 };

/* RMS norm with the residual's addition and an 8-bit output with one scale per row.
 *
 * x [rows, dim] and residual (NULL = none) in x_type (F32, BF16, F16); weight [dim] in x_type or
 * F32; q [rows, dim] in q_type (I8: Q = 127, E4M3: Q = 448); scale [rows] F32. residual_out (NULL =
 * not wanted; requires residual) receives h rounded once to x_type; it may be x or residual itself
 * (same address and stride). 0 <= eps <= 2^127.
 *
 * Everything between the loads and the stores is held in 32 bits: the norm sees the unrounded sum
 * h. Codes are the nearest (in the middle of two: the even one) to Q y / max |y|, in which the row's root cancels: they
 * follow from h * weight, however the root was rounded. Squares that would leave the range of 32 bits are summed again after an exact scaling by a
 * power of two. A row of zeros gives zeros and scale 0. A row whose y holds a NaN or an infinity
 * gets scale NaN (codes 0 for I8, NaN for E4M3), so that a product with it is NaN. */
IMD_API imd_status_t imd_norm_quantize(int64_t rows, int64_t dim, int32_t x_type, const void* x,
                                       int64_t x_stride, const void* residual,
                                       int64_t residual_stride, int32_t weight_type,
                                       const void* weight, double eps, void* residual_out,
                                       int64_t residual_out_stride, int32_t q_type, void* q,
                                       int64_t q_stride, float* scale, cudaStream_t stream);

/* Product of two 8-bit operands with a scale per row of each.
 *
 * x [rows, k] and w [n, k], both `type` (I8 or E4M3); x_scale [rows], w_scale [n] F32; out [rows, n]
 * in out_type (F32, BF16, F16). I8 sums are exact 32-bit integers (k <= 131071, else NOT_SUPPORTED);
 * E4M3 sums are 32-bit floats, to which a tensor instruction may add its aligned terms cut instead of
 * rounded (2^-23 of the partial sum). The sum, as a 32-bit float, times x_scale, times w_scale: each
 * rounded in 32 bits, then to out_type. k = 0: sums of 0. */
IMD_API imd_status_t imd_scaled_linear(int64_t rows, int64_t n, int64_t k, int32_t type,
                                       const void* x, int64_t x_stride, const void* w,
                                       int64_t w_stride, const float* x_scale,
                                       const float* w_scale, int32_t out_type, void* out,
                                       int64_t out_stride, cudaStream_t stream);

/* Product of 16-bit activations with 4-bit weights that have a scale (and a zero point) per group.
 *
 * x [rows, k] in x_type (BF16, F16); w: n rows of ceil(k / 2) bytes, element k in the low (even k)
 * or high (odd k) half of byte k / 2, w_stride bytes apart; groups of `group` (32, 64 or 128)
 * consecutive k, the last one possibly shorter; w_scale [n, ceil(k / group)] in scale_type (F32,
 * BF16, F16), its rows scale_stride elements apart; zeros [n, ceil(k / group)] one byte each, values
 * 0..15 (a larger byte is taken modulo 16), zeros_stride bytes apart, NULL = 8 everywhere; out
 * [rows, n] in out_type (F32 or x_type), rounded once from 32 bits. w - zero is exact, sums are 32-bit floats,
 * the scale multiplies a group's sum in 32 bits. k = 0 gives zeros. */
IMD_API imd_status_t imd_linear_w4(int64_t rows, int64_t n, int64_t k, int32_t group,
                                   int32_t x_type, const void* x, int64_t x_stride, const void* w,
                                   int64_t w_stride, int32_t scale_type, const void* w_scale,
                                   int64_t scale_stride, const void* zeros, int64_t zeros_stride,
                                   int32_t out_type, void* out, int64_t out_stride,
                                   cudaStream_t stream);

/* The sticky error word of this library on the current device, read into *word and cleared. Every wait
 * inside its kernels is bounded; one that gives up sets bit 0 and the kernel ends with its output
 * incomplete. Synchronises the device: a diagnostic, not part of a step. NULL -> INVALID_VALUE. */
IMD_API imd_status_t imd_linear_device_error(unsigned int* word);

#ifdef __cplusplus
}
#endif
#endif /* IMMERDINK_B200_LINEAR_H */
