/* C ABI of 8-bit integer linears on MI355X (gfx950): products of int8 codes with a scale for
 * every token (row of x) and every output channel (row of w), and what makes the codes.
 *
 * The integer counterpart of sdxl_linear_e4m3, sdxl_linear_act and sdxl_gated_linear, for the
 * same places of the UNet's transformer block (src/cuda/unet.cpp:98-149) and text encoders:
 *   z[i, j] = (sum over k of x[i, k] * w[j, k]) * x_scale[i] * w_scale[j] + bias[j]
 *   sdxl_linear_i8:        out = act(z) + residual
 *   sdxl_gated_linear_i8:  out = value * act(gate), [value | gate] = z
 *
 * Codes of a row v of values (weights by output channel, tokens by token): scale = amax > 0 ?
 * max(amax / 127, 1e-12) : 1 with amax the largest magnitude of v's finite values, code = v /
 * scale rounded to nearest, ties to even, at most 127 in magnitude (so infinities become +-127).
 * A row with a NaN has a NaN for its scale, which makes its whole row of z NaN; its codes are
 * unspecified. Products take codes from -128 on. Sums are exact 32-bit integers (k at most
 * 131071), scaled in fp32, and every output is rounded once.
 *
 * Any m, n, k >= 0 and any row strides of at least a row; tensors need only their element's
 * alignment. Rows of codes that 16-byte accesses divide (pointers, row strides and k multiples
 * of 16) run the fast kernels; other rows of 16 bytes or more take about twice as long, shorter
 * ones and strides above 2^20 elements the general kernel.
 *
 * All calls are stream-ordered, allocate nothing, never synchronise and may be captured into a
 * HIP graph; the stream's device must be the current one. Each call in flight needs a workspace
 * of its own. Outputs and workspace must not overlap the inputs or each other, except where a
 * call says otherwise. Errors as in attention.h (sdxl_last_error()).
 */
#ifndef SDXL_HIP_INT8_H
#define SDXL_HIP_INT8_H

#include <stddef.h>
#include <stdint.h>

#include "attention.h"
#include "feed_forward.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Codes q [rows, cols] (row stride in bytes, 0 = cols) and scales q_scale [rows] of x [rows,
 * cols] (dtype SDXL_DTYPE_F16 or SDXL_DTYPE_BF16; row stride in elements, 0 = cols): tokens, or
 * a weight [out, in] by output channel. */
sdxl_status sdxl_quantize_i8_rows(int64_t rows, int64_t cols, int32_t dtype, const void* x, int64_t x_row_stride,
                                  int8_t* q, int64_t q_row_stride, float* q_scale, void* stream);

/* LayerNorm quantised for the projection that consumes it (as sdxl_layer_norm_e4m3; any width,
 * fp16 or bf16): the codes of (x - mean) / sqrt(var + eps) * gamma + beta before it would be
 * rounded to x's type. eps 0 means 1e-5. */
sdxl_status sdxl_layer_norm_i8(int64_t rows, int64_t width, int32_t dtype, const void* x, int64_t x_row_stride,
                               const void* gamma, const void* beta, float eps, int8_t* q, int64_t q_row_stride,
                               float* q_scale, void* stream);

typedef struct sdxl_i8_desc {
    int64_t m; /* rows of x */
    int64_t n; /* columns of out: w has n rows (linear) or 2 n rows (gated) */
    int64_t k; /* columns of x and w */
    /* Row strides in elements; 0 means dense. */
    int64_t x_row_stride;
    int64_t w_row_stride;
    int64_t out_row_stride;
    int64_t residual_row_stride;
    int32_t dtype;      /* of bias, residual and out: SDXL_DTYPE_F16 or SDXL_DTYPE_BF16 */
    int32_t x_dtype;    /* SDXL_DTYPE_I8: codes with x_scale; dtype: tokens in 16 bits, which the call quantises by row */
    int32_t activation; /* sdxl_activation */
    int32_t gate_first; /* gated: 0: rows 0 .. n-1 of w are the value projection, n .. 2n-1 the gate's; 1: the other way round */
    int32_t reserved;   /* must be 0 */
} sdxl_i8_desc;

/* Workspace of the calls below, 256-byte aligned: codes and scales of 16-bit tokens (0 for codes,
 * for up to four tokens, whose product quantises them on the way, and for a descriptor that the call
 * refuses). */
size_t sdxl_linear_i8_workspace_bytes(const sdxl_i8_desc* desc);
size_t sdxl_gated_linear_i8_workspace_bytes(const sdxl_i8_desc* desc);

/* The kernels that a call of this descriptor runs on the current device (without one: on 256 CUs), on
 * tensors aligned to 16 bytes: those of sdxl_linear_i8 or (gated 1) sdxl_gated_linear_i8, named as by
 * sdxl_ff_kernels (feed_forward.h), "quantise; " before the product of 16-bit tokens, " tokens" behind
 * that which quantises them itself. Text, size and result as there. */
size_t sdxl_i8_kernels(const sdxl_i8_desc* desc, int32_t gated, char* text, size_t size);

/* out = act((x . w^T) * x_scale * w_scale + bias) + residual: x [m, k] codes with x_scale [m], or
 * 16-bit tokens (x_scale NULL), as if quantised by sdxl_quantize_i8_rows first; w [n, k] codes
 * with w_scale [n]. bias [n] and residual [m, n] are optional (NULL); residual may equal out
 * (with out's row stride). desc->gate_first must be 0. */
sdxl_status sdxl_linear_i8(const sdxl_i8_desc* desc, const void* x, const float* x_scale, const int8_t* w,
                           const float* w_scale, const void* bias, const void* residual, void* out, void* workspace,
                           size_t workspace_bytes, void* stream);

/* out = value * act(gate) with [value | gate] = (x . w^T) * x_scale * w_scale + bias, w [2n, k],
 * w_scale and bias [2n]: both projections, the activation and the product in one kernel. */
sdxl_status sdxl_gated_linear_i8(const sdxl_i8_desc* desc, const void* x, const float* x_scale, const int8_t* w,
                                 const float* w_scale, const void* bias, void* out, void* workspace,
                                 size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SDXL_HIP_INT8_H */
