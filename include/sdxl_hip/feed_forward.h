/* C ABI of the transformer block's feed-forward half on MI355X (gfx950), and of the
 * linear layers with an activation beside it.
 *
 * The reference's UNet transformer block ends with (src/cuda/unet.cpp:98-149)
 *   normalized = Ops::layer_norm(hidden, norm3.weight, norm3.bias)
 *   hidden    += ff.net.2(GEGLU(ff.net.0.proj(normalized)))
 * and its text encoders run linear -> activation -> linear (src/cuda/text_encoder.cpp).
 * Here: the gated projection as one kernel (sdxl_gated_linear), a linear with bias,
 * activation and residual in its epilogue (sdxl_linear_act), the gradients of both, and
 * the whole half as one call (sdxl_ff_sublayer).
 *
 * Types: x, bias, residual, out, dout and the gradients are fp16 or bf16 (desc->dtype);
 * w has that type or holds FP8 E4M3 codes with per-row fp32 scales (forward only).
 * Products are summed in fp32 and every output is rounded once; the backward calls round
 * dz (below) to the tensors' type in between, since it is an operand of the 16-bit matrix
 * cores: the gradients made of it are about 1.4 times as far from exact as one rounding
 * leaves them. In fp16 dz also has the type's range: beyond 65504 it is infinite, below
 * 2^-25 zero. dbias, its column sum, leaves that range with it unless terms cancel, and
 * what is lost below is at most 2^-25 of every term; scale the loss as for any fp16
 * gradient. Any m, n, k >= 0 and any row strides of at least a row; tensors need only their
 * element's alignment. Rows that 16-byte accesses divide (pointers and row strides
 * multiples of 16 bytes, k a multiple of 8 and with E4M3 weights of 16) run the fast
 * kernels; other rows of 16 bytes or more take about twice as long, shorter ones and
 * strides above 2^20 elements the general kernel (the sums' order differs).
 * An infinite pre-activation takes the activation's limit; NaN stays NaN (and relu's slope
 * at NaN is 1).
 *
 * All calls are stream-ordered, allocate nothing, never synchronise and may be captured
 * into a HIP graph; the stream's device must be the current one. Outputs and workspace
 * must not overlap the inputs or each other, except where a call says otherwise: refused
 * wherever the strides are equal or one of the two is contiguous, else by their first and
 * last rows (column slices of one tensor do not overlap). Errors as in attention.h (sdxl_last_error()).
 */
#ifndef SDXL_HIP_FEED_FORWARD_H
#define SDXL_HIP_FEED_FORWARD_H

#include <stddef.h>
#include <stdint.h>

#include "attention.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum sdxl_activation {
    SDXL_ACT_NONE = 0,
    SDXL_ACT_RELU = 1,       /* max(z, 0); slope 0 at 0 */
    SDXL_ACT_GELU = 2,       /* z Phi(z), Phi the normal distribution function */
    SDXL_ACT_GELU_TANH = 3,  /* z / 2 (1 + tanh(sqrt(2 / pi) (z + 0.044715 z^3))) */
    SDXL_ACT_QUICK_GELU = 4, /* z sigmoid(1.702 z) */
    SDXL_ACT_SILU = 5        /* z sigmoid(z) */
} sdxl_activation;

typedef struct sdxl_ff_desc {
    int64_t m; /* rows of x */
    int64_t n; /* columns of out: w has n rows (linear) or 2 n rows (gated) */
    int64_t k; /* columns of x and w */
    /* Row strides in elements; 0 means dense. dout has the stride of out. */
    int64_t x_row_stride;
    int64_t w_row_stride;
    int64_t out_row_stride;
    int64_t residual_row_stride;
    int64_t dx_row_stride; /* backward */
    int64_t dw_row_stride; /* backward */
    int32_t dtype;         /* SDXL_DTYPE_F16 or SDXL_DTYPE_BF16 */
    int32_t w_dtype;       /* dtype, or SDXL_DTYPE_E4M3 (forward only) */
    int32_t activation;    /* sdxl_activation */
    int32_t gate_first;    /* gated: 0: rows 0 .. n-1 of w are the value projection, n .. 2n-1 the
                              gate's (the GEGLU checkpoint layout); 1: the other way round */
    int32_t reserved;      /* must be 0 */
} sdxl_ff_desc;

/* out = act((x . w^T) * w_scale + bias) + residual. w_scale [n] fp32: required for E4M3
 * weights, else optional (NULL = 1). bias [n] and residual [m, n] are optional (NULL);
 * residual may equal out (with out's row stride). desc->gate_first must be 0. */
sdxl_status sdxl_linear_act(const sdxl_ff_desc* desc, const void* x, const void* w, const float* w_scale,
                            const void* bias, const void* residual, void* out, void* stream);

/* out = value * act(gate) with [value | gate] = (x . w^T) * w_scale + bias, w [2n, k],
 * w_scale and bias [2n]: both projections, the activation and the product in one kernel. */
sdxl_status sdxl_gated_linear(const sdxl_ff_desc* desc, const void* x, const void* w, const float* w_scale,
                              const void* bias, void* out, void* stream);

/* Workspace of the backward calls (dz, and up to 32 MiB of partial sums where a product of few
 * tiles splits its sum), 256-byte aligned, the same whichever gradients are asked for, so that
 * each is summed alike; 0 for a descriptor that the call refuses. */
size_t sdxl_linear_act_backward_workspace_bytes(const sdxl_ff_desc* desc);
size_t sdxl_gated_linear_backward_workspace_bytes(const sdxl_ff_desc* desc);

/* Gradients of sdxl_linear_act for dout [m, n]: with z = x . w^T + bias (formed again here),
 * dz = dout * act'(z): dx = dz . w [m, k], dw = dz^T . x [n, k], dbias = column sums of dz [n].
 * The residual's gradient is dout itself. dx, dw and dbias are each optional (NULL: not
 * computed); bias as in the forward call (NULL if it had none). There is no w_scale: a forward
 * call with scales of 16-bit weights has its gradients through the scaled weights. */
sdxl_status sdxl_linear_act_backward(const sdxl_ff_desc* desc, const void* dout, const void* x, const void* w,
                                     const void* bias, void* dx, void* dw, void* dbias, void* workspace,
                                     size_t workspace_bytes, void* stream);

/* Gradients of sdxl_gated_linear: dvalue = dout * act(gate), dgate = dout * value * act'(gate),
 * dz = [dvalue | dgate] in the order of w's rows; dx = dz . w [m, k], dw = dz^T . x [2n, k],
 * dbias = column sums of dz [2n], each optional. */
sdxl_status sdxl_gated_linear_backward(const sdxl_ff_desc* desc, const void* dout, const void* x, const void* w,
                                       const void* bias, void* dx, void* dw, void* dbias, void* workspace,
                                       size_t workspace_bytes, void* stream);

/* The kernels that a call of this descriptor runs on the current device (without one: on 256 CUs), on tensors
 * aligned to 16 bytes: those of sdxl_linear_act or sdxl_gated_linear (gated 1), or with gradients (1: dx, 2: dw,
 * 4: dbias, added up) those of its backward. "tile 256x320" is the tiled kernel's tile, "deep 32x32/8" a tile whose
 * eight waves share the depth, "rows/4" the kernel of few rows with four waves a workgroup, "staged" what takes rows
 * that 16-byte accesses do not divide, "general" the rest; "; " stands between launches, " + " between products of one
 * launch, "in 2 shares" where a depth is split and joined. Writes at most size bytes with the terminating zero to text
 * (may be NULL) and returns the length without it; 0 where the call would be refused or launch nothing. Launches
 * nothing itself. */
size_t sdxl_ff_kernels(const sdxl_ff_desc* desc, int32_t gated, int32_t gradients, char* text, size_t size);

typedef struct sdxl_ff_sublayer_desc {
    int64_t rows;  /* batch * seq */
    int64_t width; /* even, at most 2048 */
    int64_t inner; /* SDXL: 4 * width */
    int32_t w_in_dtype;  /* SDXL_DTYPE_F16 or SDXL_DTYPE_E4M3 */
    int32_t w_out_dtype; /* SDXL_DTYPE_F16 or SDXL_DTYPE_E4M3 */
    int32_t activation;  /* sdxl_activation; SDXL: SDXL_ACT_GELU */
    int32_t gate_first;
    float ln_eps;        /* 0 means 1e-5 */
    int32_t reserved;    /* must be 0 */
} sdxl_ff_sublayer_desc;

/* rows * (width + inner) * 2 bytes, each part rounded up to 256 (0 for a descriptor that the call
 * refuses). */
size_t sdxl_ff_sublayer_workspace_bytes(const sdxl_ff_sublayer_desc* desc);

/* The feed-forward half of the transformer block, fp16, after sdxl_attn_sublayer and
 * sdxl_cross_attn_sublayer: y = x + gated(LN(x), w_in, b_in) . w_out^T + b_out, for x [rows, width];
 * w_in [2 inner, width] and b_in [2 inner] (value | gate), w_out [width, inner], b_out [width],
 * w_in_scale / w_out_scale for E4M3 weights. b_in and b_out are optional (NULL). y may equal x.
 * A refused call launches nothing. */
sdxl_status sdxl_ff_sublayer(const sdxl_ff_sublayer_desc* desc, const void* x, const void* ln_gamma,
                             const void* ln_beta, const void* w_in, const float* w_in_scale, const void* b_in,
                             const void* w_out, const float* w_out_scale, const void* b_out, void* y,
                             void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SDXL_HIP_FEED_FORWARD_H */
