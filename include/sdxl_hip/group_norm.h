/* C ABI of group norm with an activation, channels last, on MI355X (gfx950).
 *
 * The reference's UNet runs a group norm of 32 groups at the entry of every spatial
 * transformer (src/cuda/unet.cpp:151-181, eps 1e-6) and two with SiLU in every residual
 * block (eps 1e-5), its VAE the same in fp32. Here, for x [batch, pixels, channels]:
 *   y = act((x - mean) * rstd * gamma + beta)
 * with the mean and the (biased) variance of the pixels and channels of a group, rstd =
 * 1 / sqrt(var + eps); the gradients; and the norm whose pixels come out as 8-bit integers
 * with a scale each, for the projection that follows (sdxl_linear_i8).
 *
 * Types: x, gamma, beta, y, dy and the gradients are fp16, bf16 or fp32 (desc->dtype), the
 * statistics, sums and scales fp32, and every output is rounded once. A group's variance is
 * summed about values of its own, so that neither a mean far from zero nor a value far from the
 * others costs digits; sums of squared distances from the mean have to stay within fp32. Any batch,
 * pixels and channels, any row strides of at least a row; image b follows image b - 1 after
 * pixels * row_stride elements. Tensors need only their element's alignment. Kernels work on slabs
 * of whole groups, as many as the smallest divisor of the groups that makes 512 bytes of a row (all
 * of a shorter row). Slabs of more than 8 KiB (groups that wide; 37 groups of 256 bytes, which no
 * divisor cuts), rows shorter than 16 bytes, more than 4096 groups, some millions of images and
 * strides above 2^20 elements take general kernels, many times as long (sdxl_group_norm_i8: rows
 * of more than 20 KiB too).
 * A NaN or an infinity in a group makes its rows NaN, and no other group's.
 *
 * All calls are stream-ordered, allocate nothing, never synchronise and may be captured into
 * a HIP graph; the stream's device must be the current one. Each call in flight needs a
 * workspace of its own. Outputs and workspace must not overlap the inputs or each other,
 * except where a call says otherwise. Errors as in attention.h (sdxl_last_error()).
 */
#ifndef SDXL_HIP_GROUP_NORM_H
#define SDXL_HIP_GROUP_NORM_H

#include <stddef.h>
#include <stdint.h>

#include "attention.h"
#include "feed_forward.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct sdxl_group_norm_desc {
    int64_t batch;
    int64_t pixels;   /* of an image: height * width */
    int64_t channels; /* a multiple of groups */
    int64_t groups;
    /* Row (pixel) strides in elements; 0 means channels. */
    int64_t x_row_stride;
    int64_t y_row_stride;  /* of y; backward: of dx */
    int64_t dy_row_stride; /* backward */
    int32_t dtype;         /* SDXL_DTYPE_F16, _BF16 or _F32 */
    int32_t activation;    /* sdxl_activation */
    float eps;             /* 0 means 1e-5 */
    int32_t reserved;      /* must be 0 */
} sdxl_group_norm_desc;

/* Workspaces of the calls below (parts of the sums), 256-byte aligned; 0 where a call needs none
 * (sdxl_group_norm of small images) and for a descriptor that the call refuses. They hold 8 bytes
 * for every image, chunk of its pixels (at least one) and group, for the gradients every channel
 * too: below 2 MiB for the UNet's and the VAE's sizes, but 8 * batch * channels bytes at least,
 * more than the tensor itself where images have fewer than four pixels of a 16-bit type. */
size_t sdxl_group_norm_workspace_bytes(const sdxl_group_norm_desc* desc);
size_t sdxl_group_norm_i8_workspace_bytes(const sdxl_group_norm_desc* desc);
size_t sdxl_group_norm_backward_workspace_bytes(const sdxl_group_norm_desc* desc);

/* y = act((x - mean) * rstd * gamma + beta), gamma and beta [channels]. stats (NULL: not
 * wanted) [batch, groups, 2] fp32 receives mean and rstd of every group, which the backward
 * call takes. y may equal x (with x's row stride). */
sdxl_status sdxl_group_norm(const sdxl_group_norm_desc* desc, const void* x, const void* gamma, const void* beta,
                            void* y, float* stats, void* workspace, size_t workspace_bytes, void* stream);

/* Gradients of sdxl_group_norm for dy [batch, pixels, channels], with stats as the forward
 * call left them: with n = (x - mean) * rstd, z = n * gamma + beta, dz = dy * act'(z),
 *   dbeta = sum dz, dgamma = sum dz * n   (over batch and pixels), and
 *   dx = rstd * (gamma dz - mean(gamma dz) - n * mean(gamma dz n))   (means over a group).
 * dx, dgamma and dbeta are each optional (NULL). Sums are made in an order that the
 * sizes alone decide: the same inputs give the same bits. */
sdxl_status sdxl_group_norm_backward(const sdxl_group_norm_desc* desc, const void* dy, const void* x,
                                     const void* gamma, const void* beta, const float* stats, void* dx,
                                     void* dgamma, void* dbeta, void* workspace, size_t workspace_bytes,
                                     void* stream);

/* sdxl_group_norm whose pixels are quantised by row (fp16 and bf16 x): codes q [batch *
 * pixels, channels] int8 (row stride in bytes, 0 = channels) and scales q_scale [batch *
 * pixels] of the values before they would be rounded to x's type, by the rule of
 * sdxl_quantize_i8_rows (int8.h). */
sdxl_status sdxl_group_norm_i8(const sdxl_group_norm_desc* desc, const void* x, const void* gamma, const void* beta,
                               int8_t* q, int64_t q_row_stride, float* q_scale, float* stats, void* workspace,
                               size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SDXL_HIP_GROUP_NORM_H */
