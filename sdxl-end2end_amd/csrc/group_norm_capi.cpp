// C ABI of group norm (include/sdxl_hip/group_norm.h): validation, workspaces
// and stream-ordered launches (reference src/cuda/unet.cpp:151-181).
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "../../include/sdxl_hip/group_norm.h"
#include "capi_areas.hpp"
#include "capi_internal.hpp"
#include "group_norm_kernels.hpp"

namespace {

using sdxl_hip::Area;
using sdxl_hip::GnParams;
using sdxl_hip::GnPlan;
using sdxl_hip::GnType;
using sdxl_hip::matrix;
using sdxl_hip::overlap;
using sdxl_hip::overlaps_one;
using sdxl_hip::vector;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

sdxl_status fail(const char* name, sdxl_status status, const char* what) {
    return sdxl_hip_fail(status, std::string(name) + ": " + what);
}

// A descriptor with its strides resolved: sizes, strides, activation and eps of p are filled in.
struct Call {
    GnParams p;
    GnType type;
    int64_t elem, rows;
    bool empty;
};

sdxl_status resolve(const sdxl_group_norm_desc* d, const char* name, Call& c) {
    if (d == nullptr) return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "null descriptor");
    if (d->reserved != 0) return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "reserved field must be 0");
    if (d->dtype != SDXL_DTYPE_F16 && d->dtype != SDXL_DTYPE_BF16 && d->dtype != SDXL_DTYPE_F32)
        return fail(name, SDXL_STATUS_INVALID_SHAPE, "tensors must be fp16, bf16 or fp32");
    if (d->activation < SDXL_ACT_NONE || d->activation > SDXL_ACT_SILU)
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "unknown activation");
    if (!(d->eps >= 0.0f) || std::isinf(d->eps)) return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "eps must be finite and not negative");
    if (d->batch < 0 || d->pixels < 0 || d->channels < 0 || d->batch > INT32_MAX || d->pixels > INT32_MAX ||
        d->channels > INT32_MAX)
        return fail(name, SDXL_STATUS_INVALID_SHAPE, "dimensions out of range");
    if (d->groups <= 0 || d->groups > INT32_MAX || d->channels % d->groups != 0)
        return fail(name, SDXL_STATUS_INVALID_SHAPE, "channels must be a multiple of groups");
    c = Call{};
    const int64_t given[3] = {d->x_row_stride, d->y_row_stride, d->dy_row_stride};
    int64_t* to[3] = {&c.p.ld_x, &c.p.ld_y, &c.p.ld_dy};
    c.rows = d->batch * d->pixels;
    for (int i = 0; i < 3; ++i) {
        *to[i] = given[i] == 0 ? d->channels : given[i];
        if (*to[i] < d->channels) return fail(name, SDXL_STATUS_INVALID_SHAPE, "row stride smaller than the row");
        if (*to[i] > INT32_MAX || (__int128)c.rows * *to[i] > INT64_MAX / 8)
            return fail(name, SDXL_STATUS_INVALID_SHAPE, "row stride out of range");
    }
    c.p.batch = (int32_t)d->batch;
    c.p.pixels = d->pixels;
    c.p.channels = (int32_t)d->channels;
    c.p.groups = (int32_t)d->groups;
    c.p.group_channels = (int32_t)(d->channels / d->groups);
    c.p.activation = d->activation;
    c.p.eps = d->eps == 0.0f ? 1e-5f : d->eps;
    c.type = d->dtype == SDXL_DTYPE_F16 ? sdxl_hip::kGnF16 : d->dtype == SDXL_DTYPE_BF16 ? sdxl_hip::kGnBf16 : sdxl_hip::kGnF32;
    c.elem = d->dtype == SDXL_DTYPE_F32 ? 4 : 2;
    c.empty = c.rows == 0 || d->channels == 0;
    return SDXL_STATUS_OK;
}

size_t round256(size_t v) { return (v + 255) / 256 * 256; }

// The workspace: the chunks' statistics; backward: their sums by group, then by channel.
size_t group_bytes(const GnParams& p, const GnPlan& plan) {
    return round256((size_t)p.batch * (size_t)plan.chunks * (size_t)p.groups * 8);
}
size_t channel_bytes(const GnParams& p, const GnPlan& plan) {
    return round256((size_t)p.batch * (size_t)plan.chunks * (size_t)p.channels * 8);
}
size_t workspace_of(const Call& c, const GnPlan& plan, bool backward) {
    return group_bytes(c.p, plan) + (backward ? channel_bytes(c.p, plan) : 0);
}

size_t workspace_bytes_of(const sdxl_group_norm_desc* d, sdxl_hip::GnCall call, const char* name) {
    Call c;
    if (resolve(d, name, c) != SDXL_STATUS_OK || c.empty) return 0;
    if (call == sdxl_hip::kGnRows && c.type == sdxl_hip::kGnF32) return 0;  // (which the call refuses)
    return workspace_of(c, gn_plan(c.p, c.type, call), call == sdxl_hip::kGnBackward);
}

void use_workspace(GnParams& p, const GnPlan& plan, void* workspace) {
    p.chunks = plan.chunks;
    p.chunk_pixels = plan.chunk_pixels;
    p.partial = static_cast<float*>(workspace);
    p.channel_sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + group_bytes(p, plan));
}

sdxl_status launched(hipError_t err, const char* name) {
    return err == hipSuccess ? SDXL_STATUS_OK : fail(name, SDXL_STATUS_LAUNCH_FAILED, hipGetErrorString(err));
}

// y, or codes q with their scales.
sdxl_status forward(const sdxl_group_norm_desc* d, const char* name, const void* x, const void* gamma, const void* beta,
                    void* y, int8_t* q, int64_t q_row_stride, float* q_scale, bool codes, float* stats, void* workspace,
                    size_t workspace_bytes, void* stream) {
    Call c;
    const sdxl_status st = resolve(d, name, c);
    if (st != SDXL_STATUS_OK) return st;
    GnParams& p = c.p;
    if (codes) {
        if (c.type == sdxl_hip::kGnF32) return fail(name, SDXL_STATUS_INVALID_SHAPE, "tensors must be fp16 or bf16");
        p.ld_q = q_row_stride == 0 ? p.channels : q_row_stride;
        if (p.ld_q < p.channels) return fail(name, SDXL_STATUS_INVALID_SHAPE, "row stride smaller than the row");
        if (p.ld_q > INT32_MAX) return fail(name, SDXL_STATUS_INVALID_SHAPE, "row stride out of range");
    }
    if (c.empty) return SDXL_STATUS_OK;
    if (x == nullptr || gamma == nullptr || beta == nullptr || (codes ? q == nullptr || q_scale == nullptr : y == nullptr))
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "null tensor pointer");
    const uintptr_t e = (uintptr_t)c.elem;
    if (!aligned(x, e) || !aligned(gamma, e) || !aligned(beta, e) || !aligned(y, e) || !aligned(q_scale, 4) || !aligned(stats, 4))
        return fail(name, SDXL_STATUS_UNSUPPORTED, "tensor not aligned to its elements");
    const GnPlan plan = gn_plan(p, c.type, codes ? sdxl_hip::kGnRows : sdxl_hip::kGnForward);
    const size_t need = workspace_of(c, plan, false);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 256)))
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "workspace missing, small or misaligned");
    const Area in = matrix(x, c.rows, p.channels, p.ld_x, c.elem), g = vector(gamma, p.channels, c.elem), b = vector(beta, p.channels, c.elem);
    const Area out[4] = {codes ? matrix(q, c.rows, p.channels, p.ld_q, 1) : matrix(y, c.rows, p.channels, p.ld_y, c.elem),
                         vector(codes ? q_scale : nullptr, c.rows, 4), vector(stats, 2 * (int64_t)p.batch * p.groups, 4),
                         vector(need > 0 ? workspace : nullptr, (int64_t)need, 1)};
    const bool in_place = !codes && x == y && p.ld_x == p.ld_y;
    for (int i = 0; i < 4; ++i) {
        if (overlaps_one(out[i], {g, b}) || (!(i == 0 && in_place) && overlap(out[i], in)))
            return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "an output or the workspace overlaps an input");
        for (int j = 0; j < i; ++j)
            if (overlap(out[i], out[j])) return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "an output overlaps another one or the workspace");
    }
    p.x = x;
    p.gamma = gamma;
    p.beta = beta;
    p.y = y;
    p.q = codes ? q : nullptr;
    p.q_scale = q_scale;
    p.stats_out = stats;
    use_workspace(p, plan, workspace);
    return launched(launch_gn_forward(plan, p, c.type, reinterpret_cast<hipStream_t>(stream)), name);
}

}  // namespace

extern "C" {

size_t sdxl_group_norm_workspace_bytes(const sdxl_group_norm_desc* d) {
    return workspace_bytes_of(d, sdxl_hip::kGnForward, "sdxl_group_norm");
}

size_t sdxl_group_norm_i8_workspace_bytes(const sdxl_group_norm_desc* d) {
    return workspace_bytes_of(d, sdxl_hip::kGnRows, "sdxl_group_norm_i8");
}

size_t sdxl_group_norm_backward_workspace_bytes(const sdxl_group_norm_desc* d) {
    return workspace_bytes_of(d, sdxl_hip::kGnBackward, "sdxl_group_norm_backward");
}

sdxl_status sdxl_group_norm(const sdxl_group_norm_desc* d, const void* x, const void* gamma, const void* beta, void* y,
                            float* stats, void* workspace, size_t workspace_bytes, void* stream) {
    return forward(d, "sdxl_group_norm", x, gamma, beta, y, nullptr, 0, nullptr, false, stats, workspace, workspace_bytes,
                   stream);
}

sdxl_status sdxl_group_norm_i8(const sdxl_group_norm_desc* d, const void* x, const void* gamma, const void* beta,
                               int8_t* q, int64_t q_row_stride, float* q_scale, float* stats, void* workspace,
                               size_t workspace_bytes, void* stream) {
    return forward(d, "sdxl_group_norm_i8", x, gamma, beta, nullptr, q, q_row_stride, q_scale, true, stats, workspace,
                   workspace_bytes, stream);
}

sdxl_status sdxl_group_norm_backward(const sdxl_group_norm_desc* d, const void* dy, const void* x, const void* gamma,
                                     const void* beta, const float* stats, void* dx, void* dgamma, void* dbeta,
                                     void* workspace, size_t workspace_bytes, void* stream) {
    const char* name = "sdxl_group_norm_backward";
    Call c;
    const sdxl_status st = resolve(d, name, c);
    if (st != SDXL_STATUS_OK) return st;
    GnParams& p = c.p;
    if (p.channels == 0 || (c.empty && dgamma == nullptr && dbeta == nullptr) ||
        (dx == nullptr && dgamma == nullptr && dbeta == nullptr))
        return SDXL_STATUS_OK;
    if (!c.empty && (dy == nullptr || x == nullptr || gamma == nullptr || beta == nullptr || stats == nullptr))
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "null tensor pointer");
    const uintptr_t e = (uintptr_t)c.elem;
    if (!aligned(dy, e) || !aligned(x, e) || !aligned(gamma, e) || !aligned(beta, e) || !aligned(dx, e) ||
        !aligned(dgamma, e) || !aligned(dbeta, e) || !aligned(stats, 4))
        return fail(name, SDXL_STATUS_UNSUPPORTED, "tensor not aligned to its elements");
    const GnPlan plan = gn_plan(p, c.type, sdxl_hip::kGnBackward);
    const size_t need = c.empty ? 0 : workspace_of(c, plan, true);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 256)))
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "workspace missing, small or misaligned");
    const Area out[4] = {matrix(dx, c.rows, p.channels, p.ld_y, c.elem), vector(dgamma, p.channels, c.elem),
                         vector(dbeta, p.channels, c.elem), vector(need > 0 ? workspace : nullptr, (int64_t)need, 1)};
    for (int i = 0; i < 4; ++i) {
        if (!c.empty && overlaps_one(out[i], {matrix(x, c.rows, p.channels, p.ld_x, c.elem), matrix(dy, c.rows, p.channels, p.ld_dy, c.elem),
                                              vector(gamma, p.channels, c.elem), vector(beta, p.channels, c.elem),
                                              vector(stats, 2 * (int64_t)p.batch * p.groups, 4)}))
            return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "a gradient or the workspace overlaps an input");
        for (int j = 0; j < i; ++j)
            if (overlap(out[i], out[j])) return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "a gradient overlaps another one or the workspace");
    }
    p.dy = dy;
    p.x = x;
    p.gamma = gamma;
    p.beta = beta;
    p.stats = stats;
    p.y = dx;
    p.dgamma = dgamma;
    p.dbeta = dbeta;
    use_workspace(p, plan, workspace);
    if (c.empty) p.chunks = 0;  // no sums: zeros
    return launched(launch_gn_backward(plan, p, c.type, reinterpret_cast<hipStream_t>(stream)), name);
}

}  // extern "C"
