// C ABI of the feed-forward operators (include/sdxl_hip/feed_forward.h):
// validation, workspaces and stream-ordered launches of the projections, their
// gradients and the feed-forward half of the transformer block (reference
// src/cuda/unet.cpp:98-149).
#include <hip/hip_runtime.h>

#include <cstdint>
#include <initializer_list>
#include <string>

#include "../../include/sdxl_hip/feed_forward.h"
#include "../../include/sdxl_hip/sublayer.h"
#include "capi_internal.hpp"
#include "feed_forward_kernels.hpp"

namespace {

using sdxl_hip::FfParams;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

sdxl_status fail(const char* name, sdxl_status status, const char* what) {
    return sdxl_hip_fail(status, std::string(name) + ": " + what);
}

// What a tensor occupies: rows of `row` bytes, `stride` bytes apart.
struct Area {
    const void* p;
    int64_t rows, row, stride;
};

Area matrix(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t elem = 2) {
    return {p, rows, cols * elem, ld * elem};
}
Area vector(const void* p, int64_t n, int64_t elem = 2) { return {p, 1, n * elem, n * elem}; }

using i128 = __int128;  // (offsets of two 63-bit areas)

i128 floor_div(i128 a, i128 b) { return a >= 0 ? a / b : -((-a + b - 1) / b); }

// Whether two areas share a byte. Slices of one wide tensor lie between each other's rows and share none: seen where
// the strides are equal or one of the areas is a single run of bytes. Of others, which lie between each other with
// different strides, only the first and last rows are looked at.
bool overlap(Area a, Area b) {
    if (a.p == nullptr || b.p == nullptr || a.rows <= 0 || b.rows <= 0 || a.row <= 0 || b.row <= 0) return false;
    const i128 d = (i128)(uintptr_t)b.p - (i128)(uintptr_t)a.p;  // b's begin from a's
    for (Area* t : {&a, &b})
        if (t->rows == 1 || t->stride == t->row) *t = {t->p, 1, t->rows * t->row, 0};
    if (a.rows > 1 && b.rows > 1 && a.stride != b.stride) {
        const auto row = [](const Area& t, int64_t r) { return Area{(const char*)t.p + r * t.stride, 1, t.row, 0}; };
        return overlap(row(a, 0), b) || overlap(row(a, a.rows - 1), b) || overlap(row(b, 0), a) || overlap(row(b, b.rows - 1), a);
    }
    if (a.rows == 1 && b.rows == 1) return d - a.row < 0 && d + b.row > 0;
    // a's row i meets b's row j where (i - j) stride lies in (d - a.row, d + b.row): the least such i - j
    const i128 stride = a.rows > 1 ? a.stride : b.stride;
    i128 t = floor_div(d - a.row, stride) + 1;
    if (t < -(i128)(b.rows - 1)) t = -(i128)(b.rows - 1);
    return t <= a.rows - 1 && t * stride < d + b.row;
}

bool overlaps_one(Area out, std::initializer_list<Area> inputs) {
    for (const Area& in : inputs)
        if (overlap(out, in)) return true;
    return false;
}

sdxl_status launch_status(hipError_t err, const char* name) {
    if (err != hipSuccess) return fail(name, SDXL_STATUS_LAUNCH_FAILED, hipGetErrorString(err));
    return SDXL_STATUS_OK;
}

// A descriptor with its strides resolved.
struct Call {
    int64_t m, n, k, features;  // features: rows of w
    int64_t ldx, ldw, ldo, ldr, lddx, lddw;
    bool gated, bf16, w_fp8;
    int32_t activation, gate_first;
};

sdxl_status resolve(const sdxl_ff_desc* d, bool gated, bool backward, const char* name, Call& c) {
    if (d == nullptr) return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "null descriptor");
    if (d->reserved != 0) return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "reserved field must be 0");
    if (d->dtype != SDXL_DTYPE_F16 && d->dtype != SDXL_DTYPE_BF16)
        return fail(name, SDXL_STATUS_INVALID_SHAPE, "tensors must be fp16 or bf16");
    if (d->w_dtype != d->dtype && d->w_dtype != SDXL_DTYPE_E4M3)
        return fail(name, SDXL_STATUS_INVALID_SHAPE, "weights must have the tensors' type or be E4M3");
    if (backward && d->w_dtype == SDXL_DTYPE_E4M3)
        return fail(name, SDXL_STATUS_UNSUPPORTED, "no gradients through E4M3 weights");
    if (d->activation < SDXL_ACT_NONE || d->activation > SDXL_ACT_SILU)
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "unknown activation");
    if (d->gate_first < 0 || d->gate_first > (gated ? 1 : 0))
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, gated ? "gate_first must be 0 or 1" : "gate_first must be 0");
    const int64_t n_max = gated ? INT32_MAX / 2 : INT32_MAX;
    if (d->m < 0 || d->n < 0 || d->k < 0 || d->m > INT32_MAX || d->n > n_max || d->k > INT32_MAX)
        return fail(name, SDXL_STATUS_INVALID_SHAPE, "dimensions out of range");
    c.m = d->m;
    c.n = d->n;
    c.k = d->k;
    c.gated = gated;
    c.features = gated ? 2 * d->n : d->n;
    c.bf16 = d->dtype == SDXL_DTYPE_BF16;
    c.w_fp8 = d->w_dtype == SDXL_DTYPE_E4M3;
    c.activation = d->activation;
    c.gate_first = d->gate_first;
    const int64_t given[6] = {d->x_row_stride,        d->w_row_stride,  d->out_row_stride,
                              d->residual_row_stride, d->dx_row_stride, d->dw_row_stride};
    const int64_t row[6] = {d->k, d->k, d->n, d->n, d->k, d->k};
    int64_t* to[6] = {&c.ldx, &c.ldw, &c.ldo, &c.ldr, &c.lddx, &c.lddw};
    for (int i = 0; i < 6; ++i) {
        *to[i] = given[i] == 0 ? row[i] : given[i];
        if (*to[i] < row[i]) return fail(name, SDXL_STATUS_INVALID_SHAPE, "row stride smaller than the row");
        if (*to[i] > INT32_MAX) return fail(name, SDXL_STATUS_INVALID_SHAPE, "row stride out of range");
    }
    return SDXL_STATUS_OK;
}

// A projection, or dz.
sdxl_status product(const FfParams& p, sdxl_hip::FfEpilogue epilogue, const Call& c, bool w_fp8, hipStream_t stream,
                    const char* name) {
    const int cus = sdxl_hip_compute_units();
    hipError_t err;
    if (sdxl_hip::ff_rows_supported(p, epilogue, w_fp8))
        err = sdxl_hip::launch_ff_rows(p, epilogue, c.bf16, w_fp8, stream);
    else if (sdxl_hip::ff_tiled_supported(p, epilogue, false, false, w_fp8))
        err = sdxl_hip::launch_ff_tiled(p, epilogue, false, c.bf16, w_fp8, cus, stream);
    else if (sdxl_hip::ff_staged_supported(p, epilogue, false, false, w_fp8))
        err = sdxl_hip::launch_ff_staged(p, epilogue, c.bf16, w_fp8, cus, stream);
    else
        err = sdxl_hip::launch_ff_general(p, epilogue, false, false, c.bf16, w_fp8, stream);
    return launch_status(err, name);
}

// The projections and their epilogue's inputs, shared by both directions.
FfParams projection(const Call& c, const void* x, const void* w, const float* w_scale, const void* bias) {
    FfParams p{};
    p.ip = x;
    p.jp = w;
    p.ld_i = c.ldx;
    p.ld_j = c.ldw;
    p.j_scale = w_scale;
    p.bias = bias;
    p.rows = c.m;
    p.cols = c.n;
    p.depth = c.k;
    p.activation = c.activation;
    p.gate_first = c.gate_first;
    return p;
}

sdxl_status forward(const sdxl_ff_desc* d, bool gated, const char* name, const void* x, const void* w,
                    const float* w_scale, const void* bias, const void* residual, void* out, void* stream) {
    Call c;
    const sdxl_status st = resolve(d, gated, false, name, c);
    if (st != SDXL_STATUS_OK) return st;
    if (c.m == 0 || c.n == 0) return SDXL_STATUS_OK;
    if (c.w_fp8 && w_scale == nullptr)
        return sdxl_hip_fail(SDXL_STATUS_INVALID_ARGUMENT, "FP8 weight has invalid scaling metadata");
    if (out == nullptr || (c.k > 0 && (x == nullptr || w == nullptr)))
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "null tensor pointer");
    if (!aligned(x, 2) || !aligned(w, c.w_fp8 ? 1 : 2) || !aligned(w_scale, 4) || !aligned(bias, 2) ||
        !aligned(residual, 2) || !aligned(out, 2))
        return fail(name, SDXL_STATUS_UNSUPPORTED, "tensor not aligned to its elements");
    const Area to = matrix(out, c.m, c.n, c.ldo);
    const bool in_place = out == residual && c.ldr == c.ldo;
    if (overlaps_one(to, {matrix(x, c.m, c.k, c.ldx), matrix(w, c.features, c.k, c.ldw, c.w_fp8 ? 1 : 2),
                          vector(bias, c.features), vector(w_scale, c.features, 4),
                          matrix(in_place ? nullptr : residual, c.m, c.n, c.ldr)}))
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "out overlaps an input");
    FfParams p = projection(c, x, w, w_scale, bias);
    p.residual = residual;
    p.ld_res = c.ldr;
    p.out = out;
    p.ld_out = c.ldo;
    return product(p, gated ? sdxl_hip::kFfGated : sdxl_hip::kFfLinear, c, c.w_fp8,
                   reinterpret_cast<hipStream_t>(stream), name);
}

size_t round256(size_t v) { return (v + 255) / 256 * 256; }

// Backward workspace: dz [m, features] with rows of a multiple of 8 elements
// (16 bytes), unless the product can take dout itself (no activation).
int64_t dz_stride(const Call& c) { return (c.features + 7) / 8 * 8; }
bool needs_dz(const Call& c) { return c.gated || c.activation != SDXL_ACT_NONE; }
size_t dz_bytes(const Call& c) { return needs_dz(c) ? (size_t)c.m * (size_t)dz_stride(c) * 2 : 0; }

// then the partial sums of products whose depth is split
size_t backward_workspace(const Call& c) {
    return round256(dz_bytes(c)) + sdxl_hip::ff_partial_bytes(c.m, c.features, c.k);
}

size_t workspace_of(const sdxl_ff_desc* d, bool gated, const char* name) {
    Call c;
    return resolve(d, gated, true, name, c) == SDXL_STATUS_OK ? backward_workspace(c) : 0;
}

sdxl_status backward(const sdxl_ff_desc* d, bool gated, const char* name, const void* dout, const void* x,
                     const void* w, const void* bias, void* dx, void* dw, void* dbias, void* workspace,
                     size_t workspace_bytes, void* stream_ptr) {
    Call c;
    sdxl_status st = resolve(d, gated, true, name, c);
    if (st != SDXL_STATUS_OK) return st;
    const bool want_dx = dx != nullptr && c.m > 0 && c.k > 0, want_dw = dw != nullptr && c.n > 0 && c.k > 0;
    const bool want_db = dbias != nullptr && c.n > 0;
    if (!want_dx && !want_dw && !want_db) return SDXL_STATUS_OK;
    const bool inputs = c.m > 0 && c.n > 0;  // else every sum is empty
    const bool dz_needed = inputs && needs_dz(c);
    // w: for z and dx; x: for z and dw
    if (inputs && (dout == nullptr || (c.k > 0 && ((w == nullptr && (dz_needed || want_dx)) ||
                                                   (x == nullptr && (dz_needed || want_dw))))))
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "null tensor pointer");
    if (!aligned(x, 2) || !aligned(w, 2) || !aligned(dout, 2) || !aligned(bias, 2) || !aligned(dx, 2) ||
        !aligned(dw, 2) || !aligned(dbias, 2))
        return fail(name, SDXL_STATUS_UNSUPPORTED, "tensor not aligned to its elements");
    const size_t need = inputs ? backward_workspace(c) : 0;
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 256)))
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "workspace missing, small or misaligned");
    const Area grads[3] = {matrix(want_dx ? dx : nullptr, c.m, c.k, c.lddx),
                           matrix(want_dw ? dw : nullptr, c.features, c.k, c.lddw),
                           vector(want_db ? dbias : nullptr, c.features)};
    const Area read[4] = {matrix(dout, c.m, c.n, c.ldo), matrix(x, c.m, c.k, c.ldx), matrix(w, c.features, c.k, c.ldw),
                          vector(bias, c.features)};
    const Area work = vector(need > 0 ? workspace : nullptr, (int64_t)need, 1);
    for (int i = 0; i < 3; ++i) {
        if (inputs && overlaps_one(grads[i], {read[0], read[1], read[2], read[3]}))
            return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "a gradient overlaps an input");
        if (overlaps_one(grads[i], {grads[(i + 1) % 3], work}))
            return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "a gradient overlaps another one or the workspace");
    }
    if (inputs && overlaps_one(work, {read[0], read[1], read[2], read[3]}))
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "the workspace overlaps an input");
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_ptr);

    const void* dz = dout;
    int64_t lddz = c.ldo;
    if (dz_needed) {
        FfParams p = projection(c, x, w, nullptr, bias);
        p.dout = dout;
        p.ld_dout = c.ldo;
        p.out = workspace;
        p.ld_out = p.out_cols_padded = dz_stride(c);
        st = product(p, gated ? sdxl_hip::kFfGatedDz : sdxl_hip::kFfLinearDz, c, false, stream, name);
        if (st != SDXL_STATUS_OK) return st;
        dz = workspace;
        lddz = dz_stride(c);
    }
    FfParams pw{}, px{};
    pw.ip = dz;
    pw.jp = x;
    pw.ld_i = lddz;
    pw.ld_j = c.ldx;
    pw.rows = c.features;
    pw.cols = c.k;
    pw.depth = c.m;
    pw.out = dw;
    pw.ld_out = c.lddw;
    pw.row_sums = want_db ? dbias : nullptr;
    px.ip = dz;
    px.jp = w;
    px.ld_i = lddz;
    px.ld_j = c.ldw;
    px.rows = c.m;
    px.cols = c.k;
    px.depth = c.features;
    px.out = dx;
    px.ld_out = c.lddx;
    if (dz_needed) pw.i_row = px.i_row = lddz;
    float* partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + round256(dz_bytes(c)));
    const size_t partial_bytes = sdxl_hip::ff_partial_bytes(c.m, c.features, c.k);
    // the gradients that the tiled kernels take, then the others
    const bool w_fast = want_dw && sdxl_hip::ff_staged_supported(pw, sdxl_hip::kFfStore, true, true, false);
    const bool x_fast = want_dx && sdxl_hip::ff_staged_supported(px, sdxl_hip::kFfStore, false, true, false);
    if (w_fast || x_fast) {
        st = launch_status(sdxl_hip::launch_ff_gradients(w_fast ? &pw : nullptr, x_fast ? &px : nullptr, c.bf16, partial,
                                                         partial_bytes, sdxl_hip_compute_units(), stream), name);
        if (st != SDXL_STATUS_OK) return st;
    }
    if (want_db && !want_dw)
        st = launch_status(sdxl_hip::launch_ff_row_sums(pw, c.bf16, partial, partial_bytes, sdxl_hip_compute_units(), stream), name);
    else if (want_dw && !w_fast)
        st = launch_status(sdxl_hip::launch_ff_general(pw, sdxl_hip::kFfStore, true, true, c.bf16, false, stream), name);
    if (st == SDXL_STATUS_OK && want_dx && !x_fast)
        st = launch_status(sdxl_hip::launch_ff_general(px, sdxl_hip::kFfStore, false, true, c.bf16, false, stream), name);
    return st;
}

sdxl_status sublayer_shape(const sdxl_ff_sublayer_desc* d) {
    const char* name = "sdxl_ff_sublayer";
    if (d == nullptr) return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "null descriptor");
    if (d->reserved != 0) return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "reserved field must be 0");
    if (d->rows < 0 || d->rows > INT32_MAX || d->width <= 0 || d->inner < 0 || d->inner > INT32_MAX / 2)
        return fail(name, SDXL_STATUS_INVALID_SHAPE, "invalid shape");
    if (d->width % 2 != 0 || d->width > 2048)
        return fail(name, SDXL_STATUS_UNSUPPORTED, "width must be even and <= 2048");
    for (int32_t t : {d->w_in_dtype, d->w_out_dtype})
        if (t != SDXL_DTYPE_F16 && t != SDXL_DTYPE_E4M3)
            return fail(name, SDXL_STATUS_INVALID_SHAPE, "weights must be fp16 or E4M3");
    if (d->activation < SDXL_ACT_NONE || d->activation > SDXL_ACT_SILU)
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "unknown activation");
    if (d->gate_first < 0 || d->gate_first > 1)
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "gate_first must be 0 or 1");
    return SDXL_STATUS_OK;
}

// The sublayer's workspace: the normalised rows, then the gated activations.
size_t sublayer_workspace(const sdxl_ff_sublayer_desc* d) {
    return round256((size_t)d->rows * (size_t)d->width * 2) + round256((size_t)d->rows * (size_t)d->inner * 2);
}

}  // namespace

extern "C" {

sdxl_status sdxl_linear_act(const sdxl_ff_desc* d, const void* x, const void* w, const float* w_scale,
                            const void* bias, const void* residual, void* out, void* stream) {
    return forward(d, false, "sdxl_linear_act", x, w, w_scale, bias, residual, out, stream);
}

sdxl_status sdxl_gated_linear(const sdxl_ff_desc* d, const void* x, const void* w, const float* w_scale,
                              const void* bias, void* out, void* stream) {
    return forward(d, true, "sdxl_gated_linear", x, w, w_scale, bias, nullptr, out, stream);
}

size_t sdxl_linear_act_backward_workspace_bytes(const sdxl_ff_desc* d) {
    return workspace_of(d, false, "sdxl_linear_act_backward");
}

size_t sdxl_gated_linear_backward_workspace_bytes(const sdxl_ff_desc* d) {
    return workspace_of(d, true, "sdxl_gated_linear_backward");
}

sdxl_status sdxl_linear_act_backward(const sdxl_ff_desc* d, const void* dout, const void* x, const void* w,
                                     const void* bias, void* dx, void* dw, void* dbias, void* workspace,
                                     size_t workspace_bytes, void* stream) {
    return backward(d, false, "sdxl_linear_act_backward", dout, x, w, bias, dx, dw, dbias, workspace, workspace_bytes,
                    stream);
}

sdxl_status sdxl_gated_linear_backward(const sdxl_ff_desc* d, const void* dout, const void* x, const void* w,
                                       const void* bias, void* dx, void* dw, void* dbias, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    return backward(d, true, "sdxl_gated_linear_backward", dout, x, w, bias, dx, dw, dbias, workspace,
                    workspace_bytes, stream);
}

size_t sdxl_ff_sublayer_workspace_bytes(const sdxl_ff_sublayer_desc* d) {
    return sublayer_shape(d) == SDXL_STATUS_OK ? sublayer_workspace(d) : 0;
}

sdxl_status sdxl_ff_sublayer(const sdxl_ff_sublayer_desc* d, const void* x, const void* ln_gamma,
                             const void* ln_beta, const void* w_in, const float* w_in_scale, const void* b_in,
                             const void* w_out, const float* w_out_scale, const void* b_out, void* y,
                             void* workspace, size_t workspace_bytes, void* stream) {
    sdxl_status st = sublayer_shape(d);
    if (st != SDXL_STATUS_OK) return st;
    if (d->rows == 0) return SDXL_STATUS_OK;
    // checked before the first launch: a refused call writes nothing
    if (x == nullptr || ln_gamma == nullptr || ln_beta == nullptr || y == nullptr ||
        (d->inner > 0 && (w_in == nullptr || w_out == nullptr)))
        return fail("sdxl_ff_sublayer", SDXL_STATUS_INVALID_ARGUMENT, "null tensor pointer");
    if ((d->inner > 0 && d->w_in_dtype == SDXL_DTYPE_E4M3 && w_in_scale == nullptr) ||
        (d->w_out_dtype == SDXL_DTYPE_E4M3 && w_out_scale == nullptr))
        return sdxl_hip_fail(SDXL_STATUS_INVALID_ARGUMENT, "FP8 weight has invalid scaling metadata");
    if (!aligned(x, 4) || !aligned(ln_gamma, 4) || !aligned(ln_beta, 4) || !aligned(y, 2) || !aligned(b_in, 2) ||
        !aligned(b_out, 2) || !aligned(w_in_scale, 4) || !aligned(w_out_scale, 4) ||
        !aligned(w_in, d->w_in_dtype == SDXL_DTYPE_E4M3 ? 1 : 2) ||
        !aligned(w_out, d->w_out_dtype == SDXL_DTYPE_E4M3 ? 1 : 2))
        return fail("sdxl_ff_sublayer", SDXL_STATUS_UNSUPPORTED, "misaligned tensor");
    if (workspace == nullptr || workspace_bytes < sublayer_workspace(d) || !aligned(workspace, 256))
        return fail("sdxl_ff_sublayer", SDXL_STATUS_INVALID_ARGUMENT, "workspace missing, small or misaligned");
    const int64_t in_elem = d->w_in_dtype == SDXL_DTYPE_E4M3 ? 1 : 2, out_elem = d->w_out_dtype == SDXL_DTYPE_E4M3 ? 1 : 2;
    const Area to = matrix(y, d->rows, d->width, d->width), work = vector(workspace, (int64_t)sublayer_workspace(d), 1);
    for (const Area& area : {to, work})
        if (overlaps_one(area, {vector(ln_gamma, d->width), vector(ln_beta, d->width),
                                matrix(w_in, 2 * d->inner, d->width, d->width, in_elem), vector(w_in_scale, 2 * d->inner, 4),
                                vector(b_in, 2 * d->inner), matrix(w_out, d->width, d->inner, d->inner, out_elem),
                                vector(w_out_scale, d->width, 4), vector(b_out, d->width)}))
            return fail("sdxl_ff_sublayer", SDXL_STATUS_INVALID_ARGUMENT, "y or the workspace overlaps an input");
    const Area from = matrix(x, d->rows, d->width, d->width);
    if ((x != y && overlap(to, from)) || overlap(work, from) || overlap(work, to))
        return fail("sdxl_ff_sublayer", SDXL_STATUS_INVALID_ARGUMENT, "one of x, y and the workspace overlaps another");
    char* normed = static_cast<char*>(workspace);
    char* gated = normed + round256((size_t)d->rows * (size_t)d->width * 2);
    st = sdxl_layer_norm(d->rows, d->width, x, 0, ln_gamma, ln_beta, d->ln_eps, normed, 0, stream);
    if (st != SDXL_STATUS_OK) return st;
    sdxl_ff_desc g{};
    g.m = d->rows;
    g.n = d->inner;
    g.k = d->width;
    g.dtype = SDXL_DTYPE_F16;
    g.w_dtype = d->w_in_dtype;
    g.activation = d->activation;
    g.gate_first = d->gate_first;
    st = sdxl_gated_linear(&g, normed, w_in, w_in_scale, b_in, gated, stream);
    if (st != SDXL_STATUS_OK) return st;
    sdxl_ff_desc o{};
    o.m = d->rows;
    o.n = d->width;
    o.k = d->inner;
    o.dtype = SDXL_DTYPE_F16;
    o.w_dtype = d->w_out_dtype;
    return sdxl_linear_act(&o, gated, w_out, w_out_scale, b_out, x, y, stream);
}

}  // extern "C"
