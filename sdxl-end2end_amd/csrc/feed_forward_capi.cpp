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
    const sdxl_hip::FfChoice choice = sdxl_hip::choose_ff(p, epilogue, w_fp8, sdxl_hip_compute_units());
    return launch_status(sdxl_hip::launch_ff(choice, p, epilogue, c.bf16, w_fp8, stream), name);
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
//
// dz is held in the tensors' type. Its rounding adds as much to a gradient's distance from exact as the output's own (in
// all 2.1e-4 -> 3.0e-4 of its norm in fp16, 1.65e-3 -> 2.34e-3 in bf16), which is what the gradient of the activation has
// anywhere that it is an fp16 or bf16 tensor. Two 16-bit planes would take it away for twice the matrix instructions of
// dx and dw, the longer part of the call (dw and dx of [2048, 1280], 2 x 5120: 130 us of 192). dbias sums the rounded dz
// too: it is made beside dw, so that the three gradients belong to one dz.
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

// The products of a backward call and the kernels that they run on.
struct Backward {
    FfParams z, w, x;
    bool with_z, with_w, with_x, sums_alone;  // sums_alone: dbias without dw
    sdxl_hip::FfEpilogue z_epilogue;
    sdxl_hip::FfChoice z_choice;
    sdxl_hip::FfGradients gradients;
    float* partial;
};

Backward backward_plan(const Call& c, const void* dout, const void* x, const void* w, const void* bias, void* dx, void* dw,
                       void* dbias, void* workspace) {
    Backward b{};
    const int cus = sdxl_hip_compute_units();
    b.with_z = c.m > 0 && c.n > 0 && needs_dz(c);
    b.with_x = dx != nullptr;
    b.with_w = dw != nullptr;
    b.sums_alone = dbias != nullptr && dw == nullptr;
    const void* dz = dout;
    int64_t lddz = c.ldo;
    if (b.with_z) {
        b.z = projection(c, x, w, nullptr, bias);
        b.z.dout = dout;
        b.z.ld_dout = c.ldo;
        b.z.out = workspace;
        b.z.ld_out = b.z.out_cols_padded = dz_stride(c);
        b.z_epilogue = c.gated ? sdxl_hip::kFfGatedDz : sdxl_hip::kFfLinearDz;
        b.z_choice = sdxl_hip::choose_ff(b.z, b.z_epilogue, false, cus);
        dz = workspace;
        lddz = dz_stride(c);
    }
    b.w.ip = dz;
    b.w.jp = x;
    b.w.ld_i = lddz;
    b.w.ld_j = c.ldx;
    b.w.rows = c.features;
    b.w.cols = c.k;
    b.w.depth = c.m;
    b.w.out = dw;
    b.w.ld_out = c.lddw;
    b.w.row_sums = dbias;
    b.x.ip = dz;
    b.x.jp = w;
    b.x.ld_i = lddz;
    b.x.ld_j = c.ldw;
    b.x.rows = c.m;
    b.x.cols = c.k;
    b.x.depth = c.features;
    b.x.out = dx;
    b.x.ld_out = c.lddx;
    if (b.with_z) b.w.i_row = b.x.i_row = lddz;
    b.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + round256(dz_bytes(c)));
    b.gradients = sdxl_hip::choose_ff_gradients(b.with_w ? &b.w : nullptr, b.with_x ? &b.x : nullptr,
                                                b.sums_alone ? &b.w : nullptr,
                                                sdxl_hip::ff_partial_bytes(c.m, c.features, c.k), cus);
    return b;
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

    const Backward b = backward_plan(c, dout, x, w, bias, want_dx ? dx : nullptr, want_dw ? dw : nullptr,
                                     want_db ? dbias : nullptr, workspace);
    if (b.with_z) {
        st = launch_status(sdxl_hip::launch_ff(b.z_choice, b.z, b.z_epilogue, c.bf16, false, stream), name);
        if (st != SDXL_STATUS_OK) return st;
    }
    return launch_status(sdxl_hip::launch_ff_gradients(b.gradients, b.with_w ? &b.w : nullptr, b.with_x ? &b.x : nullptr,
                                                       b.sums_alone ? &b.w : nullptr, c.bf16, b.partial, stream), name);
}

std::string kernel_text(const sdxl_hip::FfChoice& c) {
    using sdxl_hip::FfKernel;
    static const char* const tiles[sdxl_hip::kFfTiles] = {"256x320", "256x256", "128x256", "128x192", "128x128", "64x128", "64x64"};
    static const char* const deep[] = {"32x32/8", "32x32/4", "64x64/4"};
    const std::string through = c.staged ? " staged" : "";
    switch (c.kernel) {
    case FfKernel::kGeneral: break;
    case FfKernel::kRows: return "rows/" + std::to_string(c.variant) + through;
    case FfKernel::kDeep: return std::string("deep ") + deep[c.variant] + through;
    case FfKernel::kTile: return std::string("tile ") + tiles[c.variant];
    case FfKernel::kStaged: return c.variant == 128 ? "staged 128x128" : "staged 64x64";
    }
    return "general";
}

std::string shares_text(int shares) { return shares > 1 ? " in " + std::to_string(shares) + " shares" : ""; }

std::string kernels_text(const Call& c, int32_t gradients) {
    const auto at = reinterpret_cast<void*>(uintptr_t{256});  // aligned to everything, never followed
    if (gradients == 0) {
        FfParams p = projection(c, at, at, nullptr, nullptr);
        p.ld_res = c.ldr;
        p.out = at;
        p.ld_out = c.ldo;
        return kernel_text(sdxl_hip::choose_ff(p, c.gated ? sdxl_hip::kFfGated : sdxl_hip::kFfLinear, c.w_fp8, sdxl_hip_compute_units()));
    }
    const auto wanted = [&](int32_t bit, bool any) { return (gradients & bit) != 0 && any ? at : nullptr; };
    const Backward b = backward_plan(c, at, at, at, nullptr, wanted(1, c.m > 0 && c.k > 0), wanted(2, c.n > 0 && c.k > 0),
                                     wanted(4, c.n > 0), at);
    if (!b.with_x && !b.with_w && !b.sums_alone) return "";
    const sdxl_hip::FfGradients& g = b.gradients;
    std::string text = b.with_z ? "dz " + kernel_text(b.z_choice) : "";
    const auto add = [&](const std::string& what, const char* joint) { text += (text.empty() ? "" : joint) + what; };
    const std::string dw = "dw " + kernel_text(g.w.choice) + shares_text(g.w.splits);
    const std::string dx = "dx " + kernel_text(g.x.choice) + shares_text(g.x.splits);
    const bool together = g.one_launch && b.with_w && b.with_x && g.w.choice.kernel == g.x.choice.kernel;
    if (together) {
        add((g.w_first ? dw + " + " + dx : dx + " + " + dw), "; ");
    } else {
        if (b.with_w) add(dw, "; ");
        if (b.with_x) add(dx, "; ");
    }
    if (b.sums_alone) add("dbias" + shares_text(g.sum_shares), "; ");
    return text;
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

size_t sdxl_ff_kernels(const sdxl_ff_desc* d, int32_t gated, int32_t gradients, char* text, size_t size) {
    const char* name = "sdxl_ff_kernels";
    if (text != nullptr && size > 0) text[0] = '\0';
    Call c;
    if (gradients < 0 || gradients > 7 || (gated != 0 && gated != 1)) {
        fail(name, SDXL_STATUS_INVALID_ARGUMENT, "gated must be 0 or 1, gradients 0 to 7");
        return 0;
    }
    if (resolve(d, gated == 1, gradients != 0, name, c) != SDXL_STATUS_OK) return 0;
    if (gradients == 0 && (c.m == 0 || c.n == 0)) return 0;
    const std::string kernels = kernels_text(c, gradients);
    if (text != nullptr && size > 0) text[kernels.copy(text, size - 1)] = '\0';
    return kernels.size();
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
