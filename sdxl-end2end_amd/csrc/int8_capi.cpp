// C ABI of the 8-bit integer linears (include/sdxl_hip/int8.h): validation,
// workspaces and stream-ordered launches of the quantisers and of the products,
// which run on the feed-forward kernels.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "../../include/sdxl_hip/int8.h"
#include "capi_areas.hpp"
#include "capi_internal.hpp"
#include "feed_forward_kernels.hpp"
#include "int8_kernels.hpp"

namespace {

using sdxl_hip::Area;
using sdxl_hip::FfParams;
using sdxl_hip::I8RowsParams;
using sdxl_hip::matrix;
using sdxl_hip::overlap;
using sdxl_hip::overlaps_one;
using sdxl_hip::vector;

constexpr int64_t kMaxDepth = 131071;  // 128 * 128 * k stays below 2^31

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

sdxl_status fail(const char* name, sdxl_status status, const char* what) {
    return sdxl_hip_fail(status, std::string(name) + ": " + what);
}

sdxl_status launched(hipError_t err, const char* name) {
    return err == hipSuccess ? SDXL_STATUS_OK : fail(name, SDXL_STATUS_LAUNCH_FAILED, hipGetErrorString(err));
}

bool is_half(int32_t dtype) { return dtype == SDXL_DTYPE_F16 || dtype == SDXL_DTYPE_BF16; }

// Codes of rows, or of their LayerNorm (norm).
sdxl_status quantize(const char* name, bool norm, int64_t rows, int64_t cols, int32_t dtype, const void* x, int64_t ldx,
                     const void* gamma, const void* beta, float eps, int8_t* q, int64_t ldq, float* q_scale, void* stream) {
    if (!is_half(dtype)) return fail(name, SDXL_STATUS_INVALID_SHAPE, "tensors must be fp16 or bf16");
    if (norm && (!(eps >= 0.0f) || std::isinf(eps))) return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "eps must be finite and not negative");
    if (rows < 0 || cols < 0 || rows > INT32_MAX || cols > INT32_MAX) return fail(name, SDXL_STATUS_INVALID_SHAPE, "dimensions out of range");
    if (ldx == 0) ldx = cols;
    if (ldq == 0) ldq = cols;
    if (ldx < cols || ldq < cols) return fail(name, SDXL_STATUS_INVALID_SHAPE, "row stride smaller than the row");
    if (ldx > INT32_MAX || ldq > INT32_MAX) return fail(name, SDXL_STATUS_INVALID_SHAPE, "row stride out of range");
    if (rows == 0) return SDXL_STATUS_OK;
    if (q_scale == nullptr || (cols > 0 && (x == nullptr || q == nullptr || (norm && (gamma == nullptr || beta == nullptr)))))
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "null tensor pointer");
    if (!aligned(x, 2) || !aligned(gamma, 2) || !aligned(beta, 2) || !aligned(q_scale, 4))
        return fail(name, SDXL_STATUS_UNSUPPORTED, "tensor not aligned to its elements");
    const Area in = matrix(x, rows, cols, ldx), g = vector(norm ? gamma : nullptr, cols), b = vector(norm ? beta : nullptr, cols);
    const Area codes = matrix(q, rows, cols, ldq, 1), scales = vector(q_scale, rows, 4);
    if (overlaps_one(codes, {in, g, b}) || overlaps_one(scales, {in, g, b}))
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "an output overlaps an input");
    if (overlap(codes, scales)) return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "the codes overlap the scales");
    I8RowsParams p{};
    p.x = x;
    p.gamma = norm ? (cols > 0 ? gamma : nullptr) : nullptr;
    p.beta = beta;
    p.q = q;
    p.q_scale = q_scale;
    p.rows = rows;
    p.cols = p.q_cols = cols;
    p.ld_x = ldx;
    p.ld_q = ldq;
    p.eps = eps == 0.0f ? 1e-5f : eps;
    return launched(launch_i8_rows(p, dtype == SDXL_DTYPE_BF16, reinterpret_cast<hipStream_t>(stream)), name);
}

// A descriptor with its strides resolved.
struct Call {
    int64_t m, n, k, features;  // features: rows of w
    int64_t ldx, ldw, ldo, ldr;
    bool bf16, tokens;          // tokens: x in 16 bits
};

sdxl_status resolve(const sdxl_i8_desc* d, bool gated, const char* name, Call& c) {
    if (d == nullptr) return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "null descriptor");
    if (d->reserved != 0) return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "reserved field must be 0");
    if (!is_half(d->dtype)) return fail(name, SDXL_STATUS_INVALID_SHAPE, "tensors must be fp16 or bf16");
    if (d->x_dtype != SDXL_DTYPE_I8 && d->x_dtype != d->dtype)
        return fail(name, SDXL_STATUS_INVALID_SHAPE, "x must be 8-bit integers or have the tensors' type");
    if (d->activation < SDXL_ACT_NONE || d->activation > SDXL_ACT_SILU)
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "unknown activation");
    if (d->gate_first < 0 || d->gate_first > (gated ? 1 : 0))
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, gated ? "gate_first must be 0 or 1" : "gate_first must be 0");
    if (d->m < 0 || d->n < 0 || d->k < 0 || d->m > INT32_MAX || d->n > (gated ? INT32_MAX / 2 : INT32_MAX) || d->k > INT32_MAX)
        return fail(name, SDXL_STATUS_INVALID_SHAPE, "dimensions out of range");
    if (d->k > kMaxDepth) return fail(name, SDXL_STATUS_UNSUPPORTED, "k must be at most 131071 (32-bit sums)");
    c = {d->m, d->n, d->k, gated ? 2 * d->n : d->n, 0, 0, 0, 0, d->dtype == SDXL_DTYPE_BF16, d->x_dtype != SDXL_DTYPE_I8};
    const int64_t given[4] = {d->x_row_stride, d->w_row_stride, d->out_row_stride, d->residual_row_stride};
    const int64_t row[4] = {d->k, d->k, d->n, d->n};
    int64_t* to[4] = {&c.ldx, &c.ldw, &c.ldo, &c.ldr};
    for (int i = 0; i < 4; ++i) {
        *to[i] = given[i] == 0 ? row[i] : given[i];
        if (*to[i] < row[i]) return fail(name, SDXL_STATUS_INVALID_SHAPE, "row stride smaller than the row");
        if (*to[i] > INT32_MAX) return fail(name, SDXL_STATUS_INVALID_SHAPE, "row stride out of range");
    }
    return SDXL_STATUS_OK;
}

size_t round256(size_t v) { return (v + 255) / 256 * 256; }

// The workspace of 16-bit tokens: their codes, in rows that 16-byte accesses divide, then the scales.
int64_t code_stride(const Call& c) { return (c.k + 15) / 16 * 16; }
size_t code_bytes(const Call& c) { return round256((size_t)c.m * (size_t)code_stride(c)); }
// The product of the call, without its tensors; tokens: its x is theirs.
FfParams product_of(const Call& c, const sdxl_i8_desc* d, bool tokens) {
    FfParams p{};
    p.i8 = tokens ? sdxl_hip::kFfI8Tokens : sdxl_hip::kFfI8Codes;
    p.ld_i = c.tokens && !tokens ? code_stride(c) : c.ldx;
    p.ld_j = c.ldw;
    p.ld_res = c.ldr;
    p.ld_out = c.ldo;
    p.rows = c.m;
    p.cols = c.n;
    p.depth = c.k;
    p.activation = d->activation;
    p.gate_first = d->gate_first;
    return p;
}
// Tokens that the product's kernel quantises itself.
bool quantises(const Call& c, const sdxl_i8_desc* d, bool gated) {
    return c.tokens && ff_rows_tokens(product_of(c, d, true), gated ? sdxl_hip::kFfGated : sdxl_hip::kFfLinear);
}
size_t workspace_of(const Call& c, const sdxl_i8_desc* d, bool gated) {
    return !c.tokens || c.m == 0 || c.n == 0 || quantises(c, d, gated) ? 0 : code_bytes(c) + round256((size_t)c.m * 4);
}

size_t workspace_bytes_of(const sdxl_i8_desc* d, bool gated, const char* name) {
    Call c;
    return resolve(d, gated, name, c) == SDXL_STATUS_OK ? workspace_of(c, d, gated) : 0;
}

sdxl_status product(const sdxl_i8_desc* d, bool gated, const char* name, const void* x, const float* x_scale,
                    const int8_t* w, const float* w_scale, const void* bias, const void* residual, void* out,
                    void* workspace, size_t workspace_bytes, void* stream_ptr) {
    Call c;
    const sdxl_status st = resolve(d, gated, name, c);
    if (st != SDXL_STATUS_OK) return st;
    if (c.m == 0 || c.n == 0) return SDXL_STATUS_OK;
    if (c.tokens ? x_scale != nullptr : x_scale == nullptr)
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, c.tokens ? "x_scale belongs to 8-bit x" : "8-bit x needs x_scale");
    if (out == nullptr || w_scale == nullptr || (c.k > 0 && (x == nullptr || w == nullptr)))
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "null tensor pointer");
    if (!aligned(x, c.tokens ? 2 : 1) || !aligned(x_scale, 4) || !aligned(w_scale, 4) || !aligned(bias, 2) ||
        !aligned(residual, 2) || !aligned(out, 2))
        return fail(name, SDXL_STATUS_UNSUPPORTED, "tensor not aligned to its elements");
    const size_t need = workspace_of(c, d, gated);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 256)))
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "workspace missing, small or misaligned");
    const Area to = matrix(out, c.m, c.n, c.ldo), work = vector(need > 0 ? workspace : nullptr, (int64_t)need, 1);
    const Area res = matrix(residual, c.m, c.n, c.ldr);
    const bool in_place = out == residual && c.ldr == c.ldo;
    for (const Area& area : {to, work})
        if (overlaps_one(area, {matrix(x, c.m, c.k, c.ldx, c.tokens ? 2 : 1), vector(x_scale, c.m, 4),
                                matrix(w, c.features, c.k, c.ldw, 1), vector(w_scale, c.features, 4), vector(bias, c.features)}))
            return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "out or the workspace overlaps an input");
    if ((!in_place && overlap(to, res)) || overlap(work, res) || overlap(work, to))
        return fail(name, SDXL_STATUS_INVALID_ARGUMENT, "one of out, residual and the workspace overlaps another");
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_ptr);
    FfParams p = product_of(c, d, quantises(c, d, gated));
    p.ip = x;
    p.i_scale = x_scale;
    if (need > 0) {
        I8RowsParams q{};
        q.x = x;
        q.q = static_cast<int8_t*>(workspace);
        q.q_scale = reinterpret_cast<float*>(static_cast<char*>(workspace) + code_bytes(c));
        q.rows = c.m;
        q.cols = c.k;
        q.ld_x = c.ldx;
        q.ld_q = q.q_cols = code_stride(c);
        const hipError_t err = launch_i8_rows(q, c.bf16, stream);
        if (err != hipSuccess) return launched(err, name);
        p.ip = q.q;
        p.i_scale = q.q_scale;
    }
    p.jp = w;
    p.j_scale = w_scale;
    p.bias = bias;
    p.residual = residual;
    p.out = out;
    const sdxl_hip::FfEpilogue epilogue = gated ? sdxl_hip::kFfGated : sdxl_hip::kFfLinear;
    const sdxl_hip::FfChoice choice = sdxl_hip::choose_ff(p, epilogue, false, sdxl_hip_compute_units());
    return launched(sdxl_hip::launch_ff(choice, p, epilogue, c.bf16, false, stream), name);
}

}  // namespace

extern "C" {

sdxl_status sdxl_quantize_i8_rows(int64_t rows, int64_t cols, int32_t dtype, const void* x, int64_t x_row_stride,
                                  int8_t* q, int64_t q_row_stride, float* q_scale, void* stream) {
    return quantize("sdxl_quantize_i8_rows", false, rows, cols, dtype, x, x_row_stride, nullptr, nullptr, 0.0f, q,
                    q_row_stride, q_scale, stream);
}

sdxl_status sdxl_layer_norm_i8(int64_t rows, int64_t width, int32_t dtype, const void* x, int64_t x_row_stride,
                               const void* gamma, const void* beta, float eps, int8_t* q, int64_t q_row_stride,
                               float* q_scale, void* stream) {
    return quantize("sdxl_layer_norm_i8", true, rows, width, dtype, x, x_row_stride, gamma, beta, eps, q, q_row_stride,
                    q_scale, stream);
}

size_t sdxl_linear_i8_workspace_bytes(const sdxl_i8_desc* d) { return workspace_bytes_of(d, false, "sdxl_linear_i8"); }

size_t sdxl_gated_linear_i8_workspace_bytes(const sdxl_i8_desc* d) {
    return workspace_bytes_of(d, true, "sdxl_gated_linear_i8");
}

size_t sdxl_i8_kernels(const sdxl_i8_desc* d, int32_t gated, char* text, size_t size) {
    const char* name = "sdxl_i8_kernels";
    if (text != nullptr && size > 0) text[0] = '\0';
    Call c;
    if (gated != 0 && gated != 1) {
        fail(name, SDXL_STATUS_INVALID_ARGUMENT, "gated must be 0 or 1");
        return 0;
    }
    if (resolve(d, gated == 1, name, c) != SDXL_STATUS_OK || c.m == 0 || c.n == 0) return 0;
    const auto at = reinterpret_cast<void*>(uintptr_t{256});  // aligned to everything, never followed
    const bool tokens = quantises(c, d, gated == 1);
    FfParams p = product_of(c, d, tokens);
    p.ip = p.jp = p.out = at;
    const sdxl_hip::FfEpilogue epilogue = gated == 1 ? sdxl_hip::kFfGated : sdxl_hip::kFfLinear;
    std::string kernels = sdxl_hip::kernel_text(sdxl_hip::choose_ff(p, epilogue, false, sdxl_hip_compute_units()));
    if (tokens) kernels += " tokens";
    else if (c.tokens) kernels = "quantise; " + kernels;
    if (text != nullptr && size > 0) text[kernels.copy(text, size - 1)] = '\0';
    return kernels.size();
}

sdxl_status sdxl_linear_i8(const sdxl_i8_desc* d, const void* x, const float* x_scale, const int8_t* w,
                           const float* w_scale, const void* bias, const void* residual, void* out, void* workspace,
                           size_t workspace_bytes, void* stream) {
    return product(d, false, "sdxl_linear_i8", x, x_scale, w, w_scale, bias, residual, out, workspace, workspace_bytes,
                   stream);
}

sdxl_status sdxl_gated_linear_i8(const sdxl_i8_desc* d, const void* x, const float* x_scale, const int8_t* w,
                                 const float* w_scale, const void* bias, void* out, void* workspace,
                                 size_t workspace_bytes, void* stream) {
    return product(d, true, "sdxl_gated_linear_i8", x, x_scale, w, w_scale, bias, nullptr, out, workspace,
                   workspace_bytes, stream);
}

}  // extern "C"
