// Ops over the C ABI (see ops.hpp). Validation, eligibility errors and the
// profile labels follow the reference's Ops::attention
// (src/cuda/ops_kernels.cu:1912-1973), Ops::layer_norm (:1428-1460) and
// Ops::linear (src/cuda/ops_blas.cpp).
#include "sdxl_hip/ops.hpp"

#include "sdxl_hip/attention.h"
#include "sdxl_hip/feed_forward.h"
#include "sdxl_hip/group_norm.h"
#include "sdxl_hip/int8.h"
#include "sdxl_hip/sublayer.h"

#include <sstream>

namespace sdxl::hip {

namespace {

std::int32_t dtype_code(ScalarType type) {
    switch (type) {
    case ScalarType::Float16: return SDXL_DTYPE_F16;
    case ScalarType::BFloat16: return SDXL_DTYPE_BF16;
    case ScalarType::Float32: return SDXL_DTYPE_F32;
    default: throw HipError("CUDA attention mismatch");
    }
}

void validate(const Tensor& query, const Tensor& key, const Tensor& value, std::size_t heads, const Tensor* key_mask) {
    if (query.rank() != 3 || key.rank() != 3 || value.shape() != key.shape() || query.type() != key.type() ||
        value.type() != key.type() ||
        (query.type() != ScalarType::Float16 && query.type() != ScalarType::BFloat16 &&
         query.type() != ScalarType::Float32) ||
        query.size(0) != key.size(0) || query.size(2) != key.size(2) || heads == 0 || query.size(2) % heads != 0)
        throw HipError("CUDA attention mismatch");
    const std::size_t head_dimension = query.size(2) / heads;
    if (head_dimension == 0 || head_dimension > 1024)
        throw HipError("CUDA attention head dimension must be in [1,1024]");
    if (key_mask != nullptr && (key_mask->type() != ScalarType::Int32 || key_mask->rank() != 2 ||
                                key_mask->size(0) != key.size(0) || key_mask->size(1) != key.size(1)))
        throw HipError("CUDA attention key mask mismatch");
}

}  // namespace

Ops::Ops(const Runtime& runtime) : runtime_(&runtime) {}

Tensor Ops::attention(const Tensor& query, const Tensor& key, const Tensor& value, std::size_t heads, bool causal,
                      const Tensor* key_mask) const {
    validate(query, key, value, heads, key_mask);
    Tensor output = Tensor::allocate(*runtime_, query.shape(), query.type());
    attention_into(query, key, value, heads, output, causal, key_mask);
    return output;
}

void Ops::attention_into(const Tensor& query, const Tensor& key, const Tensor& value, std::size_t heads,
                         Tensor& output, bool causal, const Tensor* key_mask) const {
    validate(query, key, value, heads, key_mask);
    if (output.shape() != query.shape() || output.type() != query.type()) throw HipError("CUDA attention mismatch");

    sdxl_attn_desc desc{};
    desc.batch = static_cast<std::int64_t>(query.size(0));
    desc.q_seq = static_cast<std::int64_t>(query.size(1));
    desc.k_seq = static_cast<std::int64_t>(key.size(1));
    desc.heads = static_cast<std::int64_t>(heads);
    desc.head_dim = static_cast<std::int64_t>(query.size(2) / heads);
    desc.dtype = dtype_code(query.type());
    desc.causal = causal ? 1 : 0;
    desc.backend = static_cast<std::int32_t>(runtime_->options().attention_backend);

    std::int32_t resolved = 0;
    if (sdxl_attn_resolve_backend(&desc, key_mask != nullptr, &resolved) != SDXL_STATUS_OK)
        throw HipError(sdxl_last_error());

    std::ostringstream label;
    label << "ops/attention/" << sdxl_attn_backend_name(resolved) << "/q" << query.size(1) << "_k" << key.size(1)
          << "_h" << heads << "_d" << desc.head_dim << (causal ? "_causal" : "_full");
    const int scope = runtime_->begin_profile(label.str());
    const sdxl_status status =
        sdxl_attn_fwd(&desc, query.data(), key.data(), value.data(), key_mask ? key_mask->int32_data() : nullptr,
                      output.data(), runtime_->stream());
    runtime_->end_profile(scope);
    if (status != SDXL_STATUS_OK) throw HipError(sdxl_last_error());
}

namespace {

std::size_t rows_of(const Tensor& t) {
    const std::size_t last = t.shape().back();
    return last == 0 ? 0 : t.elements() / last;
}

void check(sdxl_status status) {
    if (status != SDXL_STATUS_OK) throw HipError(sdxl_last_error());
}

sdxl_linear_desc linear_desc(const Tensor& input, const Tensor& weight) {
    if (input.type() != ScalarType::Float16 || input.rank() < 2 || weight.rank() != 2 ||
        (weight.type() != ScalarType::Float16 && weight.type() != ScalarType::Float8E4M3))
        throw HipError("linear requires an fp16 input and an fp16 or FP8 E4M3 rank-2 weight");
    if (weight.size(1) != input.shape().back()) throw HipError("linear feature mismatch");
    const bool fp8 = weight.type() == ScalarType::Float8E4M3;
    if (fp8 && (!weight.has_dequant_scale() || weight.dequant_scale_count() != weight.size(0)))
        throw HipError("FP8 weight has invalid scaling metadata");
    sdxl_linear_desc d{};
    d.m = static_cast<std::int64_t>(rows_of(input));
    d.n = static_cast<std::int64_t>(weight.size(0));
    d.k = static_cast<std::int64_t>(weight.size(1));
    d.w_dtype = fp8 ? SDXL_DTYPE_E4M3 : SDXL_DTYPE_F16;
    return d;
}

void check_bias(const Tensor* bias, std::size_t n) {
    if (bias != nullptr && (bias->type() != ScalarType::Float16 || bias->rank() != 1 || bias->size(0) != n))
        throw HipError("linear bias mismatch");
}

std::string linear_label(const sdxl_linear_desc& d) {
    std::ostringstream label;
    label << "ops/linear/" << (d.w_dtype == SDXL_DTYPE_E4M3 ? "e4m3" : "f16") << "/m" << d.m << "_n" << d.n << "_k"
          << d.k;
    return label.str();
}

}  // namespace

Tensor Ops::layer_norm(const Tensor& input, const Tensor& weight, const Tensor& bias, float epsilon) const {
    if (input.type() != ScalarType::Float16 || weight.type() != ScalarType::Float16 ||
        bias.type() != ScalarType::Float16 || input.rank() < 2 || weight.rank() != 1 || bias.rank() != 1 ||
        weight.size(0) != input.shape().back() || bias.size(0) != input.shape().back())
        throw HipError("CUDA layer norm shape/type mismatch");
    Tensor output = Tensor::allocate(*runtime_, input.shape(), ScalarType::Float16);
    const int scope = runtime_->begin_profile("ops/layer_norm/w" + std::to_string(input.shape().back()));
    const sdxl_status st = sdxl_layer_norm(static_cast<std::int64_t>(rows_of(input)),
                                           static_cast<std::int64_t>(input.shape().back()), input.data(), 0,
                                           weight.data(), bias.data(), epsilon, output.data(), 0, runtime_->stream());
    runtime_->end_profile(scope);
    check(st);
    return output;
}

Tensor Ops::linear(const Tensor& input, const Tensor& weight, const Tensor* bias) const {
    const sdxl_linear_desc d = linear_desc(input, weight);
    check_bias(bias, weight.size(0));
    std::vector<std::size_t> shape = input.shape();
    shape.back() = weight.size(0);
    Tensor output = Tensor::allocate(*runtime_, shape, ScalarType::Float16);
    const int scope = runtime_->begin_profile(linear_label(d));
    const sdxl_status st =
        sdxl_linear(&d, input.data(), weight.data(), weight.has_dequant_scale() ? weight.dequant_scale_data() : nullptr,
                    bias ? bias->data() : nullptr, nullptr, output.data(), runtime_->stream());
    runtime_->end_profile(scope);
    check(st);
    return output;
}

Tensor Ops::layer_norm_linear(const Tensor& input, const Tensor& norm_weight, const Tensor& norm_bias,
                              const Tensor& weight, const Tensor* bias, float epsilon) const {
    const sdxl_linear_desc d = linear_desc(input, weight);
    check_bias(bias, weight.size(0));
    if (norm_weight.type() != ScalarType::Float16 || norm_bias.type() != ScalarType::Float16 ||
        norm_weight.rank() != 1 || norm_bias.rank() != 1 || norm_weight.size(0) != input.shape().back() ||
        norm_bias.size(0) != input.shape().back())
        throw HipError("CUDA layer norm shape/type mismatch");
    const bool fused = d.w_dtype == SDXL_DTYPE_E4M3 && d.k == 640 && d.n % 128 == 0;
    if (!fused) return linear(layer_norm(input, norm_weight, norm_bias, epsilon), weight, bias);
    std::vector<std::size_t> shape = input.shape();
    shape.back() = weight.size(0);
    Tensor output = Tensor::allocate(*runtime_, shape, ScalarType::Float16);
    const int scope = runtime_->begin_profile("ops/layer_norm_linear/e4m3/m" + std::to_string(d.m) + "_n" +
                                              std::to_string(d.n) + "_k" + std::to_string(d.k));
    const sdxl_status st = sdxl_layer_norm_linear(&d, input.data(), norm_weight.data(), norm_bias.data(), epsilon,
                                                  weight.data(), weight.dequant_scale_data(),
                                                  bias ? bias->data() : nullptr, output.data(), runtime_->stream());
    runtime_->end_profile(scope);
    // the fused kernel's alignment and stride conditions are checked by the call itself (nothing is
    // launched when it declines): fall back to the two-launch composition, the same values
    if (st == SDXL_STATUS_UNSUPPORTED) return linear(layer_norm(input, norm_weight, norm_bias, epsilon), weight, bias);
    check(st);
    return output;
}

void Ops::linear_residual_into(const Tensor& input, const Tensor& weight, const Tensor* bias, Tensor& hidden) const {
    const sdxl_linear_desc d = linear_desc(input, weight);
    check_bias(bias, weight.size(0));
    if (hidden.type() != ScalarType::Float16 || hidden.shape().back() != weight.size(0) ||
        rows_of(hidden) != rows_of(input))
        throw HipError("linear residual shape mismatch");
    const int scope = runtime_->begin_profile(linear_label(d) + "_residual");
    const sdxl_status st =
        sdxl_linear(&d, input.data(), weight.data(), weight.has_dequant_scale() ? weight.dequant_scale_data() : nullptr,
                    bias ? bias->data() : nullptr, hidden.data(), hidden.data(), runtime_->stream());
    runtime_->end_profile(scope);
    check(st);
}

Tensor Ops::pack_e4m3(const Tensor& weight) const {
    if (weight.type() != ScalarType::Float16 || weight.rank() != 2)
        throw HipError("FP8 weight packing requires an fp16 rank-2 weight");
    Tensor codes = Tensor::allocate(*runtime_, weight.shape(), ScalarType::Float8E4M3);
    Tensor scales = Tensor::allocate(*runtime_, {weight.size(0)}, ScalarType::Float32);
    check(sdxl_quantize_e4m3_rows(static_cast<std::int64_t>(weight.size(0)), static_cast<std::int64_t>(weight.size(1)),
                                  weight.data(), static_cast<std::uint8_t*>(codes.data()),
                                  static_cast<float*>(scales.data()), runtime_->stream()));
    codes.attach_dequant_scale(std::move(scales));
    return codes;
}

Tensor Ops::concat_rows(const Tensor& a, const Tensor& b, const Tensor& c) const {
    for (const Tensor* t : {&a, &b, &c})
        if (t->rank() != 2 || t->type() != a.type() || t->size(1) != a.size(1))
            throw HipError("concat_rows requires rank-2 tensors of one type and width");
    Tensor out = Tensor::allocate(*runtime_, {a.size(0) + b.size(0) + c.size(0), a.size(1)}, a.type());
    char* dst = static_cast<char*>(out.data());
    for (const Tensor* t : {&a, &b, &c}) {
        if (t->bytes() > 0)
            SDXL_HIP_CHECK(hipMemcpyAsync(dst, t->data(), t->bytes(), hipMemcpyDeviceToDevice, runtime_->stream()));
        dst += t->bytes();
    }
    return out;
}

Tensor Ops::concat_rows(const Tensor& a, const Tensor& b) const {
    for (const Tensor* t : {&a, &b})
        if (t->rank() != 2 || t->type() != a.type() || t->size(1) != a.size(1))
            throw HipError("concat_rows requires rank-2 tensors of one type and width");
    Tensor out = Tensor::allocate(*runtime_, {a.size(0) + b.size(0), a.size(1)}, a.type());
    char* dst = static_cast<char*>(out.data());
    for (const Tensor* t : {&a, &b}) {
        if (t->bytes() > 0)
            SDXL_HIP_CHECK(hipMemcpyAsync(dst, t->data(), t->bytes(), hipMemcpyDeviceToDevice, runtime_->stream()));
        dst += t->bytes();
    }
    return out;
}

void Ops::cross_attention_sublayer(Tensor& hidden, const Tensor& norm_weight, const Tensor& norm_bias,
                                   const Tensor& q_weight, const Tensor& context_kv, const Tensor& out_weight,
                                   const Tensor& out_bias, std::size_t heads, bool fp8_activations) const {
    if (hidden.type() != ScalarType::Float16 || hidden.rank() != 3 || heads == 0 || hidden.size(2) != heads * 64)
        throw HipError("attention sublayer requires fp16 hidden [B, S, 64 * heads]");
    const std::size_t W = hidden.size(2);
    if (q_weight.rank() != 2 || q_weight.size(0) != W || q_weight.size(1) != W ||
        out_weight.type() != ScalarType::Float16 || out_weight.rank() != 2 || out_weight.size(0) != W ||
        out_weight.size(1) != W || norm_weight.elements() != W || norm_bias.elements() != W ||
        out_bias.elements() != W)
        throw HipError("attention sublayer weight mismatch");
    if (context_kv.type() != ScalarType::Float16 || context_kv.rank() != 3 || context_kv.size(0) != hidden.size(0) ||
        context_kv.size(2) != 2 * W)
        throw HipError("cross attention requires context K|V [B, L, 2W] fp16");
    const bool fp8 = q_weight.type() == ScalarType::Float8E4M3;
    if (fp8 && (!q_weight.has_dequant_scale() || q_weight.dequant_scale_count() != W))
        throw HipError("FP8 weight has invalid scaling metadata");
    if (fp8_activations && !fp8) throw HipError("FP8 activations require a packed E4M3 q weight");
    sdxl_cross_sublayer_desc d{};
    d.batch = static_cast<std::int64_t>(hidden.size(0));
    d.seq = static_cast<std::int64_t>(hidden.size(1));
    d.heads = static_cast<std::int64_t>(heads);
    d.ctx_len = static_cast<std::int64_t>(context_kv.size(1));
    d.w_q_dtype = fp8 ? SDXL_DTYPE_E4M3 : SDXL_DTYPE_F16;
    d.attn_backend = static_cast<std::int32_t>(runtime_->options().attention_backend);
    d.q_activations = fp8_activations ? SDXL_DTYPE_E4M3 : SDXL_DTYPE_F16;
    const std::size_t ws_bytes = sdxl_cross_attn_sublayer_workspace_bytes(&d);
    Tensor workspace = Tensor::allocate(*runtime_, {ws_bytes}, ScalarType::Float8E4M3);  // raw bytes
    std::ostringstream label;
    label << "unet/cross_attention_sublayer/s" << hidden.size(1) << "_k" << context_kv.size(1) << "_h" << heads
          << (fp8_activations ? "_e4m3a" : fp8 ? "_e4m3" : "_f16");
    const int scope = runtime_->begin_profile(label.str());
    const sdxl_status st = sdxl_cross_attn_sublayer(
        &d, hidden.data(), norm_weight.data(), norm_bias.data(), q_weight.data(),
        fp8 ? q_weight.dequant_scale_data() : nullptr, context_kv.data(), 0, out_weight.data(), out_bias.data(),
        hidden.data(), workspace.data(), ws_bytes, runtime_->stream());
    runtime_->end_profile(scope);
    check(st);
}

void Ops::attention_sublayer(Tensor& hidden, const Tensor& norm_weight, const Tensor& norm_bias,
                             const Tensor& qkv_weight, const Tensor& out_weight, const Tensor& out_bias,
                             std::size_t heads, bool fp8_activations) const {
    if (hidden.type() != ScalarType::Float16 || hidden.rank() != 3 || heads == 0 || hidden.size(2) != heads * 64)
        throw HipError("attention sublayer requires fp16 hidden [B, S, 64 * heads]");
    const std::size_t W = hidden.size(2);
    if (qkv_weight.rank() != 2 || qkv_weight.size(0) != 3 * W || qkv_weight.size(1) != W ||
        out_weight.type() != ScalarType::Float16 || out_weight.rank() != 2 || out_weight.size(0) != W ||
        out_weight.size(1) != W || norm_weight.elements() != W || norm_bias.elements() != W ||
        out_bias.elements() != W)
        throw HipError("attention sublayer weight mismatch");
    const bool fp8 = qkv_weight.type() == ScalarType::Float8E4M3;
    if (fp8 && (!qkv_weight.has_dequant_scale() || qkv_weight.dequant_scale_count() != 3 * W))
        throw HipError("FP8 weight has invalid scaling metadata");
    if (fp8_activations && !fp8) throw HipError("FP8 activations require a packed E4M3 qkv weight");
    sdxl_sublayer_desc d{};
    d.batch = static_cast<std::int64_t>(hidden.size(0));
    d.seq = static_cast<std::int64_t>(hidden.size(1));
    d.heads = static_cast<std::int64_t>(heads);
    d.w_qkv_dtype = fp8 ? SDXL_DTYPE_E4M3 : SDXL_DTYPE_F16;
    d.attn_backend = static_cast<std::int32_t>(runtime_->options().attention_backend);
    d.qkv_activations = fp8_activations ? SDXL_DTYPE_E4M3 : SDXL_DTYPE_F16;
    const std::size_t ws_bytes = sdxl_attn_sublayer_workspace_bytes(&d);
    Tensor workspace = Tensor::allocate(*runtime_, {ws_bytes}, ScalarType::Float8E4M3);  // raw bytes
    std::ostringstream label;
    label << "unet/attention_sublayer/s" << hidden.size(1) << "_h" << heads << (fp8_activations ? "_e4m3a" : fp8 ? "_e4m3" : "_f16");
    const int scope = runtime_->begin_profile(label.str());
    const sdxl_status st = sdxl_attn_sublayer(
        &d, hidden.data(), norm_weight.data(), norm_bias.data(), qkv_weight.data(),
        fp8 ? qkv_weight.dequant_scale_data() : nullptr, out_weight.data(), out_bias.data(), hidden.data(),
        workspace.data(), ws_bytes, runtime_->stream());
    runtime_->end_profile(scope);
    check(st);
    // The workspace is released when `workspace` goes out of scope; hipFree
    // waits for the work queued on it.
}

namespace {

std::int32_t activation_code(Activation activation) {
    switch (activation) {
    case Activation::None: return SDXL_ACT_NONE;
    case Activation::Relu: return SDXL_ACT_RELU;
    case Activation::Gelu: return SDXL_ACT_GELU;
    case Activation::GeluTanh: return SDXL_ACT_GELU_TANH;
    case Activation::QuickGelu: return SDXL_ACT_QUICK_GELU;
    case Activation::Silu: return SDXL_ACT_SILU;
    }
    throw HipError("feed-forward: unknown activation");
}

// E4M3 weights need a scale per row.
const float* weight_scales(const Tensor& weight) {
    if (weight.type() != ScalarType::Float8E4M3) return nullptr;
    if (!weight.has_dequant_scale() || weight.dequant_scale_count() != weight.size(0))
        throw HipError("FP8 weight has invalid scaling metadata");
    return weight.dequant_scale_data();
}

sdxl_ff_desc feed_forward_desc(const Tensor& input, const Tensor& weight, const Tensor* bias, bool gated,
                               Activation activation, bool gate_first) {
    if ((input.type() != ScalarType::Float16 && input.type() != ScalarType::BFloat16) || input.rank() < 2 ||
        weight.rank() != 2 || (weight.type() != input.type() && weight.type() != ScalarType::Float8E4M3))
        throw HipError("feed-forward requires an fp16 or bf16 input and a rank-2 weight of its type or FP8 E4M3");
    if (weight.size(1) != input.shape().back() || (gated && weight.size(0) % 2 != 0))
        throw HipError("feed-forward feature mismatch");
    if (bias != nullptr && (bias->type() != input.type() || bias->rank() != 1 || bias->size(0) != weight.size(0)))
        throw HipError("feed-forward bias mismatch");
    sdxl_ff_desc d{};
    d.m = 1;  // rows: also where the input has no columns
    for (std::size_t i = 0; i + 1 < input.rank(); ++i) d.m *= static_cast<std::int64_t>(input.size(i));
    d.n = static_cast<std::int64_t>(gated ? weight.size(0) / 2 : weight.size(0));
    d.k = static_cast<std::int64_t>(weight.size(1));
    d.dtype = dtype_code(input.type());
    d.w_dtype = weight.type() == ScalarType::Float8E4M3 ? SDXL_DTYPE_E4M3 : d.dtype;
    d.activation = activation_code(activation);
    d.gate_first = gate_first ? 1 : 0;
    return d;
}

// The 8-bit integer product (weight: Int8), which gated_linear and linear_activation share.
Tensor int8_product(const Runtime& runtime, const Tensor& input, const Tensor& weight, const Tensor* bias, const Tensor* residual,
                    bool gated, Activation activation, bool gate_first) {
    const bool codes = input.type() == ScalarType::Int8;
    const ScalarType type = !codes ? input.type() : bias != nullptr ? bias->type() : residual != nullptr ? residual->type() : ScalarType::Float16;
    if ((type != ScalarType::Float16 && type != ScalarType::BFloat16) || input.rank() < 2 || weight.rank() != 2)
        throw HipError("8-bit linear requires an fp16, bf16 or Int8 input and a rank-2 weight");
    if (weight.size(1) != input.shape().back() || (gated && weight.size(0) % 2 != 0))
        throw HipError("8-bit linear feature mismatch");
    sdxl_i8_desc d{};
    d.m = 1;
    for (std::size_t i = 0; i + 1 < input.rank(); ++i) d.m *= static_cast<std::int64_t>(input.size(i));
    d.n = static_cast<std::int64_t>(gated ? weight.size(0) / 2 : weight.size(0));
    d.k = static_cast<std::int64_t>(weight.size(1));
    d.dtype = dtype_code(type);
    d.x_dtype = codes ? SDXL_DTYPE_I8 : d.dtype;
    d.activation = activation_code(activation);
    d.gate_first = gate_first ? 1 : 0;
    if (!weight.has_dequant_scale() || weight.dequant_scale_count() != weight.size(0) ||
        (codes && (!input.has_dequant_scale() || input.dequant_scale_count() != static_cast<std::size_t>(d.m))))
        throw HipError("8-bit linear requires a scale for every row of 8-bit integers");
    std::vector<std::size_t> shape = input.shape();
    shape.back() = static_cast<std::size_t>(d.n);
    if (bias != nullptr && (bias->type() != type || bias->rank() != 1 || bias->size(0) != weight.size(0)))
        throw HipError("8-bit linear bias mismatch");
    if (residual != nullptr && (residual->type() != type || residual->shape() != shape))
        throw HipError("8-bit linear residual mismatch");
    Tensor output = Tensor::allocate(runtime, shape, type);
    const std::size_t ws_bytes = gated ? sdxl_gated_linear_i8_workspace_bytes(&d) : sdxl_linear_i8_workspace_bytes(&d);
    Tensor workspace = Tensor::allocate(runtime, {ws_bytes}, ScalarType::Int8);  // raw bytes
    std::ostringstream label;
    label << "ops/" << (gated ? "gated_linear" : "linear_activation") << "/i8/m" << d.m << "_n" << d.n << "_k" << d.k;
    const int scope = runtime.begin_profile(label.str());
    const float* x_scale = codes ? input.dequant_scale_data() : nullptr;
    const auto* w = static_cast<const std::int8_t*>(weight.data());
    const void* b = bias != nullptr ? bias->data() : nullptr;
    const sdxl_status st =
        gated ? sdxl_gated_linear_i8(&d, input.data(), x_scale, w, weight.dequant_scale_data(), b, output.data(),
                                     workspace.data(), ws_bytes, runtime.stream())
              : sdxl_linear_i8(&d, input.data(), x_scale, w, weight.dequant_scale_data(), b,
                               residual != nullptr ? residual->data() : nullptr, output.data(), workspace.data(), ws_bytes,
                               runtime.stream());
    runtime.end_profile(scope);
    check(st);
    return output;
}

std::string feed_forward_label(const char* name, const sdxl_ff_desc& d) {
    std::ostringstream label;
    label << "ops/" << name << '/'
          << (d.w_dtype == SDXL_DTYPE_E4M3 ? "e4m3" : d.w_dtype == SDXL_DTYPE_BF16 ? "bf16" : "f16") << "/m" << d.m
          << "_n" << d.n << "_k" << d.k;
    return label.str();
}

}  // namespace

Tensor Ops::gated_linear(const Tensor& input, const Tensor& weight, const Tensor* bias, Activation activation,
                         bool gate_first) const {
    if (weight.type() == ScalarType::Int8)
        return int8_product(*runtime_, input, weight, bias, nullptr, true, activation, gate_first);
    const sdxl_ff_desc d = feed_forward_desc(input, weight, bias, true, activation, gate_first);
    const float* scales = weight_scales(weight);
    std::vector<std::size_t> shape = input.shape();
    shape.back() = weight.size(0) / 2;
    Tensor output = Tensor::allocate(*runtime_, shape, input.type());
    const int scope = runtime_->begin_profile(feed_forward_label("gated_linear", d));
    const sdxl_status st = sdxl_gated_linear(&d, input.data(), weight.data(), scales, bias ? bias->data() : nullptr,
                                             output.data(), runtime_->stream());
    runtime_->end_profile(scope);
    check(st);
    return output;
}

Tensor Ops::linear_activation(const Tensor& input, const Tensor& weight, const Tensor* bias, Activation activation,
                              const Tensor* residual) const {
    if (weight.type() == ScalarType::Int8)
        return int8_product(*runtime_, input, weight, bias, residual, false, activation, false);
    const sdxl_ff_desc d = feed_forward_desc(input, weight, bias, false, activation, false);
    const float* scales = weight_scales(weight);
    std::vector<std::size_t> shape = input.shape();
    shape.back() = weight.size(0);
    if (residual != nullptr && (residual->type() != input.type() || residual->shape() != shape))
        throw HipError("feed-forward residual mismatch");
    Tensor output = Tensor::allocate(*runtime_, shape, input.type());
    const int scope = runtime_->begin_profile(feed_forward_label("linear_activation", d));
    const sdxl_status st = sdxl_linear_act(&d, input.data(), weight.data(), scales, bias ? bias->data() : nullptr,
                                           residual ? residual->data() : nullptr, output.data(), runtime_->stream());
    runtime_->end_profile(scope);
    check(st);
    return output;
}

void Ops::feed_forward_sublayer(Tensor& hidden, const Tensor& norm_weight, const Tensor& norm_bias,
                                const Tensor& in_weight, const Tensor* in_bias, const Tensor& out_weight,
                                const Tensor* out_bias, Activation activation, float epsilon, bool gate_first) const {
    if (hidden.type() != ScalarType::Float16 || hidden.rank() < 2)
        throw HipError("feed-forward sublayer requires fp16 hidden [..., W]");
    const sdxl_ff_desc in = feed_forward_desc(hidden, in_weight, in_bias, true, activation, gate_first);
    const std::size_t W = hidden.shape().back(), inner = in_weight.size(0) / 2;
    if (out_weight.rank() != 2 || out_weight.size(0) != W || out_weight.size(1) != inner ||
        (out_weight.type() != ScalarType::Float16 && out_weight.type() != ScalarType::Float8E4M3) ||
        (out_bias != nullptr &&
         (out_bias->type() != ScalarType::Float16 || out_bias->rank() != 1 || out_bias->size(0) != W)) ||
        norm_weight.type() != ScalarType::Float16 || norm_bias.type() != ScalarType::Float16 ||
        norm_weight.elements() != W || norm_bias.elements() != W)
        throw HipError("feed-forward sublayer weight mismatch");
    sdxl_ff_sublayer_desc d{};
    d.rows = in.m;
    d.width = static_cast<std::int64_t>(W);
    d.inner = static_cast<std::int64_t>(inner);
    d.w_in_dtype = in.w_dtype;
    d.w_out_dtype = out_weight.type() == ScalarType::Float8E4M3 ? SDXL_DTYPE_E4M3 : SDXL_DTYPE_F16;
    d.activation = in.activation;
    d.gate_first = in.gate_first;
    d.ln_eps = epsilon;
    const float *in_scales = weight_scales(in_weight), *out_scales = weight_scales(out_weight);
    const std::size_t ws_bytes = sdxl_ff_sublayer_workspace_bytes(&d);
    Tensor workspace = Tensor::allocate(*runtime_, {ws_bytes}, ScalarType::Float8E4M3);  // raw bytes
    std::ostringstream label;
    label << "unet/feed_forward_sublayer/m" << d.rows << "_w" << W << "_i" << inner
          << (in_scales != nullptr ? "_e4m3" : "_f16");
    const int scope = runtime_->begin_profile(label.str());
    const sdxl_status st = sdxl_ff_sublayer(
        &d, hidden.data(), norm_weight.data(), norm_bias.data(), in_weight.data(), in_scales,
        in_bias ? in_bias->data() : nullptr, out_weight.data(), out_scales, out_bias ? out_bias->data() : nullptr,
        hidden.data(), workspace.data(), ws_bytes, runtime_->stream());
    runtime_->end_profile(scope);
    check(st);
}

namespace {

sdxl_group_norm_desc group_norm_desc(const Tensor& input, const Tensor& weight, const Tensor& bias, std::size_t groups,
                                     Activation activation, float epsilon) {
    if ((input.type() != ScalarType::Float16 && input.type() != ScalarType::BFloat16 && input.type() != ScalarType::Float32) ||
        input.rank() < 3 || weight.type() != input.type() || bias.type() != input.type() || weight.rank() != 1 ||
        bias.rank() != 1 || weight.size(0) != input.shape().back() || bias.size(0) != input.shape().back())
        throw HipError("group norm shape/type mismatch");
    sdxl_group_norm_desc d{};
    d.batch = static_cast<std::int64_t>(input.size(0));
    d.pixels = 1;
    for (std::size_t i = 1; i + 1 < input.rank(); ++i) d.pixels *= static_cast<std::int64_t>(input.size(i));
    d.channels = static_cast<std::int64_t>(input.shape().back());
    d.groups = static_cast<std::int64_t>(groups);
    d.dtype = dtype_code(input.type());
    d.activation = activation_code(activation);
    d.eps = epsilon;
    return d;
}

std::string group_norm_label(const char* name, const sdxl_group_norm_desc& d) {
    std::ostringstream label;
    label << "ops/" << name << "/b" << d.batch << "_p" << d.pixels << "_c" << d.channels << "_g" << d.groups;
    return label.str();
}

// Codes like the input, with a scale by row attached.
Tensor int8_like(const Runtime& runtime, const Tensor& input) {
    std::size_t rows = 1;
    for (std::size_t i = 0; i + 1 < input.rank(); ++i) rows *= input.size(i);
    Tensor codes = Tensor::allocate(runtime, input.shape(), ScalarType::Int8);
    codes.attach_dequant_scale(Tensor::allocate(runtime, {rows}, ScalarType::Float32));
    return codes;
}

float* scales_of(const Tensor& codes) { return const_cast<float*>(codes.dequant_scale_data()); }

}  // namespace

Tensor Ops::group_norm(const Tensor& input, const Tensor& weight, const Tensor& bias, std::size_t groups,
                       Activation activation, float epsilon) const {
    const sdxl_group_norm_desc d = group_norm_desc(input, weight, bias, groups, activation, epsilon);
    Tensor output = Tensor::allocate(*runtime_, input.shape(), input.type());
    const std::size_t ws_bytes = sdxl_group_norm_workspace_bytes(&d);
    Tensor workspace = Tensor::allocate(*runtime_, {ws_bytes}, ScalarType::Int8);  // raw bytes
    const int scope = runtime_->begin_profile(group_norm_label("group_norm", d));
    const sdxl_status st = sdxl_group_norm(&d, input.data(), weight.data(), bias.data(), output.data(), nullptr,
                                           workspace.data(), ws_bytes, runtime_->stream());
    runtime_->end_profile(scope);
    check(st);
    return output;
}

Tensor Ops::group_norm_int8(const Tensor& input, const Tensor& weight, const Tensor& bias, std::size_t groups,
                            Activation activation, float epsilon) const {
    const sdxl_group_norm_desc d = group_norm_desc(input, weight, bias, groups, activation, epsilon);
    Tensor codes = int8_like(*runtime_, input);
    const std::size_t ws_bytes = sdxl_group_norm_i8_workspace_bytes(&d);
    Tensor workspace = Tensor::allocate(*runtime_, {ws_bytes}, ScalarType::Int8);  // raw bytes
    const int scope = runtime_->begin_profile(group_norm_label("group_norm_i8", d));
    const sdxl_status st = sdxl_group_norm_i8(&d, input.data(), weight.data(), bias.data(), static_cast<std::int8_t*>(codes.data()),
                                              0, scales_of(codes), nullptr, workspace.data(), ws_bytes, runtime_->stream());
    runtime_->end_profile(scope);
    check(st);
    return codes;
}

Tensor Ops::layer_norm_int8(const Tensor& input, const Tensor& weight, const Tensor& bias, float epsilon) const {
    if ((input.type() != ScalarType::Float16 && input.type() != ScalarType::BFloat16) || input.rank() < 2 ||
        weight.type() != input.type() || bias.type() != input.type() || weight.rank() != 1 || bias.rank() != 1 ||
        weight.size(0) != input.shape().back() || bias.size(0) != input.shape().back())
        throw HipError("CUDA layer norm shape/type mismatch");
    Tensor codes = int8_like(*runtime_, input);
    const int scope = runtime_->begin_profile("ops/layer_norm_i8/w" + std::to_string(input.shape().back()));
    const sdxl_status st = sdxl_layer_norm_i8(static_cast<std::int64_t>(codes.dequant_scale_count()),
                                              static_cast<std::int64_t>(input.shape().back()), dtype_code(input.type()),
                                              input.data(), 0, weight.data(), bias.data(), epsilon,
                                              static_cast<std::int8_t*>(codes.data()), 0, scales_of(codes), runtime_->stream());
    runtime_->end_profile(scope);
    check(st);
    return codes;
}

Tensor Ops::pack_int8(const Tensor& input) const {
    if ((input.type() != ScalarType::Float16 && input.type() != ScalarType::BFloat16) || input.rank() < 2)
        throw HipError("8-bit packing requires an fp16 or bf16 tensor of rank 2 or more");
    Tensor codes = int8_like(*runtime_, input);
    check(sdxl_quantize_i8_rows(static_cast<std::int64_t>(codes.dequant_scale_count()),
                                static_cast<std::int64_t>(input.shape().back()), dtype_code(input.type()), input.data(), 0,
                                static_cast<std::int8_t*>(codes.data()), 0, scales_of(codes), runtime_->stream()));
    return codes;
}

}  // namespace sdxl::hip
