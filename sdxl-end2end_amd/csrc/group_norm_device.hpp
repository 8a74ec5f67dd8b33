// Device helpers shared by the group norm kernels: the activation by element
// type, and a row quantised to 8-bit integers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "feed_forward_device.hpp"
#include "group_norm_kernels.hpp"

namespace sdxl_hip {
namespace {

// act(z). The feed-forward kernels' forms, but for gelu of fp32 tensors: the polynomial behind ff_tail is good to
// 1.1e-5, a fortieth of an fp16 half-step and 180 fp32 ones.
template <typename T, FfFamily kFam>
__device__ __forceinline__ float gn_value(const FfAct& a, float z) {
    if constexpr (__is_same(T, float) && kFam == kFamErf) {
        const float zc = __builtin_fmaxf(z, -30.0f);  // (0 there; -infinity too)
        return zc != zc ? z : zc * (0.5f * erfcf(zc * -0.7071067811865476f));
    } else {
        return ff_value<kFam>(a, z);
    }
}

// act'(z)
template <typename T, FfFamily kFam>
__device__ __forceinline__ float gn_slope(const FfAct& a, float z) {
    if constexpr (__is_same(T, float) && kFam == kFamErf) {
        const float zc = __builtin_amdgcn_fmed3f(z, -30.0f, 30.0f);
        return z != z ? z : __builtin_fmaf(zc * 0.3989422804014327f, __expf(-0.5f * zc * zc), 0.5f * erfcf(zc * -0.7071067811865476f));
    } else {
        float value;
        return ff_slope<kFam>(a, z, value);
    }
}

// What one step of a row's codes stands for, and the code of a value: the rule of sdxl_quantize_i8_rows. amax is over
// the row's finite values; a row with a NaN has a NaN for its scale.
__device__ __forceinline__ float i8_scale(float amax, bool has_nan) {
    const float s = amax > 0.0f ? __builtin_fmaxf(amax / 127.0f, 1e-12f) : 1.0f;
    return has_nan ? __builtin_nanf("") : s;
}
// (scale NaN: 0)
__device__ __forceinline__ int i8_code(float v, float scale) {
    return (int)__builtin_rintf(__builtin_amdgcn_fmed3f(v / scale, -127.0f, 127.0f));
}

}  // namespace
}  // namespace sdxl_hip
