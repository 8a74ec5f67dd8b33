// Device helpers shared by the group norm kernels: the activation by element
// type, 16 bytes of a row as fp32 values.
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
        const float zc = z < -30.0f ? -30.0f : z;  // (0 there, -infinity too; NaN stays, which a maximum would drop)
        return zc * (0.5f * erfcf(zc * -0.7071067811865476f));
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

// 16 bytes of a row as fp32 values
template <typename T>
struct GnVec {
    static constexpr int kV = 16 / (int)sizeof(T);
    static __device__ __forceinline__ u32x4 load(const char* at) { return ((const Unaligned<sizeof(T)>*)at)->v; }
    static __device__ __forceinline__ void store(char* at, u32x4 d) { ((Unaligned<sizeof(T)>*)at)->v = d; }
    // what nobody reads again before the caches are full of it
    static __device__ __forceinline__ void store_through(char* at, u32x4 d) {
        typedef u32x4 __attribute__((aligned(2))) u32x4_element;
        __builtin_nontemporal_store(d, (u32x4_element*)at);
    }
    static __device__ __forceinline__ void unpack(u32x4 d, float (&v)[kV]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (sizeof(T) == 4) {
                v[e] = __uint_as_float(d[e]);
            } else {
                v[2 * e] = FfType<T>::lo(d[e]);
                v[2 * e + 1] = FfType<T>::hi(d[e]);
            }
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&v)[kV]) {
        u32x4 d;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (sizeof(T) == 4) d[e] = __float_as_uint(v[e]);
            else d[e] = FfType<T>::pack(v[2 * e], v[2 * e + 1]);
        }
        return d;
    }
};

}  // namespace
}  // namespace sdxl_hip
