// Device helpers shared by the feed-forward kernels: element types, matrix
// instructions by type, the activations and their slopes.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/sdxl_hip/feed_forward.h"
#include "sublayer_device.hpp"

namespace sdxl_hip {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct FfType;
template <>
struct FfType<_Float16> {
    static __device__ __forceinline__ f32x16 mfma(i16x8 a, i16x8 b, f32x16 c) { return mfma32(a, b, c); }
    // two values rounded to nearest even
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const f16x2 v{(_Float16)a, (_Float16)b};
        return __builtin_bit_cast(uint32_t, v);
    }
    static __device__ __forceinline__ float lo(uint32_t v) { return (float)__builtin_bit_cast(f16x2, v)[0]; }
    static __device__ __forceinline__ float hi(uint32_t v) { return (float)__builtin_bit_cast(f16x2, v)[1]; }
    // the sum of two packed values and s
    static __device__ __forceinline__ float dot_ones(uint32_t v, float s) {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, v), f16x2{(_Float16)1.0f, (_Float16)1.0f}, s, false);
    }
    // four E4M3 codes, every one exact in the type
    static __device__ __forceinline__ uint2 decode(uint32_t codes) { return e4m3x4_to_f16(codes); }
};
template <>
struct FfType<__bf16> {
    static __device__ __forceinline__ f32x16 mfma(i16x8 a, i16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const bf16x2 v{(__bf16)a, (__bf16)b};
        return __builtin_bit_cast(uint32_t, v);
    }
    static __device__ __forceinline__ float lo(uint32_t v) { return __uint_as_float(v << 16); }
    static __device__ __forceinline__ float hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }
    static __device__ __forceinline__ float dot_ones(uint32_t v, float s) {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, v), bf16x2{(__bf16)1.0f, (__bf16)1.0f}, s, false);
    }
    static __device__ __forceinline__ uint2 decode(uint32_t codes) {
        const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, false);
        const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, true);
        return uint2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
    }
};

// 16 bytes at any element's address
template <int kAlign>
struct __attribute__((packed, aligned(kAlign))) Unaligned {
    u32x4 v;
};

// A chunk of 16 bytes (kAll elements) of a row that 16-byte accesses do not divide, of which the row has `valid` elements
// (none: 0 or less; rows have at least kAll). One that the row ends in is read as the row's last 16 bytes and shifted
// by settle_chunk, which waits for the read.
template <int kAll>
__device__ __forceinline__ u32x4 fetch_chunk(const char* at, int valid) {
    constexpr int kElem = 16 / kAll;
    u32x4 d{};
    if (valid > 0) d = ((const Unaligned<kElem>*)(at - (valid < kAll ? kAll - valid : 0) * kElem))->v;
    return d;
}

template <int kAll>
__device__ __forceinline__ u32x4 settle_chunk(u32x4 d, int valid) {
    const int bits = valid < kAll && valid > 0 ? (kAll - valid) * (128 / kAll) : 0;
    uint64_t lo = d[0] | (uint64_t)d[1] << 32, hi = d[2] | (uint64_t)d[3] << 32;
    if (bits >= 64) {
        lo = hi >> (bits - 64);
        hi = 0;
    } else if (bits > 0) {
        lo = lo >> bits | hi << (64 - bits);
        hi >>= bits;
    }
    return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// An operand's window as a buffer descriptor (raw, byte offsets): reads at or
// past `size` return zero.
struct Window {
    const char* base;
    uint32_t size;
};

__device__ __forceinline__ u32x4 window_rsrc(Window w) {
    const uint64_t b = (uint64_t)(uintptr_t)w.base;
    return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)b),
                 (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32) & 0xFFFFu),
                 (uint32_t)__builtin_amdgcn_readfirstlane(w.size), 0x00020000u};
}

// 1-KiB transfer: lane l's 16 bytes at offset voff of the window go to lds +
// 16 l. Ordered by explicit waits and barriers, as the attention kernel's.
__device__ __forceinline__ void window_to_lds(u32x4 rsrc, uint32_t voff, uint32_t lds) {
    lds = __builtin_amdgcn_readfirstlane(lds);
    asm volatile(
        "s_nop 4\n\t"
        "buffer_load_dwordx4 %0, %1, 0 offen lds"
        :
        : "v"(voff), "s"(rsrc), "{m0}"(lds));
}

constexpr uint32_t kOutside = 0x80000000u;  // past every window (their sizes stay below 2^31)

// ---- activations, in families that a workgroup chooses from once (the
// activation is uniform): z and relu; z sigmoid(c0 z), which is silu and quick
// gelu; z sigmoid(z (c0 + c1 z^2)), the tanh form of gelu (1 + tanh u = 2
// sigmoid(2u)); and gelu. Infinite z takes the limit, NaN stays NaN.
struct FfAct {
    float lo, kink;  // z < lo becomes lo; slope 0 at z <= kink (NaN: nowhere)
    float c0, c1;    // of the sigmoid's argument
};

enum FfFamily { kFamLinear, kFamSigmoid, kFamTanh, kFamErf };

__device__ __forceinline__ FfFamily ff_family(int32_t activation) {
    return activation == SDXL_ACT_GELU ? kFamErf : activation <= SDXL_ACT_RELU ? kFamLinear : activation == SDXL_ACT_GELU_TANH ? kFamTanh : kFamSigmoid;
}

__device__ __forceinline__ FfAct ff_act(int32_t activation) {
    FfAct a;
    const bool relu = activation == SDXL_ACT_RELU;
    a.lo = relu ? 0.0f : -__builtin_inff();
    a.kink = relu ? 0.0f : __builtin_nanf("");
    const float tanh_c = 1.5957691216057308f;  // 2 sqrt(2 / pi)
    a.c0 = activation == SDXL_ACT_QUICK_GELU ? 1.702f : activation == SDXL_ACT_GELU_TANH ? tanh_c : 1.0f;
    a.c1 = tanh_c * 0.044715f;
    return a;
}

// Upper tail of the normal distribution, Q(x) = erfc(|x| / sqrt 2) / 2 =
// e^(-x^2 / 2) R(|x|): R is a degree-6 polynomial without constant term in
// t = 1 / (1 + 0.32 |x|), fitted to erfcx(|x| / sqrt 2) / 2 (reweighted least
// squares towards the smallest relative error). Relative error 1.1e-5 for
// every |x|, a fortieth of an fp16 half-step, so that gelu keeps its relative
// precision in the negative tail; e is e^(-x^2 / 2), ax = min(|x|, 40).
__device__ __forceinline__ float ff_tail(float x, float& e, float& ax) {
    ax = __builtin_fminf(__builtin_fabsf(x), 40.0f);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.32f, ax, 1.0f));
    e = __builtin_amdgcn_exp2f(x * x * -0.7213475204444817f);
    float r = __builtin_fmaf(t, -0.06677360087633133f, 0.13958339393138885f);
    r = __builtin_fmaf(t, r, 0.04961634799838066f);
    r = __builtin_fmaf(t, r, 0.12305037677288055f);
    r = __builtin_fmaf(t, r, 0.12682831287384033f);
    r = __builtin_fmaf(t, r, 0.12768970429897308f);
    return e * (t * r);
}

// sigmoid of the two families' argument; z2 (tanh form): min(z^2, 1e30), so that c1 z^2 stays finite
template <FfFamily kFam>
__device__ __forceinline__ float ff_sigmoid(const FfAct& a, float z, float z2) {
    const float c = kFam == kFamTanh ? __builtin_fmaf(a.c1, z2, a.c0) : a.c0;
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * (c * -1.4426950408889634f)));
}

template <FfFamily kFam>
__device__ __forceinline__ float ff_value(const FfAct& a, float z) {
    if constexpr (kFam == kFamLinear) {
        return z < a.lo ? a.lo : z;
    } else if constexpr (kFam != kFamErf) {
        return __builtin_fmaxf(z, -1.0e30f) * ff_sigmoid<kFam>(a, z, __builtin_fminf(z * z, 1.0e30f));
    } else {
        float e, ax;
        const float q = ff_tail(z, e, ax);
        return __builtin_fmaf(-ax, q, __builtin_fmaxf(z, 0.0f));  // z Phi(z) = max(z, 0) - |z| Q(|z|)
    }
}

// act(z) and act'(z)
template <FfFamily kFam>
__device__ __forceinline__ float ff_slope(const FfAct& a, float z, float& value) {
    if constexpr (kFam == kFamLinear) {
        value = z < a.lo ? a.lo : z;
        return z <= a.kink ? 0.0f : 1.0f;
    } else if constexpr (kFam != kFamErf) {
        const float z2 = __builtin_fminf(z * z, 1.0e30f);
        const float s = ff_sigmoid<kFam>(a, z, z2);
        value = __builtin_fmaxf(z, -1.0e30f) * s;
        const float zc = __builtin_amdgcn_fmed3f(z, -1.0e30f, 1.0e30f);
        return __builtin_fmaf((zc * s) * (1.0f - s), kFam == kFamTanh ? __builtin_fmaf(3.0f * a.c1, z2, a.c0) : a.c0, s);
    } else {
        float e, ax;
        const float q = ff_tail(z, e, ax);
        value = __builtin_fmaf(-ax, q, __builtin_fmaxf(z, 0.0f));
        const float zc = __builtin_amdgcn_fmed3f(z, -40.0f, 40.0f);
        return __builtin_fmaf(zc * 0.3989422804014327f, e, z > 0.0f ? 1.0f - q : q);
    }
}

// act(z) where the family is not a constant
__device__ __forceinline__ float ff_value_of(const FfAct& a, FfFamily fam, float z) {
    switch (fam) {
    case kFamErf: return ff_value<kFamErf>(a, z);
    case kFamTanh: return ff_value<kFamTanh>(a, z);
    case kFamSigmoid: return ff_value<kFamSigmoid>(a, z);
    default: return ff_value<kFamLinear>(a, z);
    }
}

// the same of act'(z), with act(z)
__device__ __forceinline__ float ff_slope_of(const FfAct& a, FfFamily fam, float z, float& value) {
    switch (fam) {
    case kFamErf: return ff_slope<kFamErf>(a, z, value);
    case kFamTanh: return ff_slope<kFamTanh>(a, z, value);
    case kFamSigmoid: return ff_slope<kFamSigmoid>(a, z, value);
    default: return ff_slope<kFamLinear>(a, z, value);
    }
}

// f.operator()<family>() of the activation
template <typename Fn>
__device__ __forceinline__ void ff_with_family(int32_t activation, Fn&& f) {
    switch (ff_family(activation)) {
    case kFamErf: f.template operator()<kFamErf>(); break;
    case kFamTanh: f.template operator()<kFamTanh>(); break;
    case kFamSigmoid: f.template operator()<kFamSigmoid>(); break;
    default: f.template operator()<kFamLinear>(); break;
    }
}

}  // namespace
}  // namespace sdxl_hip
