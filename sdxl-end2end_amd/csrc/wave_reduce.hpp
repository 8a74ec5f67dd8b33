// Reductions over 16 lanes and over a wave of 64, to every lane, in registers: DPP within rows of 16, then the row and half
// swaps. One order, whichever lanes hold what.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sdxl_hip {
namespace {

template <int kControl>
__device__ __forceinline__ float lanes_moved(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kControl, 0xf, 0xf, false));
}

template <typename Fn>
__device__ __forceinline__ float reduce16(float v, Fn&& f) {
    v = f(v, lanes_moved<0xB1>(v));   // lane ^ 1
    v = f(v, lanes_moved<0x4E>(v));   // lane ^ 2
    v = f(v, lanes_moved<0x141>(v));  // the other four of eight
    return f(v, lanes_moved<0x140>(v));
}

// of what reduce16 left
template <typename Fn>
__device__ __forceinline__ float reduce_rows(float v, Fn&& f) {
    const uint32_t d = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane16_swap(d, d, false, false);
    v = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const uint32_t h = __float_as_uint(v);
    const auto s = __builtin_amdgcn_permlane32_swap(h, h, false, false);
    return f(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

template <typename Fn>
__device__ __forceinline__ float reduce64(float v, Fn&& f) {
    return reduce_rows(reduce16(v, f), f);
}

struct Add {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct Max {
    __device__ __forceinline__ float operator()(float a, float b) const { return __builtin_fmaxf(a, b); }
};

}  // namespace
}  // namespace sdxl_hip
