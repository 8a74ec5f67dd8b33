// Device helpers of the kernels that quantise rows to 8-bit integers: the rule,
// and a row that one wave or a workgroup's four hold in registers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "feed_forward_device.hpp"
#include "wave_reduce.hpp"

namespace sdxl_hip {
namespace {

// What one step of a row's codes stands for, and the code of a value: the rule of sdxl_quantize_i8_rows. amax is over
// the row's finite values; a row with a NaN has a NaN for its scale.
__device__ __forceinline__ float i8_scale(float amax, bool has_nan) {
    const float s = amax > 0.0f ? __builtin_fmaxf(amax / 127.0f, 1e-12f) : 1.0f;
    return has_nan ? __builtin_nanf("") : s;
}
// (scale NaN: any code)
__device__ __forceinline__ int i8_code(float v, float scale) {
    return (int)__builtin_rintf(__builtin_amdgcn_fmed3f(v / scale, -127.0f, 127.0f));
}
// The same of a v of at most 127 steps, in the low byte: the quotient from the scale's reciprocal, one residual step
// from which leaves it correctly rounded (Markstein), then rounded to an integer (ties to even) by the addition.
__device__ __forceinline__ uint32_t i8_code_bits(float v, float scale, float over) {
    const float q = v * over;
    return __float_as_uint(__builtin_fmaf(__builtin_fmaf(-q, scale, v), over, q) + 12582912.0f);  // 3 * 2^22
}

// Eight codes: the low bytes of two, then of all.
__device__ __forceinline__ u32x2 i8_codes(const float (&v)[8], float scale, float over, float limit) {
    u32x2 d;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = i8_code_bits(__builtin_amdgcn_fmed3f(v[4 * h + e], -limit, limit), scale, over);
        d[h] = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u) | __builtin_amdgcn_perm(c[3], c[2], 0x0c0c0400u) << 16;
    }
    return d;
}

struct __attribute__((packed, aligned(1))) Unaligned8 {
    u32x2 v;
};

// A row of 16-bit values over kWaves waves (of a workgroup of four), kVecs vectors of 8 a lane: vector `i` of the lane is
// the row's vector lane_of_row + 64 kWaves i. The row's last vector may overlap the one before; its first `skip` values
// is that one's. Lanes past the row's end hold its last vector again, which changes no maximum.
template <int kWaves, int kVecs>
struct I8Row {
    static constexpr int kLanes = 64 * kWaves;
    int cols, lane;  // lane of the row

    __device__ __forceinline__ explicit I8Row(int cols) : cols(cols), lane((int)threadIdx.x % kLanes) {}
    __device__ __forceinline__ bool has(int i) const { return (lane + kLanes * i) * 8 < cols; }
    __device__ __forceinline__ int column(int i) const { return min((lane + kLanes * i) * 8, cols - 8); }
    __device__ __forceinline__ int skip(int i) const { return (lane + kLanes * i) * 8 - column(i); }

    // over the row's lanes; part: a place for every wave
    template <typename Fn>
    static __device__ __forceinline__ float reduce(float v, float* part, Fn&& f) {
        v = reduce64(v, f);
        if constexpr (kWaves > 1) {
            static_assert(kWaves == 4, "a wave or four");
            __syncthreads();  // the part's last values are read
            if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
            __syncthreads();
            v = f(f(part[0], part[1]), f(part[2], part[3]));
        }
        return v;
    }

    // The codes of the values and their scale: codes to q, zeros from `cols` to q_cols; returns the scale.
    __device__ __forceinline__ float quantise(const float (&v)[kVecs][8], float* part, int8_t* q, int q_cols) const {
        constexpr uint32_t kInf = 0x7f800000u;
        auto largest = [&](uint32_t most) __attribute__((always_inline)) {
            uint32_t top = 0;  // magnitudes compare as their bits do, NaN above infinity
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t m = __float_as_uint(v[i][e]) & 0x7fffffffu;
                    top = max(top, m <= most ? m : 0);
                }
            }
            return __float_as_uint(reduce(__uint_as_float(top), part, [](float a, float b) __attribute__((always_inline)) {
                return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
            }));
        };
        uint32_t top = largest(0xffffffffu);
        const bool nan = top > kInf;
        if (top >= kInf) top = largest(kInf - 1);  // (all of the row's lanes)
        const float scale = i8_scale(__uint_as_float(top), nan), over = 1.0f / scale, limit = 127.0f * scale;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            if (has(i)) ((Unaligned8*)(q + column(i)))->v = i8_codes(v[i], scale, over, limit);
        }
        if (cols + lane < q_cols) q[cols + lane] = 0;  // (fewer than 16)
        return scale;
    }
};

}  // namespace
}  // namespace sdxl_hip
