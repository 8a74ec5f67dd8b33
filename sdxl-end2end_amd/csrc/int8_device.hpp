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
// (scale NaN: 0)
__device__ __forceinline__ int i8_code(float v, float scale) {
    return (int)__builtin_rintf(__builtin_amdgcn_fmed3f(v / scale, -127.0f, 127.0f));
}

struct __attribute__((packed, aligned(1))) Unaligned8 {
    u32x2 v;
};

// A row of 16-bit values over kWaves waves (of a workgroup of four), kVecs vectors of 8 a lane: vector `i` of the lane is
// the row's vector lane_of_row + 64 kWaves i. The row's last vector may overlap the one before; its first `skip` values
// are that one's.
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
        float amax = 0.0f;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            if (has(i)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float m = __builtin_fabsf(v[i][e]);
                    nan |= m != m;
                    amax = __builtin_fmaxf(amax, m < __builtin_inff() ? m : 0.0f);
                }
            }
        }
        amax = reduce(nan ? __builtin_inff() : amax, part, Max{});
        const float scale = i8_scale(amax, amax == __builtin_inff());
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            if (has(i)) {
                uint32_t d[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    d[h] = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) d[h] |= (uint32_t)(i8_code(v[i][4 * h + e], scale) & 0xff) << (8 * e);
                }
                ((Unaligned8*)(q + column(i)))->v = u32x2{d[0], d[1]};
            }
        }
        if (cols + lane < q_cols) q[cols + lane] = 0;  // (fewer than 16)
        return scale;
    }
};

}  // namespace
}  // namespace sdxl_hip
