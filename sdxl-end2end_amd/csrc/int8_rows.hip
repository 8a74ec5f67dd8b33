// Rows of 16-bit values, or of their LayerNorm, as 8-bit integers with a scale
// each (include/sdxl_hip/int8.h): scale = amax / 127, code = value / scale
// rounded to nearest even (the IEEE quotient: ties fall where the definition
// says).
#include <hip/hip_runtime.h>

#include "group_norm_device.hpp"
#include "int8_kernels.hpp"

namespace sdxl_hip {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxGrid = 1 << 16;  // more: each workgroup takes several rows

template <typename V>
__device__ __forceinline__ V block_sum(V v, V* part) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

// Any row, element by element; a workgroup a row, which is read again for every pass.
template <typename T, bool kNorm>
__global__ __launch_bounds__(kThreads) void i8_rows_general_kernel(I8RowsParams p) {
    __shared__ double part[4];
    __shared__ float max_part[4];
    __shared__ int nan_part[4];
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = (const T*)p.x + row * p.ld_x;
        float mean = 0.0f, rstd = 1.0f;
        if constexpr (kNorm) {
            double sum = 0.0, centred = 0.0;
            for (int64_t c = threadIdx.x; c < p.cols; c += kThreads) sum += (double)(float)x[c];
            const double m = block_sum(sum, part) / (double)p.cols;
            for (int64_t c = threadIdx.x; c < p.cols; c += kThreads) centred += ((double)(float)x[c] - m) * ((double)(float)x[c] - m);
            mean = (float)m;
            rstd = 1.0f / __builtin_sqrtf((float)(block_sum(centred, part) / (double)p.cols) + p.eps);
        }
        auto value = [&](int64_t c) {
            const float v = (float)x[c];
            if constexpr (kNorm) return __builtin_fmaf((v - mean) * rstd, (float)((const T*)p.gamma)[c], (float)((const T*)p.beta)[c]);
            return v;
        };
        float amax = 0.0f;
        int has_nan = 0;
        for (int64_t c = threadIdx.x; c < p.cols; c += kThreads) {
            const float v = value(c), m = __builtin_fabsf(v);
            has_nan |= v != v;
            if (m < __builtin_inff()) amax = __builtin_fmaxf(amax, m);
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            amax = __builtin_fmaxf(amax, __shfl_xor(amax, d));
            has_nan |= __shfl_xor(has_nan, d);
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            max_part[threadIdx.x >> 6] = amax;
            nan_part[threadIdx.x >> 6] = has_nan;
        }
        __syncthreads();
        amax = __builtin_fmaxf(__builtin_fmaxf(max_part[0], max_part[1]), __builtin_fmaxf(max_part[2], max_part[3]));
        const float scale = i8_scale(amax, (nan_part[0] | nan_part[1] | nan_part[2] | nan_part[3]) != 0);
        for (int64_t c = threadIdx.x; c < p.q_cols; c += kThreads) p.q[row * p.ld_q + c] = c < p.cols ? (int8_t)i8_code(value(c), scale) : (int8_t)0;
        if (threadIdx.x == 0) p.q_scale[row] = scale;
    }
}

}  // namespace

hipError_t launch_i8_rows(const I8RowsParams& p, bool bf16, hipStream_t stream) {
    const dim3 grid((unsigned)(p.rows < kMaxGrid ? p.rows : kMaxGrid));
    if (p.gamma != nullptr) {
        if (bf16) hipLaunchKernelGGL((i8_rows_general_kernel<__bf16, true>), grid, dim3(kThreads), 0, stream, p);
        else hipLaunchKernelGGL((i8_rows_general_kernel<_Float16, true>), grid, dim3(kThreads), 0, stream, p);
    } else {
        if (bf16) hipLaunchKernelGGL((i8_rows_general_kernel<__bf16, false>), grid, dim3(kThreads), 0, stream, p);
        else hipLaunchKernelGGL((i8_rows_general_kernel<_Float16, false>), grid, dim3(kThreads), 0, stream, p);
    }
    return hipGetLastError();
}

}  // namespace sdxl_hip
