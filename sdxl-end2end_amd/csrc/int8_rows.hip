// Rows of 16-bit values, or of their LayerNorm, as 8-bit integers with a scale
// each (include/sdxl_hip/int8.h): scale = amax / 127, code = value / scale
// rounded to nearest even (the IEEE quotient: ties fall where the definition
// says).
#include <hip/hip_runtime.h>

#include "int8_device.hpp"
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

// Rows in registers: a wave a row, or four.
template <typename T, bool kNorm, int kWaves, int kVecs>
__global__ __launch_bounds__(kThreads) void i8_rows_kernel(I8RowsParams p) {
    using F = FfType<T>;
    __shared__ float part[4];
    const I8Row<kWaves, kVecs> row((int)p.cols);
    constexpr int kRows = 4 / kWaves;  // of a workgroup at a time
    for (int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / (64 * kWaves); r < p.rows; r += (int64_t)gridDim.x * kRows) {
        const char* x = (const char*)p.x + r * p.ld_x * 2;
        u32x4 d[kVecs];
#pragma unroll
        for (int i = 0; i < kVecs; ++i) d[i] = ((const Unaligned<2>*)(x + row.column(i) * 2))->v;
        u32x4 g[kNorm ? kVecs : 1], b[kNorm ? kVecs : 1];  // on the way before the sums
        // the value that the mean is summed about: of a row of one value the sum is 0 and the mean that value (10239 times
        // 2047 is not a number of 24 bits: the mean was off by 1.2e-4, and codes of such rows by 7 steps)
        [[maybe_unused]] T pivot{};
        if constexpr (kNorm) {
            pivot = *(const T*)x;
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                g[i] = ((const Unaligned<2>*)((const char*)p.gamma + row.column(i) * 2))->v;
                b[i] = ((const Unaligned<2>*)((const char*)p.beta + row.column(i) * 2))->v;
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        float v[kVecs][8];
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][2 * e] = F::lo(d[i][e]), v[i][2 * e + 1] = F::hi(d[i][e]);
        if constexpr (kNorm) {
            float sum = 0.0f, centred = 0.0f;
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                const int skip = row.has(i) ? row.skip(i) : 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum += e >= skip ? v[i][e] - (float)pivot : 0.0f;
            }
            const float mean = (float)pivot + row.reduce(sum, part, Add{}) / (float)p.cols;
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                const int skip = row.has(i) ? row.skip(i) : 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float t = e >= skip ? v[i][e] - mean : 0.0f;
                    centred = __builtin_fmaf(t, t, centred);
                }
            }
            const float rstd = 1.0f / __builtin_sqrtf(row.reduce(centred, part, Add{}) / (float)p.cols + p.eps);
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[i][2 * e] = __builtin_fmaf((v[i][2 * e] - mean) * rstd, F::lo(g[i][e]), F::lo(b[i][e]));
                    v[i][2 * e + 1] = __builtin_fmaf((v[i][2 * e + 1] - mean) * rstd, F::hi(g[i][e]), F::hi(b[i][e]));
                }
            }
        }
        const float scale = row.quantise(v, part, p.q + r * p.ld_q, (int)p.q_cols);
        if (row.lane == 0) p.q_scale[r] = scale;
    }
}

template <typename T, bool kNorm, int kWaves>
hipError_t launch_vecs(const I8RowsParams& p, hipStream_t stream) {
    const int64_t blocks = (p.rows * kWaves + 3) / 4;
    const dim3 grid((unsigned)(blocks < kMaxGrid ? blocks : kMaxGrid)), block(kThreads);
    switch ((p.cols + 512 * kWaves - 1) / (512 * kWaves)) {
    case 1: hipLaunchKernelGGL((i8_rows_kernel<T, kNorm, kWaves, 1>), grid, block, 0, stream, p); break;
    case 2: hipLaunchKernelGGL((i8_rows_kernel<T, kNorm, kWaves, 2>), grid, block, 0, stream, p); break;
    case 3: hipLaunchKernelGGL((i8_rows_kernel<T, kNorm, kWaves, 3>), grid, block, 0, stream, p); break;
    case 4: hipLaunchKernelGGL((i8_rows_kernel<T, kNorm, kWaves, 4>), grid, block, 0, stream, p); break;
    case 5: hipLaunchKernelGGL((i8_rows_kernel<T, kNorm, kWaves, 5>), grid, block, 0, stream, p); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

// A wave a row up to 5 vectors a lane, four up to 20; shorter rows than a vector and longer ones: the general kernel.
template <typename T, bool kNorm>
hipError_t launch_rows(const I8RowsParams& p, hipStream_t stream) {
    if (p.cols < 8 || p.cols > 4 * 2560) {
        hipLaunchKernelGGL((i8_rows_general_kernel<T, kNorm>), dim3((unsigned)(p.rows < kMaxGrid ? p.rows : kMaxGrid)), dim3(kThreads), 0, stream, p);
        return hipGetLastError();
    }
    return p.cols <= 2560 ? launch_vecs<T, kNorm, 1>(p, stream) : launch_vecs<T, kNorm, 4>(p, stream);
}

}  // namespace

hipError_t launch_i8_rows(const I8RowsParams& p, bool bf16, hipStream_t stream) {
    if (p.gamma != nullptr) return bf16 ? launch_rows<__bf16, true>(p, stream) : launch_rows<_Float16, true>(p, stream);
    return bf16 ? launch_rows<__bf16, false>(p, stream) : launch_rows<_Float16, false>(p, stream);
}

}  // namespace sdxl_hip
