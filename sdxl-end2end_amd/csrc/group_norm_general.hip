// The general group norm kernels (include/sdxl_hip/group_norm.h): any batch,
// pixels, channels, groups, strides and alignment, element by element, sums in
// 64 bits. The fast kernels (group_norm.hip) take rows of 16 bytes and more.
// One workgroup sums a group of an image, one thread an element of the second
// pass; what bounds them is the element loads ([2, 4096, 960] fp16 is 31 MB).
#include <hip/hip_runtime.h>

#include "group_norm_device.hpp"
#include "int8_device.hpp"

namespace sdxl_hip {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxGrid = 1 << 16;  // more: each workgroup takes several

// Sum over the workgroup, to every thread; part: one place a wave.
__device__ __forceinline__ double block_sum(double v, double* part) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void gn_stats_general_kernel(GnParams p) {
    __shared__ double part[4];
    const int64_t tasks = (int64_t)p.batch * p.groups, values = p.pixels * p.group_channels;
    for (int64_t task = blockIdx.x; task < tasks; task += gridDim.x) {
        const int64_t n = task / p.groups, c0 = task % p.groups * p.group_channels;
        const T* x = (const T*)p.x + n * p.pixels * p.ld_x + c0;
        auto at = [&](int64_t e) { return (double)(float)x[e / p.group_channels * p.ld_x + e % p.group_channels]; };
        double sum = 0.0, centred = 0.0;
        for (int64_t e = threadIdx.x; e < values; e += kThreads) sum += at(e);
        const double mean = block_sum(sum, part) / (double)values;
        for (int64_t e = threadIdx.x; e < values; e += kThreads) centred += (at(e) - mean) * (at(e) - mean);
        centred = block_sum(centred, part);
        if (threadIdx.x == 0) {
            p.partial[2 * task] = (float)mean;
            p.partial[2 * task + 1] = (float)centred;
        }
    }
}

// mean and rstd of a group from its one chunk
__device__ __forceinline__ float2 stats_of(const GnParams& p, int64_t group) {
    const float var = p.partial[2 * group + 1] / ((float)p.pixels * (float)p.group_channels);
    return float2{p.partial[2 * group], 1.0f / __builtin_sqrtf(var + p.eps)};
}

template <typename T, FfFamily kFam>
__device__ __forceinline__ float normed(const GnParams& p, const FfAct& act, int64_t row, int c) {
    const float2 s = stats_of(p, row / p.pixels * p.groups + c / p.group_channels);
    const float x = (float)((const T*)p.x)[row * p.ld_x + c];
    return gn_value<T, kFam>(act, __builtin_fmaf((x - s.x) * s.y, (float)((const T*)p.gamma)[c], (float)((const T*)p.beta)[c]));
}

template <typename T>
__global__ __launch_bounds__(kThreads) void gn_apply_general_kernel(GnParams p) {
    const FfAct act = ff_act(p.activation);
    const int64_t all = p.batch * p.pixels * p.channels, step = (int64_t)gridDim.x * kThreads;
    const int64_t first = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    ff_with_family(p.activation, [&]<FfFamily kFam>() {
        for (int64_t e = first; e < all; e += step) {
            const int64_t row = e / p.channels;
            const int c = (int)(e % p.channels);
            ((T*)p.y)[row * p.ld_y + c] = (T)normed<T, kFam>(p, act, row, c);
        }
    });
    if (p.stats_out != nullptr)
        for (int64_t g = first; g < (int64_t)p.batch * p.groups; g += step) {
            const float2 s = stats_of(p, g);
            p.stats_out[2 * g] = s.x;
            p.stats_out[2 * g + 1] = s.y;
        }
}

// a workgroup a row
template <typename T>
__global__ __launch_bounds__(kThreads) void gn_apply_i8_general_kernel(GnParams p) {
    __shared__ float part[4];
    __shared__ int nan_part[4];
    const FfAct act = ff_act(p.activation);
    const int64_t rows = p.batch * p.pixels;
    ff_with_family(p.activation, [&]<FfFamily kFam>() {
        for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
            float amax = 0.0f;
            int has_nan = 0;
            for (int c = threadIdx.x; c < p.channels; c += kThreads) {
                const float v = normed<T, kFam>(p, act, row, c), m = __builtin_fabsf(v);
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
                part[threadIdx.x >> 6] = amax;
                nan_part[threadIdx.x >> 6] = has_nan;
            }
            __syncthreads();
            amax = __builtin_fmaxf(__builtin_fmaxf(part[0], part[1]), __builtin_fmaxf(part[2], part[3]));
            const float scale = i8_scale(amax, (nan_part[0] | nan_part[1] | nan_part[2] | nan_part[3]) != 0);
            for (int c = threadIdx.x; c < p.channels; c += kThreads)
                p.q[row * p.ld_q + c] = (int8_t)i8_code(normed<T, kFam>(p, act, row, c), scale);
            if (threadIdx.x == 0) p.q_scale[row] = scale;
        }
    });
    if (p.stats_out != nullptr)
        for (int64_t g = (int64_t)blockIdx.x * kThreads + threadIdx.x; g < (int64_t)p.batch * p.groups; g += (int64_t)gridDim.x * kThreads) {
            const float2 s = stats_of(p, g);
            p.stats_out[2 * g] = s.x;
            p.stats_out[2 * g + 1] = s.y;
        }
}

// dz and n of an element
template <typename T, FfFamily kFam>
__device__ __forceinline__ float2 dz_of(const GnParams& p, const FfAct& act, int64_t row, int c) {
    const float* s = p.stats + 2 * (row / p.pixels * p.groups + c / p.group_channels);
    const float n = ((float)((const T*)p.x)[row * p.ld_x + c] - s[0]) * s[1];
    const float z = __builtin_fmaf(n, (float)((const T*)p.gamma)[c], (float)((const T*)p.beta)[c]);
    return float2{(float)((const T*)p.dy)[row * p.ld_dy + c] * gn_slope<T, kFam>(act, z), n};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void gn_sums_general_kernel(GnParams p) {
    __shared__ double part[4];
    const FfAct act = ff_act(p.activation);
    const int64_t tasks = (int64_t)p.batch * p.groups;
    ff_with_family(p.activation, [&]<FfFamily kFam>() {
        for (int64_t task = blockIdx.x; task < tasks; task += gridDim.x) {
            const int64_t n = task / p.groups;
            double first = 0.0, second = 0.0;
            for (int i = 0; i < p.group_channels; ++i) {
                const int c = (int)(task % p.groups) * p.group_channels + i;
                double s1 = 0.0, s2 = 0.0;
                for (int64_t pixel = threadIdx.x; pixel < p.pixels; pixel += kThreads) {
                    const float2 d = dz_of<T, kFam>(p, act, n * p.pixels + pixel, c);
                    s1 += (double)d.x;
                    s2 += (double)d.x * (double)d.y;
                }
                s1 = block_sum(s1, part);
                s2 = block_sum(s2, part);
                if (threadIdx.x == 0) {
                    p.channel_sums[2 * (n * p.channels + c)] = (float)s1;
                    p.channel_sums[2 * (n * p.channels + c) + 1] = (float)s2;
                }
                const double gamma = (double)(float)((const T*)p.gamma)[c];
                first += gamma * s1;
                second += gamma * s2;
            }
            if (threadIdx.x == 0) {
                p.partial[2 * task] = (float)first;
                p.partial[2 * task + 1] = (float)second;
            }
        }
    });
}

template <typename T>
__global__ __launch_bounds__(kThreads) void gn_dx_general_kernel(GnParams p) {
    const FfAct act = ff_act(p.activation);
    const int64_t all = p.batch * p.pixels * p.channels, step = (int64_t)gridDim.x * kThreads;
    const float over = 1.0f / ((float)p.pixels * (float)p.group_channels);
    ff_with_family(p.activation, [&]<FfFamily kFam>() {
        for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < all; e += step) {
            const int64_t row = e / p.channels;
            const int c = (int)(e % p.channels);
            const int64_t group = row / p.pixels * p.groups + c / p.group_channels;
            const float2 d = dz_of<T, kFam>(p, act, row, c);
            const float a = p.partial[2 * group] * over, b = p.partial[2 * group + 1] * over;
            ((T*)p.y)[row * p.ld_y + c] =
                (T)(p.stats[2 * group + 1] * (__builtin_fmaf(-d.y, b, d.x * (float)((const T*)p.gamma)[c]) - a));
        }
    });
}

// dgamma and dbeta of a channel: the images' and chunks' sums
template <typename T>
__global__ __launch_bounds__(kThreads) void gn_parameters_general_kernel(GnParams p) {
    const int64_t parts = (int64_t)p.batch * p.chunks;
    for (int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x; c < p.channels; c += (int64_t)gridDim.x * kThreads) {
        double s1 = 0.0, s2 = 0.0;
        for (int64_t k = 0; k < parts; ++k) {
            s1 += (double)p.channel_sums[2 * (k * p.channels + c)];
            s2 += (double)p.channel_sums[2 * (k * p.channels + c) + 1];
        }
        if (p.dbeta != nullptr) ((T*)p.dbeta)[c] = (T)(float)s1;
        if (p.dgamma != nullptr) ((T*)p.dgamma)[c] = (T)(float)s2;
    }
}

unsigned grid_of(int64_t blocks) { return (unsigned)(blocks < 1 ? 1 : blocks < kMaxGrid ? blocks : kMaxGrid); }

#define GN_LAUNCH(kernel, blocks)                                                                                          \
    do {                                                                                                                   \
        const dim3 grid(grid_of(blocks));                                                                                  \
        if (type == kGnF16) hipLaunchKernelGGL(kernel<_Float16>, grid, dim3(kThreads), 0, stream, p);                      \
        else if (type == kGnBf16) hipLaunchKernelGGL(kernel<__bf16>, grid, dim3(kThreads), 0, stream, p);                  \
        else hipLaunchKernelGGL(kernel<float>, grid, dim3(kThreads), 0, stream, p);                                        \
        return hipGetLastError();                                                                                          \
    } while (0)

int64_t threads_of(int64_t n) { return (n + kThreads - 1) / kThreads; }

}  // namespace

hipError_t launch_gn_stats_general(const GnParams& p, GnType type, hipStream_t stream) {
    GN_LAUNCH(gn_stats_general_kernel, (int64_t)p.batch * p.groups);
}

hipError_t launch_gn_apply_general(const GnParams& p, GnType type, hipStream_t stream) {
    if (p.q != nullptr) GN_LAUNCH(gn_apply_i8_general_kernel, p.batch * p.pixels);
    GN_LAUNCH(gn_apply_general_kernel, threads_of(p.batch * p.pixels * p.channels));
}

hipError_t launch_gn_sums_general(const GnParams& p, GnType type, hipStream_t stream) {
    GN_LAUNCH(gn_sums_general_kernel, (int64_t)p.batch * p.groups);
}

hipError_t launch_gn_dx_general(const GnParams& p, GnType type, hipStream_t stream) {
    GN_LAUNCH(gn_dx_general_kernel, threads_of(p.batch * p.pixels * p.channels));
}

hipError_t launch_gn_parameters_general(const GnParams& p, GnType type, hipStream_t stream) {
    GN_LAUNCH(gn_parameters_general_kernel, threads_of(p.channels));
}

}  // namespace sdxl_hip
