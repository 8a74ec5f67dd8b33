// Projections of few rows (at most 16): serving a token, a time embedding, a
// short prompt. The weights' transfer is all there is, so as much of it as LDS
// holds is on its way at once.
//
// A workgroup owns 16 rows of w (gated: 8 value rows and the 8 gate rows of the
// same columns). Its waves share the depth in blocks of 64, wave v the blocks v,
// v + waves, ..: it brings them into LDS of its own (two transfers of 8 rows x
// 128 bytes, swizzled as the tiled kernel's rows; E4M3: one of 16 rows x 64
// bytes), the same depth of x into registers (16 bytes a lane), and multiplies
// them by v_mfma_f32_16x16x32 with the weight rows as the A operand. No other
// wave touches them, so the waves meet only once, when their sums are added in
// LDS in the waves' order. Up to 32 blocks (64 KiB; a depth of 2048) are on
// their way at once; deeper products repeat that. (Weights loaded
// straight into registers, 16 rows a load, took 9.5 us for [1, 1280] x [10240,
// 1280], a plain read of those bytes 5.7, this 5.7 on the device.) Rows that 16-byte
// accesses do not divide come through registers, as many blocks at once: [16,
// 5127] x [1280, 5127] 20 us, [1, 1283] x [5120, 1283] 6.7.
#include <hip/hip_runtime.h>

#include "feed_forward_device.hpp"
#include "feed_forward_kernels.hpp"

namespace sdxl_hip {
namespace {

typedef __attribute__((address_space(3))) f32x4 lds_f32x4;

template <typename T>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (__is_same(T, _Float16))
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <typename T, bool kJFp8, int kWaves, bool kGated, bool kStaged>
__global__ __launch_bounds__(64 * kWaves) void ff_rows_kernel(FfParams p) {
    using F = FfType<T>;
    constexpr int kBlocks = 32 / kWaves;  // of a wave at a time
    extern __shared__ __attribute__((aligned(1024))) char smem[];  // [kBlocks][kWaves] of kBlockBytes; then the sums
    constexpr int kBlockBytes = kJFp8 ? 1024 : 2048, kElem = kJFp8 ? 1 : 2;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    constexpr int kCols = kGated ? 8 : 16;
    const int64_t c0 = (int64_t)blockIdx.x * kCols;
    const int64_t value_row = p.gate_first ? p.cols : 0, gate_row = p.gate_first ? 0 : p.cols;
    const int depth = (int)p.depth, blocks = (depth + 63) / 64;
    const u32x4 w_rsrc = window_rsrc({(const char*)p.jp, (uint32_t)((((kGated ? 2 : 1) * p.cols - 1) * p.ld_j + p.depth) * kElem)});
    const u32x4 x_win = window_rsrc({(const char*)p.ip, (uint32_t)(((p.rows - 1) * p.ld_i + p.depth) * 2)});
    const auto x_rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)p.ip, 0, (int)x_win[2], 0x00020000);

    // the lane's row in a transfer (rows past the last one: outside), its chunk of 16 bytes
    auto w_offset = [&](int row) __attribute__((always_inline)) {
        const int64_t c = c0 + (kGated ? row & 7 : row);
        const int64_t j = kGated ? c + (row < 8 ? value_row : gate_row) : c;
        return c < p.cols ? (uint32_t)(j * p.ld_j * kElem) : kOutside;
    };
    const int row = kJFp8 ? lane >> 2 : lane >> 3;
    const uint32_t w_at[2] = {w_offset(row), kJFp8 ? 0u : w_offset(8 + row)};
    const int chunk_at[2] = {kJFp8 ? (lane & 3) ^ ((row >> 2) & 3) : (lane & 7) ^ swz(row), (lane & 7) ^ swz(8 + row)};
    const uint32_t x_at = r16 < p.rows ? (uint32_t)(r16 * p.ld_i * 2) : kOutside;

    const uint32_t lds0 = lds_addr(smem);
    u32x4 x[kBlocks][2];
    f32x4 acc{};
    for (int first = 0; first < blocks; first += 32) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the last reads of the blocks' place are done
        if constexpr (kStaged) {
            // through registers: all reads first
            constexpr int kAll = kJFp8 ? 16 : 8, kH = kJFp8 ? 1 : 2;
            u32x4 held[kBlocks][kH];
            auto x_valid = [&](int block, int q) { return r16 < p.rows ? depth - (64 * block + 32 * q + 8 * g) : 0; };
            auto w_valid = [&](int block, int h) { return w_at[h] != kOutside ? depth - 64 * block - kAll * chunk_at[h] : 0; };
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const int block = first + b * kWaves + wave;
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    x[b][q] = fetch_chunk<8>((const char*)p.ip + (r16 * p.ld_i + 64 * block + 32 * q + 8 * g) * 2, x_valid(block, q));
#pragma unroll
                for (int h = 0; h < kH; ++h)
                    held[b][h] = fetch_chunk<kAll>((const char*)p.jp + w_at[h] + (int64_t)(64 * block + kAll * chunk_at[h]) * kElem, w_valid(block, h));
            }
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const int block = first + b * kWaves + wave;
#pragma unroll
                for (int q = 0; q < 2; ++q) x[b][q] = settle_chunk<8>(x[b][q], x_valid(block, q));
                if (block < blocks) {  // (LDS holds no others)
#pragma unroll
                    for (int h = 0; h < kH; ++h)
                        *(lds_u32x4*)(smem + (b * kWaves + wave) * kBlockBytes + 1024 * h + lane * 16) = settle_chunk<kAll>(held[b][h], w_valid(block, h));
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        } else {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const int block = first + b * kWaves + wave;
                if (block < blocks) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int k = 64 * block + 32 * q + 8 * g;
                        x[b][q] = __builtin_amdgcn_raw_buffer_load_b128(x_rsrc, k < depth && x_at != kOutside ? x_at + 2 * k : kOutside, 0, 0);
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const int block = first + b * kWaves + wave;
                if (block < blocks) {
#pragma unroll
                    for (int h = 0; h < (kJFp8 ? 1 : 2); ++h) {
                        const int k = 64 * block + (kJFp8 ? 16 : 8) * chunk_at[h];
                        window_to_lds(w_rsrc, k < depth && w_at[h] != kOutside ? w_at[h] + kElem * k : kOutside,
                                      lds0 + (b * kWaves + wave) * kBlockBytes + 1024 * h);
                    }
                }
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            if (first + b * kWaves + wave < blocks) {
                const char* from = smem + (b * kWaves + wave) * kBlockBytes;
                u32x4 a[2];
                if constexpr (kJFp8) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const u32x2 codes = *(const lds_u32x2*)(from + r16 * 64 + (((2 * q + (g >> 1)) ^ ((r16 >> 2) & 3)) << 4) + 8 * (g & 1));
                        const uint2 lo = F::decode(codes[0]), hi = F::decode(codes[1]);
                        a[q] = u32x4{lo.x, lo.y, hi.x, hi.y};
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < 2; ++q) a[q] = *(const lds_u32x4*)(from + r16 * 128 + (((4 * q + g) ^ swz(r16)) << 4));
                }
#pragma unroll
                for (int q = 0; q < 2; ++q) acc = mfma16<T>(a[q], x[b][q], acc);
            }
        }
    }
    __syncthreads();  // the sums take the blocks' place
    *(lds_f32x4*)(smem + (wave * 64 + lane) * 16) = acc;
    __syncthreads();

    // acc[e] of lane l: column (w row) 4 (l / 16) + e, row l % 16
    const FfAct act = ff_act(p.activation);
    const FfFamily fam = ff_family(p.activation);
    auto sum_of = [&](int from) {
        f32x4 s{};
        for (int v = 0; v < kWaves; ++v) s += *(const lds_f32x4*)(smem + (v * 64 + from) * 16);
        return s;
    };
    auto z_of = [&](float sum, int64_t row) {
        if (p.j_scale != nullptr) sum *= p.j_scale[row];
        if (p.bias != nullptr) sum += (float)((const T*)p.bias)[row];
        return sum;
    };
    if (threadIdx.x < (kGated ? 32 : 64)) {
        const int64_t i = r16;
        if (i >= p.rows) return;
        const f32x4 a = sum_of(lane);
        f32x4 b{};
        if constexpr (kGated) b = sum_of(lane + 32);
        T* out = (T*)p.out + i * p.ld_out;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t n = c0 + 4 * g + e;
            if (n >= p.cols) continue;
            if constexpr (kGated) {
                out[n] = (T)(z_of(a[e], value_row + n) * ff_value_of(act, fam, z_of(b[e], gate_row + n)));
            } else {
                float v = ff_value_of(act, fam, z_of(a[e], n));
                if (p.residual != nullptr) v += (float)((const T*)p.residual)[i * p.ld_res + n];
                out[n] = (T)v;
            }
        }
    }
}

template <typename T, bool kJFp8, int kWaves, bool kStaged>
hipError_t launch(const FfParams& p, bool gated, hipStream_t stream) {
    const dim3 grid((unsigned)(gated ? (p.cols + 7) / 8 : (p.cols + 15) / 16)), block(64 * kWaves);
    const int64_t blocks = (p.depth + 63) / 64, held = blocks < 32 ? (blocks + kWaves - 1) / kWaves * kWaves : 32;
    const size_t lds = (size_t)held * (kJFp8 ? 1024 : 2048);  // (the sums take 1 KiB a wave)
    if (gated) hipLaunchKernelGGL((ff_rows_kernel<T, kJFp8, kWaves, true, kStaged>), grid, block, lds, stream, p);
    else hipLaunchKernelGGL((ff_rows_kernel<T, kJFp8, kWaves, false, kStaged>), grid, block, lds, stream, p);
    return hipGetLastError();
}

template <typename T, bool kJFp8, bool kStaged>
hipError_t launch_rows(const FfParams& p, bool gated, int waves, hipStream_t stream) {
    switch (waves) {
    case 16: return launch<T, kJFp8, 16, kStaged>(p, gated, stream);
    case 8: return launch<T, kJFp8, 8, kStaged>(p, gated, stream);
    case 4: return launch<T, kJFp8, 4, kStaged>(p, gated, stream);
    }
    return hipErrorInvalidValue;
}

}  // namespace

bool ff_rows_supported(const FfParams& p, FfEpilogue epilogue, bool j_fp8) {
    // one window (below 2^31 bytes) holds w, one x
    const int64_t w_rows = epilogue == kFfGated ? 2 * p.cols : p.cols;
    return (epilogue == kFfLinear || epilogue == kFfGated) && p.rows <= 16 &&
           w_rows * p.ld_j * (j_fp8 ? 1 : 2) < (int64_t{1} << 31) && ff_staged_supported(p, epilogue, false, false, j_fp8);
}

// 2048 waves in all where there are blocks for them
int ff_rows_waves(const FfParams& p, bool gated) {
    const int64_t groups = gated ? (p.cols + 7) / 8 : (p.cols + 15) / 16, blocks = (p.depth + 63) / 64;
    return groups * 8 < 2048 && blocks > 8 ? 16 : groups * 4 < 2048 && blocks > 4 ? 8 : 4;
}

hipError_t launch_ff_rows(const FfParams& p, FfEpilogue epilogue, int waves, bool staged, bool bf16, bool j_fp8,
                          hipStream_t stream) {
    const bool gated = epilogue == kFfGated;
    auto by_type = [&]<typename T>() {
        if (staged) return j_fp8 ? launch_rows<T, true, true>(p, gated, waves, stream) : launch_rows<T, false, true>(p, gated, waves, stream);
        return j_fp8 ? launch_rows<T, true, false>(p, gated, waves, stream) : launch_rows<T, false, false>(p, gated, waves, stream);
    };
    return bf16 ? by_type.template operator()<__bf16>() : by_type.template operator()<_Float16>();
}

}  // namespace sdxl_hip
