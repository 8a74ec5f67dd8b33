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
//
// 8-bit weights with up to four tokens in 16 bits (kTokens): every workgroup quantises the tokens
// itself, into LDS, while its weights are on their way, instead of a launch before and a workspace:
// gated [1, 1280] -> 2 x 5120 13.4 us a call so, 8.0 here.
#include <hip/hip_runtime.h>

#include "feed_forward_device.hpp"
#include "int8_device.hpp"
#include "feed_forward_kernels.hpp"

namespace sdxl_hip {
namespace {

typedef __attribute__((address_space(3))) float lds_float;

constexpr int kMaxTokens = 4, kMaxTokenDepth = 8192;

template <typename T, typename Acc4>
__device__ __forceinline__ Acc4 mfma16(u32x4 a, u32x4 b, Acc4 c) {
    if constexpr (FfType<T>::kI8)
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
    else if constexpr (__is_same(T, _Float16))
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <typename T, bool kJFp8, int kWaves, bool kGated, bool kStaged, bool kTokens = false>
__global__ __launch_bounds__(64 * kWaves) void ff_rows_kernel(FfParams p) {
    using F = FfType<T>;
    using Out = typename F::Out;
    using Acc4 = typename F::Acc4;
    typedef __attribute__((address_space(3))) Acc4 lds_acc4;
    constexpr int kBlocks = 32 / kWaves;  // of a wave at a time
    extern __shared__ __attribute__((aligned(1024))) char smem[];  // [kBlocks][kWaves] of kBlockBytes; then the sums
    constexpr int kBlockBytes = kJFp8 ? 1024 : 2048, kElem = kJFp8 ? 1 : F::kElem;  // w's
    constexpr int kXElem = F::kElem, kDepth = 128 / kXElem, kChunk = 16 / kXElem;     // elements of a block, of 16 bytes of x
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    constexpr int kCols = kGated ? 8 : 16;
    const int64_t c0 = (int64_t)blockIdx.x * kCols;
    const int64_t value_row = p.gate_first ? p.cols : 0, gate_row = p.gate_first ? 0 : p.cols;
    const int depth = (int)p.depth, blocks = (depth + kDepth - 1) / kDepth;
    const u32x4 w_rsrc = window_rsrc({(const char*)p.jp, (uint32_t)((((kGated ? 2 : 1) * p.cols - 1) * p.ld_j + p.depth) * kElem)});
    const u32x4 x_win = window_rsrc({(const char*)p.ip, (uint32_t)(((p.rows - 1) * p.ld_i + p.depth) * kXElem)});
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
    // kTokens: rows of codes behind the blocks, as many bytes as the blocks' depth and 16 more, then the rows' scales
    const int code_row = blocks * 128 + 16;
    char* const codes = smem + (blocks < 32 ? (blocks + kWaves - 1) / kWaves * kWaves : 32) * kBlockBytes;
    lds_float* const code_scale = (lds_float*)(codes + kMaxTokens * code_row);
    auto quantise = [&]() __attribute__((always_inline)) {
        constexpr uint32_t kInf = 0x7f800000u;
        lds_float* const part = code_scale + kMaxTokens;
        const int vecs = blocks * 16;  // of 8 values, zeros past the depth
        for (int row = 0; row < (int)p.rows; ++row) {
            const char* x = (const char*)p.ip + row * p.ld_i * 2;
            auto values = [&](int v, float (&f)[8]) __attribute__((always_inline)) {
                const int valid = depth - 8 * v;
                const u32x4 d = settle_chunk<8>(fetch_chunk<8>(x + 16 * v, valid), valid);
#pragma unroll
                for (int e = 0; e < 4; ++e) f[2 * e] = F::lo(d[e]), f[2 * e + 1] = F::hi(d[e]);
            };
            auto largest = [&](uint32_t most) __attribute__((always_inline)) {
                uint32_t top = 0;
                for (int v = (int)threadIdx.x; v < vecs; v += 64 * kWaves) {
                    float f[8];
                    values(v, f);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t m = __float_as_uint(f[e]) & 0x7fffffffu;
                        top = max(top, m <= most ? m : 0);
                    }
                }
                auto larger = [](float a, float b) __attribute__((always_inline)) {
                    return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
                };
                const float mine = reduce64(__uint_as_float(top), larger);
                __syncthreads();  // the last values are read
                if (lane == 0) part[wave] = mine;
                __syncthreads();
                float all = part[0];
                for (int w = 1; w < kWaves; ++w) all = larger(all, part[w]);
                return __float_as_uint(all);
            };
            uint32_t top = largest(0xffffffffu);
            const bool nan = top > kInf;
            if (top >= kInf) top = largest(kInf - 1);
            const float scale = i8_scale(__uint_as_float(top), nan), over = 1.0f / scale, limit = 127.0f * scale;
            for (int v = (int)threadIdx.x; v < vecs; v += 64 * kWaves) {
                float f[8];
                values(v, f);
                *(lds_u32x2*)(codes + row * code_row + 8 * v) = i8_codes(f, scale, over, limit);
            }
            if (threadIdx.x == 0) code_scale[row] = scale;
        }
        __syncthreads();
    };
    const uint32_t x_at = r16 < p.rows ? (uint32_t)(r16 * p.ld_i * kXElem) : kOutside;

    const uint32_t lds0 = lds_addr(smem);
    u32x4 x[kBlocks][2];
    Acc4 acc{};
    for (int first = 0; first < blocks; first += 32) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the last reads of the blocks' place are done
        if constexpr (kStaged) {
            // through registers: all reads first
            constexpr int kAll = kJFp8 ? 16 : kChunk, kH = kJFp8 ? 1 : 2;
            u32x4 held[kBlocks][kH];
            auto x_valid = [&](int block, int q) { return r16 < p.rows ? depth - (kDepth * block + kChunk * (4 * q + g)) : 0; };
            auto w_valid = [&](int block, int h) { return w_at[h] != kOutside ? depth - kDepth * block - kAll * chunk_at[h] : 0; };
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const int block = first + b * kWaves + wave;
#pragma unroll
                for (int q = 0; q < (kTokens ? 0 : 2); ++q)
                    x[b][q] = fetch_chunk<kChunk>((const char*)p.ip + (r16 * p.ld_i + kDepth * block + kChunk * (4 * q + g)) * kXElem, x_valid(block, q));
#pragma unroll
                for (int h = 0; h < kH; ++h)
                    held[b][h] = fetch_chunk<kAll>((const char*)p.jp + w_at[h] + (int64_t)(kDepth * block + kAll * chunk_at[h]) * kElem, w_valid(block, h));
            }
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const int block = first + b * kWaves + wave;
#pragma unroll
                for (int q = 0; q < (kTokens ? 0 : 2); ++q) x[b][q] = settle_chunk<kChunk>(x[b][q], x_valid(block, q));
                if (block < blocks) {  // (LDS holds no others)
#pragma unroll
                    for (int h = 0; h < kH; ++h)
                        *(lds_u32x4*)(smem + (b * kWaves + wave) * kBlockBytes + 1024 * h + lane * 16) = settle_chunk<kAll>(held[b][h], w_valid(block, h));
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (kTokens && first == 0) quantise();
        } else {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const int block = first + b * kWaves + wave;
                if (!kTokens && block < blocks) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int k = kDepth * block + kChunk * (4 * q + g);
                        x[b][q] = __builtin_amdgcn_raw_buffer_load_b128(x_rsrc, k < depth && x_at != kOutside ? x_at + kXElem * k : kOutside, 0, 0);
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const int block = first + b * kWaves + wave;
                if (block < blocks) {
#pragma unroll
                    for (int h = 0; h < (kJFp8 ? 1 : 2); ++h) {
                        const int k = kDepth * block + (kJFp8 ? 16 : kChunk) * chunk_at[h];
                        window_to_lds(w_rsrc, k < depth && w_at[h] != kOutside ? w_at[h] + kElem * k : kOutside,
                                      lds0 + (b * kWaves + wave) * kBlockBytes + 1024 * h);
                    }
                }
            }
            if (kTokens && first == 0) quantise();  // (its reads wait for the weights too)
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
                for (int q = 0; q < 2; ++q) {
                    if constexpr (kTokens)  // (columns past the rows: any)
                        x[b][q] = *(const lds_u32x4*)(codes + (r16 < p.rows ? r16 : 0) * code_row + kDepth * (first + b * kWaves + wave) + kChunk * (4 * q + g));
                    acc = mfma16<T>(a[q], x[b][q], acc);
                }
            }
        }
    }
    __syncthreads();  // the sums take the blocks' place
    *(lds_acc4*)(smem + (wave * 64 + lane) * 16) = acc;
    __syncthreads();

    // acc[e] of lane l: column (w row) 4 (l / 16) + e, row l % 16
    const FfAct act = ff_act(p.activation);
    const FfFamily fam = ff_family(p.activation);
    auto sum_of = [&](int from) {
        Acc4 s{};
        for (int v = 0; v < kWaves; ++v) s += *(const lds_acc4*)(smem + (v * 64 + from) * 16);
        return s;
    };
    const float row_scale = kTokens ? code_scale[r16 < p.rows ? r16 : 0] : F::kI8 && r16 < p.rows ? p.i_scale[r16] : 1.0f;
    auto z_of = [&](float sum, int64_t row) {
        if constexpr (F::kI8) sum *= row_scale;
        if (p.j_scale != nullptr) sum *= p.j_scale[row];
        if (p.bias != nullptr) sum += (float)((const Out*)p.bias)[row];
        return sum;
    };
    if (threadIdx.x < (kGated ? 32 : 64)) {
        const int64_t i = r16;
        if (i >= p.rows) return;
        const Acc4 a = sum_of(lane);
        Acc4 b{};
        if constexpr (kGated) b = sum_of(lane + 32);
        Out* out = (Out*)p.out + i * p.ld_out;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t n = c0 + 4 * g + e;
            if (n >= p.cols) continue;
            if constexpr (kGated) {
                out[n] = (Out)(z_of((float)a[e], value_row + n) * ff_value_of(act, fam, z_of((float)b[e], gate_row + n)));
            } else {
                float v = ff_value_of(act, fam, z_of((float)a[e], n));
                if (p.residual != nullptr) v += (float)((const Out*)p.residual)[i * p.ld_res + n];
                out[n] = (Out)v;
            }
        }
    }
}

template <typename T, bool kJFp8, int kWaves, bool kStaged>
hipError_t launch(const FfParams& p, bool gated, hipStream_t stream) {
    if constexpr (FfType<T>::kI8) {
        if (p.i8 == kFfI8Tokens) {
            const int64_t blocks = ff_stages(p), held = blocks < 32 ? (blocks + kWaves - 1) / kWaves * kWaves : 32;
            const size_t lds = (size_t)held * 2048 + kMaxTokens * ((size_t)blocks * 128 + 16) + (kMaxTokens + kWaves) * 4;
            const dim3 grid((unsigned)(gated ? (p.cols + 7) / 8 : (p.cols + 15) / 16)), block(64 * kWaves);
            if (gated) hipLaunchKernelGGL((ff_rows_kernel<T, kJFp8, kWaves, true, kStaged, true>), grid, block, lds, stream, p);
            else hipLaunchKernelGGL((ff_rows_kernel<T, kJFp8, kWaves, false, kStaged, true>), grid, block, lds, stream, p);
            return hipGetLastError();
        }
    }
    const dim3 grid((unsigned)(gated ? (p.cols + 7) / 8 : (p.cols + 15) / 16)), block(64 * kWaves);
    const int64_t blocks = (p.depth + 128 / FfType<T>::kElem - 1) / (128 / FfType<T>::kElem), held = blocks < 32 ? (blocks + kWaves - 1) / kWaves * kWaves : 32;
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
           w_rows * p.ld_j * (j_fp8 || p.i8 != 0 ? 1 : 2) < (int64_t{1} << 31) && ff_staged_supported(p, epilogue, false, false, j_fp8);
}

bool ff_rows_tokens(const FfParams& p, FfEpilogue epilogue) {
    return p.rows <= kMaxTokens && p.depth <= kMaxTokenDepth && p.ld_i < (1 << 20) && ff_rows_supported(p, epilogue, false);
}

// 2048 waves in all where there are blocks for them
int ff_rows_waves(const FfParams& p, bool gated) {
    const int64_t groups = gated ? (p.cols + 7) / 8 : (p.cols + 15) / 16, blocks = ff_stages(p);
    return groups * 8 < 2048 && blocks > 8 ? 16 : groups * 4 < 2048 && blocks > 4 ? 8 : 4;
}

hipError_t launch_ff_rows(const FfParams& p, FfEpilogue epilogue, int waves, bool staged, bool bf16, bool j_fp8,
                          hipStream_t stream) {
    const bool gated = epilogue == kFfGated;
    auto by_type = [&]<typename T>() {
        if (p.i8 != 0) return staged ? launch_rows<I8<T>, false, true>(p, gated, waves, stream) : launch_rows<I8<T>, false, false>(p, gated, waves, stream);
        if (staged) return j_fp8 ? launch_rows<T, true, true>(p, gated, waves, stream) : launch_rows<T, false, true>(p, gated, waves, stream);
        return j_fp8 ? launch_rows<T, true, false>(p, gated, waves, stream) : launch_rows<T, false, false>(p, gated, waves, stream);
    };
    return bf16 ? by_type.template operator()<__bf16>() : by_type.template operator()<_Float16>();
}

}  // namespace sdxl_hip
