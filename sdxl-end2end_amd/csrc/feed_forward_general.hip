// The general product kernel of the feed-forward operators
// (include/sdxl_hip/feed_forward.h): any size, stride and alignment, either
// operand transposed, fp16 / bf16 / E4M3. The fast kernels (feed_forward.hip)
// take what has rows of 16 bytes or more and strides up to 2^20; this one takes
// the rest (depths or widths below 8, empty sums, huge strides or outputs).
//
// One workgroup of 4 waves makes 64 x 64 tiles of C = I J^T: 32-deep steps go
// through registers into LDS element by element, every element checked
// against the operand's sizes, then one v_mfma_f32_32x32x16 per wave and 16
// of depth with the J rows as the A operand, so that a lane holds 4
// consecutive columns of one row. Gated products stage 16 value rows and the
// 16 gate rows of the same columns in every 32-row J tile, so that a lane
// holds value and gate of its columns (8-bit integers: v_mfma_i32_32x32x32, one
// a step). What bounds it is the element loads and
// stores: [8192, 7] x [5120, 7] 105 us, a fifth of the copy rate on its 84 MB.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "feed_forward_device.hpp"
#include "feed_forward_kernels.hpp"

namespace sdxl_hip {
namespace {

constexpr int kGTile = 64, kGStep = 32;
constexpr int kGRow = kGStep + 8;  // LDS row, elements: 80 bytes, 16-byte operand reads

typedef __attribute__((address_space(3))) i16x8 lds_op;

template <typename T, bool kIT, bool kJT, bool kJFp8, FfEpilogue kEpi, bool kI8 = false>
__global__ __launch_bounds__(256) void ff_general_kernel(FfParams p) {
    constexpr bool kGated = kEpi == kFfGated || kEpi == kFfGatedDz;
    constexpr int kCols = kGated ? kGTile / 2 : kGTile;  // columns of C per tile
    static_assert(!kI8 || (!kIT && !kJT && !kJFp8), "8-bit integers: by rows");
    static_assert(!kJFp8 || (!kJT && (kEpi == kFfLinear || kEpi == kFfGated)), "E4M3: forward only");
    __shared__ __attribute__((aligned(16))) uint16_t tile_i[kGTile * kGRow];
    __shared__ __attribute__((aligned(16))) uint16_t tile_j[kGTile * kGRow];
    using F = FfType<T>;
    using Acc = std::conditional_t<kI8, i32x16, f32x16>;
    // 8-bit integers: rows of the same 80 bytes
    auto put = [&](uint16_t* tile, int row, int d, uint16_t v) __attribute__((always_inline)) {
        if constexpr (kI8) ((uint8_t*)tile)[row * kGRow * 2 + d] = (uint8_t)v;
        else tile[row * kGRow + d] = v;
    };
    const int tid = threadIdx.x, lane = tid & 63, hf = lane >> 5, col = lane & 31;
    const int wi = tid >> 7, wj = (tid >> 6) & 1;
    const FfAct act = ff_act(p.activation);
    const int64_t value_row = p.gate_first ? p.cols : 0, gate_row = p.gate_first ? 0 : p.cols;
    const int64_t i_blocks = (p.rows + kGTile - 1) / kGTile, j_blocks = (p.cols + kCols - 1) / kCols;

    for (int64_t task = blockIdx.x; task < i_blocks * j_blocks; task += gridDim.x) {
        const int64_t i0 = task % i_blocks * kGTile, j0 = task / i_blocks * kCols;
        // the J row that row jr of the tile holds (p.cols or more: none)
        auto j_row = [&](int jr) -> int64_t {
            if constexpr (kGated) {
                const int64_t c = j0 + 16 * (jr >> 5) + (jr & 15);
                return c >= p.cols ? -1 : c + (jr & 16 ? gate_row : value_row);
            } else {
                return j0 + jr < p.cols ? j0 + jr : -1;
            }
        };
        const bool sums = kEpi == kFfStore && p.row_sums != nullptr && j0 == 0;
        Acc acc;
        f32x16 acc_sum;
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] = acc_sum[r] = 0;

        for (int64_t d0 = 0; d0 < p.depth; d0 += kGStep) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int row = kIT ? (tid & 7) * 8 + e : tid >> 2, d = kIT ? tid >> 3 : (tid & 3) * 8 + e;
                const int64_t i = i0 + row, r = d0 + d;
                uint16_t v = 0;
                if (i < p.rows && r < p.depth) {
                    if constexpr (kI8) v = ((const uint8_t*)p.ip)[i * p.ld_i + r];
                    else v = ((const uint16_t*)p.ip)[kIT ? r * p.ld_i + i : i * p.ld_i + r];
                }
                put(tile_i, row, d, v);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int row = kJT ? (tid & 7) * 8 + e : tid >> 2, d = kJT ? tid >> 3 : (tid & 3) * 8 + e;
                const int64_t j = j_row(row), r = d0 + d;
                uint16_t v = 0;
                if (j >= 0 && r < p.depth) {
                    const int64_t at = kJT ? r * p.ld_j + j : j * p.ld_j + r;
                    if constexpr (kI8) v = ((const uint8_t*)p.jp)[at];
                    else if constexpr (kJFp8) v = (uint16_t)F::decode(((const uint8_t*)p.jp)[at]).x;
                    else v = ((const uint16_t*)p.jp)[at];
                }
                put(tile_j, row, d, v);
            }
            __syncthreads();
            if constexpr (kI8) {
                const i16x8 iop = *(const lds_op*)(tile_i + (32 * wi + col) * kGRow + 8 * hf);
                const i16x8 jop = *(const lds_op*)(tile_j + (32 * wj + col) * kGRow + 8 * hf);
                acc = mfma32_i8(jop, iop, acc);
            } else {
#pragma unroll
                for (int ks = 0; ks < kGStep / 16; ++ks) {
                    const i16x8 iop = *(const lds_op*)(tile_i + (32 * wi + col) * kGRow + 16 * ks + 8 * hf);
                    const i16x8 jop = *(const lds_op*)(tile_j + (32 * wj + col) * kGRow + 16 * ks + 8 * hf);
                    acc = F::mfma(jop, iop, acc);
                    if (sums && wj == 0) {
                        const short one = (short)__builtin_bit_cast(uint16_t, (T)1.0f);
                        acc_sum = F::mfma(i16x8{one, one, one, one, one, one, one, one}, iop, acc_sum);
                    }
                }
            }
        }

        // acc[4u + q]: row i0 + 32 wi + col, tile column 32 wj + 8u + 4hf + q
        const int64_t i = i0 + 32 * wi + col;
        if (i >= p.rows) continue;
        T* out = (T*)p.out + i * p.ld_out;
        if (sums && wj == 0 && hf == 0) ((T*)p.row_sums)[i] = (T)acc_sum[0];
        const float row_scale = kI8 ? p.i_scale[i] : 1.0f;
        auto z_of = [&](float sum, int64_t j) {
            if constexpr (kI8) sum *= row_scale;
            if (p.j_scale != nullptr) sum *= p.j_scale[j];
            if (p.bias != nullptr) sum += (float)((const T*)p.bias)[j];
            return sum;
        };
        auto epilogue = [&]<FfFamily kFam>() {
            if constexpr (kGated) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int64_t c = j0 + 16 * wj + 8 * (e >> 2) + 4 * hf + (e & 3);
                    if (c >= p.cols) continue;
                    const float v = z_of((float)acc[e], value_row + c), g = z_of((float)acc[8 + e], gate_row + c);
                    if constexpr (kEpi == kFfGated) {
                        out[c] = (T)(v * ff_value<kFam>(act, g));
                    } else {
                        const float d = (float)((const T*)p.dout)[i * p.ld_dout + c];
                        float a;
                        const float s = ff_slope<kFam>(act, g, a);
                        out[value_row + c] = (T)(d * a);
                        out[gate_row + c] = (T)(d * v * s);
                        if (c == p.cols - 1)
                            for (int64_t z = 2 * p.cols; z < p.out_cols_padded; ++z) out[z] = (T)0.0f;
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int64_t j = j0 + 32 * wj + 8 * (e >> 2) + 4 * hf + (e & 3);
                    if (j >= p.cols) continue;
                    if constexpr (kEpi == kFfStore) {
                        out[j] = (T)(float)acc[e];
                    } else if constexpr (kEpi == kFfLinear) {
                        float v = ff_value<kFam>(act, z_of((float)acc[e], j));
                        if (p.residual != nullptr) v += (float)((const T*)p.residual)[i * p.ld_res + j];
                        out[j] = (T)v;
                    } else {
                        float a;
                        const float s = ff_slope<kFam>(act, z_of((float)acc[e], j), a);
                        out[j] = (T)((float)((const T*)p.dout)[i * p.ld_dout + j] * s);
                        if (j == p.cols - 1)
                            for (int64_t z = p.cols; z < p.out_cols_padded; ++z) out[z] = (T)0.0f;
                    }
                }
            }
        };
        if constexpr (kEpi == kFfStore) epilogue.template operator()<kFamLinear>();
        else ff_with_family(p.activation, epilogue);
    }
}

template <typename T, bool kIT, bool kJT, bool kJFp8, FfEpilogue kEpi, bool kI8 = false>
hipError_t launch(const FfParams& p, hipStream_t stream) {
    constexpr int64_t cols = kEpi == kFfGated || kEpi == kFfGatedDz ? kGTile / 2 : kGTile;
    const int64_t tasks = ((p.rows + kGTile - 1) / kGTile) * ((p.cols + cols - 1) / cols);
    if (tasks == 0) return hipSuccess;
    const unsigned grid = (unsigned)(tasks < (1 << 20) ? tasks : 1 << 20);  // more: each workgroup takes several
    hipLaunchKernelGGL((ff_general_kernel<T, kIT, kJT, kJFp8, kEpi, kI8>), dim3(grid), dim3(256), 0, stream, p);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_type(const FfParams& p, FfEpilogue epilogue, bool it, bool jt, bool j_fp8, hipStream_t stream) {
    if (p.i8 != 0) {
        if (epilogue == kFfLinear) return launch<T, false, false, false, kFfLinear, true>(p, stream);
        return epilogue == kFfGated ? launch<T, false, false, false, kFfGated, true>(p, stream) : hipErrorInvalidValue;
    }
    switch (epilogue) {
    case kFfLinear: return j_fp8 ? launch<T, false, false, true, kFfLinear>(p, stream) : launch<T, false, false, false, kFfLinear>(p, stream);
    case kFfGated: return j_fp8 ? launch<T, false, false, true, kFfGated>(p, stream) : launch<T, false, false, false, kFfGated>(p, stream);
    case kFfLinearDz: return launch<T, false, false, false, kFfLinearDz>(p, stream);
    case kFfGatedDz: return launch<T, false, false, false, kFfGatedDz>(p, stream);
    case kFfStore:
        if (jt) return it ? launch<T, true, true, false, kFfStore>(p, stream) : launch<T, false, true, false, kFfStore>(p, stream);
        break;
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_ff_general(const FfParams& p, FfEpilogue epilogue, bool i_transposed, bool j_transposed, bool bf16,
                             bool j_fp8, hipStream_t stream) {
    return bf16 ? launch_type<__bf16>(p, epilogue, i_transposed, j_transposed, j_fp8, stream)
                : launch_type<_Float16>(p, epilogue, i_transposed, j_transposed, j_fp8, stream);
}

}  // namespace sdxl_hip
