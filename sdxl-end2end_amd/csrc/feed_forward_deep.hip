// Projections, and dz, of few tiles and much depth (some tens to hundreds of rows, few
// columns: the down projections of short batches). Tiles of the tiled kernel
// that fill the CUs there are so small that a stage's barrier costs more than
// its work (64 x 64: 0.3 us a 64-deep stage, 650 clocks for 64 of matrix
// instructions per wave), so here the waves of a 32 x 32 tile share the depth
// and never meet before the end: wave v takes the 64-deep blocks v, v + kWaves,
// .., brings both operands' rows of a block into LDS of its own (8 KiB, the
// tiled kernel's layouts) through a ring of two blocks, and multiplies all of
// the tile. The waves' sums are added in LDS in the waves' order. Eight waves
// where every CU has at most one tile, else four and two tiles a CU: [64, 5120] x
// [1280, 5120] 10.3 us with eight, 13.5 with four, 31 on 64 x 64 tiles; [600, 640]
// x [640, 640] 6.4, 4.9 and 8. Rows that 16-byte accesses do not divide come
// through registers, two blocks ahead: [40, 5127] x [1280, 5127] 20 us. dz of 19
// rows, 2 x 736 deep 2048: 7.3 us here, 16 on 64 x 64 tiles. 64 x 64 tiles whose
// four waves share the depth in the same way halve the reads of the caches where
// CUs would get several of the small ones: gated [248, 8192] -> 2 x 2048 33 us,
// 48 on 32 x 32 and on 64 x 64 tiles with barriers.
#include <hip/hip_runtime.h>

#include "feed_forward_device.hpp"
#include "feed_forward_kernels.hpp"

namespace sdxl_hip {
namespace {

typedef __attribute__((address_space(3))) i16x8 lds_op;

template <typename T, bool kJFp8, int kSide, int kWaves, FfEpilogue kEpi, bool kStaged>
__global__ __launch_bounds__(64 * kWaves) void ff_deep_kernel(FfParams p) {
    using F = FfType<T>;
    using Out = typename F::Out;
    using Acc = typename F::Acc;
    using Acc4 = typename F::Acc4;
    typedef __attribute__((address_space(3))) Acc4 lds_acc4;
    constexpr int kElem = F::kElem, kDepth = 128 / kElem, kChunk = 16 / kElem;  // elements of a block, of 16 bytes
    constexpr bool kGated = kEpi == kFfGated || kEpi == kFfGatedDz, kDz = kEpi == kFfLinearDz || kEpi == kFfGatedDz;
    constexpr int kT = kSide / 32, kRing = 2, kCols = kGated ? kSide / 2 : kSide;
    constexpr int kIBytes = kSide * 128, kBlock = kIBytes + kSide * (kJFp8 ? 64 : 128), kXfers = kBlock / 1024, kIXfers = kIBytes / 1024;
    static_assert(kWaves * kRing * kBlock <= 160 * 1024 && kT * kT * 4096 <= kRing * kBlock, "LDS of one CU; the sums take the blocks' place");
    __shared__ __attribute__((aligned(1024))) char smem[kWaves * kRing * kBlock];  // then the sums

    const int lane = threadIdx.x & 63, hf = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t value_row = p.gate_first ? p.cols : 0, gate_row = p.gate_first ? 0 : p.cols;
    const int64_t ldi_b = p.ld_i * kElem, ldj_b = p.ld_j * (kJFp8 ? 1 : kElem);
    // tasks by XCD, rows fastest: an XCD's workgroups share their J rows in its L2
    int64_t i0, j0;
    {
        const int n = p.i_blocks * p.j_blocks;
        const int id = blockIdx.x, xcd = id & 7, slot = id >> 3;
        const int per = n >> 3, extra = n & 7;
        const int task = xcd * per + (xcd < extra ? xcd : extra) + slot;
        i0 = (int64_t)(task % p.i_blocks) * kSide;
        j0 = (int64_t)(task / p.i_blocks) * kCols;
    }
    const int64_t i_rows = min(p.rows - i0, (int64_t)kSide), j_rows = min(p.cols - j0, (int64_t)kCols);
    const int blocks = (int)((p.depth + kDepth - 1) / kDepth);
    const int mine = (blocks - wave + kWaves - 1) / kWaves;  // blocks of the wave

    // the lane's part of a transfer: 8 rows (by the parity of its number) or, of E4M3 rows, 16
    const int row8 = lane >> 3, row16 = lane >> 2;
    const int chunk8[2] = {(lane & 7) ^ swz(row8), (lane & 7) ^ swz(8 + row8)}, chunk16 = (lane & 3) ^ ((row16 >> 2) & 3);
    const uint32_t lds0 = lds_addr(smem) + wave * kRing * kBlock;
    // transfer n of J: of the gate's rows, and the lane's row from j0 on; a gated 32-row tile is 16 value and 16 gate rows
    auto gate_of = [&](int n) { return kGated && (kJFp8 ? n & 1 : n & 2); };
    auto j_row = [&](int n) {
        if (kJFp8) return 16 * (kGated ? n >> 1 : n) + row16;
        return (kGated ? 16 * (n >> 2) + 8 * (n & 1) : 8 * n) + row8;
    };
    auto request = [&](int it, int slot) __attribute__((always_inline)) {
        const int64_t at = (int64_t)(it * kWaves + wave) * kDepth, left = p.depth - at, i_left = p.i_row - at;
        const uint32_t buf = lds0 + slot * kBlock;
        const u32x4 ir = window_rsrc({(const char*)p.ip + i0 * ldi_b + at * kElem, (uint32_t)((i_rows - 1) * ldi_b + i_left * kElem)});
#pragma unroll
        for (int n = 0; n < kIXfers; ++n)
            window_to_lds(ir, kChunk * chunk8[n & 1] < i_left ? (uint32_t)((8 * n + row8) * ldi_b) + 16 * chunk8[n & 1] : kOutside, buf + n * 1024);
        const char* base = (const char*)p.jp + at * (kJFp8 ? 1 : kElem);
        const uint32_t size = (uint32_t)((j_rows - 1) * ldj_b + left * (kJFp8 ? 1 : kElem));
        const u32x4 jv = window_rsrc({base + (kGated ? value_row + j0 : j0) * ldj_b, size});
        const u32x4 jg = window_rsrc({base + (kGated ? gate_row + j0 : j0) * ldj_b, size});
#pragma unroll
        for (int n = 0; n < kXfers - kIXfers; ++n) {
            const bool gate = gate_of(n);
            uint32_t off;
            if constexpr (kJFp8) off = 16 * chunk16 < left ? (uint32_t)(j_row(n) * ldj_b) + 16 * chunk16 : kOutside;
            else off = kChunk * chunk8[n & 1] < left ? (uint32_t)(j_row(n) * ldj_b) + 16 * chunk8[n & 1] : kOutside;
            window_to_lds(gate ? jg : jv, off, buf + kIBytes + n * 1024);
        }
    };
    // operand reads: depth step ks = 2 pp + q has lane half hf supply depth 32 pp + 16 hf + 8 q .. + 7
    int row_off[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) row_off[ks] = col * 128 + (((4 * (ks >> 1) + 2 * hf + (ks & 1)) ^ swz(col)) << 4);
    Acc acc[kT][kT];  // [J][I]
#pragma unroll
    for (int t = 0; t < kT; ++t)
#pragma unroll
        for (int m = 0; m < kT; ++m)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[t][m][r] = 0;
    auto multiply = [&](int slot) __attribute__((always_inline)) {
        const char* buf = smem + (wave * kRing + slot) * kBlock;
        u32x4 codes[kT];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            i16x8 iop[kT];
#pragma unroll
            for (int m = 0; m < kT; ++m) iop[m] = *(const lds_op*)(buf + m * 4096 + row_off[ks]);
#pragma unroll
            for (int t = 0; t < kT; ++t) {
                i16x8 jop;
                if constexpr (kJFp8) {
                    if ((ks & 1) == 0)
                        codes[t] = *(const lds_u32x4*)(buf + kIBytes + t * 2048 + col * 64 + (((2 * (ks >> 1) + hf) ^ ((col >> 2) & 3)) << 4));
                    const uint2 lo = F::decode(codes[t][2 * (ks & 1)]), hi = F::decode(codes[t][2 * (ks & 1) + 1]);
                    jop = __builtin_bit_cast(i16x8, u32x4{lo.x, lo.y, hi.x, hi.y});
                } else {
                    jop = *(const lds_op*)(buf + kIBytes + t * 4096 + row_off[ks]);
                }
#pragma unroll
                for (int m = 0; m < kT; ++m) acc[t][m] = F::mfma(jop, iop[m], acc[t][m]);
            }
        }
    };
    if constexpr (kStaged) {
        // through registers, two blocks ahead, and one place in LDS
        u32x4 held[2][kXfers];
        auto part = [&](int it, int n, const char*& at) __attribute__((always_inline)) {
            const int64_t k0 = (int64_t)(it * kWaves + wave) * kDepth;
            const int left = (int)min(p.depth - k0, (int64_t)kDepth);
            if (n < kIXfers) {
                at = (const char*)p.ip + (i0 + 8 * n + row8) * ldi_b + k0 * kElem + 16 * chunk8[n & 1];
                return 8 * n + row8 < i_rows ? left - kChunk * chunk8[n & 1] : 0;
            }
            n -= kIXfers;
            const bool gate = gate_of(n);
            const int row = j_row(n);
            const int chunk = kJFp8 ? chunk16 : chunk8[n & 1];
            at = (const char*)p.jp + ((kGated ? (gate ? gate_row : value_row) : 0) + j0 + row) * ldj_b + k0 * (kJFp8 ? 1 : kElem) + 16 * chunk;
            return row < j_rows ? left - (kJFp8 ? 16 : kChunk) * chunk : 0;
        };
        auto fetch = [&](int it, u32x4 (&to)[kXfers]) __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < kXfers; ++n) {
                const char* at;
                const int valid = it < mine ? part(it, n, at) : 0;
                to[n] = kJFp8 && n >= kIXfers ? fetch_chunk<16>(at, valid) : fetch_chunk<kChunk>(at, valid);
            }
        };
        auto turn = [&](int it, u32x4 (&from)[kXfers]) __attribute__((always_inline)) {
            char* buf = smem + wave * kRing * kBlock + lane * 16;
#pragma unroll
            for (int n = 0; n < kXfers; ++n) {
                const char* at;
                const int valid = part(it, n, at);
                *(lds_u32x4*)(buf + n * 1024) = kJFp8 && n >= kIXfers ? settle_chunk<16>(from[n], valid) : settle_chunk<kChunk>(from[n], valid);
            }
            fetch(it + 2, from);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            multiply(0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the next block is put down
        };
        fetch(0, held[0]);
        fetch(1, held[1]);
        for (int it = 0; it < mine; it += 2) {
            turn(it, held[0]);
            if (it + 1 < mine) turn(it + 1, held[1]);
        }
    } else {
#pragma unroll
        for (int it = 0; it < kRing; ++it)
            if (it < mine) request(it, it);
        for (int it = 0; it < mine; ++it) {
            const int slot = it & 1;
            if (it + 1 < mine) wait_vmem<kXfers>();  // the next block's transfers may still be on their way
            else wait_vmem<0>();
            __builtin_amdgcn_sched_barrier(0);
            multiply(slot);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot is read
            if (it + kRing < mine) request(it + kRing, slot);
        }
    }
    __syncthreads();
    // the sums: [wave][J tile][I tile][4][lane] f32x4; acc[4u + q]: row col, tile column 8u + 4hf + q
    constexpr int kGroups = kT * kT * 4;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        const Acc& v = acc[g / 4 / kT][g / 4 % kT];
        *(lds_acc4*)(smem + ((wave * kGroups + g) * 64 + lane) * 16) =
            Acc4{v[4 * (g & 3)], v[4 * (g & 3) + 1], v[4 * (g & 3) + 2], v[4 * (g & 3) + 3]};
    }
    __syncthreads();

    const FfAct act = ff_act(p.activation);
    const FfFamily fam = ff_family(p.activation);
    auto sum_of = [&](int g) {
        Acc4 s{};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) s += *(const lds_acc4*)(smem + ((w * kGroups + g) * 64 + lane) * 16);
        return s;
    };
    float row_scale = 1.0f;  // 8-bit integers: of the lane's row
    auto z_of = [&](float sum, int64_t j) {
        if constexpr (F::kI8) sum *= row_scale;
        if (p.j_scale != nullptr) sum *= p.j_scale[j];
        if (p.bias != nullptr) sum += (float)((const Out*)p.bias)[j];
        return sum;
    };
    // groups of 4 columns by waves (gated: a tile's first two, with the gates of its last two)
    constexpr int kOwn = kGated ? 2 : 4;
    for (int own = wave; own < kT * kT * kOwn; own += kWaves) {
        const int tile = own / kOwn, u = own % kOwn;
        const int64_t i = i0 + 32 * (tile % kT) + col, c = j0 + (kGated ? 16 : 32) * (tile / kT) + 8 * u + 4 * hf;
        const Acc4 a = sum_of(4 * tile + u);
        Acc4 b{};
        if constexpr (kGated) b = sum_of(4 * tile + u + 2);
        if (i >= p.rows) continue;
        if constexpr (F::kI8) row_scale = p.i_scale[i];
        if constexpr (kDz) {
            const Out* dout = (const Out*)p.dout + i * p.ld_dout;
            Out* out = (Out*)p.out + i * p.ld_out;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (c + q >= p.cols) continue;
                const float d = (float)dout[c + q];
                float value;
                if constexpr (kGated) {
                    const float s = ff_slope_of(act, fam, z_of((float)b[q], gate_row + c + q), value);
                    out[value_row + c + q] = (Out)(d * value);
                    out[gate_row + c + q] = (Out)(d * z_of((float)a[q], value_row + c + q) * s);
                } else {
                    out[c + q] = (Out)(ff_slope_of(act, fam, z_of((float)a[q], c + q), value) * d);
                }
                if (c + q == p.cols - 1)  // up to the padded row
                    for (int64_t z = kGated ? 2 * p.cols : p.cols; z < p.out_cols_padded; ++z) out[z] = (Out)0.0f;
            }
        } else {
            float v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                v[q] = 0.0f;
                if (c + q >= p.cols) continue;
                if constexpr (kGated) v[q] = z_of((float)a[q], value_row + c + q) * ff_value_of(act, fam, z_of((float)b[q], gate_row + c + q));
                else v[q] = ff_value_of(act, fam, z_of((float)a[q], c + q)) + (p.residual != nullptr ? (float)((const Out*)p.residual)[i * p.ld_res + c + q] : 0.0f);
            }
            Out* out = (Out*)p.out + i * p.ld_out + c;
            if (p.vec && c < p.cols) {
                *(u32x2*)out = u32x2{F::pack(v[0], v[1]), F::pack(v[2], v[3])};
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (c + q < p.cols) out[q] = (Out)v[q];
            }
        }
    }
}

template <typename T, bool kJFp8, int kSide, int kWaves, bool kStaged>
hipError_t launch(FfParams p, FfEpilogue epilogue, hipStream_t stream) {
    p.i_blocks = (int32_t)((p.rows + kSide - 1) / kSide);
    const int64_t cols = epilogue == kFfGated || epilogue == kFfGatedDz ? kSide / 2 : kSide;
    p.j_blocks = (int32_t)((p.cols + cols - 1) / cols);
    const dim3 grid((unsigned)(p.i_blocks * p.j_blocks)), block(64 * kWaves);
    if (epilogue == kFfGated) {
        hipLaunchKernelGGL((ff_deep_kernel<T, kJFp8, kSide, kWaves, kFfGated, kStaged>), grid, block, 0, stream, p);
    } else if (epilogue == kFfLinear) {
        hipLaunchKernelGGL((ff_deep_kernel<T, kJFp8, kSide, kWaves, kFfLinear, kStaged>), grid, block, 0, stream, p);
    } else if constexpr (!kJFp8 && !FfType<T>::kI8) {
        if (epilogue == kFfGatedDz) hipLaunchKernelGGL((ff_deep_kernel<T, false, kSide, kWaves, kFfGatedDz, kStaged>), grid, block, 0, stream, p);
        else hipLaunchKernelGGL((ff_deep_kernel<T, false, kSide, kWaves, kFfLinearDz, kStaged>), grid, block, 0, stream, p);
    }
    return hipGetLastError();
}

template <typename T, bool kStaged>
hipError_t launch_type(const FfParams& p, FfEpilogue epilogue, bool j_fp8, FfDeepId id, hipStream_t stream) {
    if (p.i8 != 0) {
        switch (id) {
        case kFfDeep32x8: return launch<I8<T>, false, 32, 8, kStaged>(p, epilogue, stream);
        case kFfDeep32x4: return launch<I8<T>, false, 32, 4, kStaged>(p, epilogue, stream);
        case kFfDeep64x4: return launch<I8<T>, false, 64, 4, kStaged>(p, epilogue, stream);
        }
        return hipErrorInvalidValue;
    }
    switch (id) {
    case kFfDeep32x8: return j_fp8 ? launch<T, true, 32, 8, kStaged>(p, epilogue, stream) : launch<T, false, 32, 8, kStaged>(p, epilogue, stream);
    case kFfDeep32x4: return j_fp8 ? launch<T, true, 32, 4, kStaged>(p, epilogue, stream) : launch<T, false, 32, 4, kStaged>(p, epilogue, stream);
    case kFfDeep64x4: return j_fp8 ? launch<T, true, 64, 4, kStaged>(p, epilogue, stream) : launch<T, false, 64, 4, kStaged>(p, epilogue, stream);
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t ff_deep(const FfParams& p, FfEpilogue epilogue, bool bf16, bool j_fp8, bool staged, FfDeepId id, hipStream_t stream) {
    if (staged)
        return bf16 ? launch_type<__bf16, true>(p, epilogue, j_fp8, id, stream) : launch_type<_Float16, true>(p, epilogue, j_fp8, id, stream);
    return bf16 ? launch_type<__bf16, false>(p, epilogue, j_fp8, id, stream) : launch_type<_Float16, false>(p, epilogue, j_fp8, id, stream);
}

}  // namespace sdxl_hip
