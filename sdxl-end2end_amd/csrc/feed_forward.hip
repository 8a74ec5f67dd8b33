// The tiled product kernel of the feed-forward operators
// (include/sdxl_hip/feed_forward.h), for gfx950 (MI355X, CDNA4).
//
// C[i, j] = sum_r I(i, r) J(j, r), with the epilogue of FfEpilogue on the fp32
// sums: the projections (I = x, J = w), dx (I = dz, J = w by columns) and dw
// (I = dz by columns, J = x by columns). A workgroup of kWI x kWJ waves owns
// (32 kMI kWI) x (32 kMJ kWJ) tiles of C, each wave a (32 kMI) x (32 kMJ) block
// as kMI x kMJ v_mfma_f32_32x32x16 tiles with the J rows as the A operand, so
// that a lane ends up with 4 consecutive columns of one row of C.
//
// Depth goes in stages of 64 through two LDS buffers, filled by
// buffer_load_dwordx4 ... lds (1 KiB per wave and instruction, no registers).
// Rows with contiguous depth lie as 128-byte rows whose 16-byte chunks are
// XOR-swizzled (conflict-free 16-byte operand reads); operands taken by columns
// lie as panels of 64 columns x 64 depth rows in the same layout and reach the
// registers through the transposing ds_read_b64_tr_b16. E4M3 rows stay as codes
// (64-byte rows) and are decoded on the way to the matrix cores. What lies
// outside an operand (rows past the end, depth past the end) is read as zero:
// the descriptor's size cuts the rows off, and the last stage's chunks past the
// depth get an offset beyond it.
//
// Schedule: the operands of depth step k + 1 are read while step k's matrix
// instructions run (two register sets), across the stage boundary too: the
// barrier that frees a buffer stands before the stage's last step, whose
// operands are in registers by then, so that its matrix instructions cover the
// barrier, the next stage's first reads and the issue of the transfers.
//
// Gated products put 16 value rows and the 16 gate rows of the same columns
// into every 32-row J tile: a lane holds value and gate of its columns and the
// product needs no exchange.
#include <hip/hip_runtime.h>

#include "feed_forward_device.hpp"
#include "feed_forward_kernels.hpp"

namespace sdxl_hip {
namespace {

typedef __attribute__((address_space(3))) i16x8 lds_op;

// An operand's window as a buffer descriptor (raw, byte offsets): reads at or
// past `size` return zero.
struct Window {
    const char* base;
    uint32_t size;
};

__device__ __forceinline__ u32x4 window_rsrc(Window w) {
    const uint64_t b = (uint64_t)(uintptr_t)w.base;
    return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)b),
                 (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32) & 0xFFFFu),
                 (uint32_t)__builtin_amdgcn_readfirstlane(w.size), 0x00020000u};
}

// 1-KiB transfer: lane l's 16 bytes at offset voff of the window go to lds +
// 16 l. Ordered by explicit waits and barriers, as the attention kernel's.
__device__ __forceinline__ void window_to_lds(u32x4 rsrc, uint32_t voff, uint32_t lds) {
    lds = __builtin_amdgcn_readfirstlane(lds);
    asm volatile(
        "s_nop 4\n\t"
        "buffer_load_dwordx4 %0, %1, 0 offen lds"
        :
        : "v"(voff), "s"(rsrc), "{m0}"(lds));
}

constexpr uint32_t kOutside = 0x80000000u;  // past every window (their sizes stay below 2^31)

__device__ __forceinline__ int64_t min64(int64_t a, int64_t b) { return a < b ? a : b; }

// Exchanges the halves so that lanes 0-31 hold 8 consecutive columns made of
// both halves' a, lanes 32-63 those of b (a, b: two values each, packed).
__device__ __forceinline__ void join_halves(uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}

template <typename T, bool kIT, bool kJT, bool kJFp8, int kWI, int kWJ, int kMI, int kMJ, FfEpilogue kEpi>
__global__ __launch_bounds__(64 * kWI * kWJ, kWI * kWJ == 8 ? 2 : 1) void ff_tile_kernel(FfParams p) {
    using F = FfType<T>;
    constexpr bool kGated = kEpi == kFfGated || kEpi == kFfGatedDz;
    constexpr int kWaves = kWI * kWJ;
    constexpr int kBI = 32 * kMI * kWI, kBJ = 32 * kMJ * kWJ;
    constexpr int kCols = kGated ? kBJ / 2 : kBJ;  // columns of C per tile
    constexpr int kIBytes = kBI * 128, kJBytes = kBJ * (kJFp8 ? 64 : 128);
    constexpr int kStage = kIBytes + kJBytes;
    constexpr int kIXfers = kIBytes / 1024, kJXfers = kJBytes / 1024;
    static_assert(kWaves % 4 == 0, "the waves' transfers keep their parity and their half of the gating");
    static_assert(kIXfers % kWaves == 0 && (kJXfers % kWaves == 0 || kJFp8), "transfers per wave");
    static_assert(2 * kStage <= 160 * 1024, "LDS of one CU");
    static_assert(!kGated || (!kIT && !kJT), "gated products are projections");
    static_assert(!kJFp8 || !kJT, "E4M3: by rows");
    __shared__ __attribute__((aligned(1024))) char smem[2 * kStage];

    const int lane = threadIdx.x & 63, hf = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave % kWI, wj = wave / kWI;
    const int64_t value_row = p.gate_first ? p.cols : 0, gate_row = p.gate_first ? 0 : p.cols;
    const int n_stages = (int)((p.depth + 63) / 64);
    const int64_t ldi_b = p.ld_i * 2, ldj_b = p.ld_j * (kJFp8 ? 1 : 2);

    // ---- task: each XCD takes one contiguous range of them, in groups of
    // group_i row blocks (rows fastest, then columns), so that its workgroups
    // share I rows and J rows in its L2
    int64_t i0, j0;
    {
        const int n = p.i_blocks * p.j_blocks;
        const int id = blockIdx.x, xcd = id & 7, slot = id >> 3;
        const int per = n >> 3, extra = n & 7;
        const int task = xcd * per + (xcd < extra ? xcd : extra) + slot;
        const int in_group = p.group_i * p.j_blocks;
        const int first = (task / in_group) * p.group_i;
        const int rows = min(p.i_blocks - first, p.group_i);
        const int r = task % in_group;
        i0 = (int64_t)(first + r % rows) * kBI;
        j0 = (int64_t)(r / rows) * kCols;
    }

    // ---- transfers. Transfer n of an operand is 8 rows (E4M3: 16) of 128 (64)
    // bytes of its region; wave w takes n = w, w + kWaves, ..: the swizzle and,
    // for gated J tiles, value or gate follow from the wave.
    const int row8 = lane >> 3, chunk8 = (lane & 7) ^ swz(8 * (wave & 1) + row8);
    const int row16 = lane >> 2, chunk16 = (lane & 3) ^ ((row16 >> 2) & 3);
    Window iw, jw;
    uint32_t i_lane, j_lane;  // the lane's offset in a transfer
    if constexpr (kIT) {
        iw.base = (const char*)p.ip + i0 * 2;
        i_lane = (uint32_t)(row8 * ldi_b) + chunk8 * 16;
    } else {
        iw.base = (const char*)p.ip + i0 * ldi_b;
        i_lane = (uint32_t)(row8 * ldi_b) + chunk8 * 16;
    }
    const int64_t j_first = kGated ? j0 + ((kJFp8 ? wave & 1 : wave & 2) ? gate_row : value_row) : j0;
    if constexpr (kJT) jw.base = (const char*)p.jp + j0 * 2;
    else jw.base = (const char*)p.jp + j_first * ldj_b;
    j_lane = kJFp8 ? (uint32_t)(row16 * ldj_b) + chunk16 * 16 : (uint32_t)(row8 * ldj_b) + chunk8 * 16;
    const int64_t i_rows = min64(p.rows - i0, kBI), j_rows = min64(p.cols - j0, kGated ? kCols : kBJ);
    // window of stage st: everything from its first byte to the last valid one
    auto i_window = [&](int st) __attribute__((always_inline)) {
        if constexpr (kIT) {
            const int64_t left = min64(p.depth - (int64_t)st * 64, 64);
            return window_rsrc({iw.base + (int64_t)st * 64 * ldi_b, (uint32_t)((left - 1) * ldi_b + min64(p.i_row - i0, kBI) * 2)});
        } else {
            return window_rsrc({iw.base + st * 128, (uint32_t)((i_rows - 1) * ldi_b + (p.i_row - (int64_t)st * 64) * 2)});
        }
    };
    auto j_window = [&](int st) __attribute__((always_inline)) {
        if constexpr (kJT) {
            const int64_t left = min64(p.depth - (int64_t)st * 64, 64);
            return window_rsrc({jw.base + (int64_t)st * 64 * ldj_b, (uint32_t)((left - 1) * ldj_b + j_rows * 2)});
        } else {
            return window_rsrc({jw.base + (kJFp8 ? st * 64 : st * 128),
                                (uint32_t)((j_rows - 1) * ldj_b + (p.depth - (int64_t)st * 64) * (kJFp8 ? 1 : 2))});
        }
    };
    const uint32_t lds0 = lds_addr(smem);
    constexpr int kXfers = kIXfers / kWaves + (kJXfers + kWaves - 1) / kWaves;
    // one of the wave's kXfers transfers of stage st
    auto issue = [&](int st, int x, u32x4 irsrc, u32x4 jrsrc) __attribute__((always_inline)) {
        const uint32_t buf = lds0 + (st & 1) * kStage;
        // depth of the stage, by I's rows and by J's
        const int i_left = (int)min64(p.i_row - (int64_t)st * 64, 64), left = (int)min64(p.depth - (int64_t)st * 64, 64);
        if (x < kIXfers / kWaves) {
            const int n = x * kWaves + wave;
            uint32_t off;
            if constexpr (kIT) {
                off = (uint32_t)((8 * (n & 7)) * ldi_b) + (n >> 3) * 128 + i_lane;
            } else {
                off = (uint32_t)(8 * n * ldi_b) + i_lane;
                if (8 * chunk8 >= i_left) off = kOutside;
            }
            window_to_lds(irsrc, off, buf + n * 1024);
        } else {
            const int n = (x - kIXfers / kWaves) * kWaves + wave;
            if (kJXfers % kWaves != 0 && n >= kJXfers) return;
            uint32_t off;
            if constexpr (kJT) {
                off = (uint32_t)((8 * (n & 7)) * ldj_b) + (n >> 3) * 128 + j_lane;
            } else if constexpr (kJFp8) {
                off = (uint32_t)(16 * (kGated ? n >> 1 : n) * ldj_b) + j_lane;
                if (16 * chunk16 >= left) off = kOutside;
            } else {
                off = (uint32_t)((kGated ? 16 * (n >> 2) + 8 * (n & 1) : 8 * n) * ldj_b) + j_lane;
                if (8 * chunk8 >= left) off = kOutside;
            }
            window_to_lds(jrsrc, off, buf + kIBytes + n * 1024);
        }
    };

    // ---- operand reads. Depth order inside a stage: step ks = 2 pp + q has lane
    // half hf supply depth 32 pp + 16 hf + 8 q .. + 7 of its row (any order that
    // both operands share gives the same sum), so that a lane's E4M3 codes of two
    // steps are 16 consecutive bytes.
    int row_off[4];  // by rows: chunk 4 pp + 2 hf + q of row col
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) row_off[ks] = col * 128 + (((4 * (ks >> 1) + 2 * hf + (ks & 1)) ^ swz(col)) << 4);
    int tr_off[2][2][2];  // by columns: [q][depth group of 4][half of the panel]
    if constexpr (kIT || kJT) {
        const int s = lane & 15, g = lane >> 4;
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int row = 16 * (g >> 1) + 8 * q + 4 * h + (s >> 2);
                    const int c = 4 * b + 2 * (g & 1) + ((s & 3) >> 1);
                    tr_off[q][h][b] = row * 128 + ((c ^ swz(row)) << 4) + (s & 1) * 8;
                }
    }
    auto read_tile = [&](const char* region, bool by_columns, int t, int ks) __attribute__((always_inline)) {
        if (!by_columns) return *(const lds_op*)(region + t * 4096 + row_off[ks]);
        const char* panel = region + (t >> 1) * 8192 + (ks >> 1) * 4096;
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(panel + tr_off[ks & 1][0][t & 1]));
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(panel + tr_off[ks & 1][1][t & 1]));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    // the wave's tiles start at an even tile of the region where panels are used
    static_assert(!kIT || kMI % 2 == 0 || kWI == 1, "panels per wave");
    static_assert(!kJT || kMJ % 2 == 0 || kWJ == 1, "panels per wave");
    const int i_base = kIT ? wi * (kMI / 2) * 8192 : wi * kMI * 4096;
    const int j_base = kIBytes + (kJT ? wj * (kMJ / 2) * 8192 : wj * kMJ * (kJFp8 ? 2048 : 4096));
    i16x8 iop[2][kMI];
    u32x4 jop[2][kMJ];  // E4M3: the codes of two steps, read at the first
    auto read_ops = [&](int st, int ks) __attribute__((always_inline)) {
        const char* buf = smem + (st & 1) * kStage;
        const int set = ks & 1;
#pragma unroll
        for (int t = 0; t < kMJ; ++t) {
            if constexpr (kJFp8) {
                if ((ks & 1) == 0)
                    jop[(ks >> 1) & 1][t] = *(const lds_u32x4*)(buf + j_base + t * 2048 + col * 64 +
                                                               (((2 * (ks >> 1) + hf) ^ ((col >> 2) & 3)) << 4));
            } else {
                jop[set][t] = __builtin_bit_cast(u32x4, read_tile(buf + j_base, kJT, t, ks));
            }
        }
#pragma unroll
        for (int t = 0; t < kMI; ++t) iop[set][t] = read_tile(buf + i_base, kIT, t, ks);
    };

    f32x16 acc[kMJ][kMI];
#pragma unroll
    for (int j = 0; j < kMJ; ++j)
#pragma unroll
        for (int i = 0; i < kMI; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[j][i][r] = 0.0f;
    float sums[kMI] = {};  // row sums of the I operand (dbias)

    auto land = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    auto main_loop = [&]<bool kSums>() __attribute__((always_inline)) {
        // step ks's matrix instructions, with the transfers of stage `next` between them
        auto step = [&]<bool kIssue>(int ks, int next) __attribute__((always_inline)) {
            const int set = ks & 1;
            u32x4 irsrc, jrsrc;
            if constexpr (kIssue) {
                irsrc = i_window(next);
                jrsrc = j_window(next);
            }
            i16x8 w[kMJ];
#pragma unroll
            for (int t = 0; t < kMJ; ++t) {
                if constexpr (kJFp8) {
                    const u32x4 codes = jop[(ks >> 1) & 1][t];
                    const uint2 lo = F::decode(codes[2 * (ks & 1)]), hi = F::decode(codes[2 * (ks & 1) + 1]);
                    w[t] = __builtin_bit_cast(i16x8, u32x4{lo.x, lo.y, hi.x, hi.y});
                } else {
                    w[t] = __builtin_bit_cast(i16x8, jop[set][t]);
                }
            }
#pragma unroll
            for (int q = 0; q < kMI * kMJ; ++q) {
                const int j = q / kMI, i = q % kMI;
                acc[j][i] = F::mfma(w[j], iop[set][i], acc[j][i]);
                if constexpr (kIssue)
                    if (q < kXfers) issue(next, q, irsrc, jrsrc);
            }
            if constexpr (kIssue) {
#pragma unroll
                for (int q = kMI * kMJ; q < kXfers; ++q) issue(next, q, irsrc, jrsrc);
            }
            if constexpr (kSums) {
#pragma unroll
                for (int i = 0; i < kMI; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sums[i] = F::dot_ones(__builtin_bit_cast(u32x4, iop[set][i])[e], sums[i]);
            }
        };
        auto stage = [&]<bool kIssue>(int st) __attribute__((always_inline)) {
#pragma unroll
            for (int ks = 0; ks < 3; ++ks) {
                read_ops(st, ks + 1);
                __builtin_amdgcn_sched_barrier(0);
                step.template operator()<false>(ks, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            land();  // stage st + 1 is there, and nobody reads stage st any more
            read_ops(st + 1, 0);  // (past the last stage: unused)
            __builtin_amdgcn_sched_barrier(0);
            step.template operator()<kIssue>(3, st + 2);
            __builtin_amdgcn_sched_barrier(0);
        };
        {
            const u32x4 ir = i_window(0), jr = j_window(0);
#pragma unroll
            for (int x = 0; x < kXfers; ++x) issue(0, x, ir, jr);
        }
        land();
        read_ops(0, 0);
        if (n_stages > 1) {
            const u32x4 ir = i_window(1), jr = j_window(1);
#pragma unroll
            for (int x = 0; x < kXfers; ++x) issue(1, x, ir, jr);
        }
        int st = 0;
        for (; st < n_stages - 2; ++st) stage.template operator()<true>(st);
        for (; st < n_stages; ++st) stage.template operator()<false>(st);
    };
    const bool with_sums = kEpi == kFfStore && kIT && p.row_sums != nullptr && j0 == 0 && wj == 0;
    if constexpr (kEpi == kFfStore && kIT) {
        if (with_sums) main_loop.template operator()<true>();
        else main_loop.template operator()<false>();
    } else {
        main_loop.template operator()<false>();
    }

    // ---- epilogue. acc[t][s][4u + q]: row i0 + 32 (kMI wi + s) + col, tile column
    // 32 (kMJ wj + t) + 8u + 4hf + q. Two groups of 4 columns are rounded, packed
    // and exchanged between the lane halves, so that every lane stores 16 bytes.
    // Everything goes through windows of the tile's rows: rows past the end lie
    // outside them, columns past the end get an offset that does (loads give 0,
    // stores nothing), so that no access branches.
    const bool vec = p.vec != 0;
    const int wave_row = 32 * kMI * wi + col;                  // + 32 s: the lane's row in the tile
    const int wave_col = (kGated ? 16 : 32) * kMJ * wj;        // + (16 | 32) t: columns of C in the tile
    const int cols = (int)min64(p.cols - j0, 1 << 16);         // columns of C from j0 on
    auto rows_window = [&](const void* base, int64_t ld, int64_t first) __attribute__((always_inline)) {
        // [i_rows, ..] of a row-major 16-bit tensor, from column `first` to the end of C's columns
        const uint64_t b = (uint64_t)(uintptr_t)base + (uint64_t)((i0 * ld + first) * 2);
        return __builtin_amdgcn_make_buffer_rsrc((void*)(uintptr_t)b, 0, (int)(base == nullptr ? 0 : ((i_rows - 1) * ld + cols) * 2),
                                                 0x00020000);
    };
    auto load4 = [&](__amdgpu_buffer_rsrc_t r, uint32_t row_b, int c, float (&v)[4]) __attribute__((always_inline)) {
        if (vec) {
            const u32x2 d = __builtin_amdgcn_raw_buffer_load_b64(r, c < cols ? row_b + 2 * c : kOutside, 0, 0);
            v[0] = F::lo(d[0]), v[1] = F::hi(d[0]), v[2] = F::lo(d[1]), v[3] = F::hi(d[1]);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                v[q] = F::lo((uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, c + q < cols ? row_b + 2 * (c + q) : kOutside, 0, 0));
        }
    };
    auto load4f = [&](__amdgpu_buffer_rsrc_t r, int c, float (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            v[q] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, c + q < cols ? 4 * (c + q) : kOutside, 0, 0));
    };
    auto store8 = [&](__amdgpu_buffer_rsrc_t r, uint32_t row_b, int c, const float (&a)[4], const float (&b)[4]) __attribute__((always_inline)) {
        // a: columns c + 4hf .., b: c + 8 + 4hf ..
        uint32_t a0 = F::pack(a[0], a[1]), a1 = F::pack(a[2], a[3]), b0 = F::pack(b[0], b[1]), b1 = F::pack(b[2], b[3]);
        join_halves(a0, b0);
        join_halves(a1, b1);
        const int at = c + 8 * hf;
        const u32x4 d{a0, a1, b0, b1};
        if (vec) {
            __builtin_amdgcn_raw_buffer_store_b128(d, r, at < cols ? row_b + 2 * at : kOutside, 0, 0);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                __builtin_amdgcn_raw_buffer_store_b16((uint16_t)(d[e >> 1] >> (16 * (e & 1))), r,
                                                      at + e < cols ? row_b + 2 * (at + e) : kOutside, 0, 0);
        }
    };
    auto vector_window = [&](const void* base, int64_t first, int elem) __attribute__((always_inline)) {
        return __builtin_amdgcn_make_buffer_rsrc((void*)((uintptr_t)base + (uintptr_t)(first * elem)), 0,
                                                 base == nullptr ? 0 : cols * elem, 0x00020000);
    };
    // dz: zeros behind the last column, up to the padded row
    auto zero_pad = [&](uint32_t row, int64_t first) __attribute__((always_inline)) {
        if (j0 + kCols >= p.cols && wj == 0 && hf == 0 && (int64_t)row < i_rows)
            for (int64_t z = first; z < p.out_cols_padded; ++z) ((T*)p.out)[(i0 + row) * p.ld_out + z] = (T)0.0f;
    };
    const FfAct act = ff_act(p.activation);
    const uint32_t ldo_b = (uint32_t)(p.ld_out * 2), ldd_b = (uint32_t)(p.ld_dout * 2), ldr_b = (uint32_t)(p.ld_res * 2);
    auto epilogue = [&]<FfFamily kFam>() __attribute__((always_inline)) {
        if constexpr (kGated) {
            const auto bias_v = vector_window(p.bias, value_row + j0, 2), bias_g = vector_window(p.bias, gate_row + j0, 2);
            const auto scale_v = vector_window(p.j_scale, value_row + j0, 4), scale_g = vector_window(p.j_scale, gate_row + j0, 4);
            const auto dout = rows_window(p.dout, p.ld_dout, j0);
            const auto out_v = rows_window(p.out, p.ld_out, (kEpi == kFfGatedDz ? value_row : 0) + j0);
            const auto out_g = rows_window(p.out, p.ld_out, gate_row + j0);
#pragma unroll
            for (int t = 0; t < kMJ; ++t) {
                const int c0 = wave_col + 16 * t;
                float bv[2][4], bg[2][4], sv[2][4], sg[2][4];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    load4(bias_v, 0, c0 + 8 * u + 4 * hf, bv[u]);
                    load4(bias_g, 0, c0 + 8 * u + 4 * hf, bg[u]);
                    if (p.j_scale != nullptr) {
                        load4f(scale_v, c0 + 8 * u + 4 * hf, sv[u]);
                        load4f(scale_g, c0 + 8 * u + 4 * hf, sg[u]);
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q) sv[u][q] = sg[u][q] = 1.0f;
                    }
                }
#pragma unroll
                for (int s = 0; s < kMI; ++s) {
                    const uint32_t row = wave_row + 32 * s;
                    float va[2][4], vb[2][4];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        float d[4];
                        if constexpr (kEpi == kFfGatedDz) load4(dout, row * ldd_b, c0 + 8 * u + 4 * hf, d);
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const float v = __builtin_fmaf(acc[t][s][4 * u + q], sv[u][q], bv[u][q]);
                            const float g = __builtin_fmaf(acc[t][s][8 + 4 * u + q], sg[u][q], bg[u][q]);
                            if constexpr (kEpi == kFfGated) {
                                va[u][q] = v * ff_value<kFam>(act, g);
                            } else {
                                float a;
                                const float sl = ff_slope<kFam>(act, g, a);
                                va[u][q] = d[q] * a;
                                vb[u][q] = d[q] * v * sl;
                            }
                        }
                    }
                    store8(out_v, row * ldo_b, c0, va[0], va[1]);
                    if constexpr (kEpi == kFfGatedDz) {
                        store8(out_g, row * ldo_b, c0, vb[0], vb[1]);
                        if (t == 0) zero_pad(row, 2 * p.cols);
                    }
                }
            }
        } else {
            const auto bias = vector_window(p.bias, j0, 2), scale = vector_window(p.j_scale, j0, 4);
            const auto dout = rows_window(p.dout, p.ld_dout, j0), residual = rows_window(p.residual, p.ld_res, j0);
            const auto out = rows_window(p.out, p.ld_out, j0);
#pragma unroll
            for (int t = 0; t < kMJ; ++t) {
                const int c0 = wave_col + 32 * t;
                float b[4][4], sc[4][4];
                if constexpr (kEpi != kFfStore) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        load4(bias, 0, c0 + 8 * u + 4 * hf, b[u]);
                        if (p.j_scale != nullptr) {
                            load4f(scale, c0 + 8 * u + 4 * hf, sc[u]);
                        } else {
#pragma unroll
                            for (int q = 0; q < 4; ++q) sc[u][q] = 1.0f;
                        }
                    }
                }
#pragma unroll
                for (int s = 0; s < kMI; ++s) {
                    const uint32_t row = wave_row + 32 * s;
                    float v[4][4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        float d[4] = {};
                        if constexpr (kEpi == kFfLinearDz) {
                            load4(dout, row * ldd_b, c0 + 8 * u + 4 * hf, d);
                        } else if constexpr (kEpi == kFfLinear) {
                            if (p.residual != nullptr) load4(residual, row * ldr_b, c0 + 8 * u + 4 * hf, d);
                        }
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const float sum = acc[t][s][4 * u + q];
                            if constexpr (kEpi == kFfStore) {
                                v[u][q] = sum;
                            } else if constexpr (kEpi == kFfLinear) {
                                v[u][q] = ff_value<kFam>(act, __builtin_fmaf(sum, sc[u][q], b[u][q])) + d[q];
                            } else {
                                float a;
                                v[u][q] = ff_slope<kFam>(act, __builtin_fmaf(sum, sc[u][q], b[u][q]), a) * d[q];
                            }
                        }
                    }
                    store8(out, row * ldo_b, c0, v[0], v[1]);
                    store8(out, row * ldo_b, c0 + 16, v[2], v[3]);
                    if constexpr (kEpi == kFfLinearDz)
                        if (t == 0) zero_pad(row, p.cols);
                }
            }
        }
    };
    if constexpr (kEpi == kFfStore) {
        epilogue.template operator()<kFamLinear>();
        if constexpr (kIT) {
            if (with_sums) {
#pragma unroll
                for (int s = 0; s < kMI; ++s) {
                    const int64_t i = i0 + 32 * (kMI * wi + s) + col;
                    const float v = sums[s] + __shfl_xor(sums[s], 32);
                    if (hf == 0 && i < p.rows) ((T*)p.row_sums)[i] = (T)v;
                }
            }
        }
    } else {
        const FfFamily fam = ff_family(p.activation);
        if (fam == kFamErf) epilogue.template operator()<kFamErf>();
        else if (fam == kFamSigmoid) epilogue.template operator()<kFamSigmoid>();
        else epilogue.template operator()<kFamLinear>();
    }
}

template <typename T, bool kIT, bool kJT, bool kJFp8, int kWI, int kWJ, int kMI, int kMJ, FfEpilogue kEpi>
hipError_t launch(FfParams p, hipStream_t stream) {
    constexpr bool gated = kEpi == kFfGated || kEpi == kFfGatedDz;
    constexpr int bi = 32 * kMI * kWI, bj = 32 * kMJ * kWJ / (gated ? 2 : 1);
    p.i_blocks = (int32_t)((p.rows + bi - 1) / bi);
    p.j_blocks = (int32_t)((p.cols + bj - 1) / bj);
    p.group_i = p.i_blocks < 8 ? p.i_blocks : 8;
    hipLaunchKernelGGL((ff_tile_kernel<T, kIT, kJT, kJFp8, kWI, kWJ, kMI, kMJ, kEpi>),
                       dim3((unsigned)((int64_t)p.i_blocks * p.j_blocks)), dim3(64 * kWI * kWJ), 0, stream, p);
    return hipGetLastError();
}

#define FF_TILE 4, 2, 2, 4
template <typename T>
hipError_t launch_type(const FfParams& p, FfEpilogue epilogue, bool it, bool j_fp8, hipStream_t stream) {
    switch (epilogue) {
    case kFfLinear: return j_fp8 ? launch<T, false, false, true, FF_TILE, kFfLinear>(p, stream) : launch<T, false, false, false, FF_TILE, kFfLinear>(p, stream);
    case kFfGated: return j_fp8 ? launch<T, false, false, true, FF_TILE, kFfGated>(p, stream) : launch<T, false, false, false, FF_TILE, kFfGated>(p, stream);
    case kFfLinearDz: return launch<T, false, false, false, FF_TILE, kFfLinearDz>(p, stream);
    case kFfGatedDz: return launch<T, false, false, false, FF_TILE, kFfGatedDz>(p, stream);
    case kFfStore: return it ? launch<T, true, true, false, FF_TILE, kFfStore>(p, stream) : launch<T, false, true, false, FF_TILE, kFfStore>(p, stream);
    }
    return hipErrorInvalidValue;
}

bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

}  // namespace

bool ff_tiled_supported(const FfParams& p, FfEpilogue epilogue, bool i_transposed, bool j_transposed, bool j_fp8) {
    if (p.depth <= 0 || (epilogue == kFfStore && (!j_transposed || p.out == nullptr))) return false;
    // rows in whole 16-byte chunks: the depth, or the columns of an operand that is read by columns
    const int64_t i_row = p.i_row != 0 ? p.i_row : i_transposed ? p.rows : p.depth;
    if (!aligned(p.ip, 16) || !aligned(p.jp, 16) || p.ld_i % 8 != 0 || p.ld_j % (j_fp8 ? 16 : 8) != 0) return false;
    if (i_row % 8 != 0 || (j_transposed ? p.cols % 8 != 0 : p.depth % (j_fp8 ? 16 : 8) != 0)) return false;
    // a window (at most 512 rows) stays below 2^31 bytes, the tasks below 2^31
    if (p.ld_i > (1 << 20) || p.ld_j > (1 << 20) || p.ld_out > (1 << 20) || p.ld_dout > (1 << 20) || p.ld_res > (1 << 20))
        return false;
    return ((p.rows + 255) / 256) * ((p.cols + 127) / 128) <= 4000000;
}

hipError_t launch_ff_tiled(const FfParams& params, FfEpilogue epilogue, bool i_transposed, bool bf16, bool j_fp8,
                           hipStream_t stream) {
    FfParams p = params;
    if (p.i_row == 0) p.i_row = i_transposed ? p.rows : p.depth;
    // 16-byte stores and 8-byte loads in the epilogue
    p.vec = p.cols % 8 == 0 && p.ld_out % 8 == 0 && aligned(p.out, 16) && aligned(p.bias, 8) && aligned(p.residual, 8) &&
            aligned(p.dout, 8) && (p.residual == nullptr || p.ld_res % 4 == 0) && (p.dout == nullptr || p.ld_dout % 4 == 0);
    return bf16 ? launch_type<__bf16>(p, epilogue, i_transposed, j_fp8, stream)
                : launch_type<_Float16>(p, epilogue, i_transposed, j_fp8, stream);
}

}  // namespace sdxl_hip
