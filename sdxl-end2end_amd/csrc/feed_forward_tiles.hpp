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
// Depth goes in stages of 64 through a ring of kRing LDS buffers, filled by
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
// barrier, the next stage's first reads and the issue of the transfers. The
// reads go out one by one behind the step's first matrix instructions, in the
// order of use, the transfers evenly behind all of them: bunched before and
// behind the step they took turns with the matrix cores instead (x 2048 x 1280,
// w 10240 x 1280, loop alone: 256 x 320 tiles 37.9 us, now 36.1; 128 x 256
// tiles 18.6, now 17.6).
//
// A depth in shares (kSplit): a workgroup sums one share and leaves it in fp32
// for the joining pass. Staged operands (kStaged, rows that 16-byte accesses do
// not divide): 16-byte loads at any element's address bring a stage into
// registers a stage ahead, from where it is put down where the transfers would
// have (gated [2048, 1281] -> 2 x 5120 in bf16 109 us, 52 where 1280 allows the
// transfers).
//
// Gated products put 16 value rows and the 16 gate rows of the same columns
// into every 32-row J tile: a lane holds value and gate of its columns and the
// product needs no exchange.
#pragma once

#include <hip/hip_runtime.h>

#include <utility>

#include "feed_forward_device.hpp"
#include "feed_forward_kernels.hpp"

namespace sdxl_hip {
namespace {

typedef __attribute__((address_space(3))) i16x8 lds_op;
typedef __attribute__((address_space(3))) float lds_float;

__device__ __forceinline__ int64_t min64(int64_t a, int64_t b) { return a < b ? a : b; }

// Exchanges the halves so that lanes 0-31 hold 8 consecutive columns made of
// both halves' a, lanes 32-63 those of b (a, b: two values each, packed).
__device__ __forceinline__ void join_halves(uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}

// A tile: kWI x kWJ waves of (32 kMI) x (32 kMJ) blocks, kWK such groups of
// waves that share every stage's depth, kRing stages in LDS.
template <int kWI_, int kWJ_, int kWK_, int kMI_, int kMJ_, int kRing_, int kSpread_ = 1>
struct FfTile {
    static constexpr int kWI = kWI_, kWJ = kWJ_, kWK = kWK_, kMI = kMI_, kMJ = kMJ_, kRing = kRing_, kSpread = kSpread_;
    static constexpr int kWaves = kWI * kWJ * kWK, kBI = 32 * kMI * kWI, kBJ = 32 * kMJ * kWJ;
    static constexpr int stage_bytes(bool j_fp8) { return kBI * 128 + kBJ * (j_fp8 ? 64 : 128); }
    // the stages, or the sums of the other depth shares (one round of tiles at a time)
    static constexpr int smem_bytes(bool j_fp8) {
        const int stages = kRing * stage_bytes(j_fp8), exchange = kWI * kWJ * kWK * (kWK - 1) * 4096;
        return stages > exchange ? stages : exchange;
    }
    // 8-bit integers: behind them the columns' scales and biases
    static constexpr int constant_bytes(bool i8) { return i8 ? kBJ * 8 : 0; }
    // workgroups that one CU's LDS and registers (512 per lane and SIMD) hold
    static constexpr int waves_per_simd(bool j_fp8) {
        const int by_lds = kWaves / 4 * (160 * 1024 / smem_bytes(j_fp8));
        const int by_regs = kMI * kMJ <= 4 ? 4 : kMI * kMJ <= 10 ? 2 : 1;
        return by_lds < by_regs ? by_lds : by_regs;
    }
};

// Task `id` of a product whose tasks' numbers modulo 8 are their XCDs; smem: Tile::smem_bytes.
template <typename T, bool kIT, bool kJT, bool kJFp8, typename Tile, FfEpilogue kEpi, bool kSplit = false, bool kStaged = false>
__device__ __forceinline__ void ff_tile(const FfParams& p, int task_id, char* smem) {
    constexpr int kWI = Tile::kWI, kWJ = Tile::kWJ, kWK = Tile::kWK, kMI = Tile::kMI, kMJ = Tile::kMJ, kRing = Tile::kRing;
    using F = FfType<T>;
    using Out = typename F::Out;
    using Acc = typename F::Acc;
    using Acc4 = typename F::Acc4;
    typedef __attribute__((address_space(3))) Acc4 lds_acc4;
    constexpr int kElem = F::kElem, kDepth = 128 / kElem, kChunk = 16 / kElem;  // elements of a stage, of 16 bytes
    constexpr bool kGated = kEpi == kFfGated || kEpi == kFfGatedDz;
    constexpr int kWaves = Tile::kWaves, kBI = Tile::kBI, kBJ = Tile::kBJ;
    constexpr int kCols = kGated ? kBJ / 2 : kBJ;  // columns of C per tile
    constexpr int kSteps = 4 / kWK;                // depth steps (of 16) per wave and stage
    constexpr int kSpread = Tile::kSpread;         // steps that a stage's requests are spread over
    static_assert(kSpread <= kSteps, "steps");
    constexpr int kIBytes = kBI * 128, kStage = Tile::stage_bytes(kJFp8), kJBytes = kStage - kIBytes;
    constexpr int kIXfers = kIBytes / 1024, kJXfers = kJBytes / 1024;
    constexpr int kIX = (kIXfers + kWaves - 1) / kWaves, kXfers = kIX + (kJXfers + kWaves - 1) / kWaves;
    static_assert(kWaves % 4 == 0, "the waves' transfers keep their parity and their half of the gating");
    // waves below kMore have kXfers transfers a stage, the others one less
    constexpr int kMore = kIXfers % kWaves + kJXfers % kWaves;
    static_assert(kIXfers % kWaves == 0 || kJXfers % kWaves == 0, "one operand's transfers come out even");
    static_assert((kRing - 1) * kXfers < 64, "vmcnt range");
    static_assert(kWK == 1 || (kWK == 2 && !kJFp8), "depth shares");
    static_assert(!kGated || (!kIT && !kJT), "gated products are projections");
    static_assert(!kJFp8 || !kJT, "E4M3: by rows");
    static_assert(!F::kI8 || (!kIT && !kJT && !kJFp8 && !kSplit && (kEpi == kFfLinear || kEpi == kFfGated)), "8-bit integers: projections");
    static_assert(Tile::smem_bytes(kJFp8) <= 160 * 1024, "LDS of one CU");

    const int lane = threadIdx.x & 63, hf = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave % kWI, wj = wave / kWI % kWJ, wk = kWK > 1 ? wave / (kWI * kWJ) : 0;
    const int64_t value_row = p.gate_first ? p.cols : 0, gate_row = p.gate_first ? 0 : p.cols;
    const int64_t ldi_b = p.ld_i * kElem, ldj_b = p.ld_j * (kJFp8 ? 1 : kElem);
    // the workgroup's share of the depth: from depth0 on
    static_assert(!kSplit || kEpi == kFfStore, "shares are joined before an epilogue");
    const int n_tiles = p.i_blocks * p.j_blocks, share = kSplit ? task_id / n_tiles : 0, id = kSplit ? task_id % n_tiles : task_id;
    const int64_t depth0 = kSplit ? (int64_t)share * p.share_stages * kDepth : 0;
    const int64_t depth = kSplit ? min64(p.depth - depth0, (int64_t)p.share_stages * kDepth) : p.depth;
    const int64_t i_row = kIT ? p.i_row : p.i_row - depth0;  // (by columns the row runs along C)
    const int n_stages = (int)((depth + kDepth - 1) / kDepth);

    // ---- task: each XCD takes one contiguous range of them, in groups of
    // group_i row blocks (rows fastest, then columns), so that its workgroups
    // share I rows and J rows in its L2
    int64_t i0, j0;
    {
        const int xcd = id & 7, slot = id >> 3;
        const int per = n_tiles >> 3, extra = n_tiles & 7;
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
        iw.base = (const char*)p.ip + i0 * 2 + depth0 * ldi_b;
        i_lane = (uint32_t)(row8 * ldi_b) + chunk8 * 16;
    } else {
        iw.base = (const char*)p.ip + i0 * ldi_b + depth0 * kElem;
        i_lane = (uint32_t)(row8 * ldi_b) + chunk8 * 16;
    }
    const int64_t j_first = kGated ? j0 + ((kJFp8 ? wave & 1 : wave & 2) ? gate_row : value_row) : j0;
    if constexpr (kJT) jw.base = (const char*)p.jp + j0 * 2 + depth0 * ldj_b;
    else jw.base = (const char*)p.jp + j_first * ldj_b + depth0 * (kJFp8 ? 1 : kElem);
    j_lane = kJFp8 ? (uint32_t)(row16 * ldj_b) + chunk16 * 16 : (uint32_t)(row8 * ldj_b) + chunk8 * 16;
    const int64_t i_rows = min64(p.rows - i0, kBI), j_rows = min64(p.cols - j0, kGated ? kCols : kBJ);
    // window of stage st: everything from its first byte to the last valid one
    // (past the last stage: nothing, its transfers write zeros that nobody reads)
    auto i_window = [&](int st) __attribute__((always_inline)) {
        const int64_t left = depth - (int64_t)st * kDepth;
        const char* base = iw.base + (kIT ? (int64_t)st * 64 * ldi_b : (int64_t)st * 128);
        const int64_t size = kIT ? (min64(left, 64) - 1) * ldi_b + min64(i_row - i0, kBI) * 2
                                 : (i_rows - 1) * ldi_b + (i_row - (int64_t)st * kDepth) * kElem;
        return window_rsrc({base, left > 0 ? (uint32_t)size : 0u});
    };
    auto j_window = [&](int st) __attribute__((always_inline)) {
        const int64_t left = depth - (int64_t)st * kDepth;
        const char* base = jw.base + (kJT ? (int64_t)st * 64 * ldj_b : (int64_t)st * (kJFp8 ? 64 : 128));
        const int64_t size = kJT ? (min64(left, 64) - 1) * ldj_b + j_rows * 2 : (j_rows - 1) * ldj_b + left * (kJFp8 ? 1 : kElem);
        return window_rsrc({base, left > 0 ? (uint32_t)size : 0u});
    };
    const uint32_t lds0 = lds_addr(smem);
    // Staged: rows that 16-byte accesses do not divide come through registers, to the places that the transfers give
    // them: the wave's parts of the next stage are fetched over a stage before they are needed. A chunk that its row
    // ends in is fetched as the row's last 16 bytes and shifted when it is put down.
    static_assert(!kStaged || (kRing == 2 && kSpread == 1 && kMore == 0), "staged: one stage in LDS, one in registers");
    u32x4 held[kStaged ? kXfers : 1];
    // part x of stage st: its address, and how many of the chunk's elements its row has (none: 0 or less)
    auto part = [&](int st, int x, const char*& from) __attribute__((always_inline)) {
        const int64_t d_left = depth - (int64_t)st * kDepth;
        const int left = (int)min64(d_left, kDepth);
        int64_t off;
        int valid;
        if (x < kIX) {
            const int n = x * kWaves + wave;
            if constexpr (kIT) {
                off = (int64_t)st * 64 * ldi_b + (int64_t)(8 * (n & 7)) * ldi_b + (n >> 3) * 128 + i_lane;
                valid = 8 * (n & 7) + row8 < left ? (int)min64(i_row - i0, kBI) - 64 * (n >> 3) - 8 * chunk8 : 0;
            } else {
                off = (int64_t)st * 128 + (int64_t)(8 * n) * ldi_b + i_lane;
                valid = 8 * n + row8 < i_rows ? (int)min64(i_row - (int64_t)st * kDepth, kDepth) - kChunk * chunk8 : 0;
            }
            from = iw.base + off;
        } else {
            const int n = (x - kIX) * kWaves + wave;
            if constexpr (kJT) {
                off = (int64_t)st * 64 * ldj_b + (int64_t)(8 * (n & 7)) * ldj_b + (n >> 3) * 128 + j_lane;
                valid = 8 * (n & 7) + row8 < left ? (int)j_rows - 64 * (n >> 3) - 8 * chunk8 : 0;
            } else {
                const int first = kJFp8 ? 16 * (kGated ? n >> 1 : n) : kGated ? 16 * (n >> 2) + 8 * (n & 1) : 8 * n;
                off = (int64_t)st * (kJFp8 ? 64 : 128) + (int64_t)first * ldj_b + j_lane;
                valid = first + (kJFp8 ? row16 : row8) < j_rows ? left - (kJFp8 ? 16 * chunk16 : kChunk * chunk8) : 0;
            }
            from = jw.base + off;
        }
        return valid;
    };
    const bool inner_tile = i_rows == kBI && j_rows == (kGated ? kCols : kBJ) && (!kIT || i_row - i0 >= kBI);
    auto whole = [&](int st) __attribute__((always_inline)) { return inner_tile && depth - (int64_t)st * kDepth >= kDepth; };
    auto read16 = [&](int x, const char* from) __attribute__((always_inline)) {
        return kJFp8 && x >= kIX ? ((const Unaligned<1>*)from)->v : ((const Unaligned<kElem>*)from)->v;
    };
    auto fetch = [&](int st) __attribute__((always_inline)) {
        const char* from;
        if (whole(st)) {
#pragma unroll
            for (int x = 0; x < kXfers; ++x) {
                part(st, x, from);
                held[x] = read16(x, from);
            }
        } else {
#pragma unroll
            for (int x = 0; x < kXfers; ++x) {
                const int valid = part(st, x, from);
                held[x] = kJFp8 && x >= kIX ? fetch_chunk<16>(from, valid) : fetch_chunk<kChunk>(from, valid);
            }
        }
    };
    auto put = [&](int st, int buffer) __attribute__((always_inline)) {
        char* buf = smem + buffer * kStage + lane * 16;
        if (!whole(st)) {
#pragma unroll
            for (int x = 0; x < kXfers; ++x) {
                const char* from;
                const int valid = part(st, x, from);
                held[x] = kJFp8 && x >= kIX ? settle_chunk<16>(held[x], valid) : settle_chunk<kChunk>(held[x], valid);
            }
        }
#pragma unroll
        for (int x = 0; x < kXfers; ++x)
            *(lds_u32x4*)(buf + (x < kIX ? 0 : kIBytes) + ((x < kIX ? x : x - kIX) * kWaves + wave) * 1024) = held[x];
    };
    // one of the wave's kXfers transfers of stage st
    auto issue = [&](int st, int buffer, int x, u32x4 irsrc, u32x4 jrsrc) __attribute__((always_inline)) {
        const uint32_t buf = lds0 + buffer * kStage;
        // depth of the stage, by I's rows and by J's
        const int i_left = (int)min64(i_row - (int64_t)st * kDepth, kDepth), left = (int)min64(depth - (int64_t)st * kDepth, kDepth);
        if (x < kIX) {
            const int n = x * kWaves + wave;
            if (kIXfers % kWaves != 0 && n >= kIXfers) return;
            uint32_t off;
            if constexpr (kIT) {
                off = (uint32_t)((8 * (n & 7)) * ldi_b) + (n >> 3) * 128 + i_lane;
            } else {
                off = (uint32_t)(8 * n * ldi_b) + i_lane;
                if (kChunk * chunk8 >= i_left) off = kOutside;
            }
            window_to_lds(irsrc, off, buf + n * 1024);
        } else {
            const int n = (x - kIX) * kWaves + wave;
            if (kJXfers % kWaves != 0 && n >= kJXfers) return;
            uint32_t off;
            if constexpr (kJT) {
                off = (uint32_t)((8 * (n & 7)) * ldj_b) + (n >> 3) * 128 + j_lane;
            } else if constexpr (kJFp8) {
                off = (uint32_t)(16 * (kGated ? n >> 1 : n) * ldj_b) + j_lane;
                if (16 * chunk16 >= left) off = kOutside;
            } else {
                off = (uint32_t)((kGated ? 16 * (n >> 2) + 8 * (n & 1) : 8 * n) * ldj_b) + j_lane;
                if (kChunk * chunk8 >= left) off = kOutside;
            }
            window_to_lds(jrsrc, off, buf + kIBytes + n * 1024);
        }
    };

    // ---- operand reads. Depth order inside a stage: step ks = 2 pp + q has lane
    // half hf supply depth 32 pp + 16 hf + 8 q .. + 7 of its row (any order that
    // both operands share gives the same sum), so that a lane's E4M3 codes of two
    // steps are 16 consecutive bytes.
    // With the depth shared, group wk of the waves takes steps kSteps wk ...
    int row_off[kSteps];  // by rows: chunk 4 pp + 2 hf + q of row col
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        const int ks = kSteps * wk + k;
        row_off[k] = col * 128 + (((4 * (ks >> 1) + 2 * hf + (ks & 1)) ^ swz(col)) << 4);
    }
    // by columns: [q][depth group of 4] in the wave's half of the panel
    int tr_i[2][2], tr_j[2][2];
    if constexpr (kIT || kJT) {
        const int s = lane & 15, g = lane >> 4, pp = kSteps * wk >> 1;
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = 16 * (g >> 1) + 8 * q + 4 * h + (s >> 2);
                const int c = 2 * (g & 1) + ((s & 3) >> 1), at = pp * 4096 + row * 128 + (s & 1) * 8;
                tr_i[q][h] = at + (((c + 4 * (wi & 1)) ^ swz(row)) << 4);
                tr_j[q][h] = at + (((c + 4 * (wj & 1)) ^ swz(row)) << 4);
            }
    }
    // The wave's tile t is tile kW t + w of the region (kW waves share the
    // operand): by columns it is half w % 2 of panel (kW t + w) / 2.
    static_assert(kWI % 2 == 0 && kWJ % 2 == 0 && kSteps % 2 == 0, "half panels by wave, both depth groups by step");
    auto read_rows = [&](const char* region, int t, int k) __attribute__((always_inline)) {
        return *(const lds_op*)(region + t * 4096 + row_off[k]);
    };
    auto read_columns = [&](const char* region, int panel, int lo_off, int hi_off, int k) __attribute__((always_inline)) {
        const char* base = region + panel * 8192 + (k >> 1) * 4096;
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(base + lo_off));
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(base + hi_off));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    const int i_base = kIT ? (wi >> 1) * 8192 : wi * 4096;
    const int j_base = kIBytes + (kJT ? (wj >> 1) * 8192 : wj * (kJFp8 ? 2048 : 4096));
    i16x8 iop[2][kMI];
    u32x4 jop[2][kMJ];  // E4M3: the codes of two steps, read at the first
    // operand x of step k, in the order in which the step needs them: J tile 0, the I tiles, the other J tiles
    auto read_op = [&](int buffer, int k, int set, int x) __attribute__((always_inline)) {
        const char* buf = smem + buffer * kStage;
        if (x == 0 || x > kMI) {
            const int t = x == 0 ? 0 : x - kMI;
            if constexpr (kJFp8) {
                if ((k & 1) == 0)
                    jop[(k >> 1) & 1][t] = *(const lds_u32x4*)(buf + j_base + t * kWJ * 2048 + col * 64 +
                                                              (((2 * (k >> 1) + hf) ^ ((col >> 2) & 3)) << 4));
            } else {
                if constexpr (kJT) jop[set][t] = __builtin_bit_cast(u32x4, read_columns(buf + j_base, t * kWJ / 2, tr_j[k & 1][0], tr_j[k & 1][1], k));
                else jop[set][t] = __builtin_bit_cast(u32x4, read_rows(buf + j_base, t * kWJ, k));
            }
        } else {
            const int t = x - 1;
            if constexpr (kIT) iop[set][t] = read_columns(buf + i_base, t * kWI / 2, tr_i[k & 1][0], tr_i[k & 1][1], k);
            else iop[set][t] = read_rows(buf + i_base, t * kWI, k);
        }
    };

    // 8-bit integers: thread t's column constants and the lane's row scales, loaded ahead of the main loop and put down (read)
    // behind it. Loaded tile by tile there, each round of them waited for the caches: gated [8192, 2048] -> 2 x 5456 228 us, 200 so.
    constexpr int kConstants = F::kI8 ? (kCols + 64 * kWaves - 1) / (64 * kWaves) : 0;
    float column[kConstants > 0 ? kConstants : 1][4], row_scale[F::kI8 ? kMI : 1];
    if constexpr (F::kI8) {
#pragma unroll
        for (int n = 0; n < kConstants; ++n) {
            const int64_t c = j0 + n * 64 * kWaves + threadIdx.x;
            const bool there = c < p.cols && n * 64 * kWaves + (int)threadIdx.x < kCols;
            const int64_t v = (kGated ? value_row : 0) + c, g = gate_row + c;
            column[n][0] = there ? p.j_scale[v] : 0.0f;
            column[n][1] = there && p.bias != nullptr ? (float)((const Out*)p.bias)[v] : 0.0f;
            column[n][2] = kGated && there ? p.j_scale[g] : 0.0f;
            column[n][3] = kGated && there && p.bias != nullptr ? (float)((const Out*)p.bias)[g] : 0.0f;
        }
#pragma unroll
        for (int s = 0; s < kMI; ++s) {
            const int64_t i = i0 + 32 * (kWI * s + wi) + col;
            row_scale[s] = i < p.rows ? p.i_scale[i] : 0.0f;
        }
    }

    Acc acc[kMJ][kMI];
#pragma unroll
    for (int j = 0; j < kMJ; ++j)
#pragma unroll
        for (int i = 0; i < kMI; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[j][i][r] = 0;
    float sums[kMI] = {};  // row sums of the I operand (dbias)

    // at most kFlying stages' transfers of the wave are still on their way, and no wave reads LDS any more
    auto land = [&]<int kFlying>() __attribute__((always_inline)) {
        if (kFlying == 0 || kMore == 0 || wave < kMore) wait_vmem<kFlying * kXfers>();
        else wait_vmem<kFlying * (kXfers - 1)>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    auto main_loop = [&]<bool kSums>() __attribute__((always_inline)) {
        // Step k's matrix instructions; between them the operand reads of step next_k (from buffer `from`) and part
        // kPart of the transfers of stage `next` (-1: none), evenly spread.
        auto step = [&]<int kPart>(int k, int from, int next_k, int next, int buffer) __attribute__((always_inline)) {
            constexpr int kFrom = kPart < 0 ? 0 : kPart * kXfers / kSpread, kTo = kPart < 0 ? 0 : (kPart + 1) * kXfers / kSpread;
            constexpr int kQs = kMI * kMJ, kReads = kMI + kMJ, kReadQs = kQs > 4 ? kQs / 2 : kQs;
            const int set = k & 1;
            u32x4 irsrc{}, jrsrc{};
            if constexpr (kTo > kFrom) {
                irsrc = i_window(next);
                jrsrc = j_window(next);
            }
            i16x8 w[kMJ];
#pragma unroll
            for (int t = 0; t < kMJ; ++t) {
                if constexpr (kJFp8) {
                    const u32x4 codes = jop[(k >> 1) & 1][t];
                    const uint2 lo = F::decode(codes[2 * (k & 1)]), hi = F::decode(codes[2 * (k & 1) + 1]);
                    w[t] = __builtin_bit_cast(i16x8, u32x4{lo.x, lo.y, hi.x, hi.y});
                } else {
                    w[t] = __builtin_bit_cast(i16x8, jop[set][t]);
                }
            }
#pragma unroll
            for (int q = 0; q < kQs; ++q) {
                const int j = q / kMI, i = q % kMI;
                acc[j][i] = F::mfma(w[j], iop[set][i], acc[j][i]);
#pragma unroll
                for (int x = kReads * q / kReadQs; x < kReads * (q + 1) / kReadQs && x < kReads; ++x) read_op(from, next_k, next_k & 1, x);
#pragma unroll
                for (int x = kFrom + (kTo - kFrom) * q / kQs; x < kFrom + (kTo - kFrom) * (q + 1) / kQs; ++x) issue(next, buffer, x, irsrc, jrsrc);
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (kSums) {
#pragma unroll
                for (int i = 0; i < kMI; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sums[i] = F::dot_ones(__builtin_bit_cast(u32x4, iop[set][i])[e], sums[i]);
            }
        };
        // Stage st in `buffer`: part 0 of the requests of stage st + kRing follows the barrier that frees
        // the buffer, the other parts the next stage's first steps.
        auto stage = [&](int st, int buffer) __attribute__((always_inline)) {
            const int before = buffer == 0 ? kRing - 1 : buffer - 1, after = buffer + 1 == kRing ? 0 : buffer + 1;
            [&]<int... k>(std::integer_sequence<int, k...>) __attribute__((always_inline)) {
                ((step.template operator()<(k + 1 < kSpread ? k + 1 : -1)>(k, buffer, k + 1, st - 1 + kRing, before),
                  __builtin_amdgcn_sched_barrier(0)), ...);
            }(std::make_integer_sequence<int, kSteps - 1>{});
            if constexpr (kStaged) put(st + 1, before);
            land.template operator()<kRing - 2>();  // stage st + 1 is there, and nobody reads stage st any more
            if constexpr (kStaged) fetch(st + kRing);
            step.template operator()<kStaged ? -1 : 0>(kSteps - 1, after, 0, st + kRing, buffer);  // (past the last stage: reads unused)
            __builtin_amdgcn_sched_barrier(0);
        };
        if constexpr (kStaged) {
            fetch(0);
            put(0, 0);
            fetch(1);
        } else {
#pragma unroll
            for (int st = 0; st < kRing; ++st) {
                const u32x4 ir = i_window(st), jr = j_window(st);
#pragma unroll
                for (int x = 0; x < (st == kRing - 1 ? kXfers / kSpread : kXfers); ++x) issue(st, st, x, ir, jr);
            }
        }
        land.template operator()<kRing - 2>();
#pragma unroll
        for (int x = 0; x < kMI + kMJ; ++x) read_op(0, 0, 0, x);
        for (int st = 0, buffer = 0; st < n_stages; ++st, buffer = buffer + 1 == kRing ? 0 : buffer + 1) stage(st, buffer);
        wait_vmem<0>();  // LDS outlives the transfers
    };
    const bool with_sums = kEpi == kFfStore && kIT && p.row_sums != nullptr && j0 == 0 && wj == 0;  // (every depth share)
    if constexpr (kEpi == kFfStore && kIT) {
        if (with_sums) main_loop.template operator()<true>();
        else main_loop.template operator()<false>();
    } else {
        main_loop.template operator()<false>();
    }

    // ---- epilogue. acc[t][s][4u + q]: row i0 + 32 (kWI s + wi) + col, tile column
    // 32 (kWJ t + wj) + 8u + 4hf + q. Two groups of 4 columns are rounded, packed
    // and exchanged between the lane halves, so that every lane stores 16 bytes.
    // Everything goes through windows of the tile's rows: rows past the end lie
    // outside them, columns past the end get an offset that does (loads give 0,
    // stores nothing), so that no access branches.
    const bool vec = p.vec != 0;
    const int wave_row = 32 * wi + col;             // + 32 kWI s: the lane's row in the tile
    const int wave_col = (kGated ? 16 : 32) * wj;   // + (16 | 32) kWJ t: columns of C in the tile
    const int cols = (int)min64(p.cols - j0, 1 << 16);         // columns of C from j0 on
    const uint32_t ldo_b = (uint32_t)(p.ld_out * 2), ldd_b = (uint32_t)(p.ld_dout * 2), ldr_b = (uint32_t)(p.ld_res * 2);
    auto rows_at = [&](const void* base, int64_t ld, int64_t first) __attribute__((always_inline)) { return (char*)base + (i0 * ld + first) * 2; };
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
    // 16 columns from c on of the lane's row: as loaded, 8 a lane, and as the sums lie (columns 8u + 4hf ..).
    // Rows that 16 bytes do not divide: 16 bytes at any address where the row has them, elements at its end
    // (elements alone: gated [2048, 2 x 5123] deep 1280 96 us, dw [10240, 1283] of one row 240).
    auto load16 = [&](__amdgpu_buffer_rsrc_t r, const char* base, uint32_t row, uint32_t ld_b, int c) __attribute__((always_inline)) {
        const int at = c + 8 * hf;
        const uint32_t row_b = row * ld_b;
        if (vec) return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at < cols ? row_b + 2 * at : kOutside, 0, 0));
        if ((int64_t)row < i_rows && at + 8 <= cols) return ((const Unaligned<2>*)(base + row_b + 2 * at))->v;
        u32x4 d{};
#pragma unroll
        for (int e = 0; e < 8; ++e)
            d[e >> 1] |= (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, at + e < cols ? row_b + 2 * (at + e) : kOutside, 0, 0)
                         << (16 * (e & 1));
        return d;
    };
    auto values16 = [&](u32x4 d, float (&v)[2][4]) __attribute__((always_inline)) {
        uint32_t a0 = d[0], a1 = d[1], b0 = d[2], b1 = d[3];
        join_halves(a0, b0);
        join_halves(a1, b1);
        v[0][0] = F::lo(a0), v[0][1] = F::hi(a0), v[0][2] = F::lo(a1), v[0][3] = F::hi(a1);
        v[1][0] = F::lo(b0), v[1][1] = F::hi(b0), v[1][2] = F::lo(b1), v[1][3] = F::hi(b1);
    };
    auto load4f = [&](__amdgpu_buffer_rsrc_t r, int c, float (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            v[q] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, c + q < cols ? 4 * (c + q) : kOutside, 0, 0));
    };
    auto store8 = [&](__amdgpu_buffer_rsrc_t r, char* base, uint32_t row, int c, const float (&a)[4], const float (&b)[4]) __attribute__((always_inline)) {
        // a: columns c + 4hf .., b: c + 8 + 4hf ..
        uint32_t a0 = F::pack(a[0], a[1]), a1 = F::pack(a[2], a[3]), b0 = F::pack(b[0], b[1]), b1 = F::pack(b[2], b[3]);
        join_halves(a0, b0);
        join_halves(a1, b1);
        const int at = c + 8 * hf;
        const u32x4 d{a0, a1, b0, b1};
        const uint32_t row_b = row * ldo_b;
        if (vec) {
            __builtin_amdgcn_raw_buffer_store_b128(d, r, at < cols ? row_b + 2 * at : kOutside, 0, 0);
        } else if ((int64_t)row < i_rows && at + 8 <= cols) {
            ((Unaligned<2>*)(base + row_b + 2 * at))->v = d;
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
            for (int64_t z = first; z < p.out_cols_padded; ++z) ((Out*)p.out)[(i0 + row) * p.ld_out + z] = (Out)0.0f;
    };
    lds_float* const constant = (lds_float*)(smem + Tile::smem_bytes(kJFp8));  // [4][kCols]: scale, bias, the gate's
    if constexpr (F::kI8) {
#pragma unroll
        for (int n = 0; n < kConstants; ++n) {
            const int c = n * 64 * kWaves + threadIdx.x;
            if (c < kCols) {
#pragma unroll
                for (int e = 0; e < (kGated ? 4 : 2); ++e) constant[e * kCols + c] = column[n][e];
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }
    const auto dout = rows_window(p.dout, p.ld_dout, j0), residual = rows_window(p.residual, p.ld_res, j0);
    const auto out = rows_window(p.out, p.ld_out, (kEpi == kFfGatedDz ? value_row : 0) + j0);
    const auto out_g = rows_window(p.out, p.ld_out, (kEpi == kFfGatedDz ? gate_row : 0) + j0);
    const char *dout_at = rows_at(p.dout, p.ld_dout, j0), *residual_at = rows_at(p.residual, p.ld_res, j0);
    char *out_at = rows_at(p.out, p.ld_out, (kEpi == kFfGatedDz ? value_row : 0) + j0);
    char *out_g_at = rows_at(p.out, p.ld_out, (kEpi == kFfGatedDz ? gate_row : 0) + j0);
    // What the epilogue reads of a tile (dout, or the residual): requested for all of the wave's tiles first where the
    // registers hold that, so that its latency passes once (256 x 256, dz [8192, 10240] 258 -> 239 us), else tile by tile.
    constexpr int kSets = kGated ? 1 : 2;  // of 16 columns
    constexpr bool kReads = kEpi == kFfLinear || kEpi == kFfLinearDz || kEpi == kFfGatedDz;
    constexpr bool kAhead = kReads && kWK == 1 && kMI * kMJ * kSets <= 8;
    u32x4 ahead[kAhead ? kMJ : 1][kAhead ? kMI : 1][kSets];
    auto read_tile = [&](uint32_t row, int c0, u32x4 (&d)[kSets]) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < kSets; ++h) {
            if constexpr (kEpi == kFfLinear) {
                if (p.residual != nullptr) d[h] = load16(residual, residual_at, row, ldr_b, c0 + 16 * h);
                else d[h] = u32x4{};
            } else {
                d[h] = load16(dout, dout_at, row, ldd_b, c0 + 16 * h);
            }
        }
    };
    if constexpr (kAhead) {
#pragma unroll
        for (int t = 0; t < kMJ; ++t)
#pragma unroll
            for (int s = 0; s < kMI; ++s) read_tile(wave_row + 32 * kWI * s, wave_col + (kGated ? 16 : 32) * kWJ * t, ahead[t][s]);
        __builtin_amdgcn_sched_barrier(0);
    }
    const FfAct act = ff_act(p.activation);
    constexpr int kHalves = kGated ? 2 : 4;  // groups of 4 columns of a lane: value (and gate) columns 8u + 4hf ..
    float bias[kHalves][4], scale[kHalves][4], bias_g[2][4], scale_g[2][4];
    // the columns' constants of the tile from column c0 of C's tile on
    auto constants = [&](int c0) __attribute__((always_inline)) {
        if constexpr (kEpi == kFfStore) return;
        if constexpr (F::kI8) {
            auto from = [&](int e, int c, float (&v)[4]) __attribute__((always_inline)) {
                typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
                const f32x4 d = *(const lds_f32x4*)(constant + e * kCols + c);
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] = d[q];
            };
#pragma unroll
            for (int u = 0; u < kHalves; ++u) {
                const int c = c0 + 8 * u + 4 * hf;
                from(0, c, scale[u]);
                from(1, c, bias[u]);
                if constexpr (kGated) {
                    from(2, c, scale_g[u]);
                    from(3, c, bias_g[u]);
                }
            }
            return;
        }
        const int64_t first = kGated ? value_row : 0;
        const auto b = vector_window(p.bias, first + j0, 2), sc = vector_window(p.j_scale, first + j0, 4);
        const auto bg = vector_window(p.bias, gate_row + j0, 2), sg = vector_window(p.j_scale, gate_row + j0, 4);
#pragma unroll
        for (int u = 0; u < kHalves; ++u) {
            const int c = c0 + 8 * u + 4 * hf;
            load4(b, 0, c, bias[u]);
            if constexpr (kGated) load4(bg, 0, c, bias_g[u]);
            if (p.j_scale != nullptr) {
                load4f(sc, c, scale[u]);
                if constexpr (kGated) load4f(sg, c, scale_g[u]);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    scale[u][q] = 1.0f;
                    if constexpr (kGated) scale_g[u][q] = 1.0f;
                }
            }
        }
    };
    // one 32 x 32 tile of sums: the lane's row of C's tile, first column c0, what read_tile gave
    auto finish = [&]<FfFamily kFam>(const Acc& tile_sums, uint32_t row, [[maybe_unused]] float of_row, int c0, const u32x4 (&in)[kSets]) __attribute__((always_inline)) {
        f32x16 z;
        if constexpr (F::kI8) {  // with the row's scale
#pragma unroll
            for (int r = 0; r < 16; ++r) z[r] = (float)tile_sums[r] * of_row;
        } else {
            z = tile_sums;
        }
        if constexpr (kGated) {
            float va[2][4], vb[2][4], d[2][4];
            if constexpr (kEpi == kFfGatedDz) values16(in[0], d);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float v = __builtin_fmaf(z[4 * u + q], scale[u][q], bias[u][q]);
                    const float g = __builtin_fmaf(z[8 + 4 * u + q], scale_g[u][q], bias_g[u][q]);
                    if constexpr (kEpi == kFfGated) {
                        va[u][q] = v * ff_value<kFam>(act, g);
                    } else {
                        float a;
                        const float sl = ff_slope<kFam>(act, g, a);
                        va[u][q] = d[u][q] * a;
                        vb[u][q] = d[u][q] * v * sl;
                    }
                }
            }
            store8(out, out_at, row, c0, va[0], va[1]);
            if constexpr (kEpi == kFfGatedDz) store8(out_g, out_g_at, row, c0, vb[0], vb[1]);
        } else {
            float v[4][4], d[2][2][4] = {};
            if (kEpi == kFfLinearDz || (kEpi == kFfLinear && p.residual != nullptr)) {
                values16(in[0], d[0]);
                values16(in[kSets - 1], d[1]);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float sum = z[4 * u + q];
                    if constexpr (kEpi == kFfStore) {
                        v[u][q] = sum;
                    } else if constexpr (kEpi == kFfLinear) {
                        v[u][q] = ff_value<kFam>(act, __builtin_fmaf(sum, scale[u][q], bias[u][q])) + d[u >> 1][u & 1][q];
                    } else {
                        float a;
                        v[u][q] = ff_slope<kFam>(act, __builtin_fmaf(sum, scale[u][q], bias[u][q]), a) * d[u >> 1][u & 1][q];
                    }
                }
            }
            store8(out, out_at, row, c0, v[0], v[1]);
            store8(out, out_at, row, c0 + 16, v[2], v[3]);
        }
    };
    // a share's sums, 4 columns a lane
    auto store_share = [&](const Acc& z, uint32_t row, int c0) __attribute__((always_inline)) {
        const uint64_t b = (uint64_t)(uintptr_t)p.partial + (uint64_t)(((share * p.rows + i0) * p.ld_partial + j0) * 4);
        const auto r = __builtin_amdgcn_make_buffer_rsrc((void*)(uintptr_t)b, 0, (int)((i_rows * p.ld_partial - j0) * 4), 0x00020000);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int c = c0 + 8 * u + 4 * hf;
            const Acc4 v{z[4 * u], z[4 * u + 1], z[4 * u + 2], z[4 * u + 3]};
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, c < cols ? (uint32_t)(row * p.ld_partial + c) * 4 : kOutside, 0, 0);
        }
    };
    auto epilogue = [&]<FfFamily kFam, bool kShare = false>() __attribute__((always_inline)) {
        if constexpr (kWK == 1) {
#pragma unroll
            for (int t = 0; t < kMJ; ++t) {
                const int c0 = wave_col + (kGated ? 16 : 32) * kWJ * t;
                constants(c0);
#pragma unroll
                for (int s = 0; s < kMI; ++s) {
                    const uint32_t row = wave_row + 32 * kWI * s;
                    if constexpr (kShare) {
                        store_share(acc[t][s], row, c0);
                    } else if constexpr (kAhead) {
                        finish.template operator()<kFam>(acc[t][s], row, row_scale[F::kI8 ? s : 0], c0, ahead[t][s]);
                    } else {
                        u32x4 in[kSets];
                        if constexpr (kReads) read_tile(row, c0, in);
                        finish.template operator()<kFam>(acc[t][s], row, row_scale[F::kI8 ? s : 0], c0, in);
                    }
                }
            }
        } else {
            // The depth shares' sums meet in LDS, kWK tiles a round: group wk of the
            // waves finishes tile kWK r + wk of round r, adding the shares in their order.
            char* mine = smem + (wi + kWI * wj) * (kWK * (kWK - 1) * 4096) + lane * 16;
            auto slot = [&](int owner, int from) __attribute__((always_inline)) {
                return mine + (owner * (kWK - 1) + (from < owner ? from : from - 1)) * 4096;
            };
            constexpr int kTiles = kMI * kMJ;
#pragma unroll
            for (int r = 0; r < (kTiles + kWK - 1) / kWK; ++r) {
                land.template operator()<0>();  // the stage buffers, or the last round's sums, are free
                Acc own{};
#pragma unroll
                for (int o = 0; o < kWK; ++o) {
                    const int q = r * kWK + o;
                    if (q >= kTiles) continue;
                    if (o == wk) {
                        own = acc[q / kMI][q % kMI];
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            *(lds_acc4*)(slot(o, wk) + e * 1024) = Acc4{acc[q / kMI][q % kMI][4 * e], acc[q / kMI][q % kMI][4 * e + 1],
                                                                         acc[q / kMI][q % kMI][4 * e + 2], acc[q / kMI][q % kMI][4 * e + 3]};
                    }
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                const int q = r * kWK + wk;
                if (q < kTiles) {
                    Acc sum{};
#pragma unroll
                    for (int from = 0; from < kWK; ++from) {
                        Acc part = own;
                        if (from != wk) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const Acc4 v = *(const lds_acc4*)(slot(wk, from) + e * 1024);
#pragma unroll
                                for (int x = 0; x < 4; ++x) part[4 * e + x] = v[x];
                            }
                        }
#pragma unroll
                        for (int x = 0; x < 16; ++x) sum[x] += part[x];
                    }
                    const int c0 = wave_col + (kGated ? 16 : 32) * kWJ * (q / kMI);
                    constants(c0);
                    const uint32_t row = wave_row + 32 * kWI * (q % kMI);
                    if constexpr (kShare) {
                        store_share(sum, row, c0);
                    } else {
                        u32x4 in[kSets];
                        if constexpr (kReads) read_tile(row, c0, in);
                        finish.template operator()<kFam>(sum, row, row_scale[F::kI8 ? q % kMI : 0], c0, in);
                    }
                }
            }
        }
        if constexpr (kEpi == kFfLinearDz || kEpi == kFfGatedDz) {
            if (wk == 0)
#pragma unroll
                for (int s = 0; s < kMI; ++s) zero_pad(wave_row + 32 * kWI * s, kGated ? 2 * p.cols : p.cols);
        }
    };
    if constexpr (kEpi == kFfStore) {
        if (kSplit && p.splits > 1) epilogue.template operator()<kFamLinear, kSplit>();
        else epilogue.template operator()<kFamLinear>();
        if constexpr (kIT) {
            const bool tile_sums = p.row_sums != nullptr && j0 == 0;
            if constexpr (kWK > 1) {
                if (tile_sums) {
                    land.template operator()<0>();
                    float* part = (float*)smem + lane;  // [kMI][kWI][kWK][64]
                    if (wj == 0)
#pragma unroll
                        for (int s = 0; s < kMI; ++s) *(lds_float*)(part + 64 * (kWK * (kWI * s + wi) + wk)) = sums[s];
                    land.template operator()<0>();
#pragma unroll
                    for (int s = 0; s < kMI; ++s) {
                        sums[s] = 0.0f;
#pragma unroll
                        for (int w = 0; w < kWK; ++w) sums[s] += *(const lds_float*)(part + 64 * (kWK * (kWI * s + wi) + w));
                    }
                }
            }
            if (with_sums && wk == 0) {
#pragma unroll
                for (int s = 0; s < kMI; ++s) {
                    const int64_t i = i0 + 32 * (kWI * s + wi) + col;
                    const float v = sums[s] + __shfl_xor(sums[s], 32);
                    if (hf == 0 && i < p.rows) {
                        if (kSplit && p.splits > 1) p.partial[(p.splits * p.ld_partial + share) * p.rows + i] = v;
                        else ((Out*)p.row_sums)[i] = (Out)v;
                    }
                }
            }
        }
    } else {
        ff_with_family(p.activation, epilogue);
    }
}

template <typename T, bool kIT, bool kJT, bool kJFp8, typename Tile, FfEpilogue kEpi>
__global__ __launch_bounds__(64 * Tile::kWaves, Tile::waves_per_simd(kJFp8)) void ff_tile_kernel(FfParams p) {
    __shared__ __attribute__((aligned(1024))) char smem[Tile::smem_bytes(kJFp8) + Tile::constant_bytes(FfType<T>::kI8)];
    ff_tile<T, kIT, kJT, kJFp8, Tile, kEpi>(p, blockIdx.x, smem);
}

// Rows that 16-byte accesses do not divide.
template <typename T, bool kIT, bool kJT, bool kJFp8, typename Tile, FfEpilogue kEpi>
__global__ __launch_bounds__(64 * Tile::kWaves, Tile::kMI * Tile::kMJ > 1 ? 2 : 4) void ff_staged_kernel(FfParams p) {
    __shared__ __attribute__((aligned(1024))) char smem[Tile::smem_bytes(kJFp8) + Tile::constant_bytes(FfType<T>::kI8)];
    ff_tile<T, kIT, kJT, kJFp8, Tile, kEpi, kEpi == kFfStore, true>(p, blockIdx.x, smem);
}

// dw and dx in one launch, one workgroup per CU at a time: the tasks of the
// product with the longer ones first, so that the shorter ones fill the CUs
// that the last round of the longer ones leaves idle.
template <typename T, typename TileW, typename TileX>
__global__ __launch_bounds__(512, 2) void ff_pair_kernel(FfParams w, FfParams x, int w_first) {
    static_assert(TileW::kWaves == 8 && TileX::kWaves == 8, "waves");
    constexpr int kW = TileW::smem_bytes(false), kX = TileX::smem_bytes(false);
    __shared__ __attribute__((aligned(1024))) char smem[kW > kX ? kW : kX];
    const int w_tasks = w.i_blocks * w.j_blocks * w.splits, x_tasks = x.i_blocks * x.j_blocks * x.splits;
    const int id = blockIdx.x;
    if (w_first ? id < w_tasks : id >= x_tasks) ff_tile<T, true, true, false, TileW, kFfStore, true>(w, w_first ? id : id - x_tasks, smem);
    else ff_tile<T, false, true, false, TileX, kFfStore, true>(x, w_first ? id - w_tasks : id, smem);
}

// Tiles of C and the tasks' groups.
template <typename Tile>
void ff_blocks(FfParams& p, bool gated) {
    const int cols = Tile::kBJ / (gated ? 2 : 1);
    p.i_blocks = (int32_t)((p.rows + Tile::kBI - 1) / Tile::kBI);
    p.j_blocks = (int32_t)((p.cols + cols - 1) / cols);
    p.group_i = p.i_blocks < 8 ? p.i_blocks : 8;
}

template <typename T, bool kIT, bool kJT, bool kJFp8, typename Tile, FfEpilogue kEpi>
hipError_t ff_launch(FfParams p, hipStream_t stream) {
    ff_blocks<Tile>(p, kEpi == kFfGated || kEpi == kFfGatedDz);
    hipLaunchKernelGGL((ff_tile_kernel<T, kIT, kJT, kJFp8, Tile, kEpi>), dim3((unsigned)((int64_t)p.i_blocks * p.j_blocks)),
                       dim3(64 * Tile::kWaves), 0, stream, p);
    return hipGetLastError();
}

template <typename T, bool kIT, bool kJT, bool kJFp8, typename Tile, FfEpilogue kEpi>
hipError_t ff_launch_staged(FfParams p, hipStream_t stream) {
    ff_blocks<Tile>(p, kEpi == kFfGated || kEpi == kFfGatedDz);
    hipLaunchKernelGGL((ff_staged_kernel<T, kIT, kJT, kJFp8, Tile, kEpi>), dim3((unsigned)((int64_t)p.i_blocks * p.j_blocks * p.splits)),
                       dim3(64 * Tile::kWaves), 0, stream, p);
    return hipGetLastError();
}

template <typename T, typename TileW, typename TileX>
hipError_t ff_launch_pair(FfParams w, FfParams x, bool w_first, hipStream_t stream) {
    ff_blocks<TileW>(w, false);
    ff_blocks<TileX>(x, false);
    hipLaunchKernelGGL((ff_pair_kernel<T, TileW, TileX>),
                       dim3((unsigned)(w.i_blocks * w.j_blocks * w.splits + x.i_blocks * x.j_blocks * x.splits)), dim3(512), 0, stream, w, x,
                       w_first ? 1 : 0);
    return hipGetLastError();
}

// The tiles that the launcher chooses from (feed_forward.hip), and their products by direction.
typedef FfTile<4, 2, 1, 2, 5, 2, 2> FfTile256x320;
typedef FfTile<4, 2, 1, 2, 4, 2, 2> FfTile256x256;
typedef FfTile<4, 2, 1, 2, 3, 2, 2> FfTile256x192;  // 8-bit integers alone
typedef FfTile<2, 4, 1, 2, 2, 3, 2> FfTile128x256;
typedef FfTile<4, 2, 1, 1, 3, 3, 2> FfTile128x192;
typedef FfTile<2, 2, 2, 2, 2, 4, 2> FfTile128x128;
typedef FfTile<2, 2, 1, 1, 2, 3, 3> FfTile64x128;
typedef FfTile<2, 2, 1, 1, 1, 4, 4> FfTile64x64;

template <typename T, typename Tile>
hipError_t ff_forward_tile(const FfParams& p, FfEpilogue epilogue, bool j_fp8, hipStream_t stream) {
    if constexpr (Tile::kWK == 1) {
        if (j_fp8)
            return epilogue == kFfGated ? ff_launch<T, false, false, true, Tile, kFfGated>(p, stream)
                                        : ff_launch<T, false, false, true, Tile, kFfLinear>(p, stream);
    }
    return j_fp8 ? hipErrorInvalidValue
           : epilogue == kFfGated ? ff_launch<T, false, false, false, Tile, kFfGated>(p, stream)
                                  : ff_launch<T, false, false, false, Tile, kFfLinear>(p, stream);
}

template <typename T, typename Tile>
hipError_t ff_backward_tile(const FfParams& p, FfEpilogue epilogue, bool i_transposed, hipStream_t stream) {
    if (epilogue == kFfGatedDz) return ff_launch<T, false, false, false, Tile, kFfGatedDz>(p, stream);
    if (epilogue == kFfLinearDz) return ff_launch<T, false, false, false, Tile, kFfLinearDz>(p, stream);
    return i_transposed ? ff_launch<T, true, true, false, Tile, kFfStore>(p, stream)
                        : ff_launch<T, false, true, false, Tile, kFfStore>(p, stream);
}

template <typename T, typename TileW>
hipError_t ff_pair_tile(const FfParams& w, const FfParams& x, int x_tile, bool w_first, hipStream_t stream) {
    return x_tile == kFf256x256   ? ff_launch_pair<T, TileW, FfTile256x256>(w, x, w_first, stream)
           : x_tile == kFf128x256 ? ff_launch_pair<T, TileW, FfTile128x256>(w, x, w_first, stream)
           : x_tile == kFf128x128 ? ff_launch_pair<T, TileW, FfTile128x128>(w, x, w_first, stream)
                                  : hipErrorInvalidValue;
}

template <typename T>
hipError_t ff_pair(const FfParams& w, const FfParams& x, int w_tile, int x_tile, bool w_first, hipStream_t stream) {
    return w_tile == kFf256x256   ? ff_pair_tile<T, FfTile256x256>(w, x, x_tile, w_first, stream)
           : w_tile == kFf128x256 ? ff_pair_tile<T, FfTile128x256>(w, x, x_tile, w_first, stream)
           : w_tile == kFf128x128 ? ff_pair_tile<T, FfTile128x128>(w, x, x_tile, w_first, stream)
                                  : hipErrorInvalidValue;
}

template <typename T>
hipError_t ff_forward(const FfParams& p, FfEpilogue epilogue, bool j_fp8, int tile, hipStream_t stream) {
    switch (tile) {
    case kFf256x320: return ff_forward_tile<T, FfTile256x320>(p, epilogue, j_fp8, stream);
    case kFf256x256: return ff_forward_tile<T, FfTile256x256>(p, epilogue, j_fp8, stream);
    case kFf128x256: return ff_forward_tile<T, FfTile128x256>(p, epilogue, j_fp8, stream);
    case kFf128x192: return ff_forward_tile<T, FfTile128x192>(p, epilogue, j_fp8, stream);
    case kFf128x128: return ff_forward_tile<T, FfTile128x128>(p, epilogue, j_fp8, stream);
    case kFf64x128: return ff_forward_tile<T, FfTile64x128>(p, epilogue, j_fp8, stream);
    case kFf64x64: return ff_forward_tile<T, FfTile64x64>(p, epilogue, j_fp8, stream);
    }
    return hipErrorInvalidValue;
}

// Projections of 8-bit integers, on tiles and through registers (below).
template <typename T>
hipError_t ff_i8_forward(const FfParams& p, FfEpilogue epilogue, int tile, hipStream_t stream) {
    const bool gated = epilogue == kFfGated;
    auto by_tile = [&]<typename Tile>() {
        return gated ? ff_launch<I8<T>, false, false, false, Tile, kFfGated>(p, stream)
                     : ff_launch<I8<T>, false, false, false, Tile, kFfLinear>(p, stream);
    };
    switch (tile) {
    case kFf256x320: return by_tile.template operator()<FfTile256x320>();
    case kFf256x256: return by_tile.template operator()<FfTile256x256>();
    case kFf256x192: return by_tile.template operator()<FfTile256x192>();
    case kFf128x256: return by_tile.template operator()<FfTile128x256>();
    case kFf128x192: return by_tile.template operator()<FfTile128x192>();
    case kFf128x128: return by_tile.template operator()<FfTile128x128>();
    case kFf64x128: return by_tile.template operator()<FfTile64x128>();
    case kFf64x64: return by_tile.template operator()<FfTile64x64>();
    }
    return hipErrorInvalidValue;
}

template <typename T>
hipError_t ff_backward(const FfParams& p, FfEpilogue epilogue, bool i_transposed, int tile, hipStream_t stream) {
    switch (tile) {
    case kFf256x320: return ff_backward_tile<T, FfTile256x320>(p, epilogue, i_transposed, stream);
    case kFf256x256: return ff_backward_tile<T, FfTile256x256>(p, epilogue, i_transposed, stream);
    case kFf128x256: return ff_backward_tile<T, FfTile128x256>(p, epilogue, i_transposed, stream);
    case kFf128x192: return ff_backward_tile<T, FfTile128x192>(p, epilogue, i_transposed, stream);
    case kFf128x128: return ff_backward_tile<T, FfTile128x128>(p, epilogue, i_transposed, stream);
    case kFf64x128: return ff_backward_tile<T, FfTile64x128>(p, epilogue, i_transposed, stream);
    case kFf64x64: return ff_backward_tile<T, FfTile64x64>(p, epilogue, i_transposed, stream);
    }
    return hipErrorInvalidValue;
}

// The tiles of rows that come through registers.
typedef FfTile<2, 2, 1, 2, 2, 2, 1> FfStaged128x128;
typedef FfTile<2, 2, 1, 1, 1, 2, 1> FfStaged64x64;

template <typename T, typename Tile>
hipError_t ff_staged_tile(const FfParams& p, FfEpilogue epilogue, bool i_transposed, bool j_fp8, hipStream_t stream) {
    switch (epilogue) {
    case kFfLinear:
        return j_fp8 ? ff_launch_staged<T, false, false, true, Tile, kFfLinear>(p, stream)
                     : ff_launch_staged<T, false, false, false, Tile, kFfLinear>(p, stream);
    case kFfGated:
        return j_fp8 ? ff_launch_staged<T, false, false, true, Tile, kFfGated>(p, stream)
                     : ff_launch_staged<T, false, false, false, Tile, kFfGated>(p, stream);
    case kFfLinearDz: return ff_launch_staged<T, false, false, false, Tile, kFfLinearDz>(p, stream);
    case kFfGatedDz: return ff_launch_staged<T, false, false, false, Tile, kFfGatedDz>(p, stream);
    case kFfStore:
        return i_transposed ? ff_launch_staged<T, true, true, false, Tile, kFfStore>(p, stream)
                            : ff_launch_staged<T, false, true, false, Tile, kFfStore>(p, stream);
    }
    return hipErrorInvalidValue;
}

template <typename T>
hipError_t ff_staged(const FfParams& p, FfEpilogue epilogue, bool i_transposed, bool j_fp8, bool large, hipStream_t stream) {
    return large ? ff_staged_tile<T, FfStaged128x128>(p, epilogue, i_transposed, j_fp8, stream)
                 : ff_staged_tile<T, FfStaged64x64>(p, epilogue, i_transposed, j_fp8, stream);
}

template <typename T>
hipError_t ff_i8_staged(const FfParams& p, FfEpilogue epilogue, bool large, hipStream_t stream) {
    const bool gated = epilogue == kFfGated;
    auto by_tile = [&]<typename Tile>() {
        return gated ? ff_launch_staged<I8<T>, false, false, false, Tile, kFfGated>(p, stream)
                     : ff_launch_staged<I8<T>, false, false, false, Tile, kFfLinear>(p, stream);
    };
    return large ? by_tile.template operator()<FfStaged128x128>() : by_tile.template operator()<FfStaged64x64>();
}

}  // namespace
}  // namespace sdxl_hip
