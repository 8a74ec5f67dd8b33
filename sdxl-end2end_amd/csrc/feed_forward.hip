// Which kernel and tile a product of the feed-forward operators runs on whose
// rows have 16 bytes (feed_forward_tiles.hpp, feed_forward_deep.hip), and what goes
// with the gradients: shares of a depth, their joining pass, row sums alone.
#include <hip/hip_runtime.h>

#include "feed_forward_device.hpp"
#include "feed_forward_kernels.hpp"

namespace sdxl_hip {

hipError_t ff_forward_f16(const FfParams& p, FfEpilogue epilogue, bool j_fp8, int tile, hipStream_t stream);
hipError_t ff_forward_bf16(const FfParams& p, FfEpilogue epilogue, bool j_fp8, int tile, hipStream_t stream);
hipError_t ff_backward_f16(const FfParams& p, FfEpilogue epilogue, bool i_transposed, int tile, hipStream_t stream);
hipError_t ff_backward_bf16(const FfParams& p, FfEpilogue epilogue, bool i_transposed, int tile, hipStream_t stream);
hipError_t ff_pair_f16(const FfParams& w, const FfParams& x, int w_tile, int x_tile, bool w_first, hipStream_t stream);
hipError_t ff_pair_bf16(const FfParams& w, const FfParams& x, int w_tile, int x_tile, bool w_first, hipStream_t stream);
hipError_t ff_staged_f16(const FfParams& p, FfEpilogue epilogue, bool i_transposed, bool j_fp8, bool large, hipStream_t stream);
hipError_t ff_staged_bf16(const FfParams& p, FfEpilogue epilogue, bool i_transposed, bool j_fp8, bool large, hipStream_t stream);
hipError_t ff_i8_forward_f16(const FfParams& p, FfEpilogue epilogue, int tile, hipStream_t stream);
hipError_t ff_i8_forward_bf16(const FfParams& p, FfEpilogue epilogue, int tile, hipStream_t stream);
hipError_t ff_i8_staged_f16(const FfParams& p, FfEpilogue epilogue, bool large, hipStream_t stream);
hipError_t ff_i8_staged_bf16(const FfParams& p, FfEpilogue epilogue, bool large, hipStream_t stream);
hipError_t ff_deep(const FfParams& p, FfEpilogue epilogue, bool bf16, bool j_fp8, bool staged, FfDeepId id, hipStream_t stream);

namespace {

bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// Time of a product on a tile, in microseconds: rounds of tiles over the CUs,
// each of so many 64-deep stages and a start and end (first stage, epilogue).
// `alone` is a stage's time of the one tile that a CU holds, `pair` that of two
// tiles that share a CU (0: LDS holds one). Measured on an MI355X in bf16,
// products of 160, 128 and 32 stages on 40 to 2752 tiles:
//   256 x 320  dx [8192, 1280] deep 10240 234 us, [2048, 10240] deep 1280 gated 51
//   256 x 256  dx 200, dw [10240, 1280] deep 8192 178 (1200 TFLOP/s), gated 71
//   128 x 256  dw [5120, 1280] deep 2464 39 (256 x 256: 55, 128 x 128: 48)
//   128 x 192  [8192, 640] deep 2560 39 (128 x 256: 42), [512, 10240] deep 1280 gated 21 (128 x 256: 23, 128 x 128: 32)
//   128 x 128  dx [2048, 1280] deep 10240 69 (256 x 256: 207, 128 x 256: 116)
//    64 x 128  dw [640, 2560] deep 8192 51 (128 x 128: 56, 128 x 256: 95)
//    64 x  64  [154, 5120] deep 1280 10 (128 x 128: 15, 256 x 256: 32)
// The constants have no terms for bytes, caches or power and one end for every epilogue: they rank tiles, and miss the
// times of whole chips by up to a fifth (gated [8192, 2048] -> 2 x 5456 316 for 340, [8192, 2560] -> 640 31 for 36).
struct TileCost {
    int rows, cols;
    float alone, pair, ends;
};
constexpr TileCost kTiles[kFfTiles] = {{256, 320, 1.60f, 0.0f, 15.0f}, {256, 256, 1.32f, 0.0f, 10.5f},
                                       {128, 256, 0.76f, 0.0f, 7.2f},  {128, 192, 0.62f, 0.0f, 6.5f},
                                       {128, 128, 0.45f, 0.0f, 5.5f},
                                       {64, 128, 0.35f, 0.58f, 5.0f},  {64, 64, 0.30f, 0.46f, 4.5f}};

// The same of 8-bit integers, by stages of 128, and a tile more: their stages take the same bytes and nearly the same time for
// twice the products, so that starts and ends (a conversion and a scale more for every sum) weigh more. Measured in fp16 out:
//   256 x 320  gated [2048, 1280] -> 2 x 5120 32 us (256 x 256: 45, 128 x 256: 42)
//   256 x 256  gated [8192, 2048] -> 2 x 5456 195 (1.88 POP/s), [16384, 2048] x [2048, 2048] 76-80
//   256 x 192  [8192, 5120] x [1280, 5120] 66 (256 x 256: 72, 128 x 192: 73)
//   128 x 256  [2048, 1280] x [3840, 1280] 19 (256 x 256: 25)
//   128 x 192  [8192, 640] x [640, 640] 11.9 (128 x 256: 13.7, 64 x 128: 14.5), [4096, 2560] x [1280, 2560] 23.5 (25.2, 30.2)
//   128 x 128  [2048, 5120] x [1280, 5120] 26.7 (64 x 128: 28.6, 128 x 192: 31.9)
//    64 x 128  [4940, 640] x [640, 640] 9.2 (128 x 128: 10.4)
//    64 x  64  [154, 1280] x [5120, 1280] 7.7 (32 x 32, shared depth: 10.1)
// On a whole chip the matrix cores' power holds the long products back, the library's too (8192 cubed 1.97 POP/s).
constexpr TileCost kI8Tiles[kFfI8Tiles] = {{256, 320, 1.65f, 0.0f, 16.5f}, {256, 256, 1.47f, 0.0f, 11.8f},
                                           {128, 256, 0.69f, 0.0f, 10.2f}, {128, 192, 0.55f, 0.0f, 9.0f},
                                           {128, 128, 0.44f, 0.0f, 8.3f},
                                           {64, 128, 0.39f, 0.55f, 6.5f},  {64, 64, 0.33f, 0.49f, 4.4f},
                                           {256, 192, 1.05f, 0.0f, 11.3f}};

// Time of two kinds of tasks, a tasks of a_time each before b of b_time, on CUs that take the next task when
// they are free: the CUs as groups that become free together.
float list_time(int64_t a, float a_time, int64_t b, float b_time, int64_t cus) {
    // after the a tasks: `late` CUs free at a_end, the others one a_time earlier
    const int64_t rounds = a / cus, late = a % cus;
    float early_at = (float)rounds * a_time, late_at = early_at + a_time;
    if (b == 0) return late > 0 ? late_at : early_at;
    // b tasks go round by round to whichever group is free first; a group moves as one
    int64_t early_cus = cus - late, late_cus = late;
    float end = late > 0 ? late_at : early_at;
    while (b > 0) {
        const bool to_early = late_cus == 0 || (early_cus > 0 && early_at <= late_at);
        float& at = to_early ? early_at : late_at;
        const int64_t n = to_early ? early_cus : late_cus;
        // as many rounds at once as stay ahead of the other group
        int64_t times = 1;
        if (early_cus > 0 && late_cus > 0) {
            const float gap = (to_early ? late_at : early_at) - at;
            times = gap > b_time ? (int64_t)(gap / b_time) : 1;
        } else {
            times = (b + n - 1) / n;
        }
        const int64_t needed = (b + n - 1) / n;
        if (times > needed) times = needed;
        at += (float)times * b_time;
        b -= times * n;
        if (at > end) end = at;
    }
    return end;
}

// The same for the tiles whose waves share the depth (feed_forward_deep.hip), by 64-deep blocks: 32 x 32 with eight
// waves where every CU has at most one, else with four and two tiles a CU, or 64 x 64 with four. Measured in bf16, us
// (the best tile with barriers behind): [248, 8192] x [2048, 8192] 26 on 32 x 32, 31 on 64 x 64 (47); gated the same,
// 256 tiles of 64 x 64, 48 and 33 (48); [462, 5120] x [1280, 5120] 26 and 23 (32); [2048, 1280] x [1280, 1280] 37 and
// 34 (19); gated [8192, 64] -> 2 x 5120, 160 rounds of 32 x 32, 420 (58). Staged rows: [617, 3411] x [1280, 3411] 49 and
// 43 (55), [136, 5458] x [2048, 5458] 36 and 61.
FfDeepId deep_choice(const FfParams& p, FfEpilogue epilogue, int64_t cus, bool staged, float& time) {
    const int64_t cols = epilogue == kFfGated || epilogue == kFfGatedDz ? 2 * p.cols : p.cols;
    const int64_t small = ((p.rows + 31) / 32) * ((cols + 31) / 32), large = ((p.rows + 63) / 64) * ((cols + 63) / 64);
    const float blocks = (float)ff_stages(p), rounds = (float)small / (float)(2 * cus);
    FfDeepId id = kFfDeep32x4;
    if (small <= cus) {
        id = kFfDeep32x8;
        time = staged ? 5.0f + 0.19f * blocks : 3.0f + 0.095f * blocks;
    } else if (rounds <= 1.0f) {
        time = 3.0f + (staged ? 0.6f : 0.19f) * blocks;
    } else {
        time = 3.0f + (staged ? 0.6f : 0.24f) * rounds * blocks + 2.2f * (rounds - 1.0f);
    }
    const float large_time = (float)((large + cus - 1) / cus) * (7.0f + (staged ? 0.65f : 0.19f) * blocks);
    if (large_time < time) {
        id = kFfDeep64x4;
        time = large_time;
    }
    if (p.i8 != 0) time += 2.0f;
    return id;
}

int choose_tile(const FfParams& p, FfEpilogue epilogue, bool j_fp8, int64_t cus, float& best_time) {
    const int64_t cols = epilogue == kFfGated || epilogue == kFfGatedDz ? 2 * p.cols : p.cols;
    const float stages = (float)ff_stages(p);
    int best = 0;
    for (int t = 0; t < (p.i8 != 0 ? (int)kFfI8Tiles : (int)kFfTiles); ++t) {
        if (j_fp8 && t == kFf128x128) continue;  // its waves share a stage's depth, E4M3 codes come in pairs of steps
        const TileCost& c = p.i8 != 0 ? kI8Tiles[t] : kTiles[t];
        const int64_t tiles = ((p.rows + c.rows - 1) / c.rows) * ((cols + c.cols - 1) / c.cols);
        float time;
        if (c.pair == 0.0f) {
            time = (float)((tiles + cus - 1) / cus) * (stages * c.alone + c.ends);
        } else {
            const int64_t full = tiles / (2 * cus), rest = tiles % (2 * cus);
            time = (float)full * (stages * c.pair + c.ends);
            if (rest > 0) time += stages * (rest > cus ? c.pair : c.alone) + c.ends;
        }
        if (t == 0 || time < best_time) {
            best = t;
            best_time = time;
        }
    }
    return best;
}

// Fills in what the tiled kernels' launchers leave to the dispatch.
FfParams prepared(const FfParams& params, bool i_transposed) {
    FfParams p = params;
    if (p.i_row == 0) p.i_row = i_transposed ? p.rows : p.depth;
    p.splits = 1;
    p.share_stages = (int32_t)((p.depth + 63) / 64);
    p.ld_partial = (p.cols + 7) / 8 * 8;
    // 16-byte accesses in the epilogue (bias: 8)
    p.vec = p.cols % 8 == 0 && p.ld_out % 8 == 0 && aligned(p.out, 16) && aligned(p.bias, 8) && aligned(p.residual, 16) &&
            aligned(p.dout, 16) && (p.residual == nullptr || p.ld_res % 8 == 0) && (p.dout == nullptr || p.ld_dout % 8 == 0);
    return p;
}

// 128 x 128 tiles where every CU gets one, else 64 x 64: [8192, 2561] x [640, 2561], 320 of the large tiles, 62 us (small: 84);
// [2632, 2567] x [640, 2567], 105, 66 (45); gated [2632, 2567] -> 2 x 640, 210, 68 (64).
bool staged_large(const FfParams& p, int64_t cols, int64_t cus) {
    return ((p.rows + 127) / 128) * ((cols + 127) / 128) >= cus;
}

// Rows through registers on 64 x 64 tiles, microseconds: a stage waits for its reads (0.85; more with over 256 tiles).
// [40, 5127] x [1280, 5127] 72 (32 x 32, shared depth: 20), [600, 645] x [645, 645] 14.2 (10.3), gated [1000, 323] -> 2 x
// 1280 12 (33).
float staged_time(const FfParams& p, int64_t cols) {
    const int64_t tiles = ((p.rows + 63) / 64) * ((cols + 63) / 64);
    return 4.5f + (float)ff_stages(p) * (tiles > 256 ? 0.85f + 0.0012f * (float)(tiles - 256) : 0.85f);
}

// ---- dw and dx in one launch. A side of it: a product on a tile, its depth in so many shares.
constexpr int kPairTiles = 3, kPairTile[kPairTiles] = {kFf256x256, kFf128x256, kFf128x128};
constexpr int kSplitSteps = 4, kMaxSplits = 1 << (kSplitSteps - 1);
constexpr size_t kMaxPartial = 32 << 20;  // partial sums of a call, bytes
// the joining pass: start and microseconds a byte
constexpr float kJoinStart = 3.0f, kJoinPerByte = 0.4e-6f;

struct PairSide {
    int64_t tasks, partial;  // bytes
    float time;              // of a task
};

int share_stages(const FfParams& p, int splits) { return (int)(((p.depth + 63) / 64 + splits - 1) / splits); }

PairSide pair_side(const FfParams& p, int tile, int splits) {
    const TileCost& c = kTiles[tile];
    const int64_t tiles = ((p.rows + c.rows - 1) / c.rows) * ((p.cols + c.cols - 1) / c.cols);
    const int stages = share_stages(p, splits);
    // (no share may be empty, and few stages are not worth a start)
    const bool ok = splits == 1 || (stages >= 8 && (int64_t)stages * 64 * (splits - 1) < p.depth);
    const int64_t sums = splits == 1 ? 0 : splits * p.rows * (p.ld_partial + (p.row_sums != nullptr ? 1 : 0));
    return {ok ? tiles * splits : (int64_t)1 << 30, (sums * 4 + 255) / 256 * 256, (float)stages * c.alone + c.ends - 2.0f};
}

void set_splits(FfParams& p, int splits, float* partial) {
    p.splits = splits;
    p.share_stages = share_stages(p, splits);
    p.partial = partial;
}

FfJoin join_of(const FfParams& p) {
    if (p.splits == 1) return {};
    const int64_t threads = p.rows * (p.ld_partial / 8) + (p.row_sums != nullptr ? p.rows : 0);
    return {p.partial, p.out, p.row_sums, p.ld_out, (int32_t)p.rows, (int32_t)p.cols, (int32_t)p.ld_partial, p.splits, p.vec,
            (int32_t)((threads + 255) / 256)};
}

// Adds the shares in their order, 8 columns a thread (or one row sum), and rounds once. Bound by the reads, which come
// out of the Infinity Cache: 5.7 MB 4.1 us.
template <typename T>
__global__ __launch_bounds__(256) void ff_join_kernel(FfJoin a, FfJoin b) {
    using F = FfType<T>;
    const bool second = (int)blockIdx.x >= a.blocks;
    const FfJoin& p = second ? b : a;
    const uint32_t at = (blockIdx.x - (second ? a.blocks : 0)) * 256 + threadIdx.x;
    const uint32_t chunks = p.ld / 8, all = p.rows * chunks;
    const size_t share = (size_t)p.rows * p.ld;
    if (at < all) {
        float v[8] = {};
        for (int s = 0; s < p.splits; ++s) {
            const f32x4* from = (const f32x4*)(p.partial + s * share + (size_t)at * 8);
            const f32x4 lo = from[0], hi = from[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += lo[e], v[4 + e] += hi[e];
        }
        const int c = (at % chunks) * 8;
        T* out = (T*)p.out + (int64_t)(at / chunks) * p.ld_out + c;
        if (p.vec) {
            *(u32x4*)out = u32x4{F::pack(v[0], v[1]), F::pack(v[2], v[3]), F::pack(v[4], v[5]), F::pack(v[6], v[7])};
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < p.cols) out[e] = (T)v[e];
        }
    } else if (p.row_sums != nullptr && at - all < (uint32_t)p.rows) {
        const float* sums = p.partial + p.splits * share + (at - all);
        float v = 0.0f;
        for (int s = 0; s < p.splits; ++s) v += sums[(size_t)s * p.rows];
        ((T*)p.row_sums)[at - all] = (T)v;
    }
}

// Sums of I's rows alone (a bias gradient without its weights'): I = dz by columns, depth x rows. 8 columns a thread, 4 rows
// of them a workgroup at a time, the depth in shares of `span`; one share writes the sums, more their parts. Bound by
// the read: [8192, 5120] in 32 shares 24 us with the joining pass (316 as a product's by-product on the general kernel).
constexpr int kSumsMaxShares = 32;

template <typename T>
__global__ __launch_bounds__(256) void ff_row_sums_kernel(FfParams p, int64_t span) {
    using F = FfType<T>;
    __shared__ float part[4][64][8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = ((int64_t)blockIdx.x * 64 + lane) * 8, first = (int64_t)blockIdx.y * span;
    const int64_t last = first + span < p.depth ? first + span : p.depth;
    const int n = (int)(p.rows - c < 8 ? p.rows - c : 8);
    float v[8] = {};
    const char* from = (const char*)p.ip + c * 2;
    if (n == 8) {
#pragma unroll 8
        for (int64_t r = first + wave; r < last; r += 4) {
            const u32x4 d = ((const Unaligned<2>*)(from + r * p.ld_i * 2))->v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[2 * e] += F::lo(d[e]), v[2 * e + 1] += F::hi(d[e]);
        }
    } else {
        for (int64_t r = first + wave; r < last; r += 4)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < n) v[e] += (float)((const T*)(from + r * p.ld_i * 2))[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) part[wave][lane][e] = v[e];
    __syncthreads();
    for (int at = threadIdx.x; at < 512; at += 256) {
        const int64_t i = (int64_t)blockIdx.x * 512 + at;
        if (i >= p.rows) continue;
        const float* x = &part[0][0][0] + at;
        const float sum = (x[0] + x[512]) + (x[1024] + x[1536]);
        if (gridDim.y > 1) p.partial[blockIdx.y * p.rows + i] = sum;
        else ((T*)p.row_sums)[i] = (T)sum;
    }
}

}  // namespace

bool ff_staged_supported(const FfParams& p, FfEpilogue epilogue, bool i_transposed, bool j_transposed, bool j_fp8) {
    if (p.depth <= 0 || (epilogue == kFfStore && !j_transposed)) return false;
    // rows of 16 bytes or more: a row's last chunk is read as its last 16 bytes
    if (p.i8 != 0) j_fp8 = true;  // (both operands in bytes)
    if ((i_transposed ? p.rows : p.depth) < (p.i8 != 0 ? 16 : 8) || (j_transposed ? p.cols : p.depth) < (j_fp8 ? 16 : 8)) return false;
    // a window (at most 320 rows) stays below 2^31 bytes, the threads of a launch below 2^32
    if (p.ld_i > (1 << 20) || p.ld_j > (1 << 20) || p.ld_out > (1 << 20) || p.ld_dout > (1 << 20) || p.ld_res > (1 << 20))
        return false;
    return ((p.rows + 63) / 64) * ((p.cols + 31) / 32) <= (1 << 23);
}

namespace {

bool ff_tiled_supported(const FfParams& p, FfEpilogue epilogue, bool i_transposed, bool j_transposed, bool j_fp8) {
    if (!ff_staged_supported(p, epilogue, i_transposed, j_transposed, j_fp8)) return false;
    // rows in whole 16-byte chunks: the depth, or the columns of an operand that is read by columns
    const int64_t i_row = p.i_row != 0 ? p.i_row : i_transposed ? p.rows : p.depth;
    if (p.i8 != 0)  // (tokens are quantised on the way)
        return aligned(p.jp, 16) && p.ld_j % 16 == 0 && p.depth % 16 == 0 && (p.i8 == kFfI8Tokens || (aligned(p.ip, 16) && p.ld_i % 16 == 0));
    if (!aligned(p.ip, 16) || !aligned(p.jp, 16) || p.ld_i % 8 != 0 || p.ld_j % (j_fp8 ? 16 : 8) != 0) return false;
    return i_row % 8 == 0 && (j_transposed ? p.cols % 8 == 0 : p.depth % (j_fp8 ? 16 : 8) == 0);
}

int64_t units(int compute_units) { return compute_units > 0 ? compute_units : 256; }

}  // namespace

FfChoice choose_ff(const FfParams& p, FfEpilogue epilogue, bool j_fp8, int compute_units) {
    if (!ff_staged_supported(p, epilogue, false, false, j_fp8)) return {FfKernel::kGeneral, 0, false};
    const bool staged = !ff_tiled_supported(p, epilogue, false, false, j_fp8);
    if (ff_rows_supported(p, epilogue, j_fp8)) return {FfKernel::kRows, ff_rows_waves(p, epilogue == kFfGated), staged};
    const int64_t cus = units(compute_units);
    const int64_t cols = epilogue == kFfGated || epilogue == kFfGatedDz ? 2 * p.cols : p.cols;
    float deep_time, time = 0.0f;
    const FfDeepId deep = deep_choice(p, epilogue, cus, staged, deep_time);
    if (staged) {
        const bool large = staged_large(p, cols, cus);
        if (!large && deep_time < staged_time(p, cols)) return {FfKernel::kDeep, deep, true};
        return {FfKernel::kStaged, large ? 128 : 64, true};
    }
    const int tile = choose_tile(p, epilogue, j_fp8, cus, time);
    if (deep_time < time) return {FfKernel::kDeep, deep, false};
    return {FfKernel::kTile, tile, false};
}

hipError_t launch_ff(const FfChoice& choice, const FfParams& params, FfEpilogue epilogue, bool bf16, bool j_fp8, hipStream_t stream) {
    const FfParams p = prepared(params, false);
    switch (choice.kernel) {
    case FfKernel::kGeneral: return launch_ff_general(params, epilogue, false, false, bf16, j_fp8, stream);
    case FfKernel::kRows: return launch_ff_rows(params, epilogue, choice.variant, choice.staged, bf16, j_fp8, stream);
    case FfKernel::kDeep: return ff_deep(p, epilogue, bf16, j_fp8, choice.staged, (FfDeepId)choice.variant, stream);
    case FfKernel::kStaged:
        if (p.i8 != 0) return (bf16 ? ff_i8_staged_bf16 : ff_i8_staged_f16)(p, epilogue, choice.variant == 128, stream);
        return (bf16 ? ff_staged_bf16 : ff_staged_f16)(p, epilogue, false, j_fp8, choice.variant == 128, stream);
    case FfKernel::kTile: break;
    }
    if (p.i8 != 0) return (bf16 ? ff_i8_forward_bf16 : ff_i8_forward_f16)(p, epilogue, choice.variant, stream);
    if (epilogue == kFfLinear || epilogue == kFfGated)
        return (bf16 ? ff_forward_bf16 : ff_forward_f16)(p, epilogue, j_fp8, choice.variant, stream);
    return (bf16 ? ff_backward_bf16 : ff_backward_f16)(p, epilogue, false, choice.variant, stream);
}

size_t ff_partial_bytes(int64_t m, int64_t features, int64_t k) {
    const double all = 4.0 * kMaxSplits * ((double)m * (double)k + (double)features * (double)(k + 1)) + 1024.0;
    return m <= 0 || features <= 0 || k <= 0 ? 0 : all < (double)kMaxPartial ? ((size_t)all + 255) / 256 * 256 : kMaxPartial;
}

namespace {

hipError_t launch_join(const FfParams& w, const FfParams& x, bool bf16, hipStream_t stream) {
    if (w.splits == 1 && x.splits == 1) return hipSuccess;
    const FfJoin jw = join_of(w), jx = join_of(x);
    const dim3 grid((unsigned)(jw.blocks + jx.blocks));
    if (bf16) hipLaunchKernelGGL(ff_join_kernel<__bf16>, grid, dim3(256), 0, stream, jw, jx);
    else hipLaunchKernelGGL(ff_join_kernel<_Float16>, grid, dim3(256), 0, stream, jw, jx);
    return hipGetLastError();
}

// dw and dx on the tiled kernel, or one of them (the other's pointer null).
void choose_pair(const FfParams* dw, const FfParams* dx, size_t partial_bytes, int64_t cus, FfGradients& plan) {
    FfParams w{}, x{};  // (no rows: no tasks)
    // apart, or together on the best pair of tiles that take a CU each, of whole depths or of shares of them.
    // Measured on an MI355X, dw and dx of x [m, k], w [f, k]: m 2048, k 1280, f 10240 apart 142 us, together 117;
    // m 8192 apart 459, together 368; m 1111, k 640, f 5120 together 42 (105 tasks for 256 CUs), with dx's depth in 2
    // shares 28.6 and 4 for the joining pass; dx alone of m 154, k 1280, f 5120 whole 31, in shares 18.
    float best = 0.0f, apart;
    if (dw != nullptr) {
        w = prepared(*dw, true);
        plan.w.choice = {FfKernel::kTile, choose_tile(w, kFfStore, false, cus, apart), false};
        best += apart;
    }
    if (dx != nullptr) {
        x = prepared(*dx, false);
        plan.x.choice = {FfKernel::kTile, choose_tile(x, kFfStore, false, cus, apart), false};
        best += apart;
    }
    PairSide sides[2][kPairTiles][kSplitSteps];
    for (int side = 0; side < 2; ++side)
        for (int t = 0; t < kPairTiles; ++t)
            for (int s = 0; s < kSplitSteps; ++s) sides[side][t][s] = pair_side(side == 0 ? w : x, kPairTile[t], 1 << s);
    for (int i = 0; i < kPairTiles * kSplitSteps * kPairTiles * kSplitSteps; ++i) {
        const int tw = i / (kSplitSteps * kPairTiles * kSplitSteps), tx = i / kSplitSteps % kPairTiles;
        const int sw = i / (kPairTiles * kSplitSteps) % kSplitSteps, sx = i % kSplitSteps;
        if ((dw == nullptr && (tw > 0 || sw > 0)) || (dx == nullptr && (tx > 0 || sx > 0))) continue;
        const PairSide &a = sides[0][tw][sw], &b = sides[1][tx][sx];
        const int64_t partial_size = a.partial + b.partial;
        if (a.tasks + b.tasks > (1 << 23) || partial_size > (int64_t)partial_bytes) continue;
        const float join = partial_size == 0 ? 0.0f : kJoinStart + (float)partial_size * kJoinPerByte;
        const float least = ((float)a.tasks * a.time + (float)b.tasks * b.time) / (float)cus;
        if (2.0f + join + least >= best) continue;
        const bool first = dx == nullptr || (dw != nullptr && a.time >= b.time);
        const float time = 2.0f + join + (first ? list_time(a.tasks, a.time, b.tasks, b.time, cus)
                                                : list_time(b.tasks, b.time, a.tasks, a.time, cus));
        if (time < best) {
            best = time;
            plan.one_launch = true;
            plan.w_first = first;
            if (dw != nullptr) plan.w = {true, {FfKernel::kTile, kPairTile[tw], false}, 1 << sw};
            if (dx != nullptr) plan.x = {true, {FfKernel::kTile, kPairTile[tx], false}, 1 << sx};
        }
    }
}

// One gradient through registers.
FfGradient choose_staged_gradient(const FfParams& p, size_t& partial_bytes, int64_t cus) {
    const bool large = staged_large(p, p.cols, cus);
    // few tiles: shares of at least 16 stages until every CU has one (gradients of one row, w [10240, 1283]: 212 us, 76 so)
    int splits = 1;
    if (!large) {
        const int64_t tiles = ((p.rows + 63) / 64) * ((p.cols + 63) / 64);
        while (splits < kMaxSplits && tiles * splits < cus && share_stages(p, 2 * splits) >= 16 &&
               pair_side(p, kFf64x64, 2 * splits).partial <= (int64_t)partial_bytes)
            splits *= 2;
    }
    if (splits > 1) partial_bytes -= (size_t)pair_side(p, kFf64x64, splits).partial;
    return {true, {FfKernel::kStaged, large ? 128 : 64, true}, splits};
}

// The depth in shares whose sums begin at `partial`, which moves behind them.
void take_shares(FfParams& p, const FfGradient& g, float*& partial) {
    if (g.splits == 1) return;
    set_splits(p, g.splits, partial);
    partial += (size_t)pair_side(p, kFf64x64, g.splits).partial / 4;
}

hipError_t launch_row_sums(const FfParams& params, int shares, bool bf16, float* partial, hipStream_t stream) {
    FfParams p = params;
    const int64_t blocks = (p.rows + 511) / 512, span = (p.depth + shares - 1) / shares;
    p.partial = partial;
    const dim3 grid((unsigned)blocks, (unsigned)shares);
    if (bf16) hipLaunchKernelGGL(ff_row_sums_kernel<__bf16>, grid, dim3(256), 0, stream, p, span);
    else hipLaunchKernelGGL(ff_row_sums_kernel<_Float16>, grid, dim3(256), 0, stream, p, span);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess || shares == 1) return err;
    FfParams none{};
    none.splits = 1;
    p.cols = p.ld_partial = 0;
    p.splits = (int32_t)shares;
    return launch_join(p, none, bf16, stream);
}

}  // namespace

FfGradients choose_ff_gradients(const FfParams* dw, const FfParams* dx, const FfParams* sums, size_t partial_bytes,
                                int compute_units) {
    const int64_t cus = units(compute_units);
    FfGradients plan{};
    plan.w = {dw != nullptr, {}, 1};
    plan.x = {dx != nullptr, {}, 1};
    const bool w_staged = dw != nullptr && ff_staged_supported(*dw, kFfStore, true, true, false);
    const bool x_staged = dx != nullptr && ff_staged_supported(*dx, kFfStore, false, true, false);
    const bool w_tiled = w_staged && ff_tiled_supported(*dw, kFfStore, true, true, false);
    const bool x_tiled = x_staged && ff_tiled_supported(*dx, kFfStore, false, true, false);
    // (each launch's shares are joined before the next one sums its own: they have one place)
    if (w_tiled || x_tiled) choose_pair(w_tiled ? dw : nullptr, x_tiled ? dx : nullptr, partial_bytes, cus, plan);
    size_t left = partial_bytes;
    if (w_staged && !w_tiled) plan.w = choose_staged_gradient(prepared(*dw, true), left, cus);
    if (x_staged && !x_tiled) plan.x = choose_staged_gradient(prepared(*dx, false), left, cus);
    if (sums != nullptr) {
        // shares of at least 64 rows until there are four workgroups a CU
        const int64_t blocks = (sums->rows + 511) / 512;
        plan.sum_shares = 1;
        while (plan.sum_shares < kSumsMaxShares && blocks * plan.sum_shares < 4 * cus && sums->depth >= 128 * plan.sum_shares &&
               8 * plan.sum_shares * (size_t)sums->rows <= partial_bytes)
            plan.sum_shares *= 2;
    }
    return plan;
}

hipError_t launch_ff_gradients(const FfGradients& plan, const FfParams* dw, const FfParams* dx, const FfParams* sums,
                               bool bf16, float* partial, hipStream_t stream) {
    const auto on = [](const FfGradient& g, FfKernel kernel) { return g.wanted && g.choice.kernel == kernel; };
    hipError_t err = hipSuccess;
    for (FfKernel kernel : {FfKernel::kTile, FfKernel::kStaged}) {
        FfParams w{}, x{};  // (no rows: no tasks)
        w.splits = x.splits = 1;
        float* at = partial;
        const bool with_w = on(plan.w, kernel), with_x = on(plan.x, kernel);
        if (with_w) {
            w = prepared(*dw, true);
            take_shares(w, plan.w, at);
        }
        if (with_x) {
            x = prepared(*dx, false);
            take_shares(x, plan.x, at);
        }
        if (kernel == FfKernel::kTile && plan.one_launch) {
            err = (bf16 ? ff_pair_bf16 : ff_pair_f16)(w, x, with_w ? plan.w.choice.variant : kPairTile[0],
                                                     with_x ? plan.x.choice.variant : kPairTile[0], plan.w_first, stream);
        } else {
            const auto one = [&](const FfParams& p, const FfGradient& g, bool i_transposed) {
                if (kernel == FfKernel::kTile) return (bf16 ? ff_backward_bf16 : ff_backward_f16)(p, kFfStore, i_transposed, g.choice.variant, stream);
                return (bf16 ? ff_staged_bf16 : ff_staged_f16)(p, kFfStore, i_transposed, false, g.choice.variant == 128, stream);
            };
            if (with_w) err = one(w, plan.w, true);
            if (err == hipSuccess && with_x) err = one(x, plan.x, false);
        }
        if (err == hipSuccess) err = launch_join(w, x, bf16, stream);
        if (err != hipSuccess) return err;
    }
    if (sums != nullptr) err = launch_row_sums(*sums, plan.sum_shares, bf16, partial, stream);
    if (err == hipSuccess && on(plan.w, FfKernel::kGeneral)) err = launch_ff_general(*dw, kFfStore, true, true, bf16, false, stream);
    if (err == hipSuccess && on(plan.x, FfKernel::kGeneral)) err = launch_ff_general(*dx, kFfStore, false, true, bf16, false, stream);
    return err;
}

}  // namespace sdxl_hip
