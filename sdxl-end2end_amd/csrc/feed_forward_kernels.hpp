// Internal launch interface of the feed-forward kernels (feed_forward*.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

namespace sdxl_hip {

// What a product's epilogue makes of its sums.
enum FfEpilogue : int32_t {
    kFfLinear = 0,    // out = act(z) + residual
    kFfGated = 1,     // out = value * act(gate)
    kFfLinearDz = 2,  // out (dz) = dout * act'(z)
    kFfGatedDz = 3,   // out (dz) = [dout * act(gate) | dout * value * act'(gate)]
    kFfStore = 4      // out = the sums (dx, dw); optional row sums of the I operand (dbias)
};

// C[i, j] = sum_r I(i, r) J(j, r), then the epilogue. Operand X(i, r) is
// element i * ld + r of its tensor, or r * ld + i where it is transposed. The
// forward projections are I = x, J = w; dx is I = dz, J = w transposed; dw is
// I = dz transposed, J = x transposed. J holds E4M3 codes if j_fp8.
struct FfParams {
    const void* ip;
    const void* jp;
    int64_t ld_i, ld_j;       // elements (E4M3: bytes)
    const float* j_scale;     // nullable: fp32 scale of every J row
    const void* bias;         // nullable, by J rows
    const void* residual;     // nullable (kFfLinear)
    const void* dout;         // kFfLinearDz, kFfGatedDz
    void* out;
    void* row_sums;           // nullable (kFfStore): sums over r of every I row
    int64_t ld_res, ld_dout, ld_out;
    int64_t rows, cols, depth;  // of C before the gating: gated products have 2 n J rows, cols = n
    // I's row as it may be read, where its columns are padded with zeros up to a multiple of 8 (dz): the row's
    // depth, or its columns where I is transposed; 0: as given
    int64_t i_row;
    int64_t out_cols_padded;    // dz: columns up to here are written, zeros past the last one
    int32_t activation;         // sdxl_activation
    int32_t gate_first;
    // filled by the tiled kernel's launcher: wide epilogue accesses, tiles of C, row blocks per task group
    int32_t vec, i_blocks, j_blocks, group_i;
    // kFfStore: the depth in `splits` shares of 64 * share_stages: share s leaves its sums in partial
    // [splits][rows][ld_partial], its row sums behind them in [splits][rows]; one share: as ever.
    int32_t splits, share_stages;
    int64_t ld_partial;  // cols, up to a multiple of 8
    float* partial;
    // both operands hold 8-bit integers (forward epilogues): ld_i, ld_j and depth in bytes, i_scale the fp32 scale of every
    // I row, j_scale that of every J row; or an FfI8: I holds 16-bit values, which the kernel of few rows quantises
    int32_t i8;
    const float* i_scale;
};

enum FfI8 : int32_t { kFfI8None = 0, kFfI8Codes = 1, kFfI8Tokens = 2 };

// The joining pass of a product whose depth was split.
struct FfJoin {
    const float* partial;
    void *out, *row_sums;
    int64_t ld_out;
    int32_t rows, cols, ld, splits, vec, blocks;
};

// The depth in the kernels' stages of 128 bytes.
inline int64_t ff_stages(const FfParams& p) { return p.i8 != 0 ? (p.depth + 127) / 128 : (p.depth + 63) / 64; }

// The general kernel: any size, stride and alignment.
hipError_t launch_ff_general(const FfParams& p, FfEpilogue epilogue, bool i_transposed, bool j_transposed, bool bf16,
                             bool j_fp8, hipStream_t stream);

// Tiles of the tiled kernel, rows x columns of sums; the last for 8-bit integers alone.
enum FfTileId : int { kFf256x320, kFf256x256, kFf128x256, kFf128x192, kFf128x128, kFf64x128, kFf64x64, kFfTiles, kFf256x192 = kFfTiles, kFfI8Tiles };

// Tiles whose waves share the depth (feed_forward_deep.hip), side x waves.
enum FfDeepId : int { kFfDeep32x8, kFfDeep32x4, kFfDeep64x4 };

// The kernel that a product runs on, and which of its variants: an FfTileId (tile), an FfDeepId (deep), the waves of a
// workgroup (rows), the tile's side (staged).
enum class FfKernel : int { kGeneral, kRows, kDeep, kTile, kStaged };
struct FfChoice {
    FfKernel kernel;
    int variant;
    bool staged;  // rows and deep: operands through registers
};

// Its name, as sdxl_ff_kernels and sdxl_i8_kernels have it.
inline std::string kernel_text(const FfChoice& c) {
    static const char* const tiles[kFfI8Tiles] = {"256x320", "256x256", "128x256", "128x192", "128x128", "64x128", "64x64", "256x192"};
    static const char* const deep[] = {"32x32/8", "32x32/4", "64x64/4"};
    const std::string through = c.staged ? " staged" : "";
    switch (c.kernel) {
    case FfKernel::kGeneral: break;
    case FfKernel::kRows: return "rows/" + std::to_string(c.variant) + through;
    case FfKernel::kDeep: return std::string("deep ") + deep[c.variant] + through;
    case FfKernel::kTile: return std::string("tile ") + tiles[c.variant];
    case FfKernel::kStaged: return c.variant == 128 ? "staged 128x128" : "staged 64x64";
    }
    return "general";
}

// Projections and dz, by sizes, strides and alignment.
FfChoice choose_ff(const FfParams& p, FfEpilogue epilogue, bool j_fp8, int compute_units);
hipError_t launch_ff(const FfChoice& choice, const FfParams& p, FfEpilogue epilogue, bool bf16, bool j_fp8, hipStream_t stream);

// The gradients of a call: dw (I transposed), dx, and a bias gradient without dw. Both may run in one launch; either may
// have its depth split, as far as the workspace's partial sums reach (ff_partial_bytes is enough for any split that is
// taken).
struct FfGradient {
    bool wanted;
    FfChoice choice;
    int splits;
};
struct FfGradients {
    FfGradient w, x;
    bool one_launch, w_first;
    int sum_shares;  // 0: no bias gradient alone
};
size_t ff_partial_bytes(int64_t m, int64_t features, int64_t k);
// dw and dx: null where not wanted; sums: dw's parameters for a bias gradient alone, else null.
FfGradients choose_ff_gradients(const FfParams* dw, const FfParams* dx, const FfParams* sums, size_t partial_bytes,
                                int compute_units);
hipError_t launch_ff_gradients(const FfGradients& plan, const FfParams* dw, const FfParams* dx, const FfParams* sums,
                               bool bf16, float* partial, hipStream_t stream);

// Few rows (feed_forward_rows.hip): waves of a workgroup.
bool ff_rows_supported(const FfParams& p, FfEpilogue epilogue, bool j_fp8);
int ff_rows_waves(const FfParams& p, bool gated);
// Whether it takes 16-bit tokens of a product of 8-bit weights (i8: kFfI8Tokens).
bool ff_rows_tokens(const FfParams& p, FfEpilogue epilogue);
hipError_t launch_ff_rows(const FfParams& p, FfEpilogue epilogue, int waves, bool staged, bool bf16, bool j_fp8,
                          hipStream_t stream);

// Whether a product's rows have the 16 bytes that all kernels but the general one need.
bool ff_staged_supported(const FfParams& p, FfEpilogue epilogue, bool i_transposed, bool j_transposed, bool j_fp8);

}  // namespace sdxl_hip
