// Internal launch interface of the group norm kernels (group_norm*.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sdxl_hip {

// One call. Images are cut into `chunks` runs of chunk_pixels pixels (the last one shorter); every chunk leaves its
// part of the sums in the workspace, and whoever needs the whole adds the chunks in their order.
struct GnParams {
    const void *x, *gamma, *beta, *dy;
    void* y;  // backward: dx (nullable)
    void *dgamma, *dbeta;
    int8_t* q;             // y as codes, with a scale by row; null: y
    float* q_scale;
    const float* stats;    // backward: [batch][groups] {mean, rstd}
    float* stats_out;      // forward, nullable
    float* partial;        // [batch][groups][chunks] {mean, sum of squares about it}; backward: {sum gamma dz, sum gamma dz n}
    float* channel_sums;   // backward [batch][chunks][channels] {sum dz, sum dz n}
    int64_t ld_x, ld_y, ld_dy;  // elements
    int64_t ld_q;               // bytes
    int64_t pixels, chunk_pixels;
    int32_t batch, channels, groups, group_channels, chunks;
    int32_t activation;
    float eps;
    // of the fast kernels, filled in by their launcher: slabs of whole groups, vectors of 16 bytes a slab's row, rows of the
    // workgroup at a time, lanes that add a group's parts; chunks of the second pass
    int32_t slabs, slab_groups, vecs, rows_at_once, team;
    int32_t columns;  // images by slabs
    int32_t apply_chunks;
    int64_t apply_pixels;
};

enum GnType : int { kGnF16, kGnBf16, kGnF32 };

// The general kernels: any sizes, strides and alignment. Statistics and sums leave one chunk an image.
hipError_t launch_gn_stats_general(const GnParams& p, GnType type, hipStream_t stream);
hipError_t launch_gn_apply_general(const GnParams& p, GnType type, hipStream_t stream);
hipError_t launch_gn_sums_general(const GnParams& p, GnType type, hipStream_t stream);
hipError_t launch_gn_dx_general(const GnParams& p, GnType type, hipStream_t stream);
hipError_t launch_gn_parameters_general(const GnParams& p, GnType type, hipStream_t stream);

// How a call is cut and which kernels it runs on, by sizes and strides alone (a call's sums have one order everywhere).
enum GnCall : int { kGnForward, kGnRows, kGnBackward };
struct GnPlan {
    bool fast;
    int32_t hold;  // vectors that a thread of the one-launch kernel holds; 0: two passes
    int32_t chunks;
    int64_t chunk_pixels;
};
GnPlan gn_plan(const GnParams& p, GnType type, GnCall call);

// With p.chunks and p.chunk_pixels of the plan.
hipError_t launch_gn_forward(const GnPlan& plan, const GnParams& p, GnType type, hipStream_t stream);
hipError_t launch_gn_backward(const GnPlan& plan, const GnParams& p, GnType type, hipStream_t stream);

}  // namespace sdxl_hip
