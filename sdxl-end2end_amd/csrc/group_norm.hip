// Which kernels a group norm call runs on (include/sdxl_hip/group_norm.h).
#include <hip/hip_runtime.h>

#include "group_norm_device.hpp"

namespace sdxl_hip {

GnPlan gn_plan(const GnParams& p, GnType, bool) { return {false, 1, p.pixels}; }

hipError_t launch_gn_forward(const GnPlan&, const GnParams& p, GnType type, hipStream_t stream) {
    const hipError_t err = launch_gn_stats_general(p, type, stream);
    return err != hipSuccess ? err : launch_gn_apply_general(p, type, stream);
}

hipError_t launch_gn_backward(const GnPlan&, const GnParams& p, GnType type, hipStream_t stream) {
    hipError_t err = hipSuccess;
    if (p.batch > 0 && p.pixels > 0) {
        err = launch_gn_sums_general(p, type, stream);
        if (err == hipSuccess && p.y != nullptr) err = launch_gn_dx_general(p, type, stream);
    }
    if (err == hipSuccess && (p.dgamma != nullptr || p.dbeta != nullptr)) err = launch_gn_parameters_general(p, type, stream);
    return err;
}

}  // namespace sdxl_hip
