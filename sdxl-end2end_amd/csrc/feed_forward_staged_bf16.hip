// Products of the feed-forward operators whose rows 16-byte accesses do not divide, bf16.
#include "feed_forward_tiles.hpp"

namespace sdxl_hip {

hipError_t ff_staged_bf16(const FfParams& p, FfEpilogue epilogue, bool i_transposed, bool j_fp8, bool large, hipStream_t stream) {
    return ff_staged<__bf16>(p, epilogue, i_transposed, j_fp8, large, stream);
}

}  // namespace sdxl_hip
