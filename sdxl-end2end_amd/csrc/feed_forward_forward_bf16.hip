// The tiled products of the feed-forward operators: projections, bf16.
#include "feed_forward_tiles.hpp"

namespace sdxl_hip {

hipError_t ff_forward_bf16(const FfParams& p, FfEpilogue epilogue, bool j_fp8, int tile, hipStream_t stream) {
    return ff_forward<__bf16>(p, epilogue, j_fp8, tile, stream);
}

}  // namespace sdxl_hip
