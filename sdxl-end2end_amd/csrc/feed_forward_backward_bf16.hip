// The tiled products of the feed-forward operators: dz, dx and dw, bf16.
#include "feed_forward_tiles.hpp"

namespace sdxl_hip {

hipError_t ff_backward_bf16(const FfParams& p, FfEpilogue epilogue, bool i_transposed, int tile, hipStream_t stream) {
    return ff_backward<__bf16>(p, epilogue, i_transposed, tile, stream);
}

}  // namespace sdxl_hip
