// dw and dx of the feed-forward operators in one launch, bf16.
#include "feed_forward_tiles.hpp"

namespace sdxl_hip {

hipError_t ff_pair_bf16(const FfParams& w, const FfParams& x, int w_tile, int x_tile, bool w_first, hipStream_t stream) {
    return ff_pair<__bf16>(w, x, w_tile, x_tile, w_first, stream);
}

}  // namespace sdxl_hip
