// The tiled products of 8-bit integers, out of type fp16.
#include "feed_forward_tiles.hpp"

namespace sdxl_hip {

hipError_t ff_i8_forward_f16(const FfParams& p, FfEpilogue epilogue, int tile, hipStream_t stream) {
    return ff_i8_forward<_Float16>(p, epilogue, tile, stream);
}

hipError_t ff_i8_staged_f16(const FfParams& p, FfEpilogue epilogue, bool large, hipStream_t stream) {
    return ff_i8_staged<_Float16>(p, epilogue, large, stream);
}

}  // namespace sdxl_hip
