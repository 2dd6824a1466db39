// ranged_tiles_f32.hip — ranged_tiles.h over f32 pools.
#include "ranged_tiles_kernel.h"

namespace flour {

int launch_ranged_tiles_f32(const RtArgs& r, int halves, int last, hipStream_t stream) {
    return launch_ranged_tiles<float>(r, halves, last, stream);
}

}  // namespace flour
