// ranged_tiles_bf16.hip — ranged_tiles.h over bf16 pools.
#include "ranged_tiles_kernel.h"

namespace flour {

int launch_ranged_tiles_bf16(const RtArgs& r, int halves, int last, hipStream_t stream) {
    return launch_ranged_tiles<bf16_t>(r, halves, last, stream);
}

}  // namespace flour
