// ranged_decode_f32.hip — ranged_decode.h over f32 pools.
#include "ranged_decode.h"

namespace flour {

int launch_ranged_decode_f32(const RangedAttn& a, const RangedStream& st, hipStream_t stream) {
    return launch_ranged_decode<float>(a, st, stream);
}

}  // namespace flour
