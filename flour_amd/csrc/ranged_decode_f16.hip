// ranged_decode_f16.hip — ranged_decode.h over f16 pools.
#include "ranged_decode.h"

namespace flour {

int launch_ranged_decode_f16(const RangedAttn& a, const RangedStream& st, hipStream_t stream) {
    return launch_ranged_decode<f16_t>(a, st, stream);
}

}  // namespace flour
