// ranged_decode_bf16.hip — ranged_decode.h over bf16 pools.
#include "ranged_decode.h"

namespace flour {

int launch_ranged_decode_bf16(const RangedAttn& a, const RangedStream& st, hipStream_t stream) {
    return launch_ranged_decode<bf16_t>(a, st, stream);
}

}  // namespace flour
