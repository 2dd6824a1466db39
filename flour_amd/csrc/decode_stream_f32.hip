// decode_stream_f32.hip — decode_stream.h for fp32 queries.
#include "decode_stream.h"

namespace flour {

int launch_decode_stream_f32(const DpArgs& a, int pool_dtype, int head_dim, void* ws, int max_rows,
                           int rows, hipStream_t s) {
    return launch_stream_q<float>(a, pool_dtype, head_dim, ws, max_rows, rows, s);
}

}  // namespace flour
