// decode_stream_bf16.hip — decode_stream.h for bf16 queries.
#include "decode_stream.h"

namespace flour {

int launch_decode_stream_bf16(const DpArgs& a, int pool_dtype, int head_dim, void* ws, int max_rows,
                           int rows, hipStream_t s) {
    return launch_stream_q<bf16_t>(a, pool_dtype, head_dim, ws, max_rows, rows, s);
}

}  // namespace flour
