// decode_stream_f16.hip — decode_stream.h for f16 queries.
#include "decode_stream.h"

namespace flour {

int launch_decode_stream_f16(const DpArgs& a, int pool_dtype, int head_dim, void* ws, int max_rows,
                           int rows, hipStream_t s) {
    return launch_stream_q<f16_t>(a, pool_dtype, head_dim, ws, max_rows, rows, s);
}

size_t decode_stream_bytes(int batch, int64_t max_cols, int head_dim) {
    return stream_bytes_for(batch, max_cols, head_dim);
}

}  // namespace flour
