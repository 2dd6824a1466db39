// ranged_decode.h — decode steps over a window with sinks: the stream of paged_decode.hip over the chunks that
// hold visible positions. Instantiated per type in ranged_decode_*.hip.
#pragma once

#include "paged_decode_kernel.h"

namespace flour {

// The stream of a step: its workspace's parts, its waves.
struct RangedStream {
    DecodeWs ws;
    int grid;
};

int launch_ranged_decode_f32(const RangedAttn& a, const RangedStream& st, hipStream_t stream);
int launch_ranged_decode_bf16(const RangedAttn& a, const RangedStream& st, hipStream_t stream);
int launch_ranged_decode_f16(const RangedAttn& a, const RangedStream& st, hipStream_t stream);

template <typename T>
static int launch_ranged_decode(const RangedAttn& a, const RangedStream& st, hipStream_t stream) {
    const int n_rep = a.num_heads / a.kv_heads, batch = a.num_seqs;
    const size_t lds = (size_t)(batch + 1) * sizeof(int);
    auto of_dim = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        return a.block_size == 16 ? paged_decode_mfma_kernel<T, AnyOut, true, D, false, false, true>
                                  : paged_decode_mfma_kernel<T, AnyOut, false, D, false, false, true>;
    };
    using d64 = std::integral_constant<int, 64>;
    using d128 = std::integral_constant<int, 128>;
    auto kern = a.head_dim == 64 ? of_dim(d64{}) : of_dim(d128{});
    kern<<<dim3(st.grid), dim3(64), lds, stream>>>(
        static_cast<AnyOut*>(a.out), static_cast<const T*>(a.q), static_cast<const T*>(a.k_pool),
        static_cast<const T*>(a.v_pool), a.block_tables, a.max_blocks, a.kv_lens, batch, a.num_heads,
        a.kv_heads, n_rep, a.block_size, a.num_slots, a.max_kv, a.scale * LOG2E, st.ws);
    const int rc = check_hip(hipGetLastError(), "decode over a window launch");
    if (rc != FLOUR_OK) return rc;
    auto merge = a.head_dim == 64 ? paged_decode_merge_kernel<AnyOut, 64, false, false>
                                  : paged_decode_merge_kernel<AnyOut, 128, false, false>;
    merge<<<dim3(a.num_heads, batch), dim3(64 * decode_merge_waves(st.grid, batch, a.kv_heads)), 0,
            stream>>>(static_cast<AnyOut*>(a.out), batch, a.num_heads, a.kv_heads, n_rep, st.grid, st.ws);
    return check_hip(hipGetLastError(), "decode over a window merge launch");
}

}  // namespace flour
