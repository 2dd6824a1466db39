// ranged_decode.h — decode steps over a window with sinks: the stream of paged_decode.hip over the chunks that
// hold visible positions. Instantiated per type in ranged_decode_*.hip. Bound by memory: 64 x 512-4,096 tokens,
// window 1,024, 32 / 8 heads of 128 in bf16 42.0 us (6.2 TB/s of the 259 MB that are visible); 8 x 16-32K, window
// 4,096 with 16 sinks, 64 / 8 heads in f16 26.5 us (5.1) and its merge 4.6.
#pragma once

#include "paged_decode_kernel.h"

namespace flour {

// The stream of a step: its workspace's parts, its workgroups, and whether those are a pair each (or waves of
// ranges).
struct RangedStream {
    DecodeWs ws;
    int grid;
    bool pairs;
};

int launch_ranged_decode_f32(const RangedAttn& a, const RangedStream& st, hipStream_t stream);
int launch_ranged_decode_bf16(const RangedAttn& a, const RangedStream& st, hipStream_t stream);
int launch_ranged_decode_f16(const RangedAttn& a, const RangedStream& st, hipStream_t stream);

template <typename T, int D>
static void launch_ranged_decode_d(const RangedAttn& a, const RangedStream& st, hipStream_t stream) {
    auto kern = a.block_size == 16
                    ? (st.pairs ? paged_decode_mfma_kernel<T, AnyOut, true, D, false, false, true, DEC_PAIRS>
                                     : paged_decode_mfma_kernel<T, AnyOut, true, D, false, false, true>)
                    : (st.pairs ? paged_decode_mfma_kernel<T, AnyOut, false, D, false, false, true, DEC_PAIRS>
                                     : paged_decode_mfma_kernel<T, AnyOut, false, D, false, false, true>);
    const size_t lds = st.pairs ? (size_t)DEC_PAIR_WAVES * dec_pair_lds(D, sizeof(T))
                                     : (size_t)(a.num_seqs + 1) * sizeof(int);
    kern<<<dim3(st.grid), dim3(st.pairs ? 64 * DEC_PAIR_WAVES : 64), lds, stream>>>(
        static_cast<AnyOut*>(a.out), static_cast<const T*>(a.q), static_cast<const T*>(a.k_pool),
        static_cast<const T*>(a.v_pool), a.block_tables, a.max_blocks, a.kv_lens, a.num_seqs, a.num_heads,
        a.kv_heads, a.num_heads / a.kv_heads, a.block_size, a.num_slots, a.max_kv, a.scale * LOG2E, st.ws);
}

template <typename T>
static int launch_ranged_decode(const RangedAttn& a, const RangedStream& st, hipStream_t stream) {
    if (a.head_dim == 64)
        launch_ranged_decode_d<T, 64>(a, st, stream);
    else
        launch_ranged_decode_d<T, 128>(a, st, stream);
    const int rc = check_hip(hipGetLastError(), "decode over a window launch");
    if (rc != FLOUR_OK || st.pairs) return rc;
    const int batch = a.num_seqs, n_rep = a.num_heads / a.kv_heads;
    auto merge = a.head_dim == 64 ? paged_decode_merge_kernel<AnyOut, 64, false, false>
                                  : paged_decode_merge_kernel<AnyOut, 128, false, false>;
    merge<<<dim3(a.num_heads, batch), dim3(64 * decode_merge_waves(st.grid, batch, a.kv_heads)), 0,
            stream>>>(static_cast<AnyOut*>(a.out), batch, a.num_heads, a.kv_heads, n_rep, st.grid, st.ws);
    return check_hip(hipGetLastError(), "decode over a window merge launch");
}

}  // namespace flour
