// ranged.h — attention over parts of the cached positions, as the kernels that compute it share a call:
// a sliding window with sinks, or a prefix that groups of sequences have in common.
#pragma once

#include "flour_common.h"

namespace flour {

struct RangedAttn {
    void* out;
    int out_dtype;
    int64_t o_st, o_sh;
    const void* q;
    int64_t q_st, q_sh;
    const void *k_pool, *v_pool;
    int dtype;
    const int32_t* cu;  // null: a decode step, row b of sequence b
    const int32_t* kv_lens;
    const int32_t* block_tables;
    int max_blocks, num_seqs, max_rows, rows, num_heads, kv_heads, head_dim, block_size;
    int64_t num_slots;
    int max_kv;  // bounds kv_lens
    float scale;
    // A row at position p sees j <= p with p - j < window or j < sinks.
    int window, sinks;
    // Groups of sequences with the first shared_lens[g] positions in common (num_groups 0: none).
    const int32_t *group_starts, *shared_lens;
    int num_groups, max_shared;
};

// Where the rows of sequence s start (those of num_seqs: where they end). Whatever cu holds, rows are the call's.
__device__ __forceinline__ int ranged_row(const RangedAttn& a, int s) {
    return a.cu ? max(0, min(a.cu[s], a.rows)) : s;
}
// Rows of sequence s, its kv length (0 where its rows see nothing).
struct RangedSeq {
    int row0, rows, kv;
};
__device__ __forceinline__ RangedSeq ranged_seq(const RangedAttn& a, int s) {
    const int r0 = ranged_row(a, s), n = max(0, ranged_row(a, s + 1) - r0);
    const int kv = min(a.kv_lens[s], a.max_kv);
    return RangedSeq{r0, n, kv >= n && kv > 0 ? kv : 0};
}

// The last i in [lo, hi) with at[i] <= x (lo if there is none), at not decreasing; by a whole wave, the same x
// and bounds in every lane: 64 of the range in a round.
__device__ __forceinline__ int wave_last_at(const int32_t* at, int lo, int hi, int x) {
    const int lane = threadIdx.x & 63;
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) >> 6, i = lo + min(lane * step, hi - lo);
        const int below = __builtin_popcountll(__ballot(i < hi && at[i] <= x));
        hi = min(hi, lo + max(1, below) * step);
        lo += max(0, below - 1) * step;
    }
    return lo;
}

// The sequence of packed row `row`, one for the wave: the last one that starts at or before it.
__device__ __forceinline__ int ranged_seq_of(const RangedAttn& a, int row) {
    return wave_last_at(a.cu, 0, a.num_seqs, row);
}

// The group of sequence s, one for the wave (-1: none): the last one that starts at or before it, if it has
// not ended.
__device__ __forceinline__ int ranged_group(const int32_t* starts, int num_groups, int s) {
    if (num_groups == 0 || starts[0] > s) return -1;
    const int g = wave_last_at(starts, 0, num_groups, s);
    return s < starts[g + 1] ? g : -1;
}
__device__ __forceinline__ int ranged_shared_len(const int32_t* shared_lens, int max_shared, int g) {
    return g < 0 ? 0 : max(0, min(shared_lens[g], max_shared));
}
__device__ __forceinline__ int ranged_shared_of(const RangedAttn& a, int s) {
    return ranged_shared_len(a.shared_lens, a.max_shared, ranged_group(a.group_starts, a.num_groups, s));
}

// Takes every shape (ranged_generic.hip).
int launch_ranged_generic(const RangedAttn& a, hipStream_t stream);

}  // namespace flour
