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

// Groups first + lane: where they start and end, and their prefixes' lengths.
struct RangedGroups {
    int start, end, len;
};
__device__ __forceinline__ RangedGroups ranged_groups(const RangedAttn& a, int first) {
    const int g = first + (threadIdx.x & 63);
    if (g >= a.num_groups) return RangedGroups{0, 0, 0};
    return RangedGroups{a.group_starts[g], a.group_starts[g + 1], a.shared_lens[g]};
}
// The length of the prefix of sequence s, one for the wave, which is in one of these groups (0: in none).
__device__ __forceinline__ int ranged_shared_in(const RangedAttn& a, const RangedGroups& x, int s) {
    const uint64_t hit = __ballot(x.start <= s && s < x.end);
    return hit ? max(0, min(__builtin_amdgcn_readlane(x.len, __builtin_ctzll(hit)), a.max_shared)) : 0;
}
// The same of all groups, whose first 64 have been read.
__device__ __forceinline__ int ranged_shared_of(const RangedAttn& a, const RangedGroups& x, int s) {
    if (a.num_groups <= 64) return ranged_shared_in(a, x, s);
    return ranged_shared_in(a, ranged_groups(a, wave_last_at(a.group_starts, 0, a.num_groups, s)), s);
}

// The lengths of the prefixes of sequences s, one a lane.
__device__ __forceinline__ int ranged_shared_each(const RangedAttn& a, const RangedGroups& x, int s) {
    int len = 0;
    if (a.num_groups <= 64) {
        for (int g = 0; g < a.num_groups; g++) {
            const int start = __builtin_amdgcn_readlane(x.start, g), end = __builtin_amdgcn_readlane(x.end, g);
            const int n = __builtin_amdgcn_readlane(x.len, g);
            len = start <= s && s < end ? n : len;
        }
    } else {
        int lo = 0, hi = a.num_groups;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.group_starts[mid] <= s)
                lo = mid;
            else
                hi = mid;
        }
        if (a.group_starts[lo] <= s && s < a.group_starts[lo + 1]) len = a.shared_lens[lo];
    }
    return max(0, min(len, a.max_shared));
}

// Takes every shape (ranged_generic.hip).
int launch_ranged_generic(const RangedAttn& a, hipStream_t stream);

}  // namespace flour
