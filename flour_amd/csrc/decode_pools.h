// decode_pools.h — an attention call over pools of any element type, as the kernels that take one
// share it (attn_pools.hip, decode_pools.hip).
#pragma once

#include "flour_common.h"

namespace flour {

static constexpr float LOG2_E = 1.4426950408889634f;

struct PoolAttn {
    void* out;
    int out_dtype;
    int64_t o_st, o_sh;
    const void* q;
    int dtype;
    int64_t q_st, q_sh;
    const void *k_pool, *v_pool;
    const float *k_scale, *v_scale;  // null: a plain pool, of the type of q
    int pool_dtype;
    const int32_t* cu;  // null: a decode step, row b of sequence b
    const int32_t* kv_lens;
    const int32_t* block_tables;
    int max_blocks, batch, rows, num_heads, kv_heads, head_dim, block_size;
    int64_t num_slots;
    int max_kv;
    float scale;
    // decode steps whose weights are wanted: every score in the exp2 domain, (batch, num_heads,
    // score_stride), and each head's maximum and sum
    float* scores;
    int64_t score_stride;
    float* ml;
};

// The streamed kernel (decode_pools.hip): whether it takes a call, the workspace it needs for groups of
// up to max_cols columns (rows x query heads of a kv head), and its launch (max_rows bounds the rows of
// a sequence). launch_attn_pools (attn_pools.hip) takes every shape.
bool decode_stream_takes(const PoolAttn& a);
size_t decode_stream_bytes(int batch, int max_cols, int head_dim);
int launch_decode_stream(const PoolAttn& a, int max_rows, void* workspace, hipStream_t stream);
int launch_attn_pools(const PoolAttn& a, hipStream_t stream);

bool check_pool8(const char* what, int pool_dtype, const void* k_pool, const void* v_pool,
                 const void* k_scale, const void* v_scale, int kv_heads, int head_dim,
                 int block_size, int64_t num_slots);

}  // namespace flour
