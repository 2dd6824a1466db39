// decode_pools.h — an attention call over pools of any element type, as the kernels that take one
// share it.
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

// A call of the streamed kernel (decode_stream.h).
struct DpArgs {
    void* out;
    int out_dtype;
    int64_t o_st, o_sh;
    const void* q;
    int64_t q_st, q_sh;
    const uint8_t *k_pool, *v_pool;
    const float *k_scale, *v_scale;
    const int32_t *cu, *kv_lens, *block_tables;
    int max_blocks, batch, num_heads, kv_heads, n_rep, block_size;
    int64_t num_slots;
    int max_kv, max_rows;
    float scale_log2;
    float* scores;  // kept scores (or null): (batch, num_heads, score_stride)
    int64_t score_stride;
    float* ml;    // with scores: (batch, num_heads, 2)
    int cols;     // columns of a piece that can be real
    float* p_ml;  // pieces: [2 * waves][cols][3] maximum, sum, maximum with the V scales
    float* p_o;   // pieces: [2 * waves][cols][D]
    int* pre;     // [batch + 1] chunks per kv head of the sequences before
};


// Takes every shape (attn_pools.hip).
int launch_attn_pools(const PoolAttn& a, hipStream_t stream);
// After a staged prefill with f16 queries: the rows of the heads whose values f16 does not hold.
int launch_attn_beyond_f16(const PoolAttn& a, int max_rows, hipStream_t stream);

// flour_hip_kv_dequant's kernel; out_tables null: block lb of sequence s goes to block
// s * out_max_blocks + lb, and staged_table and staged_lens (both or neither) take that table and the
// lengths cut to max_kv.
int launch_kv_dequant(void* k_out, void* v_out, int dtype, const int32_t* out_tables,
                      int out_max_blocks, int64_t out_slots, const void* k_pool,
                      const void* v_pool, const float* k_scale, const float* v_scale,
                      int pool_dtype, const int32_t* bt, int max_blocks, const int32_t* kv_lens,
                      int num_seqs, int max_kv, int kv_heads, int head_dim, int block_size,
                      int64_t num_slots, int32_t* staged_table, int32_t* staged_lens,
                      hipStream_t s);

int launch_weights_add(float* weights, int64_t width, const int32_t* weight_rows, int num_rows,
                       const int32_t* context_lens, int max_ctx, int batch, int kv_heads,
                       int n_rep, const float* scores, int64_t score_stride, const float* ml,
                       hipStream_t stream);

// Per type of the queries (decode_stream_*.hip): launches, and the workspace of calls whose sequences
// bring up to max_cols columns (rows x query heads of a kv head), whatever the type.
int launch_decode_stream_f32(const DpArgs& a, int pool_dtype, int head_dim, void* ws, int max_rows,
                             int rows, hipStream_t s);
int launch_decode_stream_bf16(const DpArgs& a, int pool_dtype, int head_dim, void* ws, int max_rows,
                              int rows, hipStream_t s);
int launch_decode_stream_f16(const DpArgs& a, int pool_dtype, int head_dim, void* ws, int max_rows,
                             int rows, hipStream_t s);
size_t decode_stream_bytes(int batch, int64_t max_cols, int head_dim);

// Decode over a plain pool that keeps its scores (paged_decode.hip): whether it takes a shape, its
// workspace, the call (scores of row b * num_heads + h at row * score_stride, in chunks of up to 64
// positions, and the row's (max, sum) at row_ml).
bool paged_decode_scores_takes(int dtype, int head_dim, int block_size, int n_rep, int batch,
                               int num_heads, int64_t num_slots, const void* out, const void* q,
                               const void* k_pool, const void* v_pool);
size_t paged_decode_scores_bytes(int batch, int n_rep, int head_dim);
int paged_decode_scores(void* out, int out_dtype, const void* q, const void* k_pool,
                        const void* v_pool, const int32_t* block_tables, int max_blocks_per_seq,
                        const int32_t* context_lens, int batch, int num_heads, int kv_heads,
                        int head_dim, int block_size, int64_t num_slots, int max_context_len,
                        float scale, int dtype, void* workspace, size_t workspace_bytes,
                        float* scores, int64_t score_stride, float* row_ml, void* stream);

// Whether the fp32 matrix cores take a prefill (attn_f32_mfma.hip).
bool prefill_f32_mfma_supported(int dtype, int head_dim, int num_seqs, int max_seqlen_q,
                                int block_size, int64_t num_slots);

bool check_pool8(const char* what, int pool_dtype, const void* k_pool, const void* v_pool,
                 const void* k_scale, const void* v_scale, int kv_heads, int head_dim,
                 int block_size, int64_t num_slots);

}  // namespace flour
