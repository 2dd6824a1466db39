// ranged_attn.cpp — C entries of the attention over a sliding window with sinks and over prefixes that
// sequences share: argument checks, workspaces and the choice of the kernel.
#include "ranged.h"

namespace flour {

static bool check_shape(const char* what, const RangedAttn& a) {
    if (!valid_dtype(a.dtype) || !valid_dtype(a.out_dtype)) {
        set_error("%s: unknown dtype (%d, out %d)", what, a.dtype, a.out_dtype);
        return false;
    }
    if (a.num_seqs < 0 || a.rows < 0 || a.max_rows < 0 || a.num_heads <= 0 || a.kv_heads <= 0 ||
        a.num_heads % a.kv_heads != 0 || a.head_dim <= 0 || a.block_size <= 0 ||
        a.num_slots <= 0 || a.num_slots % a.block_size != 0 || a.max_blocks <= 0 || a.max_kv < 0 ||
        (int64_t)a.max_kv > (int64_t)a.max_blocks * a.block_size) {
        set_error("%s: bad shape (sequences=%d rows=%d of up to %d heads=%d kv_heads=%d head_dim=%d "
                  "bs=%d num_slots=%lld max_blocks=%d max_kv=%d)",
                  what, a.num_seqs, a.rows, a.max_rows, a.num_heads, a.kv_heads, a.head_dim,
                  a.block_size, (long long)a.num_slots, a.max_blocks, a.max_kv);
        return false;
    }
    if (a.window < 1 || a.sinks < 0) {
        set_error("%s: window %d with %d sinks: a row sees its own position at least", what, a.window,
                  a.sinks);
        return false;
    }
    if (a.num_groups < 0 || a.max_shared < 0 ||
        (int64_t)a.max_shared > (int64_t)a.max_blocks * a.block_size) {
        set_error("%s: %d groups with prefixes of up to %d positions, tables of %lld", what,
                  a.num_groups, a.max_shared, (long long)a.max_blocks * a.block_size);
        return false;
    }
    return true;
}

static int ranged_call(const char* what, const RangedAttn& a, bool shared, void* workspace,
                       size_t workspace_bytes, hipStream_t stream) {
    if (!check_shape(what, a)) return FLOUR_ERR_INVALID_ARGUMENT;
    if (a.num_seqs == 0 || a.rows == 0) return FLOUR_OK;
    if (!a.out || !a.q || !a.k_pool || !a.v_pool || !a.kv_lens || !a.block_tables ||
        (shared && a.num_groups > 0 && (!a.group_starts || !a.shared_lens))) {
        set_error("%s: null pointer", what);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    return launch_ranged_generic(a, stream);
}

// A decode step's part of a call: one row a sequence, packed rows of all heads.
static RangedAttn decode_call(void* out, int out_dtype, const void* q, const void* k_pool,
                              const void* v_pool, const int32_t* block_tables, int max_blocks,
                              const int32_t* context_lens, int batch, int num_heads, int kv_heads,
                              int head_dim, int block_size, int64_t num_slots, int max_context_len,
                              float scale, int dtype) {
    RangedAttn a{};
    a.out = out, a.out_dtype = out_dtype, a.q = q, a.dtype = dtype;
    a.o_st = a.q_st = (int64_t)num_heads * head_dim;
    a.o_sh = a.q_sh = head_dim;
    a.k_pool = k_pool, a.v_pool = v_pool, a.block_tables = block_tables, a.max_blocks = max_blocks;
    a.kv_lens = context_lens, a.num_seqs = a.rows = batch, a.max_rows = 1;
    a.num_heads = num_heads, a.kv_heads = kv_heads, a.head_dim = head_dim;
    a.block_size = block_size, a.num_slots = num_slots, a.max_kv = max_context_len, a.scale = scale;
    a.window = 0x7fffffff;
    return a;
}

static RangedAttn prefill_call(void* out, int out_dtype, int64_t o_st, int64_t o_sh, const void* q,
                               int64_t q_st, int64_t q_sh, const void* k_pool, const void* v_pool,
                               const int32_t* cu, const int32_t* kv_lens,
                               const int32_t* block_tables, int max_blocks, int num_seqs,
                               int max_seqlen_q, int total_q, int num_heads, int kv_heads,
                               int head_dim, int block_size, int64_t num_slots, int max_kv_len,
                               float scale, int dtype) {
    RangedAttn a = decode_call(out, out_dtype, q, k_pool, v_pool, block_tables, max_blocks, kv_lens,
                               num_seqs, num_heads, kv_heads, head_dim, block_size, num_slots,
                               max_kv_len, scale, dtype);
    a.o_st = o_st, a.o_sh = o_sh, a.q_st = q_st, a.q_sh = q_sh;
    a.cu = cu, a.max_rows = max_seqlen_q, a.rows = total_q;
    return a;
}

static bool check_sizes(const char* what, int num_seqs, int max_seqlen_q, int total_q, int num_heads,
                        int kv_heads, int head_dim, int max_kv_len, int dtype, size_t* bytes) {
    if (!bytes || num_seqs < 0 || max_seqlen_q < 0 || total_q < 0 || num_heads <= 0 ||
        kv_heads <= 0 || num_heads % kv_heads != 0 || head_dim <= 0 || max_kv_len < 0 ||
        !valid_dtype(dtype)) {
        set_error("%s: bad arguments", what);
        return false;
    }
    return true;
}

}  // namespace flour

using namespace flour;

extern "C" int flour_hip_window_workspace_size(int num_seqs, int max_seqlen_q, int total_q,
                                               int num_heads, int kv_heads, int head_dim,
                                               int max_kv_len, int window, int sinks, int dtype,
                                               size_t* bytes) {
    clear_error();
    if (!check_sizes("window_workspace_size", num_seqs, max_seqlen_q, total_q, num_heads, kv_heads,
                     head_dim, max_kv_len, dtype, bytes))
        return FLOUR_ERR_INVALID_ARGUMENT;
    if (window < 1 || sinks < 0) {
        set_error("window_workspace_size: window %d with %d sinks", window, sinks);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    *bytes = 0;
    return FLOUR_OK;
}

extern "C" int flour_hip_shared_workspace_size(int num_seqs, int num_groups, int max_seqlen_q,
                                               int total_q, int num_heads, int kv_heads,
                                               int head_dim, int max_kv_len, int max_shared_len,
                                               int dtype, size_t* bytes) {
    clear_error();
    if (!check_sizes("shared_workspace_size", num_seqs, max_seqlen_q, total_q, num_heads, kv_heads,
                     head_dim, max_kv_len, dtype, bytes))
        return FLOUR_ERR_INVALID_ARGUMENT;
    if (num_groups < 0 || max_shared_len < 0) {
        set_error("shared_workspace_size: %d groups with prefixes of up to %d positions", num_groups,
                  max_shared_len);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    *bytes = 0;
    return FLOUR_OK;
}

extern "C" int flour_hip_paged_decode_window(
    void* out, int out_dtype, const void* q, const void* k_pool, const void* v_pool,
    const int32_t* block_tables, int max_blocks_per_seq, const int32_t* context_lens, int batch,
    int num_heads, int kv_heads, int head_dim, int block_size, int64_t num_slots,
    int max_context_len, int window, int sinks, float scale, int dtype, void* workspace,
    size_t workspace_bytes, void* stream) {
    clear_error();
    RangedAttn a = decode_call(out, out_dtype, q, k_pool, v_pool, block_tables, max_blocks_per_seq,
                               context_lens, batch, num_heads, kv_heads, head_dim, block_size,
                               num_slots, max_context_len, scale, dtype);
    a.window = window, a.sinks = sinks;
    return ranged_call("paged_decode_window", a, false, workspace, workspace_bytes,
                       static_cast<hipStream_t>(stream));
}

extern "C" int flour_hip_varlen_prefill_window(
    void* out, int out_dtype, int64_t o_stride_tok, int64_t o_stride_head, const void* q,
    int64_t q_stride_tok, int64_t q_stride_head, const void* k_pool, const void* v_pool,
    const int32_t* cu_seqlens_q, const int32_t* kv_lens, const int32_t* block_tables,
    int max_blocks_per_seq, int num_seqs, int max_seqlen_q, int total_q, int num_heads,
    int kv_heads, int head_dim, int block_size, int64_t num_slots, int max_kv_len, int window,
    int sinks, float scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    RangedAttn a = prefill_call(out, out_dtype, o_stride_tok, o_stride_head, q, q_stride_tok,
                                q_stride_head, k_pool, v_pool, cu_seqlens_q, kv_lens, block_tables,
                                max_blocks_per_seq, num_seqs, max_seqlen_q, total_q, num_heads,
                                kv_heads, head_dim, block_size, num_slots, max_kv_len, scale, dtype);
    a.window = window, a.sinks = sinks;
    if (num_seqs > 0 && total_q > 0 && !cu_seqlens_q) {
        set_error("varlen_prefill_window: null pointer");
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    return ranged_call("varlen_prefill_window", a, false, workspace, workspace_bytes,
                       static_cast<hipStream_t>(stream));
}

extern "C" int flour_hip_paged_decode_shared(
    void* out, int out_dtype, const void* q, const void* k_pool, const void* v_pool,
    const int32_t* block_tables, int max_blocks_per_seq, const int32_t* context_lens, int batch,
    const int32_t* group_starts, const int32_t* shared_lens, int num_groups, int num_heads,
    int kv_heads, int head_dim, int block_size, int64_t num_slots, int max_context_len,
    int max_shared_len, float scale, int dtype, void* workspace, size_t workspace_bytes,
    void* stream) {
    clear_error();
    RangedAttn a = decode_call(out, out_dtype, q, k_pool, v_pool, block_tables, max_blocks_per_seq,
                               context_lens, batch, num_heads, kv_heads, head_dim, block_size,
                               num_slots, max_context_len, scale, dtype);
    a.group_starts = group_starts, a.shared_lens = shared_lens, a.num_groups = num_groups;
    a.max_shared = max_shared_len;
    return ranged_call("paged_decode_shared", a, true, workspace, workspace_bytes,
                       static_cast<hipStream_t>(stream));
}

extern "C" int flour_hip_varlen_prefill_shared(
    void* out, int out_dtype, int64_t o_stride_tok, int64_t o_stride_head, const void* q,
    int64_t q_stride_tok, int64_t q_stride_head, const void* k_pool, const void* v_pool,
    const int32_t* cu_seqlens_q, const int32_t* kv_lens, const int32_t* block_tables,
    int max_blocks_per_seq, int num_seqs, const int32_t* group_starts, const int32_t* shared_lens,
    int num_groups, int max_seqlen_q, int total_q, int num_heads, int kv_heads, int head_dim,
    int block_size, int64_t num_slots, int max_kv_len, int max_shared_len, float scale, int dtype,
    void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    RangedAttn a = prefill_call(out, out_dtype, o_stride_tok, o_stride_head, q, q_stride_tok,
                                q_stride_head, k_pool, v_pool, cu_seqlens_q, kv_lens, block_tables,
                                max_blocks_per_seq, num_seqs, max_seqlen_q, total_q, num_heads,
                                kv_heads, head_dim, block_size, num_slots, max_kv_len, scale, dtype);
    a.group_starts = group_starts, a.shared_lens = shared_lens, a.num_groups = num_groups;
    a.max_shared = max_shared_len;
    if (num_seqs > 0 && total_q > 0 && !cu_seqlens_q) {
        set_error("varlen_prefill_shared: null pointer");
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    return ranged_call("varlen_prefill_shared", a, true, workspace, workspace_bytes,
                       static_cast<hipStream_t>(stream));
}
