// cache8_attn.cpp — C entries of the attention over 8-bit caches and of the attention-weight sums:
// argument checks, workspaces and the choice of the kernel.
#include <algorithm>

#include "cache8.h"
#include "decode_pools.h"

namespace flour {

static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

static int64_t score_stride_of(int max_ctx) { return ((int64_t)max_ctx + 63) / 64 * 64; }

// ---- the streamed kernel
// What the shape says of it; a call's tensors can still refuse it (stream_takes).
static bool stream_fits(int batch, int rows, int max_rows, int n_rep, int max_kv, int head_dim,
                        int block_size) {
    // (chunks of 32 positions, or more, of groups of 16 columns, or more: counted in 32 bits)
    const double chunks =
        (double)batch * (max_kv / 32 + 1.0) * ((double)max_rows * n_rep / 16 + 1.0);
    return (head_dim == 64 || head_dim == 128) && chunks < 2e9 && block_size % 16 == 0 &&
           batch <= 4096 && rows <= 65535;
}

static bool stream_takes(const PoolAttn& a, int max_rows) {
    const int es = elem_bytes(a.dtype), oes = elem_bytes(a.out_dtype);
    return valid_pool8(a.pool_dtype) &&
           stream_fits(a.batch, a.rows, max_rows, a.num_heads / a.kv_heads, a.max_kv, a.head_dim,
                       a.block_size) &&
           a.num_slots * a.head_dim <= (int64_t)0x7fffffff &&
           (((uint64_t)(uintptr_t)a.q | (uint64_t)(uintptr_t)a.out | (uint64_t)(uintptr_t)a.k_pool |
             (uint64_t)(uintptr_t)a.v_pool | (uint64_t)(a.q_st * es) | (uint64_t)(a.q_sh * es) |
             (uint64_t)(a.o_st * oes) | (uint64_t)(a.o_sh * oes)) & 15) == 0;
}

static size_t stream_bytes(int batch, int64_t max_cols, int head_dim) {
    return head_dim == 64 || head_dim == 128 ? decode_stream_bytes(batch, max_cols, head_dim) : 0;
}

static int launch_stream_call(const PoolAttn& p, int max_rows, void* ws, hipStream_t stream) {
    DpArgs a{};
    a.out = p.out, a.out_dtype = p.out_dtype, a.o_st = p.o_st, a.o_sh = p.o_sh;
    a.q = p.q, a.q_st = p.q_st, a.q_sh = p.q_sh;
    a.k_pool = static_cast<const uint8_t*>(p.k_pool);
    a.v_pool = static_cast<const uint8_t*>(p.v_pool);
    a.k_scale = p.k_scale, a.v_scale = p.v_scale;
    a.cu = p.cu, a.kv_lens = p.kv_lens, a.block_tables = p.block_tables;
    a.max_blocks = p.max_blocks, a.batch = p.batch, a.num_heads = p.num_heads;
    a.kv_heads = p.kv_heads, a.n_rep = p.num_heads / p.kv_heads, a.block_size = p.block_size;
    a.num_slots = p.num_slots, a.scale_log2 = p.scale * LOG2_E, a.max_kv = p.max_kv;
    a.scores = p.scores, a.score_stride = p.score_stride, a.ml = p.ml;
    auto launch = p.dtype == FLOUR_DTYPE_F32    ? launch_decode_stream_f32
                  : p.dtype == FLOUR_DTYPE_BF16 ? launch_decode_stream_bf16
                                                : launch_decode_stream_f16;
    return launch(a, p.pool_dtype, p.head_dim, ws, max_rows, p.rows, stream);
}

// ---- decode
// Workspace: whichever kernel's part is the larger, then (with weights) the scores' maxima and sums
// and the scores.
static size_t decode_part(int batch, int n_rep, int head_dim) {
    return up256(std::max(paged_decode_scores_bytes(batch, n_rep, head_dim),
                          stream_bytes(batch, n_rep, head_dim)));
}
static size_t weights_part(int batch, int num_heads, int max_ctx) {
    const size_t rows = (size_t)batch * num_heads;
    return up256(rows * 2 * sizeof(float)) + up256(rows * score_stride_of(max_ctx) * sizeof(float));
}

static int decode_pools(const char* what, PoolAttn a, float* weights, int64_t width,
                        const int32_t* weight_rows, int num_rows, void* workspace,
                        size_t workspace_bytes, hipStream_t stream) {
    if (!valid_dtype(a.dtype) || !valid_dtype(a.out_dtype)) {
        set_error("%s: unknown dtype (%d, out %d)", what, a.dtype, a.out_dtype);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    if (a.batch < 0 || a.num_heads <= 0 || a.kv_heads <= 0 || a.num_heads % a.kv_heads != 0 ||
        a.head_dim <= 0 || a.block_size <= 0 || a.num_slots <= 0 ||
        a.num_slots % a.block_size != 0 || a.max_blocks <= 0 || a.max_kv < 0 ||
        (int64_t)a.max_kv > (int64_t)a.max_blocks * a.block_size) {
        set_error("%s: bad shape (batch=%d heads=%d kv_heads=%d head_dim=%d bs=%d num_slots=%lld "
                  "max_blocks=%d max_ctx=%d)",
                  what, a.batch, a.num_heads, a.kv_heads, a.head_dim, a.block_size,
                  (long long)a.num_slots, a.max_blocks, a.max_kv);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    if (weights && (width < a.max_kv || num_rows < 0 || (!weight_rows && num_rows < a.batch))) {
        set_error("%s: weights of %d rows of width %lld for %d sequences of up to %d positions",
                  what, num_rows, (long long)width, a.batch, a.max_kv);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    if (weights && (a.batch > 65535 || a.kv_heads > 65535)) {
        set_error("%s: weights of %d kv heads of %d sequences are too many for one call", what,
                  a.kv_heads, a.batch);
        return FLOUR_ERR_UNSUPPORTED;
    }
    if (a.batch == 0) return FLOUR_OK;
    if (!a.out || !a.q || !a.k_pool || !a.v_pool || !a.block_tables || !a.kv_lens) {
        set_error("%s: null pointer", what);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    const int n_rep = a.num_heads / a.kv_heads;
    const size_t part = decode_part(a.batch, n_rep, a.head_dim);
    const size_t need = part + (weights ? weights_part(a.batch, a.num_heads, a.max_kv) : 0);
    if ((!workspace || workspace_bytes < need || (uintptr_t)workspace % 256 != 0)) {
        set_error("%s: workspace of %zu bytes (256-byte aligned) required, got %zu at %p", what,
                  need, workspace_bytes, workspace);
        return FLOUR_ERR_WORKSPACE;
    }
    a.rows = a.batch;
    a.q_st = a.o_st = (int64_t)a.num_heads * a.head_dim;
    a.q_sh = a.o_sh = a.head_dim;
    if (weights) {
        char* ws = static_cast<char*>(workspace) + part;
        a.ml = reinterpret_cast<float*>(ws);
        a.scores = reinterpret_cast<float*>(
            ws + up256((size_t)a.batch * a.num_heads * 2 * sizeof(float)));
        a.score_stride = score_stride_of(a.max_kv);
    }
    int rc;
    if (stream_takes(a, 1))
        rc = launch_stream_call(a, 1, workspace, stream);
    else if (!valid_pool8(a.pool_dtype) && a.score_stride <= 0x7fffffff / 16 &&  // (a lane's 32-bit offset)
             paged_decode_scores_takes(a.dtype, a.head_dim, a.block_size, n_rep, a.batch, a.num_heads,
                                       a.num_slots, a.out, a.q, a.k_pool, a.v_pool))
        rc = paged_decode_scores(a.out, a.out_dtype, a.q, a.k_pool, a.v_pool, a.block_tables,
                                 a.max_blocks, a.kv_lens, a.batch, a.num_heads, a.kv_heads,
                                 a.head_dim, a.block_size, a.num_slots, a.max_kv, a.scale, a.dtype,
                                 workspace, part, a.scores, a.score_stride, a.ml, stream);
    else
        rc = launch_attn_pools(a, stream);
    if (rc != FLOUR_OK || !weights) return rc;
    return launch_weights_add(weights, width, weight_rows, num_rows, a.kv_lens, a.max_kv, a.batch,
                              a.kv_heads, n_rep, a.scores, a.score_stride, a.ml, stream);
}

}  // namespace flour

using namespace flour;

extern "C" int flour_hip_decode_weights_workspace_size(int batch, int num_heads, int kv_heads,
                                                       int head_dim, int max_context_len,
                                                       int with_weights, size_t* bytes) {
    clear_error();
    if (!bytes || batch < 0 || num_heads <= 0 || kv_heads <= 0 || num_heads % kv_heads != 0 ||
        head_dim <= 0 || max_context_len < 0) {
        set_error("decode_weights_workspace_size: bad arguments");
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    *bytes = decode_part(batch, num_heads / kv_heads, head_dim) +
             (with_weights ? weights_part(batch, num_heads, max_context_len) : 0);
    return FLOUR_OK;
}

extern "C" int flour_hip_paged_decode_q8(
    void* out, int out_dtype, const void* q, int dtype, const void* k_pool, const void* v_pool,
    const float* k_scale, const float* v_scale, int pool_dtype, const int32_t* block_tables,
    int max_blocks_per_seq, const int32_t* context_lens, int batch, int num_heads, int kv_heads,
    int head_dim, int block_size, int64_t num_slots, int max_context_len, float scale,
    float* weights, int64_t weights_width, const int32_t* weight_rows, int num_weight_rows,
    void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    if (!check_pool8("paged_decode_q8", pool_dtype, k_pool, v_pool, k_scale, v_scale, kv_heads,
                     head_dim, block_size, num_slots))
        return FLOUR_ERR_INVALID_ARGUMENT;
    PoolAttn a{};
    a.out = out, a.out_dtype = out_dtype, a.q = q, a.dtype = dtype;
    a.k_pool = k_pool, a.v_pool = v_pool, a.k_scale = k_scale, a.v_scale = v_scale;
    a.pool_dtype = pool_dtype, a.block_tables = block_tables, a.max_blocks = max_blocks_per_seq;
    a.kv_lens = context_lens, a.batch = batch, a.num_heads = num_heads, a.kv_heads = kv_heads;
    a.head_dim = head_dim, a.block_size = block_size, a.num_slots = num_slots;
    a.max_kv = max_context_len, a.scale = scale;
    return decode_pools("paged_decode_q8", a, weights, weights_width, weight_rows, num_weight_rows,
                        workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int flour_hip_paged_decode_weights(
    void* out, int out_dtype, const void* q, const void* k_pool, const void* v_pool,
    const int32_t* block_tables, int max_blocks_per_seq, const int32_t* context_lens, int batch,
    int num_heads, int kv_heads, int head_dim, int block_size, int64_t num_slots,
    int max_context_len, float scale, int dtype, float* weights, int64_t weights_width,
    const int32_t* weight_rows, int num_weight_rows, void* workspace, size_t workspace_bytes,
    void* stream) {
    clear_error();
    if (!weights) {
        set_error("paged_decode_weights: null weights");
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    PoolAttn a{};
    a.out = out, a.out_dtype = out_dtype, a.q = q, a.dtype = dtype;
    a.k_pool = k_pool, a.v_pool = v_pool, a.pool_dtype = dtype;
    a.block_tables = block_tables, a.max_blocks = max_blocks_per_seq;
    a.kv_lens = context_lens, a.batch = batch, a.num_heads = num_heads, a.kv_heads = kv_heads;
    a.head_dim = head_dim, a.block_size = block_size, a.num_slots = num_slots;
    a.max_kv = max_context_len, a.scale = scale;
    return decode_pools("paged_decode_weights", a, weights, weights_width, weight_rows,
                        num_weight_rows, workspace, workspace_bytes,
                        static_cast<hipStream_t>(stream));
}

namespace flour {

// ---- prefill
// Few rows run on the streamed kernel, which reads the 8-bit rows once per group of up to 32 columns;
// others stage the sequences' values once as a plain pool of the queries' type, whose blocks lie in order,
// for the prefill kernels. bf16 and fp32 hold q * S of any block whose S is a power of two; f16 those
// within its range, so with f16 queries the heads that have others are computed again from the 8 bits
// (attn_beyond_f16_kernel). A batch whose staged copy would be larger than STAGE_BYTES goes slice by slice (whole
// sequences) through one copy.
static int g_prefill_q8 = 0;  // 0: by the rule, 1: streamed, 2: staged, 3: the kernel for every shape

static constexpr size_t STAGE_BYTES = (size_t)1 << 30;

struct Stage {
    int slice;        // sequences a slice
    int blocks;       // of a sequence
    int64_t slots;    // of a slice's pool
    size_t pool;      // bytes of K (and of V)
    size_t table, lens, v_stage, total;
};

// The staged copy of a call within `limit` bytes: slices of as many sequences as STAGE_BYTES and the limit
// allow, and the prefill kernel's own copy of V where it wants one; false where none fits or no such
// kernel takes the shape.
static bool stage_of(int num_seqs, int max_seqlen_q, int total_q, int max_kv, int kv_heads,
                     int head_dim, int block_size, int dtype, size_t limit, Stage* st) {
    if (num_seqs <= 0 || max_kv <= 0 || (head_dim != 64 && head_dim != 128)) return false;
    st->blocks = (int)(((int64_t)max_kv + block_size - 1) / block_size);
    const size_t seq = (size_t)st->blocks * block_size * head_dim * elem_bytes(dtype);  // of a head
    if (seq > 0x7fffffff) return false;
    // (a head's part of the pool stays below 2^31 bytes: the kernels' limit)
    const size_t fit = std::min<size_t>(STAGE_BYTES / (2 * seq * kv_heads), 0x7fffffff / seq);
    st->slice = (int)std::min<size_t>(std::max<size_t>(fit, 1), num_seqs);
    bool copy_v = prefill_wants_v_stage(num_seqs, total_q);
    for (;;) {
        size_t v = 0;
        if (copy_v &&
            flour_hip_varlen_prefill_workspace_size(st->slice, st->blocks, block_size, kv_heads,
                                                    head_dim, dtype, &v) != FLOUR_OK)
            return false;
        st->pool = up256(seq * st->slice * kv_heads);
        st->table = up256((size_t)st->slice * st->blocks * sizeof(int32_t));
        st->lens = up256((size_t)st->slice * sizeof(int32_t));
        st->v_stage = up256(v);
        st->total = 2 * st->pool + st->table + st->lens + st->v_stage;
        if (st->total <= limit) break;
        if (st->slice > 1)
            st->slice = std::max(1, std::min(st->slice - 1, (int)((double)st->slice * limit / st->total)));
        else if (copy_v)
            copy_v = false;
        else
            return false;
    }
    st->slots = (int64_t)st->slice * st->blocks * block_size;
    const bool mfma = prefill_mfma_supported(dtype, head_dim, block_size, st->slots, 1.0f, 0);
    return mfma || prefill_f32_mfma_supported(dtype, head_dim, st->slice, max_seqlen_q, block_size,
                                              st->slots);
}

// Whether a call runs streamed rather than staged: estimates of both in us, from the bounds that the host
// knows (total_q rows in all, max_kv positions of each sequence).
//  * Streamed: 10, the cache once per group of 32 columns, 7.8e-5 us a position and kv head at head_dim 128
//    (9.4e-5 with fp32 queries), 6.1e-5 at 64, and up to 14 for the pieces of the groups. Positions that a
//    group does not see are read all the same.
//  * Staged: 11 (16 in fp32; 18 in f16, whose scales are looked at again, attn_beyond_f16_kernel), the copy at
//    5 TB/s, and the prefill kernel: at least one item's walk over the kv positions (24 ns each at
//    head_dim 128, 13.5 at 64; fp32 55 and 24), or the products of the causal range at 650 TFLOP/s (fp32
//    110, rows in tiles of 32).
// Measured, streamed / staged, 32 / 8 heads of 128 in bf16: 1 x 4,096 tokens with 32 rows 35 / 109, 8 x
// 4,096 with 8 39 / 132 and with 128 268 / 159, 32 x 512 with 32 76 / 45; fp32 32 x 2,048 with 32 185 /
// 637; 14 / 2 heads of 64 8 x 1,024 with 64 41 / 26. Of 1,500 drawn calls, cold prompts among them, 58 are
// more than 10% slower than on the other path, 1.7 times the most; in the mean it is 1.7%.
static bool prefer_stream(int batch, int total_q, int max_rows, int max_kv, int num_heads, int kv_heads,
                          int head_dim, int dtype) {
    const bool f32 = dtype == FLOUR_DTYPE_F32, d64 = head_dim == 64;
    const int n_rep = num_heads / kv_heads;
    const double seqs = batch, rows = std::min((double)total_q, seqs * max_rows);
    const double groups = std::max(rows * n_rep / 32 + 0.5 * seqs, seqs);
    const double pieces = (double)(((int64_t)max_rows * n_rep + 31) / 32);
    const double streamed =
        10 + groups * kv_heads * max_kv * (d64 ? 6.1e-5 : f32 ? 9.4e-5 : 7.8e-5) +
        std::min(2 * pieces, 14.0);
    const double walk = max_kv * (f32 ? (d64 ? 0.024 : 0.055) : (d64 ? 0.0135 : 0.024));
    const double seen = std::max(max_kv - rows / seqs / 2, 0.0);  // by a row, in the mean
    const double flops = 4.0 * (rows + (f32 ? 16 * seqs : 0)) * seen * num_heads * head_dim;
    const double copy = seqs * kv_heads * max_kv * head_dim * 2 * (1 + elem_bytes(dtype)) / 5e6;
    const double staged = (f32 ? 16 : dtype == FLOUR_DTYPE_F16 ? 18 : 11) + copy +
                          std::max(walk, flops / (f32 ? 1.1e8 : 6.5e8));
    return streamed < staged;
}

static int prefill_staged(const PoolAttn& a, const Stage& st, int max_rows, char* ws,
                          hipStream_t stream) {
    void *k = ws, *v = ws + st.pool;
    int32_t* table = reinterpret_cast<int32_t*>(ws + 2 * st.pool);
    int32_t* lens = reinterpret_cast<int32_t*>(ws + 2 * st.pool + st.table);
    void* v_stage = st.v_stage ? ws + 2 * st.pool + st.table + st.lens : nullptr;
    for (int s0 = 0; s0 < a.batch; s0 += st.slice) {
        const int n = std::min(st.slice, a.batch - s0);
        int rc = launch_kv_dequant(k, v, a.dtype, nullptr, st.blocks, st.slots, a.k_pool, a.v_pool,
                                   a.k_scale, a.v_scale, a.pool_dtype,
                                   a.block_tables + (int64_t)s0 * a.max_blocks, a.max_blocks,
                                   a.kv_lens + s0, n, a.max_kv, a.kv_heads, a.head_dim, a.block_size,
                                   a.num_slots, table, lens, stream);
        if (rc != FLOUR_OK) return rc;
        // (the matrix-core kernels take a sequence's rows from cu[s], cu[s + 1] alone; total_q only guides
        // their choice: the slice's share of the rows, which the host knows in all alone)
        const int rows = (int)std::max<int64_t>(1, (int64_t)a.rows * n / a.batch);
        rc = varlen_prefill_rows(a.out, a.out_dtype, a.o_st, a.o_sh, a.q, a.q_st, a.q_sh, k, v,
                                 a.cu + s0, nullptr, lens, table, st.blocks, n, max_rows,
                                 rows, a.num_heads, a.kv_heads, a.head_dim, a.block_size,
                                 st.slots, a.scale, a.dtype, v_stage, st.v_stage, a.max_kv, stream);
        if (rc != FLOUR_OK) return rc;
    }
    return a.dtype == FLOUR_DTYPE_F16 ? launch_attn_beyond_f16(a, max_rows, stream) : FLOUR_OK;
}

// Whether the prefill kernels that read rows by cu alone take the call's q and out.
static bool stage_takes(const PoolAttn& a, const Stage& st, int max_rows) {
    const int es = elem_bytes(a.dtype), oes = elem_bytes(a.out_dtype);
    const uint64_t bits = (uint64_t)(uintptr_t)a.q | (uint64_t)(uintptr_t)a.out |
                          (uint64_t)(a.q_st * es) | (uint64_t)(a.q_sh * es) |
                          (uint64_t)(a.o_st * oes) | (uint64_t)(a.o_sh * oes);
    if (bits & 15) return false;
    return prefill_mfma_supported(a.dtype, a.head_dim, a.block_size, st.slots, a.scale, a.q_st) ||
           prefill_f32_mfma_supported(a.dtype, a.head_dim, st.slice, max_rows, a.block_size,
                                      st.slots);
}

}  // namespace flour

extern "C" int flour_hip_set_prefill_q8(int mode) {
    if (mode < 0 || mode > 3) {
        flour::set_error("set_prefill_q8: mode %d is not 0 to 3", mode);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    flour::g_prefill_q8 = mode;
    flour::switch_set();
    return FLOUR_OK;
}

extern "C" int flour_hip_varlen_prefill_q8_workspace_size(int num_seqs, int max_seqlen_q,
                                                          int total_q, int max_kv_len,
                                                          int num_heads, int kv_heads,
                                                          int head_dim, int block_size, int dtype,
                                                          size_t* bytes) {
    clear_error();
    if (!bytes || num_seqs < 0 || max_seqlen_q < 0 || total_q < 0 || max_kv_len < 0 ||
        num_heads <= 0 || kv_heads <= 0 || num_heads % kv_heads != 0 || head_dim <= 0 ||
        block_size <= 0 || !valid_dtype(dtype)) {
        set_error("varlen_prefill_q8_workspace_size: bad arguments");
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    const int n_rep = num_heads / kv_heads, mode = g_prefill_q8;
    const bool streamed = mode != 3 && stream_fits(num_seqs, total_q, max_seqlen_q, n_rep, max_kv_len,
                                                   head_dim, block_size);
    const bool preferred =
        streamed && (mode == 1 || (mode == 0 && prefer_stream(num_seqs, total_q, max_seqlen_q, max_kv_len,
                                                              num_heads, kv_heads, head_dim, dtype)));
    *bytes = streamed ? stream_bytes(num_seqs, (int64_t)max_seqlen_q * n_rep, head_dim) : 0;
    Stage st{};
    if (mode != 3 && !preferred &&
        stage_of(num_seqs, max_seqlen_q, total_q, max_kv_len, kv_heads, head_dim, block_size, dtype,
                 SIZE_MAX, &st))
        *bytes = std::max(*bytes, st.total);
    return FLOUR_OK;
}

extern "C" int flour_hip_varlen_prefill_q8(
    void* out, int out_dtype, int64_t o_stride_tok, int64_t o_stride_head, const void* q,
    int64_t q_stride_tok, int64_t q_stride_head, int dtype, const void* k_pool, const void* v_pool,
    const float* k_scale, const float* v_scale, int pool_dtype, const int32_t* cu_seqlens_q,
    const int32_t* kv_lens, const int32_t* block_tables, int max_blocks_per_seq, int num_seqs,
    int max_seqlen_q, int total_q, int num_heads, int kv_heads, int head_dim, int block_size,
    int64_t num_slots, int max_kv_len, float scale, void* workspace, size_t workspace_bytes,
    void* stream) {
    clear_error();
    if (!valid_dtype(dtype) || !valid_dtype(out_dtype)) {
        set_error("varlen_prefill_q8: unknown dtype (%d, out %d)", dtype, out_dtype);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    if (!check_pool8("varlen_prefill_q8", pool_dtype, k_pool, v_pool, k_scale, v_scale, kv_heads,
                     head_dim, block_size, num_slots))
        return FLOUR_ERR_INVALID_ARGUMENT;
    if (num_seqs < 0 || total_q < 0 || max_seqlen_q < 0 || num_heads <= 0 ||
        num_heads % kv_heads != 0 || max_blocks_per_seq <= 0 || max_kv_len < 0 ||
        (int64_t)max_kv_len > (int64_t)max_blocks_per_seq * block_size) {
        set_error("varlen_prefill_q8: bad shape (seqs=%d total_q=%d max_q=%d heads=%d kv_heads=%d "
                  "max_blocks=%d max_kv=%d)",
                  num_seqs, total_q, max_seqlen_q, num_heads, kv_heads, max_blocks_per_seq,
                  max_kv_len);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    if (num_seqs == 0 || total_q == 0 || max_seqlen_q == 0) return FLOUR_OK;
    if (!out || !q || !cu_seqlens_q || !kv_lens || !block_tables) {
        set_error("varlen_prefill_q8: null pointer");
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    PoolAttn a{};
    a.out = out, a.out_dtype = out_dtype, a.o_st = o_stride_tok, a.o_sh = o_stride_head;
    a.q = q, a.dtype = dtype, a.q_st = q_stride_tok, a.q_sh = q_stride_head;
    a.k_pool = k_pool, a.v_pool = v_pool, a.k_scale = k_scale, a.v_scale = v_scale;
    a.pool_dtype = pool_dtype, a.cu = cu_seqlens_q, a.kv_lens = kv_lens;
    a.block_tables = block_tables, a.max_blocks = max_blocks_per_seq, a.batch = num_seqs;
    a.rows = total_q, a.num_heads = num_heads, a.kv_heads = kv_heads, a.head_dim = head_dim;
    a.block_size = block_size, a.num_slots = num_slots, a.max_kv = max_kv_len, a.scale = scale;
    const int n_rep = num_heads / kv_heads, mode = g_prefill_q8;
    const bool fits = mode != 3 && stream_fits(num_seqs, total_q, max_seqlen_q, n_rep, max_kv_len,
                                               head_dim, block_size);
    // (a staged copy takes what there is beyond that: workspaces of other shapes serve)
    const size_t need = fits ? stream_bytes(num_seqs, (int64_t)max_seqlen_q * n_rep, head_dim) : 0;
    if ((workspace && (uintptr_t)workspace % 256 != 0) || workspace_bytes < need ||
        (!workspace && need > 0)) {
        set_error("varlen_prefill_q8: workspace of %zu bytes (256-byte aligned) required, got %zu at "
                  "%p",
                  need, workspace_bytes, workspace);
        return FLOUR_ERR_WORKSPACE;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    Stage st{};
    const bool streamed = fits && stream_takes(a, max_seqlen_q);
    if (streamed && (mode == 1 || (mode == 0 && prefer_stream(num_seqs, total_q, max_seqlen_q, max_kv_len,
                                                              num_heads, kv_heads, head_dim, dtype))))
        return launch_stream_call(a, max_seqlen_q, workspace, s);
    if (mode != 3 &&
        stage_of(num_seqs, max_seqlen_q, total_q, max_kv_len, kv_heads, head_dim, block_size, dtype,
                 workspace ? workspace_bytes : 0, &st) &&
        stage_takes(a, st, max_seqlen_q))
        return prefill_staged(a, st, max_seqlen_q, static_cast<char*>(workspace), s);
    if (streamed) return launch_stream_call(a, max_seqlen_q, workspace, s);
    return launch_attn_pools(a, s);
}
