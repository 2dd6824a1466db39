// paged_decode.hip — kernel (2): paged decode attention on gfx950 matrix cores.
//
// Replaces paged_attention (src/backend/cpu.rs:57-112) for one new query per sequence
// (seq_q == 1, the decode step engine.rs:259-262), batched over sequences. The block list of
// Cache::kv_blocks (cache.rs:456-458, KvCache::gather_blocks cache.rs:83-96) arrives as a
// block table; query head h reads kv head h / n_rep (repeat_kv, cpu.rs:5-13); with seq_q == 1
// the causal mask of cpu.rs:88-95 admits every cached position, so only positions past the
// context length are masked.
//
// Work decomposition (stream-K at wave granularity): the K/V to read is the list of 32-token
// chunks of every (sequence, kv head) pair, laid end to end. One resident round of one-wave
// workgroups (3 per CU) each takes an equal contiguous range of that list, so every
// wave streams the same number of bytes whatever the spread of context lengths, and no wave
// pays a launch or a ramp-up twice. A pair wholly inside one range is finished by its wave; a
// pair cut by range ends leaves one partial (max, sum, acc) row per piece, and a small second
// kernel on the same stream merges those (log-sum-exp merge, as in the running update of
// cpu.rs:96-105). The kernel boundary orders partial writes before merge reads; an in-kernel
// "last workgroup merges" scheme would need an agent-scope release/acquire per workgroup,
// which on this multi-XCD part writes back and invalidates the XCD's L2 each time.
//
// Inside a piece (bf16/f16 pools, head_dim 128 or 64, block_size a multiple of 16; the
// figures below are for head_dim 128, and head_dim 64 halves every row: 8-byte lane loads, a
// 128-byte row per 16 lanes, 16 output dims per lane instead of 32):
//  * The wave walks its piece chunk by chunk. A chunk is two 16-token MFMA tiles, each one
//    4 KB (head, 16 slots) pool run of K and of V, read with buffer loads (per-pool resource,
//    loop-invariant lane offset, per-tile SGPR offset; non-temporal, whole rows per
//    instruction; K is turned into the MFMA layout through LDS); two register buffers
//    ping-pong so the next chunk's loads are in flight while one is computed, with the loop
//    peeled so that no load is conditional. Every query head of the kv head shares each K/V
//    load (GQA reuse: K/V leave HBM once).
//  * Scores S = K Q^T on v_mfma_f32_16x16x32 (M = 16 tokens, N = 16 query-head columns, the
//    n_rep real heads padded with zero rows): lane (g, c) = (lane/16, lane%16) holds head c's
//    scores for tokens 4g..4g+3 of each tile.
//  * Those registers, for the two tiles, are exactly the B operand of v_mfma_f32_16x16x32 for
//    O^T = V^T P^T (K = the 32 tokens), so P never leaves the lane. The V^T A operand is built
//    in-lane: each lane loads V rows 4g..4g+3, dims 8c..8c+7 (a wave reads 4 whole 256 B rows
//    per instruction) and v_perm_b32 packs, per output dim 8c+n, the four tokens' values. The
//    O^T accumulator holds, in lane (g, c), query head c at dims 32g..32g+31.
//  * P is split into hi + lo 16-bit parts (two MFMAs per product) so the P.V contraction keeps
//    ~16 mantissa bits of P; products are exact in fp32 and accumulate in fp32.
//  * fp32 pools (longer steps, decode_f32_split): the same stream over 16-token chunks of the same
//    bytes, on v_mfma_f32_16x16x4 in fp32 end to end. A wave instruction reads four 256 B row
//    segments; the score registers are the B operand as they stand (one product per token group
//    and 16 dims) and V registers the A operand, so only K goes through LDS. HBM-bound: 16 x
//    256-2,048 tokens of 32 / 8 heads of 128 (129 MB) 108 us on the vector kernel, 36.8 here.
//  * Online softmax in the exp2 domain: the only cross-lane step per chunk is the max over the
//    four row groups (two v_permlane*_swap exchanges); running sums stay lane-partial until
//    the end, and the accumulator is rescaled only when some lane's max moved.
#include <math.h>

#include <atomic>
#include <mutex>
#include <type_traits>

#include "paged_decode_kernel.h"

namespace flour {

bool simt_supported(int dtype, int head_dim, const void* q, int64_t q_st, int64_t q_sh,
                    const void* k_pool, const void* v_pool);
int launch_attn_simt(int dtype, int out_dtype, void* out, int64_t o_st, int64_t o_sh,
                     const void* q, int64_t q_st, int64_t q_sh, const void* k_pool,
                     const void* v_pool, const int32_t* cu, const int32_t* kv_lens,
                     const int32_t* bt, int max_blocks, int num_seqs, int total_q, int num_heads,
                     int n_rep, int head_dim, int block_size, int64_t num_slots, int max_kv,
                     float scale, hipStream_t stream);
int launch_attn_generic(int dtype, int out_dtype, void* out, int64_t o_st, int64_t o_sh,
                        const void* q, int64_t q_st, int64_t q_sh, const void* k_pool,
                        const void* v_pool, const int32_t* cu, const int32_t* kv_lens,
                        const int32_t* bt, int max_blocks, int num_seqs, int total_q,
                        int num_heads, int n_rep, int head_dim, int block_size, int64_t num_slots,
                        int max_kv, float scale, hipStream_t stream);

static int g_wg_override = 0;  // tuning / test hook: number of waves (0 = one resident round)
// Wave-range weight w of WaveRanges (0 .. 16): even-indexed ranges (even XCDs) take w/32 more
// chunks than the mean, odd ones w/32 fewer (a tuning / test switch). Same-box sweep of w = 0 ..
// 4: 2 is best or even on every decode workload (Llama-3-8B batch 5,862 -> 5,989 GB/s, 70B
// batch 6,083 -> 6,231, head_dim-64 batch even).
static int g_xcd_weight = 2;

int decode_workgroups(int dtype) {
    const int per_cu = dtype == FLOUR_DTYPE_F32 ? DEC_WAVES_PER_CU_F32 : DEC_WAVES_PER_CU;
    const int n = g_wg_override > 0 ? g_wg_override : device_cus() * per_cu;
    return n < 4096 ? n : 4096;
}

int decode_xcd_weight() { return g_xcd_weight; }

template <typename T, typename TO, int D>
static int launch_decode_mfma_d(void* out, const void* q, const void* k_pool, const void* v_pool,
                                const int32_t* bt, int max_blocks, const int32_t* ctx_lens,
                                int batch, int num_heads, int kv_heads, int n_rep, int block_size,
                                int64_t num_slots, int max_ctx, float scale, int nwg, DecodeWs ws,
                                hipStream_t stream) {
    const size_t lds = (size_t)(batch + 1) * sizeof(int);
    const bool fuse = ws.k_new != nullptr;
    if (fuse && (block_size != 16 || std::is_same<T, float>::value)) {
        set_error("paged_decode: the fused KV write needs 16-token pages of a 16-bit pool");
        return FLOUR_ERR_UNSUPPORTED;
    }
    const bool wts = ws.scores != nullptr;
    auto kern = block_size == 16 ? paged_decode_mfma_kernel<T, TO, true, D, false, false>
                                 : paged_decode_mfma_kernel<T, TO, false, D, false, false>;
    if constexpr (!std::is_same<T, float>::value)
        if (fuse) kern = paged_decode_mfma_kernel<T, TO, true, D, true, false>;
    if (wts)
        kern = block_size == 16 ? paged_decode_mfma_kernel<T, TO, true, D, false, true>
                                : paged_decode_mfma_kernel<T, TO, false, D, false, true>;
    // no more waves than ranges (range_count) for contexts of max_ctx
    const int64_t chunk = dec_chunk(sizeof(T));
    const int64_t half = (int64_t)batch * kv_heads * ((max_ctx + chunk - 1) / chunk) / 2;
    const int grid = (int)(half < 1 ? 1 : half < nwg ? half : nwg);
    kern<<<dim3(grid), dim3(64), lds, stream>>>(
        static_cast<TO*>(out), static_cast<const T*>(q), static_cast<const T*>(k_pool),
        static_cast<const T*>(v_pool), bt, max_blocks, ctx_lens, batch, num_heads, kv_heads, n_rep,
        block_size, num_slots, max_ctx, scale * LOG2E, ws);
    int rc = check_hip(hipGetLastError(), "paged_decode launch");
    if (rc != FLOUR_OK) return rc;
    const int mw = decode_merge_waves(grid, batch, kv_heads);
    constexpr bool F32 = std::is_same<T, float>::value;
    auto merge = wts ? paged_decode_merge_kernel<TO, D, F32, true>
                     : paged_decode_merge_kernel<TO, D, F32, false>;
    merge<<<dim3(num_heads, batch), dim3(64 * mw), 0, stream>>>(
        static_cast<TO*>(out), batch, num_heads, kv_heads, n_rep, grid, ws);
    return check_hip(hipGetLastError(), "paged_decode merge launch");
}

template <typename T, typename TO>
static int launch_decode_mfma(int head_dim, void* out, const void* q, const void* k_pool,
                              const void* v_pool, const int32_t* bt, int max_blocks,
                              const int32_t* ctx_lens, int batch, int num_heads, int kv_heads,
                              int n_rep, int block_size, int64_t num_slots, int max_ctx,
                              float scale, int nwg, DecodeWs ws, hipStream_t stream) {
    if (head_dim == 64)
        return launch_decode_mfma_d<T, TO, 64>(out, q, k_pool, v_pool, bt, max_blocks, ctx_lens,
                                               batch, num_heads, kv_heads, n_rep, block_size,
                                               num_slots, max_ctx, scale, nwg, ws, stream);
    return launch_decode_mfma_d<T, TO, 128>(out, q, k_pool, v_pool, bt, max_blocks, ctx_lens,
                                            batch, num_heads, kv_heads, n_rep, block_size,
                                            num_slots, max_ctx, scale, nwg, ws, stream);
}

}  // namespace flour

using namespace flour;

namespace flour {
__global__ void empty_kernel() {}
}  // namespace flour

// One empty one-wave workgroup on `stream`: the floor of a kernel launch on this device, timed
// beside the smallest decode workloads (a measurement helper, not part of the header).
extern "C" int flour_hip_empty_launch(void* stream) {
    flour::empty_kernel<<<dim3(1), dim3(64), 0, static_cast<hipStream_t>(stream)>>>();
    return check_hip(hipGetLastError(), "empty launch");
}

extern "C" int flour_hip_set_decode_xcd_weight(int w) {
    if (w < 0 || w > 16) return FLOUR_ERR_INVALID_ARGUMENT;
    g_xcd_weight = w;
    return FLOUR_OK;
}

extern "C" int flour_hip_set_decode_workgroups(int n) {
    if (n < 0 || n > 4096) return FLOUR_ERR_INVALID_ARGUMENT;
    g_wg_override = n;
    switch_set();
    return FLOUR_OK;
}

extern "C" int flour_hip_paged_decode_workspace_size(int batch, int num_heads, int kv_heads,
                                                     int head_dim, int max_context_len,
                                                     size_t* bytes) {
    clear_error();
    if (!bytes || batch < 0 || num_heads <= 0 || kv_heads <= 0 || num_heads % kv_heads != 0 ||
        head_dim <= 0 || max_context_len < 0) {
        set_error("paged_decode_workspace_size: bad arguments");
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    *bytes = decode_ws_bytes(decode_workgroups(FLOUR_DTYPE_F32), num_heads / kv_heads, head_dim, batch);
    return FLOUR_OK;
}

namespace flour {

// Body of flour_hip_paged_decode. `workspace` == nullptr with `ws_from_scratch` set takes the
// split-context workspace from this device's copy of `scratch` (flour_hip_paged_decode_noalloc).
static int paged_decode_impl(void* out, int out_dtype, const void* q, const void* k_pool,
                             const void* v_pool, const int32_t* block_tables,
                             int max_blocks_per_seq, const int32_t* context_lens, int batch,
                             int num_heads, int kv_heads, int head_dim, int block_size,
                             int64_t num_slots, int max_context_len, float scale, int dtype,
                             void* workspace, size_t workspace_bytes, bool ws_from_scratch,
                             const int32_t* rows, const DecodeWs* fused, void* stream);

// ------------------------------------------------------------------ allocation-free variant
// The split-context workspace of flour_hip_paged_decode_noalloc lives in this file-scope device
// array: each device the library runs on holds its own copy, for the life of the process. Host
// code never passes the array's name to a kernel or a copy (on the host it is a stand-in, not a
// device address): it uses the per-device address that hipGetSymbolAddress returns, looked up
// once per device on that device's first call.
static constexpr size_t DEC_SCRATCH_BYTES = (size_t)40 << 20;
static __device__ __align__(256) unsigned char scratch[DEC_SCRATCH_BYTES];
static constexpr int DEC_MAX_DEVICES = 64;
static std::atomic<void*> g_scratch_ptr[DEC_MAX_DEVICES];
static std::mutex g_scratch_mu;

static int scratch_for_current_device(void** ptr) {
    int dev = -1;
    const hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return check_hip(e, "paged_decode_noalloc: hipGetDevice");
    if (dev < 0 || dev >= DEC_MAX_DEVICES) {
        set_error("paged_decode_noalloc: device %d out of range", dev);
        return FLOUR_ERR_UNSUPPORTED;
    }
    void* p = g_scratch_ptr[dev].load(std::memory_order_acquire);
    if (!p) {
        std::lock_guard<std::mutex> lock(g_scratch_mu);
        p = g_scratch_ptr[dev].load(std::memory_order_relaxed);
        if (!p) {
            const hipError_t r = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
            if (r != hipSuccess || !p)
                return check_hip(r != hipSuccess ? r : hipErrorInvalidSymbol,
                                 "paged_decode_noalloc: hipGetSymbolAddress(scratch)");
            g_scratch_ptr[dev].store(p, std::memory_order_release);
        }
    }
    *ptr = p;
    return FLOUR_OK;
}

}  // namespace flour

extern "C" int flour_hip_paged_decode(void* out, int out_dtype, const void* q,
                                      const void* k_pool, const void* v_pool,
                                      const int32_t* block_tables, int max_blocks_per_seq,
                                      const int32_t* context_lens, int batch, int num_heads,
                                      int kv_heads, int head_dim, int block_size,
                                      int64_t num_slots, int max_context_len, float scale,
                                      int dtype, void* workspace, size_t workspace_bytes,
                                      void* stream) {
    clear_error();
    return flour::paged_decode_impl(out, out_dtype, q, k_pool, v_pool, block_tables,
                                    max_blocks_per_seq, context_lens, batch, num_heads, kv_heads,
                                    head_dim, block_size, num_slots, max_context_len, scale, dtype,
                                    workspace, workspace_bytes, false, nullptr, nullptr, stream);
}

extern "C" size_t flour_hip_paged_decode_noalloc_max_workspace(void) {
    return flour::DEC_SCRATCH_BYTES;
}

extern "C" int flour_hip_paged_decode_noalloc(void* out, int out_dtype, const void* q,
                                              const void* k_pool, const void* v_pool,
                                              const int32_t* block_tables,
                                              int max_blocks_per_seq,
                                              const int32_t* context_lens, int batch,
                                              int num_heads, int kv_heads, int head_dim,
                                              int block_size, int64_t num_slots,
                                              int max_context_len, float scale, int dtype,
                                              void* stream) {
    clear_error();
    return flour::paged_decode_impl(out, out_dtype, q, k_pool, v_pool, block_tables,
                                    max_blocks_per_seq, context_lens, batch, num_heads, kv_heads,
                                    head_dim, block_size, num_slots, max_context_len, scale, dtype,
                                    nullptr, 0, true, nullptr, nullptr, stream);
}

namespace flour {

bool decode_mfma_supported(int dtype, int head_dim, int block_size, int n_rep, int batch,
                           int num_heads, int64_t num_slots, const void* q, const void* k_pool,
                           const void* v_pool) {
    return (dtype == FLOUR_DTYPE_BF16 || dtype == FLOUR_DTYPE_F16) &&
           (head_dim == 128 || head_dim == 64) && block_size % 16 == 0 && n_rep <= 16 &&
           batch <= DEC_MAX_BATCH && num_heads <= 65535 &&
           num_slots * head_dim * 2 <= (int64_t)0x7fffffff && ((uintptr_t)q % 16 == 0) &&
           ((uintptr_t)k_pool % 16 == 0) && ((uintptr_t)v_pool % 16 == 0);
}

// Whether an fp32 batch runs split over the chip on the matrix cores (with this workspace) rather
// than on the vector kernel, which needs no workspace but gives each (sequence, kv head) one
// workgroup.
static bool decode_f32_split(int head_dim, int block_size, int n_rep, int batch, int num_heads,
                             int64_t num_slots, int max_context_len, const void* out,
                             const void* q, const void* k_pool, const void* v_pool, bool ws_ok) {
    if (!ws_ok || (head_dim != 128 && head_dim != 64) || block_size % 16 != 0 || n_rep > 16 ||
        batch > DEC_MAX_BATCH || num_heads > 65535 ||
        num_slots * head_dim * 4 > (int64_t)0x7fffffff ||
        (((uintptr_t)out | (uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15) != 0)
        return false;  // (its output stores are up to 16 bytes wide, the vector kernel's one element)
    // The vector kernel's time goes with a workgroup's kv length x queries (n_rep, as a power of
    // two) x head_dim; a split step takes ~9 us and its bytes. Vector / split in us: 1 x 256 tokens of
    // 32 / 8 heads of 128 14.5 / 10.3 (64 tokens: 7.4 / 9.8), 14 / 2 heads of 64 13.4 / 8.8 (64: 8.3 /
    // 8.4), 16 / 16 of 128 at 1,024 18.3 / 11.8 (256: 7.7 / 10.2), 8 / 8 of 64 at 2,048 19.9 / 10.0
    // (512: 8.1 / 9.0).
    int64_t work = (int64_t)max_context_len * head_dim, least = 131072;
    int nq = 1;
    for (; nq < n_rep && nq < 8; nq *= 2) work *= 2;
    // With few queries per row and a workgroup for most CUs the vector kernel reads at HBM's rate too.
    // Up to one per CU all of them end together, and at one or two queries the split kernel is the
    // slower one at any length (16 / 16 heads of 64, 12 x 4,096 tokens: 73 / 80; 32 / 16 of 64, 12 x
    // 2,149: 38 / 49; 16 x 4,096 of 16 / 16 heads 99 / 91); otherwise it needs a longer step for its
    // 9 us (12 / 4 of 64, 128 x 512 tokens: 29 / 31, x 1,024 55 / 53; 16 / 8 of 128, 64 x 512: 46 /
    // 50, x 1,024 105 / 93). Over 26,379 batches of 16-1,200 (sequence, kv head) pairs, lengths uniform
    // and ragged, the step taken is up to 7 times as fast as the vector kernel's and 3-8% slower in 10.
    const int64_t pairs = (int64_t)batch * num_heads / n_rep, cus = device_cus();
    if (nq == 1 ? 8 * pairs >= 3 * cus : 2 * pairs >= cus) {
        if (nq <= 2 && 2 * pairs >= cus && pairs < cus) return false;
        if (nq < 8 || pairs < cus) least *= 2;
    }
    return work >= least;
}

static int paged_decode_impl(void* out, int out_dtype, const void* q, const void* k_pool,
                             const void* v_pool, const int32_t* block_tables,
                             int max_blocks_per_seq, const int32_t* context_lens, int batch,
                             int num_heads, int kv_heads, int head_dim, int block_size,
                             int64_t num_slots, int max_context_len, float scale, int dtype,
                             void* workspace, size_t workspace_bytes, bool ws_from_scratch,
                             const int32_t* rows, const DecodeWs* fused, void* stream) {
    if (!valid_dtype(dtype) || !valid_dtype(out_dtype)) {
        set_error("paged_decode: unknown dtype (%d, out %d)", dtype, out_dtype);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    if (batch < 0 || num_heads <= 0 || kv_heads <= 0 || num_heads % kv_heads != 0 ||
        head_dim <= 0 || block_size <= 0 || num_slots <= 0 || num_slots % block_size != 0 ||
        max_blocks_per_seq <= 0 || max_context_len < 0 ||
        (int64_t)max_context_len > (int64_t)max_blocks_per_seq * block_size) {
        set_error("paged_decode: bad shape (batch=%d heads=%d kv_heads=%d head_dim=%d bs=%d "
                  "num_slots=%lld max_blocks=%d max_ctx=%d)",
                  batch, num_heads, kv_heads, head_dim, block_size, (long long)num_slots,
                  max_blocks_per_seq, max_context_len);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    if (batch == 0) return FLOUR_OK;
    if (!out || !q || !k_pool || !v_pool || !block_tables || !context_lens) {
        set_error("paged_decode: null pointer");
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int n_rep = num_heads / kv_heads;
    const bool mfma = decode_mfma_supported(dtype, head_dim, block_size, n_rep, batch, num_heads,
                                            num_slots, q, k_pool, v_pool);
    if (!mfma && (rows || (fused && !fused->scores))) {
        set_error("paged_decode: row indices and the fused KV write need the matrix-core path");
        return FLOUR_ERR_UNSUPPORTED;
    }
    const int nwg = decode_workgroups(dtype);
    const size_t need = decode_ws_bytes(nwg, n_rep, head_dim, batch);
    const bool ws_ok = ws_from_scratch ? need <= DEC_SCRATCH_BYTES
                                       : workspace && workspace_bytes >= need &&
                                             ((uintptr_t)workspace % 256) == 0;
    // (an fp32 call without a workspace never touches the library's shared one)
    const bool wts = fused && fused->scores;
    const bool f32_split =
        dtype == FLOUR_DTYPE_F32 && !wts &&
        decode_f32_split(head_dim, block_size, n_rep, batch, num_heads, num_slots, max_context_len,
                         out, q, k_pool, v_pool, ws_ok && !ws_from_scratch);
    if (!mfma && !f32_split && !wts) {
        // one query row per sequence: cu_seqlens == nullptr
        const int64_t qs = (int64_t)num_heads * head_dim;
        if (simt_supported(dtype, head_dim, q, qs, head_dim, k_pool, v_pool))
            return launch_attn_simt(dtype, out_dtype, out, qs, head_dim, q, qs, head_dim, k_pool,
                                    v_pool, nullptr, context_lens, block_tables,
                                    max_blocks_per_seq, batch, batch, num_heads, n_rep, head_dim,
                                    block_size, num_slots, max_context_len, scale, s);
        return launch_attn_generic(dtype, out_dtype, out, (int64_t)num_heads * head_dim, head_dim,
                                   q, (int64_t)num_heads * head_dim, head_dim, k_pool, v_pool,
                                   nullptr, context_lens, block_tables, max_blocks_per_seq, batch,
                                   batch, num_heads, n_rep, head_dim, block_size, num_slots,
                                   max_context_len, scale, s);
    }
    if (ws_from_scratch) {
        if (need > DEC_SCRATCH_BYTES) {
            set_error("paged_decode_noalloc: this call needs %zu bytes of split-context workspace, "
                      "more than the %zu bytes of the library's scratch; use "
                      "flour_hip_paged_decode with a caller workspace",
                      need, DEC_SCRATCH_BYTES);
            return FLOUR_ERR_WORKSPACE;
        }
        const int rc = scratch_for_current_device(&workspace);
        if (rc != FLOUR_OK) return rc;
        workspace_bytes = DEC_SCRATCH_BYTES;
    }
    if (!ws_ok) {
        set_error("paged_decode: workspace of %zu bytes (256-byte aligned) required, got %zu "
                  "at %p",
                  need, workspace_bytes, workspace);
        return FLOUR_ERR_WORKSPACE;
    }
    DecodeWs ws = decode_ws_at(workspace, nwg, n_rep, head_dim);
    ws.rows = rows;
    ws.k_new = fused ? fused->k_new : nullptr;
    ws.v_new = fused ? fused->v_new : nullptr;
    ws.new_st = fused ? fused->new_st : 0;
    ws.new_sh = fused ? fused->new_sh : 0;
    ws.new_slots = fused ? fused->new_slots : nullptr;
    ws.scores = fused ? fused->scores : nullptr;
    ws.score_stride = fused ? fused->score_stride : 0;
    ws.row_ml = fused ? fused->row_ml : nullptr;
#define FLOUR_DEC(T)                                                                            \
    do {                                                                                        \
        if (out_dtype == FLOUR_DTYPE_F32)                                                       \
            return launch_decode_mfma<T, float>(head_dim, out, q, k_pool, v_pool, block_tables,           \
                                                max_blocks_per_seq, context_lens, batch,        \
                                                num_heads, kv_heads, n_rep, block_size,         \
                                                num_slots, max_context_len, scale, nwg, ws, s); \
        if (out_dtype == FLOUR_DTYPE_BF16)                                                      \
            return launch_decode_mfma<T, bf16_t>(head_dim, out, q, k_pool, v_pool, block_tables,          \
                                                 max_blocks_per_seq, context_lens, batch,       \
                                                 num_heads, kv_heads, n_rep, block_size,        \
                                                 num_slots, max_context_len, scale, nwg, ws,    \
                                                 s);                                            \
        return launch_decode_mfma<T, f16_t>(head_dim, out, q, k_pool, v_pool, block_tables,               \
                                            max_blocks_per_seq, context_lens, batch, num_heads, \
                                            kv_heads, n_rep, block_size, num_slots,             \
                                            max_context_len, scale, nwg, ws, s);                \
    } while (0)
    if (dtype == FLOUR_DTYPE_BF16) FLOUR_DEC(bf16_t);
    if (dtype == FLOUR_DTYPE_F32) FLOUR_DEC(float);
    FLOUR_DEC(f16_t);
#undef FLOUR_DEC
}

}  // namespace flour

namespace flour {

// Paged decode whose batch entry b reads q row rows[b] and writes out row rows[b] of a packed
// (rows, num_heads, head_dim) contiguous layout: the one-row sequences of a mixed
// continuous-batching step. Matrix-core shapes only (FLOUR_ERR_UNSUPPORTED otherwise, before
// any launch).
int paged_decode_rows(void* out, int out_dtype, const void* q, const void* k_pool,
                      const void* v_pool, const int32_t* block_tables, int max_blocks_per_seq,
                      const int32_t* context_lens, const int32_t* rows, int batch, int num_heads,
                      int kv_heads, int head_dim, int block_size, int64_t num_slots,
                      int max_context_len, float scale, int dtype, void* workspace,
                      size_t workspace_bytes, void* stream) {
    if (!rows) {
        set_error("paged_decode_rows: null row indices");
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    return paged_decode_impl(out, out_dtype, q, k_pool, v_pool, block_tables, max_blocks_per_seq,
                             context_lens, batch, num_heads, kv_heads, head_dim, block_size,
                             num_slots, max_context_len, scale, dtype, workspace, workspace_bytes,
                             false, rows, nullptr, stream);
}

bool paged_decode_scores_takes(int dtype, int head_dim, int block_size, int n_rep, int batch,
                               int num_heads, int64_t num_slots, const void* out, const void* q,
                               const void* k_pool, const void* v_pool) {
    if (dtype != FLOUR_DTYPE_F32)
        return decode_mfma_supported(dtype, head_dim, block_size, n_rep, batch, num_heads, num_slots,
                                     q, k_pool, v_pool);
    return (head_dim == 128 || head_dim == 64) && block_size % 16 == 0 && n_rep <= 16 &&
           batch <= DEC_MAX_BATCH && num_heads <= 65535 &&
           num_slots * head_dim * 4 <= (int64_t)0x7fffffff &&
           (((uintptr_t)out | (uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15) == 0;
}

size_t paged_decode_scores_bytes(int batch, int n_rep, int head_dim) {
    return decode_ws_bytes(decode_workgroups(FLOUR_DTYPE_F32), n_rep, head_dim, batch);
}

int paged_decode_scores(void* out, int out_dtype, const void* q, const void* k_pool,
                        const void* v_pool, const int32_t* block_tables, int max_blocks_per_seq,
                        const int32_t* context_lens, int batch, int num_heads, int kv_heads,
                        int head_dim, int block_size, int64_t num_slots, int max_context_len,
                        float scale, int dtype, void* workspace, size_t workspace_bytes,
                        float* scores, int64_t score_stride, float* row_ml, void* stream) {
    DecodeWs wz{};
    wz.scores = scores;
    wz.score_stride = score_stride;
    wz.row_ml = row_ml;
    return paged_decode_impl(out, out_dtype, q, k_pool, v_pool, block_tables, max_blocks_per_seq,
                             context_lens, batch, num_heads, kv_heads, head_dim, block_size,
                             num_slots, max_context_len, scale, dtype, workspace, workspace_bytes,
                             false, nullptr, &wz, stream);
}

int paged_decode_write_kv(void* out, int out_dtype, const void* q, void* k_pool, void* v_pool,
                          const int32_t* block_tables, int max_blocks_per_seq,
                          const int32_t* context_lens, int batch, int num_heads, int kv_heads,
                          int head_dim, int block_size, int64_t num_slots, int max_context_len,
                          float scale, int dtype, void* workspace, size_t workspace_bytes,
                          const void* k_new, const void* v_new, int64_t new_stride_tok,
                          int64_t new_stride_head, const int32_t* new_slots, void* stream) {
    const int es = (dtype == FLOUR_DTYPE_F32) ? 4 : 2;
    const uint64_t row_align = head_dim == 128 ? 16 : 8;  // a lane's share of a row
    // 16-token pages only: the fused instantiation for other page sizes spills registers in its
    // piece epilogue (a reload there waits for every chunk load in flight)
    if (!k_new || !v_new || !new_slots || batch < 1 || kv_heads <= 0 || block_size != 16 ||
        num_heads % kv_heads != 0 ||
        !decode_mfma_supported(dtype, head_dim, block_size, num_heads / kv_heads, batch,
                               num_heads, num_slots, q, k_pool, v_pool) ||
        (((uint64_t)(uintptr_t)k_new | (uint64_t)(uintptr_t)v_new |
          (uint64_t)(new_stride_tok * es) | (uint64_t)(new_stride_head * es)) &
         (row_align - 1)) != 0) {
        set_error("paged_decode_write_kv: shape not taken by the fused launch");
        return FLOUR_ERR_UNSUPPORTED;
    }
    DecodeWs fz{};
    fz.k_new = k_new;
    fz.v_new = v_new;
    fz.new_st = new_stride_tok;
    fz.new_sh = new_stride_head;
    fz.new_slots = new_slots;
    return paged_decode_impl(out, out_dtype, q, k_pool, v_pool, block_tables, max_blocks_per_seq,
                             context_lens, batch, num_heads, kv_heads, head_dim, block_size,
                             num_slots, max_context_len, scale, dtype, workspace, workspace_bytes,
                             false, nullptr, &fz, stream);
}

}  // namespace flour
