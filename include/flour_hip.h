/*
 * flour_hip.h — C-ABI of libflour_hip.so, the MI355X (gfx950) attention hot path of flour.
 *
 * The library replaces the reference's CPU attention seam (reference files cited as path:line,
 * relative to the lltsdyp/flour checkout):
 *
 *   src/backend/cpu.rs:57-112          paged_attention(q, blocks, n_rep, scale)
 *   src/models/common/paged.rs:186-204 PagedKvPool::write(layer, slots, k, v)
 *   src/models/common/paged.rs:114-121 BlockTable::slot / slots
 *   src/models/common/paged.rs:7-54    BlockAllocator
 *   src/models/common/paged.rs:138-167 PagedKvPool::new (device KV layout)
 *   src/models/common/cache.rs:429-458 Cache::allocate_kv / write_kv / kv_blocks
 *   src/models/common/cache.rs:112-159 KvCache::match_prefix / register_prefix
 *
 * Conventions
 *   - Every function returns FLOUR_OK (0) on success or a negative FLOUR_ERR_* code;
 *     flour_hip_last_error() then holds a message (per calling thread).
 *   - Device pointers are owned by the caller. Kernel launches are asynchronous and ordered on
 *     `stream` (a hipStream_t passed as void*; NULL = the default stream).
 *   - The KV pool of one layer is two device arrays, K and V, each laid out
 *     (kv_heads, num_slots, head_dim) row-major, exactly as PagedKvPool::new builds them
 *     (paged.rs:124-167). Slot s of physical block b is b * block_size + s % block_size
 *     (paged.rs:114-116), so the 16 rows of one (head, block) pair are contiguous.
 *   - Element types are given by the flour_dtype codes below. Scores, softmax and accumulators
 *     are fp32 and outputs are rounded to nearest-even. The matrix products take bf16/f16
 *     inputs exactly, with one exception: prefill over bf16 pools runs P.V on fp16 matrix
 *     cores with V converted to fp16 (exact for 2^-17 <= |v| <= 65504) and P rounded to fp16;
 *     a work item whose output is not finite or whose output block has a root mean square
 *     below 2^-25 / 5e-4 (~6e-5) is recomputed with bf16 V and P split into two bf16 parts,
 *     which small batches at head_dim 64 use throughout. Decode splits P into two 16-bit
 *     parts. fp32 pools stay fp32 throughout: prefill at
 *     head_dim 64 / 128 and longer decode steps there (with a large enough workspace) run on
 *     the fp32 matrix cores, every other fp32 call on the vector ALUs.
 */
#ifndef FLOUR_HIP_H
#define FLOUR_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum flour_dtype {
    FLOUR_DTYPE_F32 = 0,
    FLOUR_DTYPE_BF16 = 1,
    FLOUR_DTYPE_F16 = 2,
    /* elements of the 8-bit pools (the functions that take a pool_dtype; no others) */
    FLOUR_DTYPE_E4M3 = 3, /* OCP e4m3: 448 the largest, no infinities */
    FLOUR_DTYPE_I8 = 4,   /* two's complement, -127 .. 127 */
};

#define FLOUR_OK 0
#define FLOUR_ERR_INVALID_ARGUMENT (-1)
#define FLOUR_ERR_UNSUPPORTED (-2)
#define FLOUR_ERR_WORKSPACE (-3)
#define FLOUR_ERR_HIP (-4)
#define FLOUR_ERR_OUT_OF_BLOCKS (-5)
#define FLOUR_ERR_CAPACITY (-6)

/* Message describing the last error on the calling thread ("" if none). */
const char* flour_hip_last_error(void);

/* Library version string. */
const char* flour_hip_version(void);

/* ------------------------------------------------------------------------------------------
 * Kernel (1): KV-cache write.
 * Replaces PagedKvPool::write (src/models/common/paged.rs:186-204) as called through
 * KvCache::write_current (src/models/common/cache.rs:71-77).
 *
 * For every token t with slot_mapping[t] >= 0 and every kv head h:
 *     k_pool[h, slot_mapping[t], :] = k[t, h, :]     (and the same for v)
 * where element (t, h, d) of k / v sits at t*stride_tok + h*stride_head + d (elements).
 * The reference layout (1, kv_heads, seq, head_dim) is stride_tok = head_dim,
 * stride_head = seq*head_dim; a packed (tokens, kv_heads, head_dim) batch is
 * stride_tok = kv_heads*head_dim, stride_head = head_dim.
 * A negative slot marks a padding token and is skipped; a slot >= num_slots is never written.
 * The copy is bit-exact (no conversion): k/v and the pools share `dtype`.
 * Each non-negative slot may appear at most once per call (BlockTable::slots, paged.rs:118-121,
 * never repeats one): tokens are written in parallel, so for a repeated slot the stored row is
 * one of the repeating tokens' rows, chosen 16 bytes at a time, not the last token's. The cache
 * layers of flour_cache.h only build mappings without repeats.
 * ---------------------------------------------------------------------------------------- */
int flour_hip_kv_write(const void* k, const void* v, int64_t stride_tok, int64_t stride_head,
                       void* k_pool, void* v_pool, const int32_t* slot_mapping, int num_tokens,
                       int kv_heads, int head_dim, int64_t num_slots, int dtype, void* stream);

/* ------------------------------------------------------------------------------------------
 * RoPE + KV-cache write, fused (the step before kernel (1) in the reference, now one pass).
 * Replaces, at src/models/common/attention.rs:96-104, rope(q) and rope(k)
 * (candle_nn::rotary_emb::rope: the non-interleaved "rotate half" form) with the cos / sin
 * tables of Cache::new (cache.rs:377-393) read at the token's position (Cache::rope_cos /
 * rope_sin narrow them to index_pos.., cache.rs:404-410), then Cache::write_kv
 * (cache.rs:451-453 -> PagedKvPool::write's scatter, paged.rs:186-187).
 *
 * For token t with table row p = positions[t] and i < head_dim / 2, c = cos[p][i],
 * s = sin[p][i], a row x is rotated to
 *   y[i] = x[i]·c - x[i + head_dim/2]·s,   y[i + head_dim/2] = x[i]·s + x[i + head_dim/2]·c
 * with every product and sum rounded to `dtype` (fp32: no contraction). Then
 *   q_out[t, h, :] = rope(q[t, h, :])                               h < num_heads
 *   k_pool[h, slot_mapping[t], :] = rope(k[t, h, :]),  v_pool[h, slot_mapping[t], :] = v[t, h, :]
 * q and q_out share the strides (q_out may be q: in place); k and v share kv_stride_*.
 * cos_table / sin_table: (max_pos, head_dim / 2) row-major in `dtype`. head_dim must be even.
 * A token whose slot is outside [0, num_slots) writes no K/V (its q row is still rotated);
 * one whose position is outside [0, max_pos) writes nothing.
 * ---------------------------------------------------------------------------------------- */
int flour_hip_rope_kv_write(void* q_out, const void* q, int64_t q_stride_tok,
                            int64_t q_stride_head, int num_heads, const void* k, const void* v,
                            int64_t kv_stride_tok, int64_t kv_stride_head, void* k_pool,
                            void* v_pool, const int32_t* slot_mapping, const int32_t* positions,
                            const void* cos_table, const void* sin_table, int max_pos,
                            int num_tokens, int kv_heads, int head_dim, int64_t num_slots,
                            int dtype, void* stream);

/* ------------------------------------------------------------------------------------------
 * Kernel (2): paged decode attention (one new query token per sequence).
 * Replaces paged_attention (src/backend/cpu.rs:57-112) for seq_q == 1, batched over sequences,
 * with the block list of Cache::kv_blocks (cache.rs:456-458 -> KvCache::gather_blocks
 * cache.rs:83-96) given as a block table.
 *
 *   q            (batch, num_heads, head_dim) contiguous, post-RoPE
 *   out          (batch, num_heads, head_dim) contiguous, element type out_dtype
 *   block_tables [batch, max_blocks_per_seq] int32 physical block ids, logical order
 *   context_lens [batch] int32 kv length of each sequence (>= 1; 0 gives a zero row; a
 *                length above max_context_len attends the first max_context_len positions)
 *   Query head h attends kv head h / (num_heads / kv_heads) (repeat_kv, cpu.rs:5-13).
 *   scale multiplies q.k before the softmax (attention.rs:108 passes 1/sqrt(head_dim)).
 *   max_context_len bounds context_lens[] and sizes the split-context grid. Over fp32 pools it
 *                also decides whether a step is split at all: a bound far above the lengths can
 *                cost a few microseconds on short steps.
 *
 * Long contexts are split across workgroups; partial (max, sum, acc) rows and the batch's
 * per-sequence chunk prefix sums go to `workspace` (device memory, 256-byte aligned, no
 * initialisation needed) and a second kernel on the same stream merges them.
 * flour_hip_paged_decode_workspace_size gives the bytes required; calls that share a
 * workspace must not overlap in time. fp32 calls without a workspace (or with a smaller one)
 * run on the vector kernel, which needs none.
 * ---------------------------------------------------------------------------------------- */
int flour_hip_paged_decode_workspace_size(int batch, int num_heads, int kv_heads, int head_dim,
                                          int max_context_len, size_t* bytes);

int flour_hip_paged_decode(void* out, int out_dtype, const void* q, const void* k_pool,
                           const void* v_pool, const int32_t* block_tables,
                           int max_blocks_per_seq, const int32_t* context_lens, int batch,
                           int num_heads, int kv_heads, int head_dim, int block_size,
                           int64_t num_slots, int max_context_len, float scale, int dtype,
                           void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------------------------
 * Paged decode with no allocation anywhere: flour_hip_paged_decode without the workspace
 * arguments. This entry point has no counterpart in the reference; it is for callers that
 * cannot allocate device memory (code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc). The split-context workspace comes from a device array inside the
 * library, one per GPU (flour_hip_paged_decode_noalloc_max_workspace() bytes, 40 MiB, held
 * until the process ends). Arguments, results and kernels are those of flour_hip_paged_decode.
 * A call whose workspace would exceed that size fails with FLOUR_ERR_WORKSPACE before any
 * launch (at 256 CUs every shape the MFMA path takes fits; larger GQA groups or batches than
 * that would need flour_hip_paged_decode). fp32 pools run on the vector kernel here, whatever
 * the length. Every call on one GPU shares that GPU's array:
 * calls that overlap in time on one GPU (different streams, or threads without ordering) race
 * and give wrong results. Nothing needs to start at zero; the array keeps the last call's
 * contents.
 * ---------------------------------------------------------------------------------------- */
size_t flour_hip_paged_decode_noalloc_max_workspace(void);

int flour_hip_paged_decode_noalloc(void* out, int out_dtype, const void* q, const void* k_pool,
                                   const void* v_pool, const int32_t* block_tables,
                                   int max_blocks_per_seq, const int32_t* context_lens,
                                   int batch, int num_heads, int kv_heads, int head_dim,
                                   int block_size, int64_t num_slots, int max_context_len,
                                   float scale, int dtype, void* stream);

/* ------------------------------------------------------------------------------------------
 * Kernel (3): causal varlen prefill attention over the paged cache.
 * Replaces paged_attention (src/backend/cpu.rs:57-112) for seq_q >= 1, batched over packed
 * sequences. Sequence s owns query rows cu_seqlens_q[s] .. cu_seqlens_q[s+1]-1 and attends
 * kv_lens[s] cached positions (its suffix plus any prefix-cached shared blocks), with the
 * reference's causal rule (cpu.rs:68, :88-95): query i of a sequence with q_len rows sees kv
 * position j iff j <= kv_len - q_len + i.
 *
 *   q    row r, head h at r*q_stride_tok + h*q_stride_head (elements), head_dim contiguous
 *   out  row r, head h at r*o_stride_tok + h*o_stride_head, element type out_dtype
 *   cu_seqlens_q [num_seqs+1] int32, kv_lens [num_seqs] int32 (kv_len >= q_len; a sequence
 *                with kv_len < q_len attends nothing and its rows are written as zeros)
 *   block_tables [num_seqs, max_blocks_per_seq] int32
 *   max_seqlen_q bounds the per-sequence query count; total_q = cu_seqlens_q[num_seqs].
 * The K/V of the new rows must already be in the pool (flour_hip_kv_write).
 * This entry point allocates nothing and needs no workspace: the kernel gathers every K/V
 * tile through registers into LDS.
 * ---------------------------------------------------------------------------------------- */
int flour_hip_varlen_prefill(void* out, int out_dtype, int64_t o_stride_tok,
                             int64_t o_stride_head, const void* q, int64_t q_stride_tok,
                             int64_t q_stride_head, const void* k_pool, const void* v_pool,
                             const int32_t* cu_seqlens_q, const int32_t* kv_lens,
                             const int32_t* block_tables, int max_blocks_per_seq, int num_seqs,
                             int max_seqlen_q, int total_q, int num_heads, int kv_heads,
                             int head_dim, int block_size, int64_t num_slots, float scale,
                             int dtype, void* stream);

/* ------------------------------------------------------------------------------------------
 * Kernel (3) with a caller-owned workspace: flour_hip_varlen_prefill plus `workspace` (device
 * memory, 256-byte aligned, no initialisation needed). Same arguments, results and
 * replacement of paged_attention (cpu.rs:57-112, seq_q >= 1) as flour_hip_varlen_prefill.
 *
 * With long prompts (at least 1,536 new rows per sequence on average) over 16-bit pools at
 * head_dim 128 the call stages V once into the workspace (every 16-token page of each
 * sequence, widened to fp16 and transposed, by a pre-pass kernel on `stream`) and the
 * attention kernel then loads both K and V tiles straight into LDS. Otherwise, or when
 * workspace_bytes is below flour_hip_varlen_prefill_workspace_size() for the call's
 * num_seqs and max_blocks_per_seq, the call runs exactly as flour_hip_varlen_prefill (the
 * workspace is not touched). Nothing is allocated either way. Calls that share a workspace
 * must not overlap in time.
 * ---------------------------------------------------------------------------------------- */
int flour_hip_varlen_prefill_workspace_size(int num_seqs, int max_blocks_per_seq,
                                            int block_size, int kv_heads, int head_dim,
                                            int dtype, size_t* bytes);

int flour_hip_varlen_prefill_ws(void* out, int out_dtype, int64_t o_stride_tok,
                                int64_t o_stride_head, const void* q, int64_t q_stride_tok,
                                int64_t q_stride_head, const void* k_pool, const void* v_pool,
                                const int32_t* cu_seqlens_q, const int32_t* kv_lens,
                                const int32_t* block_tables, int max_blocks_per_seq,
                                int num_seqs, int max_seqlen_q, int total_q, int num_heads,
                                int kv_heads, int head_dim, int block_size, int64_t num_slots,
                                float scale, int dtype, void* workspace, size_t workspace_bytes,
                                void* stream);

/* ------------------------------------------------------------------------------------------
 * 8-bit KV pools. The reference keeps K/V in the model's dtype only; these functions have no
 * counterpart there. A pool of one layer is K and V, (kv_heads, num_slots, head_dim) in
 * pool_dtype (FLOUR_DTYPE_E4M3 or FLOUR_DTYPE_I8), with k_scale and v_scale, fp32 (kv_heads,
 * num_slots / block_size): an element of block b and kv head h stands for itself times
 * scale[h, b]. Tables, lengths, slots and q / out are those of the plain pools.
 *
 * Functions that read a pool take any scale that is 0 or a positive normal number (of subnormal ones
 * attention may make 0), and elements that are numbers (the writing ones store no others). Those that write one
 * (flour_hip_kv_write_q8, flour_hip_kv_evict) store powers of two: the smallest S >= 2^-126 with
 * which no element exceeds 448 (e4m3) or 127 (int8) times S, 0 for a block of zeros. A block that
 * takes an infinity or a NaN gets the scale NaN: whoever attends to one of its positions reads
 * NaN, until the block is started again.
 * ---------------------------------------------------------------------------------------- */

/* New rows into an 8-bit cache. As in flour_hip_varlen_prefill, sequence s brings the packed rows
 * cu_seqlens_q[s] .. cu_seqlens_q[s+1]-1, its positions kv_lens[s] - q_len .. kv_lens[s]-1; row t,
 * head h of k and v at t*stride_tok + h*stride_head (elements), in `dtype`. total_q =
 * cu_seqlens_q[num_seqs].
 * A block that the call writes gets the scale max(S_kept, S_new): S_kept the stored scale (the next power
 * of two where it is none; NaN where that is beyond 2^127) if the block holds positions of the sequence from before the call (0 otherwise, whatever the block
 * held), S_new the one the new rows need. Rows kept from before are requantised where that is
 * larger than their scale; new rows are rounded once, to nearest even. Rows of a block behind the
 * sequence's last position keep their bits.
 * Nothing is written for a sequence with kv_len < q_len, for positions past the table, or to blocks
 * whose id lies outside the pool. Several sequences may share blocks that the call only keeps
 * whole; a block that it writes must belong to one sequence of the call. */
int flour_hip_kv_write_q8(const void* k, const void* v, int64_t stride_tok, int64_t stride_head,
                          int dtype, void* k_pool, void* v_pool, float* k_scale, float* v_scale,
                          int pool_dtype, const int32_t* cu_seqlens_q, const int32_t* kv_lens,
                          const int32_t* block_tables, int max_blocks_per_seq, int num_seqs,
                          int total_q, int kv_heads, int head_dim, int block_size,
                          int64_t num_slots, void* stream);

/* The way back: positions 0 .. kv_lens[s]-1 of each sequence as the values they stand for, rounded
 * to `dtype` (f16: values beyond its largest number become that number), into the slots of a plain
 * pool (kv_heads, out_slots, head_dim) that out_tables gives them; other slots are left as they
 * are. max_kv_len bounds kv_lens (a longer sequence is read up to it). Ids of block_tables outside
 * the pool read a block inside it, as in attention; ids of out_tables outside theirs are skipped. */
int flour_hip_kv_dequant(void* k_out, void* v_out, int dtype, const int32_t* out_tables,
                         int out_max_blocks, int64_t out_slots, const void* k_pool,
                         const void* v_pool, const float* k_scale, const float* v_scale,
                         int pool_dtype, const int32_t* block_tables, int max_blocks_per_seq,
                         const int32_t* kv_lens, int num_seqs, int max_kv_len, int kv_heads,
                         int head_dim, int block_size, int64_t num_slots, void* stream);

/* flour_hip_paged_decode over an 8-bit cache: q in `dtype` (f32, bf16 or f16), the products and
 * sums as there. `weights` (NULL for none) is described at flour_hip_paged_decode_weights.
 * A workspace of flour_hip_decode_weights_workspace_size bytes is required. */
int flour_hip_paged_decode_q8(void* out, int out_dtype, const void* q, int dtype,
                              const void* k_pool, const void* v_pool, const float* k_scale,
                              const float* v_scale, int pool_dtype, const int32_t* block_tables,
                              int max_blocks_per_seq, const int32_t* context_lens, int batch,
                              int num_heads, int kv_heads, int head_dim, int block_size,
                              int64_t num_slots, int max_context_len, float scale, float* weights,
                              int64_t weights_width, const int32_t* weight_rows,
                              int num_weight_rows, void* workspace, size_t workspace_bytes,
                              void* stream);

/* flour_hip_paged_decode over a plain pool that also adds the step's attention weights to a sum
 * per cached position, what an eviction goes by:
 *     weights[r, g, j] += sum over the query heads of kv head g of softmax weight (head, j)
 * for the sequence's positions j < context_len, r = weight_rows[b] (b itself if weight_rows is
 * NULL). weights is fp32 (num_weight_rows, kv_heads, weights_width) contiguous, weights_width >=
 * max_context_len. Entries of one call must have different rows; one whose row lies outside
 * [0, num_weight_rows) adds nothing (its attention is computed all the same). A query head of which a
 * score is NaN or +inf adds NaN to every position of its kv head, also where an fp32 pool's output is a zero
 * row: such sums stay NaN until the caller writes them, and to flour_hip_kv_evict are below every number.
 * A workspace of flour_hip_decode_weights_workspace_size bytes (256-byte aligned, no
 * initialisation needed) is required; calls that share one must not overlap in time. */
int flour_hip_paged_decode_weights(void* out, int out_dtype, const void* q, const void* k_pool,
                                   const void* v_pool, const int32_t* block_tables,
                                   int max_blocks_per_seq, const int32_t* context_lens, int batch,
                                   int num_heads, int kv_heads, int head_dim, int block_size,
                                   int64_t num_slots, int max_context_len, float scale, int dtype,
                                   float* weights, int64_t weights_width,
                                   const int32_t* weight_rows, int num_weight_rows,
                                   void* workspace, size_t workspace_bytes, void* stream);

/* Workspace of the two functions above; with_weights != 0 where `weights` is given. */
int flour_hip_decode_weights_workspace_size(int batch, int num_heads, int kv_heads, int head_dim,
                                            int max_context_len, int with_weights, size_t* bytes);

/* flour_hip_varlen_prefill over an 8-bit cache, whose new rows flour_hip_kv_write_q8 has written:
 * every row attends to the quantised values, its own among them. Which kernels run goes by the shape of
 * the call; all take any scale. Calls of many rows round each value, element times scale, once to
 * `dtype` (values of power-of-two scales are exact in f32 and bf16, and in f16 but for a last half step of
 * 2^-25 near zero; a head whose blocks could hold values beyond f16's range, or so small that this half
 * step would be more than 2^-12 of their largest, is computed from the 8 bits, which takes many times
 * as long) and with 16-bit queries each probability once to f16. max_kv_len bounds kv_lens (a
 * longer sequence is taken to end there); rows behind the last sequence's, where total_q is larger
 * than cu_seqlens_q[num_seqs], leave out as it was. A workspace of
 * flour_hip_varlen_prefill_q8_workspace_size bytes (256-byte aligned, no initialisation needed) goes with
 * the call (FLOUR_ERR_WORKSPACE where it is too small for any kernel); calls that share one must not overlap in time. */
int flour_hip_varlen_prefill_q8(void* out, int out_dtype, int64_t o_stride_tok,
                                int64_t o_stride_head, const void* q, int64_t q_stride_tok,
                                int64_t q_stride_head, int dtype, const void* k_pool,
                                const void* v_pool, const float* k_scale, const float* v_scale,
                                int pool_dtype, const int32_t* cu_seqlens_q,
                                const int32_t* kv_lens, const int32_t* block_tables,
                                int max_blocks_per_seq, int num_seqs, int max_seqlen_q,
                                int total_q, int num_heads, int kv_heads, int head_dim,
                                int block_size, int64_t num_slots, int max_kv_len, float scale,
                                void* workspace, size_t workspace_bytes, void* stream);

/* What the kernels take that the shape selects. Few rows read the 8-bit cache as it is, in tens of MB. More
 * have a copy of the sequences in `dtype`, up to 1 GiB or one sequence, and for long prompts another of
 * V. A call with less than that for its copy makes it in parts, or does without, and takes longer; so does
 * one whose pool holds 2^31 bytes or more of a kv head with the size for few rows. */
int flour_hip_varlen_prefill_q8_workspace_size(int num_seqs, int max_seqlen_q, int total_q,
                                               int max_kv_len, int num_heads, int kv_heads,
                                               int head_dim, int block_size, int dtype,
                                               size_t* bytes);

/* ------------------------------------------------------------------------------------------
 * Eviction by accumulated attention weight (no counterpart in the reference). Of sequence b's L =
 * context_lens[b] positions each kv head keeps n = min(keep_lens[b], L) of its own: the last
 * min(recent, n), and of the others those with the largest weights[r, g, .], ties to the lower
 * position, NaN below every number. In their order, the kept rows of K and V go to the slots that
 * out_tables gives positions 0 .. n-1; keys keep the rotation of their old positions.
 * Blocks of out_tables must not be among any block_tables of the call, nor twice among their own;
 * rows of a destination block behind position n-1 keep their bits. The old blocks are not written:
 * shared prefix blocks may be evicted from.
 *   weights      fp32 (num_weight_rows, kv_heads, weights_width), r = weight_rows[b] (b if NULL;
 *                outside [0, num_weight_rows): the entry is skipped, its kept row is all -1);
 *                entries of one call must have different rows
 *   weights_out  same shape, or weights itself: [r, g, i] = the i-th kept position's sum for i < n
 *                and 0 for n <= i < L; the rest is left as it is
 *   kept         [batch, kv_heads, max_keep_len]: the kept positions, -1 behind the n-th
 * Plain pools (pool_dtype f32, bf16 or f16; k_scale = v_scale = NULL) are copied bit for bit. Over
 * an 8-bit pool each destination block gets a scale of its own from the kept values, which are
 * rounded once more where it differs from theirs.
 * max_context_len bounds context_lens, max_keep_len keep_lens (larger ones are clamped).
 * ---------------------------------------------------------------------------------------- */
int flour_hip_kv_evict(void* k_pool, void* v_pool, float* k_scale, float* v_scale, int pool_dtype,
                       const float* weights, float* weights_out, int64_t weights_width,
                       const int32_t* weight_rows, int num_weight_rows,
                       const int32_t* block_tables, int max_blocks_per_seq,
                       const int32_t* context_lens, const int32_t* keep_lens,
                       const int32_t* out_tables, int out_max_blocks, int32_t* kept, int batch,
                       int kv_heads, int head_dim, int block_size, int64_t num_slots,
                       int max_context_len, int max_keep_len, int recent, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FLOUR_HIP_H */
