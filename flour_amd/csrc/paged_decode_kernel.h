// paged_decode_kernel.h — the decode kernels of paged_decode.hip (what they compute and why is described there)
// and of ranged_decode.h.
#pragma once

#include <math.h>

#include <type_traits>

#include "decode_ranges.h"
#include "flour_common.h"
#include "ranged.h"

namespace flour {

static constexpr float LOG2E = 1.4426950408889634f;

// Tokens per step: two 16-token MFMA tiles of a 16-bit pool, one of an fp32 pool (the same bytes)
__host__ __device__ constexpr int dec_chunk(int elem_bytes) { return elem_bytes == 4 ? 16 : 32; }
static constexpr int DEC_SEG = 32;           // chunks per tile-slot refill (up to 64 tiles, one per lane)
static constexpr int DEC_MAX_BATCH = 4096;   // per-sequence chunk prefix sums live in LDS
// Three waves per CU. Each wave keeps one 32-token chunk in flight while it computes the
// previous one (16 KB at head_dim 128), so 768 waves hold ~12 MB of reads, about HBM's
// bandwidth-delay product; more waves only lengthen the queues and open more DRAM rows at once
// on the random 4 KB page runs (measured on the Llama-3-8B / 70B / Qwen2.5-0.5B decode batches:
// 3 per CU stream 0.3-1.5% faster than 4, which stream 3-7% faster than 8; counts that do not
// divide evenly over a CU's 4 SIMDs, 2.5, 3.5 and 5 per CU, are slower than their neighbours).
static constexpr int DEC_WAVES_PER_CU = 3;
// fp32 pools: the fp32 products of a chunk keep a SIMD's matrix core busy for ~2,050 cycles of
// every 16 KB, so every SIMD gets a wave (3 / 4 / 6 per CU: 163 / 149 / 142 us for 855 MB at 32 / 8
// heads of 128, 131 / 126 / 136 us for 806 MB at 8 heads of 64).
static constexpr int DEC_WAVES_PER_CU_F32 = 4;
static_assert(DEC_WAVES_PER_CU_F32 >= DEC_WAVES_PER_CU, "the workspace is sized for the larger");
// K is read like V, four whole 256 B rows per instruction with the non-temporal hint, and
// turned into the MFMA A-operand layout (row = lane % 16) through a per-wave LDS tile. Reading
// K directly in that layout takes a 64 B quarter of 16 rows per instruction, a pattern that
// streams at most ~6.0 TB/s from HBM against ~6.8 TB/s for whole rows (measured with the same
// 2048-wave, double-buffered access over random 4 KB runs).
// Bytes per K row in LDS: the row and 16 bytes, conflict-free 16-byte fragment reads of 16 rows.
__host__ __device__ constexpr int dec_kpitch(int d, int elem_bytes) { return d * elem_bytes + 16; }

// A step that looks at parts of its contexts (the kernels' RNG instantiations): the first `sinks` and the
// last `window` positions. The list of chunks holds those that have visible positions: of the sinks, and
// from the last multiple of 16 before the window on.
struct DecodeRange {
    int window, sinks;
    int out_dtype;  // of AnyOut outputs
};
// How a launch's waves share the chunks. DEC_PAIRS (windows): a workgroup a (sequence, kv head), whose waves
// take equal parts of its chunks and fold their states through LDS, so nothing is left to merge.
enum DecodeSplit { DEC_RANGES, DEC_PAIRS };
// The output's type is a field of the call.
struct AnyOut {
    uint8_t bits;
};

// The visible part of a context of ctx positions: those below front and from lo on.
template <int CHUNK>
struct DecodePart {
    int ctx, lo, front;
    __device__ __forceinline__ DecodePart(int ctx_, const DecodeRange& r) : ctx(ctx_) {
        lo = max(0, ctx - r.window);
        if (lo <= r.sinks) lo = 0;
        front = lo > 0 ? r.sinks : 0;
    }
    __device__ __forceinline__ int front_chunks() const { return (front + CHUNK - 1) / CHUNK; }
    __device__ __forceinline__ int base() const { return max(lo & ~15, front_chunks() * CHUNK); }
    __device__ __forceinline__ int chunks() const {
        const int b = base();
        return ctx <= 0 ? 0 : front_chunks() + (ctx > b ? (ctx - b + CHUNK - 1) / CHUNK : 0);
    }
    __device__ __forceinline__ int tok(int c) const {  // the first position of chunk c
        const int f = front_chunks();
        return c < f ? c * CHUNK : base() + (c - f) * CHUNK;
    }
};

struct DecodeWs {
    float* ml;  // [2 * num_waves][n_rep][2] (max, sum) in the exp2 domain
    float* o;   // [2 * num_waves][n_rep][D]
    int* pre;   // [batch + 1] chunk prefix sums, written by workgroup 0 for the merge kernel
    // row of q / out that batch entry b reads and writes: rows[b], or b when null (a mixed
    // continuous-batching step runs its one-row sequences, scattered among the packed rows of
    // longer ones, as one decode batch)
    const int32_t* rows;
    // Decode step of a batch with its KV write fused in (the kernel's FUSE instantiation): the
    // new K / V row of entry b and kv head g at k_new / v_new + b * new_st + g * new_sh
    // (elements), written to pool slot new_slots[b] (skipped outside [0, num_slots)) before the
    // attention reads it.
    const void* k_new;
    const void* v_new;
    int64_t new_st, new_sh;
    const int32_t* new_slots;
    int xcd_w;  // wave-range weight w (WaveRanges): even ranges 32 + w, odd 32 - w
    // A step whose attention weights are wanted (the kernels' WTS instantiations): every score in the
    // exp2 domain, row b * num_heads + h at scores + row * score_stride, and each row's (max, sum). Kept
    // rather than computed again: 64 x 512-4,096 tokens of 32 / 8 heads of 128 in bf16 105 us where a
    // step without weights takes 91, and a second pass over K would take half of that again.
    float* scores;
    int64_t score_stride;
    float* row_ml;
    DecodeRange rng;
};

// Waves of a launch at most, and the ranges' weight (switches of paged_decode.hip).
int decode_workgroups(int dtype);
int decode_xcd_weight();

static size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

static size_t decode_ws_bytes(int nwg, int n_rep, int head_dim, int batch) {
    const size_t slots = 2 * (size_t)nwg;
    return align256(slots * n_rep * 2 * sizeof(float)) +
           align256(slots * n_rep * (size_t)head_dim * sizeof(float)) +
           align256(((size_t)batch + 1) * sizeof(int));
}

// The parts of a workspace for launches of up to nwg waves.
static DecodeWs decode_ws_at(void* workspace, int nwg, int n_rep, int head_dim) {
    DecodeWs ws{};
    char* at = static_cast<char*>(workspace);
    ws.ml = reinterpret_cast<float*>(at);
    at += align256((size_t)2 * nwg * n_rep * 2 * sizeof(float));
    ws.o = reinterpret_cast<float*>(at);
    at += align256((size_t)2 * nwg * n_rep * (size_t)head_dim * sizeof(float));
    ws.pre = reinterpret_cast<int*>(at);
    ws.xcd_w = decode_xcd_weight();
    return ws;
}

template <int CHUNK>
__device__ __forceinline__ int decode_chunks(int ctx, int max_ctx) {
    ctx = min(ctx, max_ctx);
    return ctx > 0 ? (ctx + CHUNK - 1) / CHUNK : 0;
}

// What a row is divided by: its sum of weights, or 1 where that is 0 (no score above -inf: a zero
// row). Over fp32 pools an undefined sum (scores of NaN or +inf) gives a zero row too, as on the
// vector kernel (attn_simt.hip): the caller clears the row wherever !(sum > 0). The 16-bit pools
// hand a NaN on.
template <bool F32>
__device__ __forceinline__ float divisor(float sum) {
    return (F32 ? !(sum > 0.0f) : sum == 0.0f) ? 1.0f : sum;
}

__device__ __forceinline__ f32x4 mfma16x16x4_f32(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Waves of a DEC_PAIRS workgroup (eight are within 10% of four, two behind them but on large batches), and a wave's
// LDS there: its K tile, then its state.
static constexpr int DEC_PAIR_WAVES = 4;
__host__ __device__ constexpr int dec_pair_lds(int d, int elem_bytes) {
    const int k = 16 * dec_kpitch(d, elem_bytes), state = 64 * (d * 16 / 64 + 2) * 4;
    return k > state ? k : state;
}

// One wave per workgroup; each wave owns one contiguous range of the chunk list. D is the head
// dim, 128 or 64. A lane's K/V share of a 16-token tile is rows 4lg .. 4lg + 3 at 16-byte
// (D 128: dims 8lc ..) or 8-byte (D 64: dims 4lc ..) width, so a wave reads whole rows.
// RNG: the context is looked at through ws.rng.
template <typename T, typename TO, bool BS16, int D, bool FUSE, bool WTS, bool RNG = false,
          int SPLIT = DEC_RANGES>
__global__ __launch_bounds__(SPLIT == DEC_PAIRS ? 64 * DEC_PAIR_WAVES : 64, 2) void paged_decode_mfma_kernel(
    TO* __restrict__ out, const T* __restrict__ q, const T* __restrict__ k_pool,
    const T* __restrict__ v_pool, const int32_t* __restrict__ block_tables, int max_blocks,
    const int32_t* __restrict__ context_lens, int batch, int num_heads, int kv_heads, int n_rep,
    int block_size, int64_t num_slots, int max_ctx, float scale_log2, DecodeWs ws) {
    static_assert(D == 128 || D == 64, "matrix-core decode: head_dim 128 or 64");
    constexpr bool F32 = std::is_same<T, float>::value;
    constexpr int CHUNK = dec_chunk(sizeof(T));
    constexpr int TILES = CHUNK / 16;  // 16-token tiles per chunk
    constexpr int KP = dec_kpitch(D, sizeof(T));
    constexpr int NV = D / 16;  // O^T products per chunk (16 output dims each)
    // A lane's loads of K (and of V) per chunk: [NL][4] of Ld. 16-bit pools: tile t, row 4lg + j,
    // 8 (D 128) or 4 (D 64) dims. fp32 pools: row 4lg + j of the one tile, dims 64i + 4lc .. + 3,
    // so an instruction reads four 256-byte row segments in every form (128 at D 64, 16-bit).
    constexpr int NL = F32 ? D / 64 : TILES;
    typedef typename std::conditional<F32 || D == 128, u32x4, u32x2>::type Ld;
    constexpr bool PAIRS = SPLIT == DEC_PAIRS;
    // pre[b] = chunks of sequences 0..b-1; pre[batch] = all. PAIRS: the waves' LDS instead.
    extern __shared__ __attribute__((aligned(16))) int pre[];
    __shared__ __attribute__((aligned(16))) unsigned char kt_one[PAIRS ? 16 : 16 * KP];  // one K tile
    const int lane = PAIRS ? threadIdx.x & 63 : threadIdx.x, lg = lane >> 4, lc = lane & 15;
    const int w_id = PAIRS ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    unsigned char* const kt = PAIRS ? reinterpret_cast<unsigned char*>(pre) + w_id * dec_pair_lds(D, sizeof(T))
                                    : kt_one;

    // ---- exclusive prefix sum of per-sequence chunk counts. Up to 64 sequences stay in
    // registers, one per lane (clamped context length and prefix), so that locating a segment
    // is a ballot and scalar lane reads: no LDS search, no second read of a context length.
    // (16-token pages: with other page sizes those two registers spill)
    const bool in_lanes = BS16 && batch <= 64;
    const DecodeRange& rng = ws.rng;
    auto part = [&](int ctx) { return DecodePart<CHUNK>(ctx, rng); };
    auto chunks_of = [&](int ctx) -> int {
        if constexpr (RNG) return part(min(ctx, max_ctx)).chunks();
        return decode_chunks<CHUNK>(ctx, max_ctx);
    };
    int my_ctx = 0, my_pre = 0, all_chunks = 0;
    if (PAIRS) {
    } else if (in_lanes) {
        my_ctx = lane < batch ? min(context_lens[lane], max_ctx) : 0;
        const int n = chunks_of(my_ctx);
        const int incl = wave_incl_sum(n);
        my_pre = incl - n;
        all_chunks = __builtin_amdgcn_readlane(incl, 63);
        if constexpr (FUSE) {  // its walk over the pairs reads them by index
            if (lane < batch) pre[lane] = my_pre;
            if (lane == 63) pre[batch] = incl;
            __syncthreads();
        }
        if (blockIdx.x == 0) {  // for the merge kernel (ordered by the kernel boundary)
            if (lane < batch) ws.pre[lane] = my_pre;
            if (lane == 63) ws.pre[batch] = incl;
        }
    } else {  // each lane scans a slice, through LDS
        const int per = (batch + 63) / 64;
        int local = 0;
        for (int i = 0; i < per; i++) {
            const int b = lane * per + i;
            if (b < batch) local += chunks_of(context_lens[b]);
        }
        const int incl = wave_incl_sum(local);
        int run = incl - local;
        for (int i = 0; i < per; i++) {
            const int b = lane * per + i;
            if (b < batch) {
                pre[b] = run;
                run += chunks_of(context_lens[b]);
            }
        }
        if (lane == 63) pre[batch] = incl;
        __syncthreads();
        all_chunks = __builtin_amdgcn_readlane(incl, 63);
        if (blockIdx.x == 0)
            for (int b = lane; b <= batch; b += 64) ws.pre[b] = pre[b];
    }
    const int64_t total = (int64_t)kv_heads * all_chunks;
    const int64_t nwg = range_count(total, gridDim.x), wgi = blockIdx.x;
    if (!PAIRS && (total == 0 || wgi >= nwg)) return;
    // 32-bit divisions whenever they fit: a 64-bit one is ~0.3 us of instructions, and the
    // range bounds and the first segments stand before the wave's first load
    const bool narrow = ranges_narrow(total, nwg, ws.xcd_w);
    // The range is [lo, lo + len); positions in it are 32-bit offsets from lo
    // (a range of 2^31 chunks would be 16 TB of reads). Everything that selects a segment is
    // uniform and made scalar here: a divergent value would put every
    // buffer load that takes its offset into a per-lane loop.
    int64_t lo;
    int len;
    // PAIRS: the pair, its context, its chunks
    int pb = 0, pg = 0, p_ctx = 0, p_nch = 0;
    if constexpr (PAIRS) {
        pb = blockIdx.x / kv_heads, pg = blockIdx.x - pb * kv_heads;
        p_ctx = min(__builtin_amdgcn_readfirstlane(context_lens[pb]), max_ctx);
        p_nch = chunks_of(p_ctx);
        lo = (int64_t)p_nch * w_id / DEC_PAIR_WAVES;
        len = (int)((int64_t)p_nch * (w_id + 1) / DEC_PAIR_WAVES - lo);
    } else if (narrow) {
        const WaveRanges<uint32_t> wr(total, nwg, ws.xcd_w);
        const uint32_t a = wr.lo((uint32_t)wgi);
        lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)a);
        len = __builtin_amdgcn_readfirstlane((int)(wr.lo((uint32_t)wgi + 1) - a));
    } else {
        const WaveRanges<int64_t> wr(total, nwg, ws.xcd_w);
        const int64_t a = wr.lo(wgi);
        lo = ((int64_t)__builtin_amdgcn_readfirstlane((int)(a >> 32)) << 32) |
             (uint32_t)__builtin_amdgcn_readfirstlane((int)a);
        len = __builtin_amdgcn_readfirstlane((int)(wr.lo(wgi + 1) - a));
    }

    const uint32_t head_bytes = (uint32_t)(num_slots * D * (int64_t)sizeof(T));
    // K and V: instruction j of a tile reads rows 4lg + j, dims (D / 16) lc .. (4 whole rows)
    uint32_t v_off = (uint32_t)((4 * lg * D + (F32 ? 4 : D / 16) * lc) * sizeof(T));
    // opaque: with its low bits known, the row offsets become ORs held in a register each instead
    // of the loads' immediate offsets
    asm volatile("" : "+v"(v_off));
    const int64_t max_phys = num_slots / block_size - 1;

    // The wave's range is a stream of segments: up to DEC_SEG consecutive chunks of one
    // (sequence, kv head) pair. Consecutive segments of the same pair form one piece.
    struct Seg {
        int b, g, cb, ce, nch, tok_end;  // RNG: tok_end is the context's
    };
    auto seg_at = [&](int at) -> Seg {
        const int64_t x = lo + at;
        Seg sg;
        if constexpr (PAIRS) {
            sg.b = pb, sg.g = pg, sg.nch = p_nch, sg.tok_end = p_ctx;
            sg.cb = (int)x;
            sg.ce = sg.cb + min(DEC_SEG, len - at);
            return sg;
        }
        int before, ctx;  // chunks per head before sequence b, its clamped context length
        if (in_lanes) {   // largest b with kv_heads * pre[b] <= x
            const uint64_t le = __ballot(lane < batch && (int64_t)kv_heads * my_pre <= x);
            sg.b = __popcll(le) - 1;
            before = __builtin_amdgcn_readlane(my_pre, sg.b);
            ctx = __builtin_amdgcn_readlane(my_ctx, sg.b);
            sg.nch = chunks_of(ctx);
        } else {
            int l0 = 0, h0 = batch;
            while (h0 - l0 > 1) {
                const int mid = (l0 + h0) >> 1;
                if ((int64_t)kv_heads * pre[mid] <= x)
                    l0 = mid;
                else
                    h0 = mid;
            }
            sg.b = __builtin_amdgcn_readfirstlane(l0);
            before = __builtin_amdgcn_readfirstlane(pre[l0]);
            sg.nch = __builtin_amdgcn_readfirstlane(pre[l0 + 1]) - before;
            ctx = min(context_lens[sg.b], max_ctx);
            if constexpr (RNG) ctx = __builtin_amdgcn_readfirstlane(ctx);
        }
        const int64_t rel = x - (int64_t)kv_heads * before;
        sg.g = __builtin_amdgcn_readfirstlane(narrow ? (int)((uint32_t)rel / (uint32_t)sg.nch)
                                                     : (int)(rel / sg.nch));
        sg.cb = (int)(rel - (int64_t)sg.g * sg.nch);
        sg.ce = sg.cb + min(min(sg.nch - sg.cb, DEC_SEG), len - at);
        sg.tok_end = RNG ? ctx : min(ctx, sg.ce * CHUNK);
        return sg;
    };
    // Pool slot of the first token of each tile of a segment: lane i holds tile i (chunk
    // cb + i/2, half i%2), so the loop fetches it with v_readlane. Tiles past the segment are
    // clamped to its last tile: every address stays valid, their tokens are masked and their V
    // zeroed in compute_chunk.
    // The block id is kept as loaded and clamped only where a tile load reads it (one segment
    // later for the next segment): using it here would make the wave wait for this load, and
    // with it for every chunk load in flight.
    struct Slots {
        int id, off;  // lane i: block id and in-block offset of tile i's first token
    };
    const int max_id = (int)max_phys;
    auto seg_slots = [&](const Seg& sg) -> Slots {
        const int32_t* bt = block_tables + (int64_t)sg.b * max_blocks;
        const int last_tile_tok0 = ((sg.tok_end - 1) >> 4) << 4;
        int first = sg.cb * CHUNK + lane * 16;
        if constexpr (RNG) first = part(sg.tok_end).tok(sg.cb + lane / TILES) + lane % TILES * 16;
        const int tok0 = min(first, last_tile_tok0);
        const int lb = BS16 ? (tok0 >> 4) : tok0 / block_size;
        return Slots{bt[lb], BS16 ? 0 : tok0 - lb * block_size};
    };
    // Chunk loads as buffer loads: one resource per pool (the kv head's region), the
    // loop-invariant lane offset (VGPR) and the tile's byte offset (SGPR), so there is no
    // per-lane address arithmetic in the loop; non-temporal (K/V are read exactly once);
    // an out-of-region offset reads zeros instead of faulting.
    auto load_chunk = [&](int g, Slots sl, int tile0, Ld (*kd)[4], Ld (*vd)[4]) {
        const __amdgpu_buffer_rsrc_t k_rsrc = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(k_pool + (int64_t)g * num_slots * D), (short)0, (int)head_bytes, BUF_DWORD3);
        const __amdgpu_buffer_rsrc_t v_rsrc = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(v_pool + (int64_t)g * num_slots * D), (short)0, (int)head_bytes, BUF_DWORD3);
#pragma unroll
        for (int t = 0; t < TILES; t++) {
            int id = __builtin_amdgcn_readlane(sl.id, tile0 + t);
            id = id < 0 ? 0 : (id > max_id ? max_id : id);  // a bad block id never leaves the pool
            const uint32_t slot =
                BS16 ? (uint32_t)(id * 16)
                     : (uint32_t)(id * block_size + __builtin_amdgcn_readlane(sl.off, tile0 + t));
            const uint32_t soff = slot * (uint32_t)(D * sizeof(T));
            auto load_rows = [&](const __amdgpu_buffer_rsrc_t& rsrc, Ld (*d)[4]) {
#pragma unroll
                for (int i = 0; i < NL / TILES; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t off = v_off + (j * D + 64 * i) * (uint32_t)sizeof(T);
                        if constexpr (sizeof(Ld) == 16)
                            d[t + i][j] =
                                __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, soff, BUF_NT);
                        else
                            d[t + i][j] =
                                __builtin_amdgcn_raw_buffer_load_b64(rsrc, off, soff, BUF_NT);
                    }
            };
            load_rows(k_rsrc, kd);
            load_rows(v_rsrc, vd);
        }
    };
    // Q^T as the B operand: lane (lg, lc) holds head lc, dims 32kk + 8lg .. +7; fp32: dims
    // 16kk + 4lg .. + 3, one per k-step 4kk .. 4kk + 3.
    constexpr int NQ = D * (int)sizeof(T) / 64;
    u32x4 qb[NQ];
    // WTS: where the scores of a chunk at token 0 go, and the lane's there
    float* score_to = nullptr;
    const uint32_t score_lane = WTS ? (uint32_t)(lc * ws.score_stride + 4 * lg) : 0;
    auto load_q = [&](int b, int g) {
        if constexpr (WTS)
            score_to = ws.scores + ((int64_t)b * num_heads + (int64_t)g * n_rep) * ws.score_stride;
        const int64_t row = ws.rows ? (int64_t)ws.rows[b] : (int64_t)b;
        const T* qh = q + (row * num_heads + (int64_t)g * n_rep + lc) * D + (F32 ? 4 : 8) * lg;
#pragma unroll
        for (int kk = 0; kk < NQ; kk++)
            qb[kk] = (lc < n_rep) ? *reinterpret_cast<const u32x4*>(qh + (F32 ? 16 : 32) * kk)
                                  : u32x4{0, 0, 0, 0};
    };

    float m = DEC_M0, lsum = 0.0f;
    f32x4 acc[NV];
#pragma unroll
    for (int nn = 0; nn < NV; nn++) acc[nn] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    auto compute_chunk = [&](int c, int tok_end, Ld (*ka)[4], Ld (*va)[4]) {
        int tok0 = c * CHUNK, tok_lo = 0, front = 0;
        bool full = tok0 + CHUNK <= tok_end;
        if constexpr (RNG) {
            const DecodePart<CHUNK> pt = part(tok_end);
            tok0 = pt.tok(c);
            tok_lo = pt.lo;
            front = pt.front;
            full = tok0 + CHUNK <= tok_end && (tok0 >= tok_lo || tok0 + CHUNK <= front);
        }
        auto seen = [&](int tok) { return tok < tok_end && (!RNG || tok >= tok_lo || tok < front); };
        if (!full) {  // tokens past the context: zero V so garbage bits cannot leak in
#pragma unroll
            for (int t = 0; t < NL; t++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (!seen(tok0 + (F32 ? 0 : 16 * t) + 4 * lg + j)) va[t][j] = Ld{};
        }
        // K rows through LDS into the A-operand layout: lane (lg, lc) needs row lc, dims
        // 32kk + 8lg .. +7 (fp32: 16kk + 4lg .. + 3). One wave per workgroup and LDS operations
        // of a wave complete in order, so the wave barriers only keep the compiler from moving
        // LDS accesses across. The second tile's writes follow the first tile's reads in that
        // order.
        u32x4 kA[TILES][NQ];
#pragma unroll
        for (int t = 0; t < TILES; t++) {
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < NL / TILES; i++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    *reinterpret_cast<Ld*>(&kt[(4 * lg + j) * KP + 256 * i + (int)sizeof(Ld) * lc]) =
                        ka[t + i][j];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int kk = 0; kk < NQ; kk++)
                kA[t][kk] = *reinterpret_cast<const u32x4*>(&kt[lc * KP + 64 * kk + 16 * lg]);
        }
        __builtin_amdgcn_wave_barrier();
        // S tiles: s[t][r] = score of head lc for token 16t + 4lg + r of the chunk.
        f32x4 s[TILES];
#pragma unroll
        for (int t = 0; t < TILES; t++) {
            s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (F32) {
                // Sums of 8 products, added pairwise: one chain over the D products of a score has
                // ~1.3 times the vector kernel's rounding error on short contexts.
                f32x4 lvl[4];  // lvl[n]: a pending sum of 2^n k-steps
#pragma unroll
                for (int kk = 0; kk < NQ; kk++) {
                    f32x4 h[2] = {s[t], s[t]};
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        h[e >> 1] = mfma16x16x4_f32(__uint_as_float(kA[t][kk][e]),
                                                    __uint_as_float(qb[kk][e]), h[e >> 1]);
                    f32x4 x = h[0] + h[1];
                    int n = 0;
                    for (; (kk >> n) & 1; n++) x = lvl[n] + x;
                    lvl[n] = x;
                    if (kk & 1) __builtin_amdgcn_sched_barrier(0);  // (few pending sums)
                }
                s[t] = lvl[NQ == 8 ? 3 : 2];
                __builtin_amdgcn_sched_barrier(0);  // (registers: no V^T P^T before the scores)
            } else {
#pragma unroll
                for (int kk = 0; kk < NQ; kk++) s[t] = mfma16x16x32<T>(kA[t][kk], qb[kk], s[t]);
            }
        }
        float sv[4 * TILES];
        float tmax = -INFINITY;
#pragma unroll
        for (int t = 0; t < TILES; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const bool ok = full || seen(tok0 + 16 * t + 4 * lg + r);
                sv[4 * t + r] = ok ? s[t][r] * scale_log2 : -INFINITY;
                tmax = fmaxf(tmax, sv[4 * t + r]);
            }
        if constexpr (WTS) {
            if (lc < n_rep)
#pragma unroll
                for (int t = 0; t < TILES; t++)
                    *reinterpret_cast<f32x4*>(score_to + tok0 + 16 * t + score_lane) =
                        f32x4{sv[4 * t], sv[4 * t + 1], sv[4 * t + 2], sv[4 * t + 3]};
        }
        tmax = max_across_rows(tmax);
        const float m_new = fmaxf(m, tmax);
        const float alpha = fast_exp2(m - m_new);
        float p[4 * TILES];
#pragma unroll
        for (int i = 0; i < 4 * TILES; i++)  // fp32: the scaling and the difference round once
            p[i] = fast_exp2(F32 ? (sv[i] == -INFINITY ? sv[i] : fmaf(s[0][i & 3], scale_log2, -m_new))
                                 : sv[i] - m_new);
        float psum = (p[0] + p[1]) + (p[2] + p[3]);
        if constexpr (TILES == 2) psum += (p[4] + p[5]) + (p[6] + p[7]);
        lsum = lsum * alpha + psum;
        if (__builtin_amdgcn_ballot_w64(m_new > m) != 0) {
#pragma unroll
            for (int nn = 0; nn < NV; nn++) acc[nn] *= alpha;
        }
        m = m_new;
        if constexpr (F32) {
            // O^T += V^T P^T, one product per score register j and 16-dim block nn = 4i + e: B is
            // the lane's p[j] (token 4lg + j, head lc), A the lane's V at that token, dim
            // 64i + 4lc + e. The chunk is summed by itself and then added, so a long context's sum
            // is a sum of chunk sums (fp32 rounding: relative error against 64 bits of 16 x 256-
            // 2,048 tokens 2.7e-7 with one chain, the vector kernel 2.0e-7).
#pragma unroll
            for (int nn = 0; nn < NV; nn++) {
                f32x4 t = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < 4; j++)
                    t = mfma16x16x4_f32(__uint_as_float(va[nn >> 2][j][nn & 3]), p[j], t);
                acc[nn] += t;
            }
        } else {
            // P^T as the B operand over the 32 tokens: lane (lg, lc) holds head lc at
            // k-slots 8lg + j: j < 4 -> token 4lg + j (tile 0), j >= 4 -> 16 + 4lg + j - 4.
            // Split hi + lo so the product keeps ~16 mantissa bits of P.
            u32x4 PH, PL;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t hi16 = pack2<T>(p[2 * i], p[2 * i + 1]);
                PH[i] = hi16;
                PL[i] = pack2<T>(p[2 * i] - lo_f32<T>(hi16), p[2 * i + 1] - hi_f32<T>(hi16));
            }
            // V^T as the A operand: lane (lg, lc) holds output dim (D / 16) lc + nn at the same
            // k-slots, packed in-lane from its four V rows of each tile.
#pragma unroll
            for (int nn = 0; nn < NV; nn++) {
                const int wd = nn >> 1;
                u32x4 A;
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    if (nn & 1) {
                        A[2 * t] = perm_hi16(va[t][0][wd], va[t][1][wd]);
                        A[2 * t + 1] = perm_hi16(va[t][2][wd], va[t][3][wd]);
                    } else {
                        A[2 * t] = perm_lo16(va[t][0][wd], va[t][1][wd]);
                        A[2 * t + 1] = perm_lo16(va[t][2][wd], va[t][3][wd]);
                    }
                }
                acc[nn] = mfma16x16x32<T>(A, PH, acc[nn]);
                acc[nn] = mfma16x16x32<T>(A, PL, acc[nn]);
            }
        }
    };

    // Piece epilogue from registers: lane (lg, lc) holds head lc, dims (D / 4) lg + NV r + nn
    // (r < 4, nn < NV): D / 4 contiguous dims; fp32 pools: dims 64i + 16lg + 4r + e for nn = 4i + e.
    auto epilogue = [&](int b, int g, bool complete, bool first_piece) {
        if constexpr (PAIRS) return;  // (at the end, all waves together)
        lsum = sum_across_rows(lsum);
        // lg made opaque here, so the per-lane output addresses are formed at the store instead
        // of being hoisted out of the stream as 64-bit values (which spill, and a spill reload
        // waits for every chunk load in flight)
        int lgo = lg;
        asm volatile("" : "+v"(lgo));
        if (lc < n_rep) {
            // F32: undefined sums give zero rows (RNG hands them on, and clears where no score is above -inf: its
            // accumulators are 0 times values that may be NaN)
            constexpr bool CLEAR = F32 && !RNG;
            if (complete) {  // whole pair in this range: final output
                if constexpr (WTS)
                    if (lg == 0) {
                        float* ml = ws.row_ml + 2 * ((int64_t)b * num_heads + (int64_t)g * n_rep + lc);
                        ml[0] = m;
                        ml[1] = lsum;
                    }
                const int64_t row = ws.rows ? (int64_t)ws.rows[b] : (int64_t)b;
                const int64_t o_at = (row * num_heads + (int64_t)g * n_rep + lc) * D +
                                     (F32 ? 16 : D / 4) * lgo;
                TO* o = out + o_at;
                const float inv = 1.0f / divisor<CLEAR>(lsum);
                if (RNG ? lsum == 0.0f : CLEAR && !(lsum > 0.0f))
#pragma unroll
                    for (int nn = 0; nn < NV; nn++) acc[nn] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if constexpr (std::is_same<TO, AnyOut>::value) {
#pragma unroll
                        for (int h4 = 0; h4 < NV; h4 += 4) {
                            const float v[4] = {acc[h4][r] * inv, acc[h4 + 1][r] * inv,
                                                acc[h4 + 2][r] * inv, acc[h4 + 3][r] * inv};
                            store_run<4>(out, rng.out_dtype, o_at + (F32 ? 16 * h4 + 4 * r : NV * r + h4), v);
                        }
                    } else if constexpr (F32) {
#pragma unroll
                        for (int h4 = 0; h4 < NV; h4 += 4) {
                            const f32x4 v = f32x4{acc[h4][r] * inv, acc[h4 + 1][r] * inv,
                                                  acc[h4 + 2][r] * inv, acc[h4 + 3][r] * inv};
                            if constexpr (sizeof(TO) == 4)
                                *reinterpret_cast<f32x4*>(o + 16 * h4 + 4 * r) = v;
                            else
                                *reinterpret_cast<u32x2*>(o + 16 * h4 + 4 * r) =
                                    u32x2{pack2<TO>(v[0], v[1]), pack2<TO>(v[2], v[3])};
                        }
                    } else if constexpr (sizeof(TO) == 4) {
#pragma unroll
                        for (int h4 = 0; h4 < NV; h4 += 4)
                            *reinterpret_cast<f32x4*>(o + NV * r + h4) =
                                f32x4{acc[h4][r] * inv, acc[h4 + 1][r] * inv, acc[h4 + 2][r] * inv,
                                      acc[h4 + 3][r] * inv};
                    } else {
                        uint32_t v[NV / 2];
#pragma unroll
                        for (int i = 0; i < NV / 2; i++)
                            v[i] = pack2<TO>(acc[2 * i][r] * inv, acc[2 * i + 1][r] * inv);
                        if constexpr (NV == 8)
                            *reinterpret_cast<u32x4*>(o + NV * r) = u32x4{v[0], v[1], v[2], v[3]};
                        else
                            *reinterpret_cast<u32x2*>(o + NV * r) = u32x2{v[0], v[1]};
                    }
                }
            } else {  // partial row for the merge kernel
                const int64_t pidx = (2 * wgi + (first_piece ? 0 : 1)) * n_rep + lc;
                float* o = ws.o + pidx * D + (F32 ? 16 : D / 4) * lgo;
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int h4 = 0; h4 < NV; h4 += 4)
                        *reinterpret_cast<f32x4*>(o + (F32 ? 16 * h4 + 4 * r : NV * r + h4)) =
                            f32x4{acc[h4][r], acc[h4 + 1][r], acc[h4 + 2][r], acc[h4 + 3][r]};
                if (lg == 0) {
                    ws.ml[2 * pidx] = m;
                    ws.ml[2 * pidx + 1] = lsum;
                }
            }
        }
        m = DEC_M0;
        lsum = 0.0f;
#pragma unroll
        for (int nn = 0; nn < NV; nn++) acc[nn] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    };

    // ---- the chunk stream. The next segment's block-table slots are read while the current
    // one streams, and the two register buffers ping-pong across segment and piece boundaries:
    // the next chunk's loads (chosen with uniform selects, never a branch, so the compiler's
    // wait counts stay exact) are in flight while the current chunk is computed and while a
    // finished piece is written out.
    // FUSE: the new K / V row of every pair whose last chunk lies in this wave's range, written
    // to the pool before the range's first chunk load. The lanes that write a row, (lg, lc) with
    // 4 lg <= slot % 16 < 4 lg + 4 (the row's place in its 16-token tile, as the block table
    // places position context_len - 1), are the lanes that load it back in load_chunk, at the
    // same bytes (dims (D / 16) lc ..), so the wave's own program order makes the later load see
    // the row. No other wave reads the slot: the pair's last chunk, the only one holding the
    // new position, is in this range alone, and a batch's new slots are private to their
    // sequences. The first two pairs' rows are requested before the block-table and q loads
    // (their wait then overlaps those loads), stored after them; further pairs (short contexts)
    // two at a time after that.
    struct NewRows {
        int b, g, slot[2], pb[2], pg[2];
        bool pv[2], more;
        int first, nch;
        Ld kr[2], vr[2];
    };
    auto new_rows_load = [&](NewRows& nr) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            nr.pv[i] = nr.more;
            nr.pb[i] = nr.b;
            nr.pg[i] = nr.g;
            if (nr.more) {  // on to the next pair in the flattened order (sequences with chunks)
                nr.first += nr.nch;
                if (++nr.g == kv_heads) {
                    nr.g = 0;
                    do {
                        nr.b++;
                    } while (nr.b < batch && pre[nr.b + 1] == pre[nr.b]);
                }
                if (nr.b < batch) {
                    nr.nch = pre[nr.b + 1] - pre[nr.b];
                    nr.more = nr.first + nr.nch - 1 < len;
                } else {
                    nr.more = false;
                }
            }
        }
        const T* kn = static_cast<const T*>(ws.k_new);
        const T* vn = static_cast<const T*>(ws.v_new);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            nr.slot[i] = nr.pv[i] ? ws.new_slots[nr.pb[i]] : -1;
            if (nr.pv[i]) {
                const int64_t src = (int64_t)nr.pb[i] * ws.new_st + (int64_t)nr.pg[i] * ws.new_sh +
                                    (D / 16) * lc;
                nr.kr[i] = *reinterpret_cast<const Ld*>(kn + src);
                nr.vr[i] = *reinterpret_cast<const Ld*>(vn + src);
            }
        }
    };
    auto new_rows_store = [&](const NewRows& nr) {
        T* const kpw = const_cast<T*>(k_pool);
        T* const vpw = const_cast<T*>(v_pool);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int sl = nr.slot[i];
            if (nr.pv[i] && sl >= 0 && sl < num_slots && lg == ((sl & 15) >> 2)) {
                const int64_t dst = ((int64_t)nr.pg[i] * num_slots + sl) * D + (D / 16) * lc;
                *reinterpret_cast<Ld*>(kpw + dst) = nr.kr[i];
                *reinterpret_cast<Ld*>(vpw + dst) = nr.vr[i];
            }
        }
    };

    // PAIRS: the waves' states through LDS, then wave r writes dims (D / 4) lg + NV r .. (fp32: 64 i + 16 lg + 4 r ..),
    // folded over the waves.
    auto fold = [&]() {
        constexpr int WAVE = dec_pair_lds(D, sizeof(T)) / 4;
        float* const all = reinterpret_cast<float*>(pre);
        lsum = sum_across_rows(lsum);
        float* const mine = all + w_id * WAVE;
#pragma unroll
        for (int nn = 0; nn < NV; nn++) *reinterpret_cast<f32x4*>(mine + (nn * 64 + lane) * 4) = acc[nn];
        mine[NV * 256 + lane] = m;
        mine[NV * 256 + 64 + lane] = lsum;
        __syncthreads();
        static_assert(DEC_PAIR_WAVES == 4, "a wave for each of the four runs of a lane's dims");
        float M = DEC_M0, L = 0.0f;
        for (int x = 0; x < DEC_PAIR_WAVES; x++) M = fmaxf(M, all[x * WAVE + NV * 256 + lane]);
        for (int x = 0; x < DEC_PAIR_WAVES; x++)
            L += fast_exp2(all[x * WAVE + NV * 256 + lane] - M) * all[x * WAVE + NV * 256 + 64 + lane];
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        if (lc >= n_rep) return;
        const int64_t o_at = ((int64_t)pb * num_heads + (int64_t)pg * n_rep + lc) * D + (F32 ? 16 : D / 4) * lg;
        float o[NV];
#pragma unroll
        for (int nn = 0; nn < NV; nn++) o[nn] = 0.0f;
        for (int x = 0; x < DEC_PAIR_WAVES; x++) {
            const float* from = all + x * WAVE;
            const float w = fast_exp2(from[NV * 256 + lane] - M) * inv;
#pragma unroll
            for (int nn = 0; nn < NV; nn++) o[nn] = fmaf(w, from[(nn * 64 + lane) * 4 + w_id], o[nn]);
        }
        if (L == 0.0f)
#pragma unroll
            for (int nn = 0; nn < NV; nn++) o[nn] = 0.0f;
#pragma unroll
        for (int h4 = 0; h4 < NV; h4 += 4)
            store_run<4>(out, rng.out_dtype, o_at + (F32 ? 16 * h4 + 4 * w_id : NV * w_id + h4), o + h4);
    };
    if constexpr (PAIRS) {
        if (len == 0) {  // (fewer chunks than waves, or an empty context: zero rows)
            fold();
            return;
        }
    }

    Seg cur = seg_at(0);
    NewRows nr{};
    if constexpr (FUSE) {
        nr.b = cur.b;
        nr.g = cur.g;
        nr.nch = cur.nch;
        nr.first = -cur.cb;  // pair (b, g)'s first chunk, as an offset from lo
        nr.more = nr.first + nr.nch - 1 < len;
        new_rows_load(nr);
    }
    Slots cur_slots = seg_slots(cur);
    int nx = cur.ce - cur.cb;
    bool has_nxt = nx < len;
    Seg nxt = cur;
    Slots nxt_slots{0, 0};  // (not a copy of cur_slots, which would wait for its load)
    if (has_nxt) {
        nxt = seg_at(nx);
        nxt_slots = seg_slots(nxt);
    }
    int pc0 = cur.cb;  // first chunk of the current piece
    bool first_piece = true;
    int c = cur.cb;
    load_q(cur.b, cur.g);

    // One stream step: prefetch the chunk after c into (kn, vn) (PREFETCH is a compile-time
    // constant at each call, so the steady-state loop has no conditional loads), compute c
    // from (kc, vc), then advance the cursor.
    auto step = [&](auto prefetch, Ld (*kc)[4], Ld (*vc)[4], Ld (*kn)[4], Ld (*vn)[4]) {
        const bool seg_end = c + 1 >= cur.ce;
        // At a segment's last chunk the segment after the next one is looked up and its
        // block-table entries are requested before this step's chunk loads, so the rotation at
        // the end of the step waits for that load alone and not for the chunk loads behind it.
        int nn_x = nx;
        bool has_nn = false;
        Seg nn = nxt;
        Slots nn_slots = nxt_slots;
        if (seg_end && has_nxt) {
            nn_x = nx + (nxt.ce - nxt.cb);
            has_nn = nn_x < len;
            if (has_nn) {
                nn = seg_at(nn_x);
                nn_slots = seg_slots(nn);
            }
        }
        if constexpr (decltype(prefetch)::value) {
            const bool in_cur = c + 1 < cur.ce;
            const int pg = in_cur ? cur.g : nxt.g;
            const Slots pslots = in_cur ? cur_slots : nxt_slots;
            const int ptile = in_cur ? TILES * (c + 1 - cur.cb) : 0;
            load_chunk(pg, pslots, ptile, kn, vn);
        }
        compute_chunk(c, cur.tok_end, kc, vc);
        if (!seg_end) {
            c += 1;
            return;
        }
        // end of a segment
        const bool piece_end = !PAIRS && (!has_nxt || nxt.b != cur.b || nxt.g != cur.g);
        if (piece_end) epilogue(cur.b, cur.g, pc0 == 0 && cur.ce == cur.nch, first_piece);
        if (!has_nxt) return;
        if (piece_end) {
            pc0 = nxt.cb;
            first_piece = false;
            load_q(nxt.b, nxt.g);
        }
        cur = nxt;
        cur_slots = nxt_slots;
        c = cur.cb;
        nx = nn_x;
        has_nxt = has_nn;
        if (has_nn) {
            nxt = nn;
            nxt_slots = nn_slots;
        }
    };


    if constexpr (FUSE) {
        new_rows_store(nr);
        while (nr.more) {
            new_rows_load(nr);
            new_rows_store(nr);
        }
        asm volatile("" ::: "memory");  // the stores stay before the chunk loads
    }

    using pf_on = std::integral_constant<bool, true>;
    using pf_off = std::integral_constant<bool, false>;
    Ld ka[NL][4], va[NL][4], kb[NL][4], vb[NL][4];
    load_chunk(cur.g, cur_slots, 0, ka, va);
    int remaining = len;  // chunks this wave computes; all but the last prefetch one
    for (; remaining > 2; remaining -= 2) {
        step(pf_on{}, ka, va, kb, vb);
        step(pf_on{}, kb, vb, ka, va);
    }
    if (remaining == 2) {
        step(pf_on{}, ka, va, kb, vb);
        step(pf_off{}, kb, vb, ka, va);
    } else {
        step(pf_off{}, ka, va, kb, vb);
    }
    if constexpr (PAIRS) fold();
}

// Merge of the pieces of pairs cut by wave ranges, and zero rows for empty contexts: one
// workgroup per (query head, sequence), lane i owning output dims 2i and 2i + 1, locating its
// pieces from the chunk prefix sums the main kernel left in the workspace. Pieces are taken 64 at
// a time (one per lane): their (max, sum) pairs become weights through wave reductions, then every
// lane accumulates its two dims over the batch with independent loads, reading each piece's
// weight and slot from the lane that holds it; batches combine with the same online rescaling
// as the running update of cpu.rs:96-105. With many pieces per pair (few sequences) the
// workgroup's waves split them, since one wave reads them 8 rows a memory round trip, and fold
// their states through LDS; with one wave there is no LDS and no barrier.
static constexpr int DEC_MERGE_WAVES = 8;
template <typename TO, int D, bool F32, bool WTS>
__global__ __launch_bounds__(64 * DEC_MERGE_WAVES) void paged_decode_merge_kernel(
    TO* __restrict__ out, int batch, int num_heads, int kv_heads, int n_rep, int nwg_i,
    DecodeWs ws) {
    // lane i owns output dims E i .. E i + E - 1
    constexpr int E = D / 64;
    const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 63;
    const int w_id = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    // chunks before sequence b, of sequence b and in all sequences (the main kernel's sums)
    const int before = ws.pre[b], nch = ws.pre[b + 1] - before, all = ws.pre[batch];
    const int64_t orow = ws.rows ? (int64_t)ws.rows[b] : (int64_t)b;
    TO* o = out + (orow * num_heads + h) * D + E * lane;
    constexpr bool ANY = std::is_same<TO, AnyOut>::value;
    const int64_t o_at = (orow * num_heads + h) * D + E * lane;
    if (nch == 0) {
        if (w_id == 0)
#pragma unroll
            for (int i = 0; i < E; i++) {
                if constexpr (ANY)
                    store_1(out, ws.rng.out_dtype, o_at + i, 0.0f);
                else
                    o[i] = from_f32<TO>(0.0f);
            }
        return;
    }
    const int g = h / n_rep, hh = h - g * n_rep;
    const int64_t total = (int64_t)kv_heads * all, nwg = range_count(total, nwg_i);
    const int64_t s = (int64_t)kv_heads * before + (int64_t)g * nch;
    const int64_t e = s + nch;
    const bool narrow = ranges_narrow(total, nwg, ws.xcd_w);
    const WaveRanges<uint32_t> r32(narrow ? total : 1, nwg, ws.xcd_w);
    const WaveRanges<int64_t> r64(total, nwg, ws.xcd_w);
    auto range_lo = [&](int64_t i) -> int64_t {
        return narrow ? (int64_t)r32.lo((uint32_t)i) : r64.lo(i);
    };
    const int64_t f = narrow ? (int64_t)r32.owner((uint32_t)s) : r64.owner(s);
    const int64_t l = narrow ? (int64_t)r32.owner((uint32_t)(e - 1)) : r64.owner(e - 1);
    const bool f_first = s == range_lo(f);
    if (f == l) return;  // finished inside one wave range
    const int np = (int)(l - f + 1);  // ranges f..l, none of them empty

    float M = DEC_M0, L = 0.0f, O[E];
#pragma unroll
    for (int i = 0; i < E; i++) O[i] = 0.0f;
    const int fslot = (int)(f_first ? 2 * f : 2 * f + 1);  // the first piece always exists
    auto piece_slot = [&](int64_t p) -> int {  // slot of piece p (< np)
        const int64_t ij = f + p;
        return (int)((ij == f && !f_first) ? 2 * ij + 1 : 2 * ij);
    };
    typedef typename std::conditional<E == 2, f32x2, float>::type RowV;
    auto row = [&](int slot) -> RowV {  // this lane's E dims of a piece's partial row
        return *reinterpret_cast<const RowV*>(ws.o + ((int64_t)slot * n_rep + hh) * D + E * lane);
    };
    auto add = [&](float wj, RowV v) {
        if constexpr (E == 2) {
            O[0] += wj * v[0];
            O[1] += wj * v[1];
        } else {
            O[0] += wj * v;
        }
    };
    // this wave's pieces: an equal share
    const int per = waves == 1 ? np : (np + waves - 1) / waves;
    const int p_end = min(np, (w_id + 1) * per);
    for (int p0 = w_id * per; p0 < p_end; p0 += 64) {
        // The batch's first 8 pieces' rows are loaded before the (max, sum) reductions, which
        // they do not depend on (a missing piece reads the first piece's row, weight 0).
        const int slot = p0 + lane < p_end ? piece_slot(p0 + lane) : -1;
        RowV v0[8];
        int s0[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            s0[j] = p0 + j < p_end ? piece_slot(p0 + j) : -1;
            v0[j] = row(s0[j] >= 0 ? s0[j] : fslot);
        }
        float mx = -INFINITY, lx = 0.0f;
        if (slot >= 0) {
            mx = ws.ml[2 * ((int64_t)slot * n_rep + hh)];
            lx = ws.ml[2 * ((int64_t)slot * n_rep + hh) + 1];
        }
        const float m_new = fmaxf(M, wave_max(mx));
        const float w = (slot >= 0) ? fast_exp2(mx - m_new) : 0.0f;
        const float bl = wave_sum(w * lx);
        const float c_old = fast_exp2(M - m_new);
        L = L * c_old + bl;
#pragma unroll
        for (int i = 0; i < E; i++) O[i] *= c_old;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float wj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), j));
            if (s0[j] >= 0) add(wj, v0[j]);
        }
        // The rest in groups of 8 unconditional loads (a missing piece reads the first piece's
        // row) so they are all in flight together; the select drops them, so stale workspace
        // bits (even NaN) never reach the sum.
        const int nb = min(64, p_end - p0);
        for (int q = 8; q < nb; q += 8) {
            RowV v[8];
            int sl[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                sl[j] = __builtin_amdgcn_readlane(slot, q + j);
                v[j] = row(sl[j] >= 0 ? sl[j] : fslot);
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float wj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), q + j));
                if (sl[j] >= 0) add(wj, v[j]);
            }
        }
        M = m_new;
    }
    if (waves > 1) {  // the waves' states, folded by the first (it always has pieces)
        __shared__ float wM[DEC_MERGE_WAVES], wL[DEC_MERGE_WAVES];
        __shared__ float wO[DEC_MERGE_WAVES][E][64];
        if (lane == 0) {
            wM[w_id] = M;
            wL[w_id] = L;
        }
#pragma unroll
        for (int i = 0; i < E; i++) wO[w_id][i][lane] = O[i];
        __syncthreads();
        if (w_id != 0) return;
        // all states are read together; slots past the last wave with pieces read its own
        float mx[DEC_MERGE_WAVES], lx[DEC_MERGE_WAVES], ox[DEC_MERGE_WAVES][E];
        float Mt = M;
#pragma unroll
        for (int x = 1; x < DEC_MERGE_WAVES; x++) {
            const bool on = x < waves && x * per < np;
            const int y = on ? x : 0;
            mx[x] = on ? wM[y] : -INFINITY;
            lx[x] = wL[y];
#pragma unroll
            for (int i = 0; i < E; i++) ox[x][i] = wO[y][i][lane];
        }
#pragma unroll
        for (int x = 1; x < DEC_MERGE_WAVES; x++) Mt = fmaxf(Mt, mx[x]);
        const float f0 = fast_exp2(M - Mt);
        L *= f0;
#pragma unroll
        for (int i = 0; i < E; i++) O[i] *= f0;
#pragma unroll
        for (int x = 1; x < DEC_MERGE_WAVES; x++) {
            if (x < waves && x * per < np) {
                const float f = fast_exp2(mx[x] - Mt);
                L += lx[x] * f;
#pragma unroll
                for (int i = 0; i < E; i++) O[i] += ox[x][i] * f;
            }
        }
    }
    if constexpr (WTS)
        if (lane == 0) {
            ws.row_ml[2 * ((int64_t)b * num_heads + h)] = M;
            ws.row_ml[2 * ((int64_t)b * num_heads + h) + 1] = L;
        }
#pragma unroll
    for (int i = 0; i < E; i++) {
        const float x = O[i] / divisor<F32>(L);
        if constexpr (ANY)
            store_1(out, ws.rng.out_dtype, o_at + i, L == 0.0f ? 0.0f : x);
        else
            o[i] = from_f32<TO>(F32 && !(L > 0.0f) ? 0.0f : x);
    }
}

// Waves per merge workgroup: about eight pieces (one memory round trip) each, for twice the mean
// number of pieces per pair (longer contexts than the mean have more).
static int decode_merge_waves(int grid, int batch, int kv_heads) {
    const int64_t pieces = 2 * (int64_t)grid / ((int64_t)batch * kv_heads);
    int waves = 1;
    while (waves < DEC_MERGE_WAVES && 8 * waves < pieces) waves *= 2;
    return waves;
}

}  // namespace flour
