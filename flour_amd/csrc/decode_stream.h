// decode_stream.h — attention of few query rows over an 8-bit cache, streamed from HBM on the f16
// matrix cores: decode steps and short runs of new rows (drafted tokens, short turns). Instantiated
// per type of the queries in decode_stream_*.hip.
//
// With few rows per sequence the step reads each K/V byte once and is bound by that; everything
// else has to fit beside the stream. Work split: as in paged_decode.hip, the chunks of every
// (sequence, kv head, column group) laid end to end and cut into equal wave ranges, one-wave
// workgroups, pieces of pairs cut by a range end merged by a second kernel.
//
// Inside a piece, for a column = (query row, query head of the kv head), 16 to a matrix tile, NT
// tiles to a wave:
//  * A chunk is TILES tiles of 16 tokens, 2 KB of K and of V each at head_dim 128. Two register
//    buffers: the next chunk's loads are in flight while one is computed.
//  * S = K Q^T on v_mfma_f32_16x16x32_f16. K is loaded as it lies in memory, 1 KB an instruction, and
//    turned into the A layout (lane (g, c) = (lane / 16, lane % 16): bytes 16g .. of token c's row, the
//    columns of Q^T permuted to match) through LDS. Loaded in that layout, a 64-byte half of 16 rows an
//    instruction, the stream alone stops at 4.2-4.6 TB/s against 4.9-5.3. Bytes become f16 exactly:
//    e4m3 by the converter, int8 by placing x + 128 under the exponent of 1,024 and subtracting 1,152.
//  * Queries are f16: f16 ones as they are; bf16 ones times a power of two per (row, head) that puts
//    the largest element just below 2^15 (exact down to 2^-31 of it); fp32 ones as two f16 parts of that
//    (22 bits, two products).
//  * A block's K scale multiplies its 16 tokens' scores, one factor per tile. Its V scale S_v goes
//    into the exponent: P' = 2^(s + log2 S_v - m'), with a reference m' of its own (within 2^8 of the
//    running maximum) beside the maximum m of s that the sum of p = 2^(s - m) uses, formed as p times a
//    factor per tile. So f16 keeps P' relative to the row's largest contribution whatever the blocks'
//    scales (up to 2^100 apart, where p leaves fp32's range), and V stays the integers and e4m3 values
//    that it is. P' is split into two f16 parts: two products, 22 bits.
//  * The score registers are the B operand of O^T = V^T P'^T as they stand; the V^T operand is built
//    in-lane, pairs of tokens' bytes by v_perm_b32, then the same conversion.
//
// Measured, kernel + merge: decode steps, 64 x 512-4,096 tokens of 32 / 8 heads of 128 in e4m3 (278
// MB) 54 + 6.5 us, the stream at 5.1 TB/s, what its loads reach alone; 8 x 16-32K of 64 / 8 in int8 (415
// MB) 72 + 6 us, 5.7 TB/s; one sequence of 2,000 tokens 7 + 5 us, launches and dependent loads. Drafted
// rows, 32 sequences of 512-4,096 tokens with 3-8 rows of 32 / 8 heads (162 MB) 49 + 9.5 us: with two
// column tiles a SIMD holds one wave, whose vector instructions take 47% of the time and its waits the rest.
#pragma once

#include <math.h>

#include <algorithm>

#include "cache8.h"
#include "decode_pools.h"
#include "decode_ranges.h"

namespace flour {

static constexpr int DP_MAX_BATCH = 4096;  // per-sequence chunk sums live in LDS
// P' times 2^7: clear of f16's subnormals down to 2^-21 of the largest, with room for a reference that lags
// the running maximum by up to 2^8.
static constexpr float DP_SHIFT = 7.0f, DP_LAG = 8.0f;
static constexpr int DP_XCD_W = 2;         // the wave ranges' weight (paged_decode.hip)

// Rows of sequence s, its kv length (0 where its rows see nothing).
struct DpSeq {
    int row0, rows, kv;
};
__device__ __forceinline__ DpSeq dp_seq(const DpArgs& a, int s) {
    const int r0 = a.cu ? a.cu[s] : s, n = a.cu ? a.cu[s + 1] - r0 : 1;
    const int kv = min(a.kv_lens[s], a.max_kv);
    // (the pieces' slots hold the columns of max_rows rows)
    return DpSeq{r0, min(max(n, 0), a.max_rows), kv >= n && kv > 0 ? kv : 0};
}
// Column groups of n rows of n_rep heads; chunks of all of them over kv positions.
template <int NT>
__device__ __forceinline__ int dp_groups(int rows, int n_rep) {
    return (rows * n_rep + 16 * NT - 1) / (16 * NT);
}

// Four bytes to two f16 pairs.
template <typename TP>
__device__ __forceinline__ u32x2 to_f16x4(uint32_t w);
template <>
__device__ __forceinline__ u32x2 to_f16x4<e4m3_t>(uint32_t w) {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))};
}
template <>
__device__ __forceinline__ u32x2 to_f16x4<i8_t>(uint32_t w) {
    const uint32_t x = w ^ 0x80808080u;  // x + 128
    const f16x2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const uint32_t a = __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u);
    const uint32_t b = __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u);
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, a) + off),
                 __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, b) + off)};
}

// Resident waves per CU: two per SIMD, or one where a wave's registers hold several column tiles or two
// chunks of 64 tokens at head_dim 128 (and fewer waves leave fewer pieces to merge).
template <int D, int TILES, int NT>
__host__ __device__ constexpr int dp_waves() {
    return NT > 1 || (TILES == 4 && D == 128) ? 4 : 8;
}

// MULTI: several rows of a sequence, or more query heads of a kv head than a tile has columns;
// otherwise a decode step whose columns are one tile's.
template <typename TQ, typename TP, int D, int TILES, int NT, bool MULTI, bool BS16, bool W>
__global__ __launch_bounds__(64, (dp_waves<D, TILES, NT>() / 4)) void decode_pools_kernel(DpArgs a) {
    constexpr int CHUNK = 16 * TILES;
    constexpr int KL = D / 64;   // 16-byte K loads of a lane and tile
    constexpr int NV = D / 16;   // O^T products of a chunk's half
    constexpr int KK = D / 32;   // products of a score tile
    constexpr int QP = sizeof(TQ) == 4 ? 2 : 1;  // parts of a query
    typedef typename std::conditional<D == 128, u32x2, uint32_t>::type Vd;
    constexpr int KP = D + 16;  // bytes of a K row in LDS: 16-byte reads of 16 rows spread over the banks
    extern __shared__ int pre[];
    __shared__ __attribute__((aligned(16))) unsigned char kt[16 * KP];  // one K tile
    const int lane = threadIdx.x, lg = lane >> 4, lc = lane & 15;
    const int n_rep = a.n_rep, batch = a.batch;
    // (opaque: where it is known to be 0, joins with paths where it is not would make it per lane)
    int wg = blockIdx.x;
    asm volatile("" : "+s"(wg));

    auto seq_of = [&](int s) -> DpSeq {
        if constexpr (MULTI) return dp_seq(a, s);
        return DpSeq{s, 1, max(min(a.kv_lens[s], a.max_kv), 0)};
    };
    auto groups_of = [&](int rows) -> int { return MULTI ? dp_groups<NT>(rows, n_rep) : 1; };
    auto seq_chunks = [&](const DpSeq& q) -> int {
        return groups_of(q.rows) * ((q.kv + CHUNK - 1) / CHUNK);
    };
    // ---- exclusive prefix sums of the sequences' chunks (per kv head); up to 64 sequences stay in
    // registers, one a lane
    const bool in_lanes = batch <= 64;
    DpSeq my = {0, 0, 0};
    int my_pre = 0, all_chunks;
    if (in_lanes) {
        if (lane < batch) my = seq_of(lane);
        const int n = seq_chunks(my);
        const int incl = wave_incl_sum(n);
        my_pre = incl - n;
        all_chunks = __builtin_amdgcn_readlane(incl, 63);
        if (wg == 0) {
            if (lane < batch) a.pre[lane] = my_pre;
            if (lane == 63) a.pre[batch] = incl;
        }
    } else {
        const int per = (batch + 63) / 64;
        int local = 0;
        for (int i = 0; i < per; i++) {
            const int b = lane * per + i;
            if (b < batch) {
                const int n = seq_chunks(seq_of(b));
                pre[b] = n;
                local += n;
            }
        }
        const int incl = wave_incl_sum(local);
        int run = incl - local;
        for (int i = 0; i < per; i++) {
            const int b = lane * per + i;
            if (b < batch) {
                const int n = pre[b];
                pre[b] = run;
                run += n;
            }
        }
        if (lane == 63) pre[batch] = incl;
        __syncthreads();
        all_chunks = __builtin_amdgcn_readlane(incl, 63);
        if (wg == 0)
            for (int b = lane; b <= batch; b += 64) a.pre[b] = pre[b];
    }
    // (scalar again: the paths above join under per-lane stores, and a divergent value here makes
    // every branch and register of the stream per lane)
    const int64_t total = (int64_t)a.kv_heads * __builtin_amdgcn_readfirstlane(all_chunks);
    const int64_t nwg = range_count(total, gridDim.x);
    const int64_t wgi = wg;
    if (total == 0 || wgi >= nwg) return;
    const bool narrow = ranges_narrow(total, nwg, DP_XCD_W);
    int64_t lo;
    int len;
    if (narrow) {
        const WaveRanges<uint32_t> wr(total, nwg, DP_XCD_W);
        const uint32_t x = wr.lo((uint32_t)wgi);
        lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
        len = __builtin_amdgcn_readfirstlane((int)(wr.lo((uint32_t)wgi + 1) - x));
    } else {
        const WaveRanges<int64_t> wr(total, nwg, DP_XCD_W);
        const int64_t x = wr.lo(wgi);
        lo = ((int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32) |
             (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
        len = __builtin_amdgcn_readfirstlane((int)(wr.lo(wgi + 1) - x));
    }

    // ---- segments: up to SEG chunks (64 tiles, one a lane) of one (sequence, kv head, group)
    constexpr int SEG = 64 / TILES;
    struct Seg {
        int b, g, grp_, cb, ce, nch, row0_, rows_, kv;
        Seg() = default;
        // (copied by field: a copy in pieces of other widths keeps the struct in memory)
        __device__ Seg(const Seg& o) { *this = o; }
        __device__ Seg& operator=(const Seg& o) {
            b = o.b, g = o.g, grp_ = o.grp_, cb = o.cb, ce = o.ce, nch = o.nch;
            row0_ = o.row0_, rows_ = o.rows_, kv = o.kv;
            return *this;
        }
        __device__ int grp() const { return MULTI ? grp_ : 0; }
        __device__ int row0() const { return MULTI ? row0_ : b; }
        __device__ int rows() const { return MULTI ? rows_ : 1; }
    };
    auto seg_at = [&](int at) __attribute__((always_inline)) -> Seg {
        const int64_t x = lo + at;
        Seg sg;
        int before;
        if (in_lanes) {
            const uint64_t le = __ballot(lane < batch && (int64_t)a.kv_heads * my_pre <= x);
            sg.b = 63 - __builtin_clzll(le);
            before = __builtin_amdgcn_readlane(my_pre, sg.b);
            sg.kv = __builtin_amdgcn_readlane(my.kv, sg.b);
            sg.row0_ = MULTI ? __builtin_amdgcn_readlane(my.row0, sg.b) : 0;
            sg.rows_ = MULTI ? __builtin_amdgcn_readlane(my.rows, sg.b) : 0;
        } else {
            int l0 = 0, h0 = batch;
            while (h0 - l0 > 1) {
                const int mid = (l0 + h0) >> 1;
                if ((int64_t)a.kv_heads * pre[mid] <= x)
                    l0 = mid;
                else
                    h0 = mid;
            }
            sg.b = __builtin_amdgcn_readfirstlane(l0);
            before = __builtin_amdgcn_readfirstlane(pre[l0]);
            const DpSeq q = seq_of(sg.b);
            sg.kv = __builtin_amdgcn_readfirstlane(q.kv);
            sg.row0_ = MULTI ? __builtin_amdgcn_readfirstlane(q.row0) : 0;
            sg.rows_ = MULTI ? __builtin_amdgcn_readfirstlane(q.rows) : 0;
        }
        sg.nch = (sg.kv + CHUNK - 1) / CHUNK;
        const int64_t rel = x - (int64_t)a.kv_heads * before;
        const int pair = __builtin_amdgcn_readfirstlane(
            narrow ? (int)((uint32_t)rel / (uint32_t)sg.nch) : (int)(rel / sg.nch));
        sg.cb = (int)(rel - (int64_t)pair * sg.nch);
        // a head's groups next to each other: they read the same K/V
        const int groups = __builtin_amdgcn_readfirstlane(groups_of(sg.rows()));
        // (scalar: a divergent value would put every buffer load into a per-lane loop)
        sg.g = !MULTI || groups == 1 ? pair : __builtin_amdgcn_readfirstlane(pair / groups);
        sg.grp_ = MULTI ? pair - sg.g * groups : 0;
        sg.ce = sg.cb + min(min(sg.nch - sg.cb, SEG), len - at);
        return sg;
    };
    const int max_id = (int)(a.num_slots / a.block_size - 1);
    const int64_t nb = a.num_slots / a.block_size;
    struct Slots {
        int id, off;  // lane i: block id as loaded and in-block offset of tile i's first token
    };
    auto seg_slots = [&](Seg sg) -> Slots {
        const int32_t* bt = a.block_tables + (int64_t)sg.b * a.max_blocks;
        const int tok0 = min(sg.cb * CHUNK + lane * 16, ((sg.kv - 1) >> 4) << 4);
        const int lb = BS16 ? (tok0 >> 4) : tok0 / a.block_size;
        return Slots{bt[lb], BS16 ? 0 : tok0 - lb * a.block_size};
    };
    auto clamp_id = [&](int id) -> int { return id < 0 ? 0 : (id > max_id ? max_id : id); };
    struct Scales {
        float k, v;  // lane i: the scales of tile i's block
    };
    auto seg_scales = [&](Seg sg, Slots sl) -> Scales {
        const int64_t at = (int64_t)sg.g * nb + clamp_id(sl.id);
        return Scales{a.k_scale[at], a.v_scale[at]};
    };

    const uint32_t head_bytes = (uint32_t)(a.num_slots * D);
    // K: bytes 16 lane + 1024 i of the tile. V: bytes (D / 16) lc of row 4 lg + j.
    uint32_t k_off = (uint32_t)(16 * lane);
    uint32_t v_off = (uint32_t)(4 * lg * D + (D / 16) * lc);
    asm volatile("" : "+v"(k_off), "+v"(v_off));  // (row offsets stay immediates of the loads)
    auto load_chunk = [&](int head, Slots sl, int tile0, u32x4 (*kd)[KL],
                          Vd (*vd)[4]) __attribute__((always_inline)) {
        const int g = __builtin_amdgcn_readfirstlane(head);
        const __amdgpu_buffer_rsrc_t k_rsrc = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(a.k_pool + (int64_t)g * a.num_slots * D), (short)0, (int)head_bytes, BUF_DWORD3);
        const __amdgpu_buffer_rsrc_t v_rsrc = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(a.v_pool + (int64_t)g * a.num_slots * D), (short)0, (int)head_bytes, BUF_DWORD3);
#pragma unroll
        for (int t = 0; t < TILES; t++) {
            const int id = clamp_id(__builtin_amdgcn_readlane(sl.id, tile0 + t));
            const uint32_t slot =
                BS16 ? (uint32_t)(id * 16)
                     : (uint32_t)(id * a.block_size + __builtin_amdgcn_readlane(sl.off, tile0 + t));
            const uint32_t soff = slot * (uint32_t)D;
#pragma unroll
            for (int i = 0; i < KL; i++)
                kd[t][i] = __builtin_amdgcn_raw_buffer_load_b128(k_rsrc, k_off + 1024 * i, soff, BUF_NT);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (D == 128)
                    vd[t][j] = __builtin_amdgcn_raw_buffer_load_b64(v_rsrc, v_off + j * D, soff, BUF_NT);
                else
                    vd[t][j] = __builtin_amdgcn_raw_buffer_load_b32(v_rsrc, v_off + j * D, soff, BUF_NT);
            }
        }
    };

    // ---- queries: lane (lg, lc) holds column lc of each tile, dims 16 lg + 64 i + 8 h .. + 7 for
    // product kk = 2 i + h
    u32x4 qb[NT][QP][KK];
    float qf[NT];  // what turns a column's products into exp2-domain scores (times the K scale)
    int vis[NT];   // positions that the column sees
    int min_vis;   // that every column sees
    auto load_q = [&](Seg sg) __attribute__((always_inline)) {
        const TQ* q = static_cast<const TQ*>(a.q);
#pragma unroll
        for (int ct = 0; ct < NT; ct++) {
            const int col = (sg.grp() * NT + ct) * 16 + lc;
            const bool real = col < sg.rows() * n_rep;
            const int i = MULTI && real ? col / n_rep : 0, r = real ? col - i * n_rep : 0;
            vis[ct] = real ? sg.kv - sg.rows() + i + 1 : sg.kv;
            const TQ* row = q + (int64_t)(sg.row0() + i) * a.q_st + (int64_t)(sg.g * n_rep + r) * a.q_sh;
            if constexpr (std::is_same<TQ, f16_t>::value) {
                qf[ct] = a.scale_log2;
#pragma unroll
                for (int kk = 0; kk < KK; kk++)
                    qb[ct][0][kk] = real ? *reinterpret_cast<const u32x4*>(
                                               row + 64 * (kk >> 1) + 16 * lg + 8 * (kk & 1))
                                         : u32x4{0, 0, 0, 0};
            } else {
                float x[KK][8];
                float top = 0.0f;
#pragma unroll
                for (int kk = 0; kk < KK; kk++) {
                    const TQ* p = row + 64 * (kk >> 1) + 16 * lg + 8 * (kk & 1);
                    if constexpr (sizeof(TQ) == 4) {
                        const f32x4 u = *reinterpret_cast<const f32x4*>(p);
                        const f32x4 v = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
                        for (int e = 0; e < 4; e++) x[kk][e] = u[e], x[kk][4 + e] = v[e];
                    } else {
                        const u32x4 u = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            x[kk][2 * e] = lo_f32<TQ>(u[e]), x[kk][2 * e + 1] = hi_f32<TQ>(u[e]);
                    }
#pragma unroll
                    for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[kk][e]));
                }
                top = max_across_rows(top);
                // 2^up * top in [2^14, 2^15) (f16 holds twice that); infinities and NaN as they come
                const int ex = (int)(__float_as_uint(top) >> 23);
                const int up = top > 0.0f ? min(14 + 127 - ex, 126) : 0;
                const float f = __uint_as_float((uint32_t)(up + 127) << 23);
                qf[ct] = a.scale_log2 * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
                for (int kk = 0; kk < KK; kk++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float y0 = real ? x[kk][2 * e] * f : 0.0f;
                        const float y1 = real ? x[kk][2 * e + 1] * f : 0.0f;
                        const uint32_t hi = pack2<f16_t>(y0, y1);
                        qb[ct][0][kk][e] = hi;
                        if constexpr (QP == 2)
                            qb[ct][1][kk][e] =
                                pack2<f16_t>(y0 - lo_f32<f16_t>(hi), y1 - hi_f32<f16_t>(hi));
                    }
            }
        }
        min_vis = MULTI ? sg.kv - sg.rows() + 1 +
                              __builtin_amdgcn_readfirstlane(sg.grp() * NT * 16 / n_rep)
                        : sg.kv;
    };

    float m[NT], lsum[NT], mv[NT];
    f32x4 acc[NT][NV];
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int ct = 0; ct < NT; ct++) {
            m[ct] = mv[ct] = DEC_M0;
            lsum[ct] = 0.0f;
#pragma unroll
            for (int nn = 0; nn < NV; nn++) acc[ct][nn] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    };
    clear();

    auto compute_chunk = [&](Seg sg, int c, Scales sc, u32x4 (*ka)[KL],
                             Vd (*va)[4]) __attribute__((always_inline)) {
        // (several column tiles: the compiler would have all of a chunk's conversions in registers)
        auto phase = [] {
            if constexpr (NT > 1) __builtin_amdgcn_sched_barrier(0);
        };
        const int tok0 = c * CHUNK, tile0 = TILES * (c - sg.cb);
        const bool full = tok0 + CHUNK <= min_vis;
        if (tok0 + CHUNK > sg.kv) {  // tokens past the sequence: no bits of theirs
#pragma unroll
            for (int t = 0; t < TILES; t++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (tok0 + 16 * t + 4 * lg + j >= sg.kv) va[t][j] = Vd{};
        }
        f32x4 s[NT][TILES];
#pragma unroll
        for (int t = 0; t < TILES; t++) {
            // One wave a workgroup, whose LDS operations complete in order: the barriers only keep
            // the compiler from moving them.
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < KL; i++)
                *reinterpret_cast<u32x4*>(
                    &kt[(lane / (D / 16) + (1024 / D) * i) * KP + 16 * (lane % (D / 16))]) = ka[t][i];
            __builtin_amdgcn_wave_barrier();
            u32x4 kA[KK];
#pragma unroll
            for (int i = 0; i < KL; i++) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(&kt[lc * KP + 64 * i + 16 * lg]);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const u32x2 x = to_f16x4<TP>(w[2 * h]), y = to_f16x4<TP>(w[2 * h + 1]);
                    kA[2 * i + h] = u32x4{x[0], x[1], y[0], y[1]};
                }
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int ct = 0; ct < NT; ct++) {
                f32x4 z = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int p = QP - 1; p >= 0; p--)
#pragma unroll
                    for (int kk = 0; kk < KK; kk++) z = mfma16x16x32<f16_t>(kA[kk], qb[ct][p][kk], z);
                s[ct][t] = z;
            }
            phase();
        }
        float kf[TILES], lv[TILES];
#pragma unroll
        for (int t = 0; t < TILES; t++) {
            kf[t] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sc.k), tile0 + t));
            lv[t] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sc.v), tile0 + t));
        }
        u32x4 PH[NT][TILES / 2], PL[NT][TILES / 2];
        auto softmax = [&](auto all_seen, int ct) __attribute__((always_inline)) {
            float x[4 * TILES];  // scores
            float top = DEC_M0, topv = -INFINITY;
#pragma unroll
            for (int t = 0; t < TILES; t++) {
                const float f = qf[ct] * kf[t];
                float tile = -INFINITY;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    x[4 * t + r] = s[ct][t][r] * f;
                    if constexpr (!decltype(all_seen)::value)
                        if (tok0 + 16 * t + 4 * lg + r >= vis[ct]) x[4 * t + r] = -INFINITY;
                    tile = fmaxf(tile, x[4 * t + r]);
                }
                top = fmaxf(top, tile);
                // a tile that the column does not see takes nothing from its block, least of all a
                // scale of NaN (fmaxf hands that on to nothing here, so it is selected away)
                topv = fmaxf(topv, tile + lv[t]);
            }
            if constexpr (W) {
                const int r = (sg.grp() * NT + ct) * 16 + lc;  // (decode steps: the query head)
                if (r < n_rep) {
                    float* to = a.scores +
                                ((int64_t)sg.b * a.num_heads + sg.g * n_rep + r) * a.score_stride +
                                tok0 + 4 * lg;
#pragma unroll
                    for (int t = 0; t < TILES; t++)
                        *reinterpret_cast<f32x4*>(to + 16 * t) =
                            f32x4{x[4 * t], x[4 * t + 1], x[4 * t + 2], x[4 * t + 3]};
                }
            }
            const float m_new = fmaxf(m[ct], max_across_rows(top));
            // The reference of P' moves only when the maximum has left it by more than 2^8: with 16
            // columns some column's maximum rises in most chunks, and the accumulators would be
            // rescaled in each.
            const float mv_max = max_across_rows(topv);
            const bool lag = mv_max > mv[ct] + DP_LAG;
            const float mv_new = lag ? mv_max : mv[ct];
            float psum = 0.0f;
#pragma unroll
            for (int t = 0; t < TILES; t++) {
                // P' = p 2^(m + log2 S_v - m'): a factor per tile. It is at most 2^(m - the tile's
                // maximum + 15); the bound keeps it finite where every p of the tile is 0.
                const bool none = !decltype(all_seen)::value && tok0 + 16 * t >= vis[ct];
                const float e = none ? 0.0f : (m_new - mv_new) + (lv[t] + DP_SHIFT);
                const float gt = fast_exp2(e > 126.0f ? 126.0f : e);
                float p[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    p[r] = fast_exp2(x[4 * t + r] - m_new);
                    psum += p[r];
                    p[r] *= gt;
                }
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    const uint32_t hi = pack2<f16_t>(p[r], p[r + 1]);
                    PH[ct][t >> 1][2 * (t & 1) + (r >> 1)] = hi;
                    PL[ct][t >> 1][2 * (t & 1) + (r >> 1)] =
                        pack2<f16_t>(fmaf(lo_f32<f16_t>(hi), -1.0f, p[r]),
                                     fmaf(hi_f32<f16_t>(hi), -1.0f, p[r + 1]));
                }
            }
            lsum[ct] = lsum[ct] * fast_exp2(m[ct] - m_new) + psum;
            m[ct] = m_new;
            if (__builtin_amdgcn_ballot_w64(lag) != 0) {
                const float alpha = fast_exp2(mv[ct] - mv_new);
#pragma unroll
                for (int nn = 0; nn < NV; nn++) acc[ct][nn] *= alpha;
            }
            mv[ct] = mv_new;
        };
#pragma unroll
        for (int ct = 0; ct < NT; ct++) {
            if (full)
                softmax(std::integral_constant<bool, true>{}, ct);
            else
                softmax(std::integral_constant<bool, false>{}, ct);
            phase();
        }
        // V^T: lane (lg, lc) holds dim (D / 16) lc + nn of tokens 4lg .. 4lg + 3 of two tiles
#pragma unroll
        for (int u = 0; u < TILES / 2; u++)
#pragma unroll
            for (int w = 0; w < NV / 4; w++) {
                u32x4 A[4];  // of the dword's four dims
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    uint32_t r[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if constexpr (D == 128)
                            r[j] = va[2 * u + t][j][w];
                        else
                            r[j] = va[2 * u + t][j];
                    }
                    // bytes (row 0, row 1) of dims 0 and 1, of dims 2 and 3; the same of rows 2 and 3
                    const u32x2 a01 = to_f16x4<TP>(__builtin_amdgcn_perm(r[1], r[0], 0x05010400u));
                    const u32x2 a23 = to_f16x4<TP>(__builtin_amdgcn_perm(r[1], r[0], 0x07030602u));
                    const u32x2 b01 = to_f16x4<TP>(__builtin_amdgcn_perm(r[3], r[2], 0x05010400u));
                    const u32x2 b23 = to_f16x4<TP>(__builtin_amdgcn_perm(r[3], r[2], 0x07030602u));
                    A[0][2 * t] = a01[0], A[0][2 * t + 1] = b01[0];
                    A[1][2 * t] = a01[1], A[1][2 * t + 1] = b01[1];
                    A[2][2 * t] = a23[0], A[2][2 * t + 1] = b23[0];
                    A[3][2 * t] = a23[1], A[3][2 * t + 1] = b23[1];
                }
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int ct = 0; ct < NT; ct++) {
                        f32x4& o = acc[ct][4 * w + e];
                        o = mfma16x16x32<f16_t>(A[e], PH[ct][u], o);
                        o = mfma16x16x32<f16_t>(A[e], PL[ct][u], o);
                    }
                phase();
            }
    };

    // ---- a piece's end: lane (lg, lc) holds column lc, dims (D / 4) lg + NV r + nn
    auto epilogue = [&](Seg sg, bool complete, bool first_piece) __attribute__((always_inline)) {
        int lgo = lg;
        asm volatile("" : "+v"(lgo));  // (addresses formed here, not kept through the stream)
#pragma unroll
        for (int ct = 0; ct < NT; ct++) {
            const float l = sum_across_rows(lsum[ct]);
            const int col = (sg.grp() * NT + ct) * 16 + lc;
            if (col >= sg.rows() * n_rep) continue;
            const int i = MULTI ? col / n_rep : 0, r0 = col - i * n_rep;
            const int h = sg.g * n_rep + r0;
            if (complete) {
                const float f = l == 0.0f ? 0.0f : fast_exp2(mv[ct] - m[ct] - DP_SHIFT) / l;
                const int64_t at = (int64_t)(sg.row0() + i) * a.o_st + (int64_t)h * a.o_sh + (D / 4) * lgo;
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int h4 = 0; h4 < NV; h4 += 4) {
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            v[e] = l == 0.0f ? 0.0f : acc[ct][h4 + e][r] * f;
                        store_run<4>(a.out, a.out_dtype, at + NV * r + h4, v);
                    }
                if constexpr (W)
                    if (lg == 0) {
                        float* ml = a.ml + 2 * ((int64_t)(sg.row0() + i) * a.num_heads + h);
                        ml[0] = m[ct];
                        ml[1] = l;
                    }
            } else {
                const int64_t slot = (2 * wgi + (first_piece ? 0 : 1)) * a.cols + 16 * ct + lc;
                float* o = a.p_o + slot * D + (D / 4) * lgo;
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int h4 = 0; h4 < NV; h4 += 4)
                        *reinterpret_cast<f32x4*>(o + NV * r + h4) =
                            f32x4{acc[ct][h4][r], acc[ct][h4 + 1][r], acc[ct][h4 + 2][r],
                                  acc[ct][h4 + 3][r]};
                if (lg == 0) {
                    a.p_ml[3 * slot] = m[ct];
                    a.p_ml[3 * slot + 1] = l;
                    a.p_ml[3 * slot + 2] = mv[ct];
                }
            }
        }
        clear();
    };

    // ---- the stream. A segment's ids are requested two segments ahead, its scales one ahead (they
    // need the ids), and every chunk's rows one chunk ahead; waits are in the order of the requests.
    auto log_scales = [&](Scales s) -> Scales { return Scales{s.k, __builtin_amdgcn_logf(s.v)}; };
    Seg cur = seg_at(0);
    Slots cur_slots = seg_slots(cur);
    int nx = cur.ce - cur.cb;
    bool has_nxt = nx < len;
    Seg nxt = cur;
    Slots nxt_slots{0, 0};
    if (has_nxt) {
        nxt = seg_at(nx);
        nxt_slots = seg_slots(nxt);
    }
    load_q(cur);
    Scales cur_raw = seg_scales(cur, cur_slots);
    u32x4 ka[TILES][KL], kb[TILES][KL];
    Vd va[TILES][4], vb[TILES][4];
    load_chunk(cur.g, cur_slots, 0, ka, va);
    Scales nxt_raw = cur_raw;
    if (has_nxt) nxt_raw = seg_scales(nxt, nxt_slots);
    Scales cur_sc = log_scales(cur_raw);
    int pc0 = cur.cb;
    bool first_piece = true;
    int c = cur.cb;

    auto step = [&](auto prefetch, u32x4 (*kc)[KL], Vd (*vc)[4], u32x4 (*kn)[KL],
                    Vd (*vn)[4]) __attribute__((always_inline)) {
        const bool seg_end = c + 1 >= cur.ce;
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
            // (selected by value: a choice between two structs keeps them in memory)
            Slots ps;
            ps.id = in_cur ? cur_slots.id : nxt_slots.id;
            ps.off = in_cur ? cur_slots.off : nxt_slots.off;
            load_chunk(in_cur ? cur.g : nxt.g, ps, in_cur ? TILES * (c + 1 - cur.cb) : 0, kn, vn);
        }
        compute_chunk(cur, c, cur_sc, kc, vc);
        if (!seg_end) {
            c += 1;
            return;
        }
        const bool piece_end =
            !has_nxt || nxt.b != cur.b || nxt.g != cur.g || nxt.grp() != cur.grp();
        if (piece_end) epilogue(cur, pc0 == 0 && cur.ce == cur.nch, first_piece);
        if (!has_nxt) return;
        if (piece_end) {
            pc0 = nxt.cb;
            first_piece = false;
            load_q(nxt);
        }
        cur = nxt;
        cur_slots = nxt_slots;
        cur_sc = log_scales(nxt_raw);
        c = cur.cb;
        nx = nn_x;
        has_nxt = has_nn;
        if (has_nn) {
            nxt = nn;
            nxt_slots = nn_slots;
            nxt_raw = seg_scales(nxt, nxt_slots);
        }
    };
    using pf_on = std::integral_constant<bool, true>;
    using pf_off = std::integral_constant<bool, false>;
    int remaining = len;
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
}

// Merge of the pieces of cut pairs, and the rows that see nothing: one workgroup a (query head, packed
// row), its waves sharing the pieces; lane i owns dims (D / 64) i .. .
static constexpr int DP_MERGE_WAVES = 8;
template <int D, int TILES, int NT, bool W>
__global__ __launch_bounds__(64 * DP_MERGE_WAVES) void decode_pools_merge_kernel(DpArgs a, int cap) {
    constexpr int E = D / 64, CHUNK = 16 * TILES;
    const int h = blockIdx.x, row = blockIdx.y, lane = threadIdx.x & 63;
    const int w_id = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    int s = row;
    if (a.cu) s = wave_find_last(a.batch, row, [&](int i) -> int64_t { return a.cu[i]; });
    const DpSeq q = dp_seq(a, s);
    const int i = row - q.row0;
    if (i < 0 || i >= q.rows) return;  // (rows of no sequence)
    const int64_t at = (int64_t)row * a.o_st + (int64_t)h * a.o_sh + E * lane;
    auto put = [&](const float* v) {
#pragma unroll
        for (int e = 0; e < E; e++) {
            if (a.out_dtype == FLOUR_DTYPE_F32)
                static_cast<float*>(a.out)[at + e] = v[e];
            else if (a.out_dtype == FLOUR_DTYPE_BF16)
                static_cast<bf16_t*>(a.out)[at + e] = from_f32<bf16_t>(v[e]);
            else
                static_cast<f16_t*>(a.out)[at + e] = from_f32<f16_t>(v[e]);
        }
    };
    if (q.kv == 0) {
        const float zero[E] = {};
        if (w_id == 0) put(zero);
        if (W && threadIdx.x == 0) {
            a.ml[2 * ((int64_t)row * a.num_heads + h)] = DEC_M0;
            a.ml[2 * ((int64_t)row * a.num_heads + h) + 1] = 0.0f;
        }
        return;
    }
    const int n_rep = a.n_rep, g = h / n_rep, col = i * n_rep + (h - g * n_rep);
    const int grp = col / (16 * NT), cc = col - grp * (16 * NT);
    const int groups = dp_groups<NT>(q.rows, n_rep), nch = (q.kv + CHUNK - 1) / CHUNK;
    const int64_t total = (int64_t)a.kv_heads * a.pre[a.batch], nwg = range_count(total, cap);
    const int64_t from = (int64_t)a.kv_heads * a.pre[s] + ((int64_t)g * groups + grp) * nch;
    const int64_t to = from + nch;
    const bool narrow = ranges_narrow(total, nwg, DP_XCD_W);
    const WaveRanges<uint32_t> r32(narrow ? total : 1, nwg, DP_XCD_W);
    const WaveRanges<int64_t> r64(total, nwg, DP_XCD_W);
    const int64_t f = narrow ? (int64_t)r32.owner((uint32_t)from) : r64.owner(from);
    const int64_t l = narrow ? (int64_t)r32.owner((uint32_t)(to - 1)) : r64.owner(to - 1);
    if (f == l) return;  // finished inside one wave range
    const bool f_first = from == (narrow ? (int64_t)r32.lo((uint32_t)f) : r64.lo(f));
    const int np = (int)(l - f + 1);
    auto slot_of = [&](int p) -> int64_t {  // (the last piece of a range but the first: its second)
        return (2 * (f + p) + (p == 0 && !f_first ? 1 : 0)) * a.cols + cc;
    };
    float M = DEC_M0, MV = DEC_M0, L = 0.0f, O[E] = {};
    // this wave's pieces, 64 at a time (one a lane for the maxima and sums), their rows 8 at a time, the
    // first 8 requested beside the maxima
    const int per = (np + waves - 1) / waves, p_end = min(np, (w_id + 1) * per);
    typedef typename std::conditional<E == 2, f32x2, float>::type RowV;
    auto row_of = [&](int p) -> RowV {  // (past the end a row that exists, for nothing)
        return *reinterpret_cast<const RowV*>(a.p_o + slot_of(min(p, np - 1)) * D + E * lane);
    };
    auto add = [&](float w, RowV v) {
        if constexpr (E == 2) {
            O[0] = fmaf(w, v[0], O[0]);
            O[1] = fmaf(w, v[1], O[1]);
        } else {
            O[0] = fmaf(w, v, O[0]);
        }
    };
    for (int p0 = w_id * per; p0 < p_end; p0 += 64) {
        const bool on = p0 + lane < p_end;
        const float* ml = a.p_ml + 3 * slot_of(on ? p0 + lane : p0);
        const float mx = ml[0], lx = ml[1], mvx = ml[2];
        RowV v[8];
#pragma unroll
        for (int y = 0; y < 8; y++) v[y] = row_of(p0 + y);
        const float Mn = fmaxf(M, wave_max(on ? mx : DEC_M0));
        const float MVn = fmaxf(MV, wave_max(on ? mvx : DEC_M0));
        L = L * fast_exp2(M - Mn) + wave_sum(on ? fast_exp2(mx - Mn) * lx : 0.0f);
        const float w = on ? fast_exp2(mvx - MVn) : 0.0f, old = fast_exp2(MV - MVn);
#pragma unroll
        for (int e = 0; e < E; e++) O[e] *= old;
        const int n = min(64, p_end - p0);
        for (int x = 0; x < n; x += 8) {
            if (x > 0)
#pragma unroll
                for (int y = 0; y < 8; y++) v[y] = row_of(p0 + x + y);
#pragma unroll
            for (int y = 0; y < 8; y++) {
                const float wy = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), x + y));
                if (x + y < n) add(wy, v[y]);
            }
        }
        M = Mn;
        MV = MVn;
    }
    if (waves > 1) {
        __shared__ float wM[DP_MERGE_WAVES][3], wO[DP_MERGE_WAVES][E][64];
        if (lane == 0) wM[w_id][0] = M, wM[w_id][1] = L, wM[w_id][2] = MV;
#pragma unroll
        for (int e = 0; e < E; e++) wO[w_id][e][lane] = O[e];
        __syncthreads();
        if (w_id != 0) return;
        for (int x = 1; x < waves; x++) {  // (a wave without pieces: sum 0 at the lowest maximum)
            const float Mn = fmaxf(M, wM[x][0]), MVn = fmaxf(MV, wM[x][2]);
            L = L * fast_exp2(M - Mn) + wM[x][1] * fast_exp2(wM[x][0] - Mn);
            const float c0 = fast_exp2(MV - MVn), c1 = fast_exp2(wM[x][2] - MVn);
#pragma unroll
            for (int e = 0; e < E; e++) O[e] = O[e] * c0 + wO[x][e][lane] * c1;
            M = Mn;
            MV = MVn;
        }
    }
    float v[E];
#pragma unroll
    for (int e = 0; e < E; e++)
        v[e] = L == 0.0f ? 0.0f : O[e] * (fast_exp2(MV - M - DP_SHIFT) / L);
    put(v);
    if (W && lane == 0) {
        a.ml[2 * ((int64_t)row * a.num_heads + h)] = M;
        a.ml[2 * ((int64_t)row * a.num_heads + h) + 1] = L;
    }
}

// The grid's waves at most: what the workspace is sized for and what a launch is cut to.
template <int D, int TILES, int NT>
static int stream_waves() {
    return std::min(device_cus() * dp_waves<D, TILES, NT>(), 4096);
}

static constexpr size_t dp_up256(size_t x) { return (x + 255) & ~(size_t)255; }

// Bytes of a streamed call's workspace for `waves` waves; its parts go to *a if that is not null.
static size_t stream_layout(DpArgs* a, void* workspace, int waves, int batch, int cols, int head_dim) {
    const size_t slots = 2 * (size_t)waves * cols;
    const size_t ml = dp_up256(slots * 3 * sizeof(float));
    const size_t o = dp_up256(slots * head_dim * sizeof(float));
    if (a) {
        char* ws = static_cast<char*>(workspace);
        a->cols = cols;
        a->p_ml = reinterpret_cast<float*>(ws);
        a->p_o = reinterpret_cast<float*>(ws + ml);
        a->pre = reinterpret_cast<int*>(ws + ml + o);
    }
    return ml + o + dp_up256(((size_t)batch + 1) * sizeof(int));
}

template <typename TQ, typename TP, int D, int TILES, int NT, bool MULTI, bool W>
static int launch_stream(DpArgs a, void* workspace, int max_rows, int rows, hipStream_t stream) {
    const int64_t max_cols = (int64_t)max_rows * a.n_rep, groups = (max_cols + 16 * NT - 1) / (16 * NT);
    const int waves = stream_waves<D, TILES, NT>();
    a.max_rows = max_rows;
    stream_layout(&a, workspace, waves, a.batch, (int)std::min<int64_t>(max_cols, 16 * NT), D);
    const int64_t chunks = ((int64_t)a.max_kv + 16 * TILES - 1) / (16 * TILES);
    const int64_t half = (int64_t)a.batch * a.kv_heads * groups * chunks / 2;
    const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(half, waves));
    const size_t lds = a.batch <= 64 ? 0 : (size_t)(a.batch + 1) * sizeof(int);
    auto kern = a.block_size == 16 ? decode_pools_kernel<TQ, TP, D, TILES, NT, MULTI, true, W>
                                   : decode_pools_kernel<TQ, TP, D, TILES, NT, MULTI, false, W>;
    kern<<<dim3(grid), dim3(64), lds, stream>>>(a);
    const int rc = check_hip(hipGetLastError(), "8-bit attention launch");
    if (rc != FLOUR_OK) return rc;
    const int64_t pieces = 2 * (int64_t)grid / ((int64_t)a.batch * a.kv_heads * groups);
    int mw = 1;
    while (mw < DP_MERGE_WAVES && 8 * mw < pieces) mw *= 2;
    decode_pools_merge_kernel<D, TILES, NT, W>
        <<<dim3(a.num_heads, rows), dim3(64 * mw), 0, stream>>>(a, grid);
    return check_hip(hipGetLastError(), "8-bit attention merge launch");
}

// One tile of columns: chunks of 64 tokens for contexts of more than 1,024 (a bound on them, that is),
// of 32 for shorter ones, which they cut finer. 64 / 32 in us: 8 x 16-32K tokens of 64 / 8 heads of
// 128 83.5 / 87.7, 64 x 512-4,096 of 32 / 8 59.4 / 60.4, 1 x 2,000 11.0 / 11.6, 32 x 512-4,096 of 32 /
// 32 heads of 64 65.5 / 69.7; 128 x 20-300 of 32 / 8 of 128 28.8 / 26.3, 8 x 100-300 11.6 / 10.4, 16 x
// 16-1,024 of 8 / 8 of 64 12.1 / 11.4.
template <typename TQ, typename TP, int D, bool W>
static int launch_stream_1(const DpArgs& a, void* ws, int rows, hipStream_t s) {
    return a.max_kv > 1024 ? launch_stream<TQ, TP, D, 4, 1, false, W>(a, ws, 1, rows, s)
                           : launch_stream<TQ, TP, D, 2, 1, false, W>(a, ws, 1, rows, s);
}

template <typename TQ, typename TP, int D>
static int launch_stream_d(const DpArgs& a, void* ws, int max_rows, int rows, hipStream_t s) {
    const int64_t cols = (int64_t)max_rows * a.n_rep;
    if (a.scores)
        return cols <= 16 ? launch_stream_1<TQ, TP, D, true>(a, ws, rows, s)
                          : launch_stream<TQ, TP, D, 2, 2, true, true>(a, ws, max_rows, rows, s);
    if (!a.cu && cols <= 16) return launch_stream_1<TQ, TP, D, false>(a, ws, rows, s);
    // More than 32 columns: groups of 32, each of which reads the cache again (a head's groups are next to
    // each other in the list). Tiles for 64 at once spill: 32 x 2,048 tokens of 32 / 8 heads of 128, 32
    // columns 51 us, 64 as one group 161, as two 95.
    return launch_stream<TQ, TP, D, 2, 2, true, false>(a, ws, max_rows, rows, s);
}

template <typename TQ>
static int launch_stream_q(const DpArgs& a, int pool_dtype, int head_dim, void* ws, int max_rows,
                           int rows, hipStream_t s) {
    if (pool_dtype == FLOUR_DTYPE_E4M3)
        return head_dim == 64 ? launch_stream_d<TQ, e4m3_t, 64>(a, ws, max_rows, rows, s)
                              : launch_stream_d<TQ, e4m3_t, 128>(a, ws, max_rows, rows, s);
    return head_dim == 64 ? launch_stream_d<TQ, i8_t, 64>(a, ws, max_rows, rows, s)
                          : launch_stream_d<TQ, i8_t, 128>(a, ws, max_rows, rows, s);
}

// The largest workspace of the launches above for calls of up to max_cols columns.
static inline size_t stream_bytes_for(int batch, int64_t max_cols, int head_dim) {
    auto bytes = [&](int waves, int cols) {
        return stream_layout(nullptr, nullptr, waves, batch, (int)std::min<int64_t>(max_cols, cols),
                             head_dim);
    };
    size_t n = bytes(head_dim == 64 ? stream_waves<64, 2, 2>() : stream_waves<128, 2, 2>(), 32);
    if (max_cols <= 16)
        n = std::max(n, head_dim == 64 ? std::max(bytes(stream_waves<64, 2, 1>(), 16),
                                                  bytes(stream_waves<64, 4, 1>(), 16))
                                       : std::max(bytes(stream_waves<128, 2, 1>(), 16),
                                                  bytes(stream_waves<128, 4, 1>(), 16)));
    return n;
}

}  // namespace flour
