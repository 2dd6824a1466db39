// ranged_tiles_kernel.h — the kernel of ranged_tiles.h.
//
// An item is 128 columns = (row, query head) pairs of one kv head, in the order row * n_rep + head, so
// any group size fills the tiles and a wave's 32 columns span few rows: the band of positions that
// they see is narrow, and tiles outside of it are skipped wave by wave. Four waves, a column a lane
// pair (l, l + 32); the item's positions come through LDS in tiles, double-buffered, loaded one tile ahead.
// Two workgroups a CU (three of 16-bit pools at head_dim 64), whose waves are in different phases: the matrix
// cores of one run beside the softmax of the other. One wave a SIMD with twice the columns, its products
// and vector work interleaved by hand, took 1.6 times as long at head_dim 64 and did not fit the
// registers at 128.
//
//  * S^T = K Q^T on v_mfma_f32_32x32x16: K rows from LDS (A), Q^T in registers (B). A lane holds its
//    column's scores at positions 8 (e / 4) + 4 (l / 32) + e % 4 of 32.
//  * These registers, rounded to f16, are the B operand of O^T = V^T P^T as they stand, its k index
//    running over the positions in that order. V lies in LDS row by row; the transposed A operand comes
//    from ds_read_b64_tr_b16, which hands 16 lanes a 4 x 16 block by columns.
//  * Softmax in the exp2 domain, with a reference maximum that may lag by 2^8.
//  * bf16 V goes to f16 on its way to LDS: exact for 2^-17 <= |v| <= 65,504. P in f16 keeps 11 bits where
//    bf16 would keep 8. A column that is not finite at its end, or whose root mean square is below
//    2^-25 / 5e-4 (smaller values lost bits), has its item computed again with bf16 V and P as two bf16 parts.
//  * A column that is not finite after that is computed again alone, position by position: a weight of 0
//    times a V row of NaN or infinity that other columns of the tile see is NaN in the products.
//  * fp32: v_mfma_f32_32x32x2 throughout, tiles of 32 positions.
//
// 16,384 tokens, window 2,048, 28 / 4 heads of 128 in bf16: 501-527 us on several cards, 857-902 TFLOP/s of visible
// products. Matrix cores are busy for 47% of the cycles, vector instructions issue in 52% (187 a wave and tile of 32
// products: weights 96, V to f16 48, maximum 19), hardly ever both at once: a wave's tile is 4,100 cycles of steps one
// behind the other (barrier and loop 340, edge check 190, scores with V to f16 and rows to LDS between them 1,250,
// asking for the next 540, masks 260, maximum 270, the first weights 130, V products with the others between them
// 1,100).
// LDS reads have no bank conflicts. Eight prompts (256-2,048 rows, window 512, 32 / 8 heads): 69-72 us, where an item is
// ten tiles, of 4,000-4,800 cycles, and waits 10,000 for its first one. K rows straight to LDS (no registers, 16 fewer LDS writes a workgroup and tile)
// are even.
#pragma once

#include "ranged_tiles.h"

namespace flour {

typedef __attribute__((ext_vector_type(4))) short s16x4;

__device__ __forceinline__ u32x2 lds_read_tr16(const void* p) {
    return __builtin_bit_cast(
        u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                   (__attribute__((address_space(3))) s16x4*)p));
}

__device__ __forceinline__ int wave_min_i32(int x) { return -wave_max_i32(-x); }

// LDS pitches (bytes) of K and V rows: 16-byte reads of 16 rows, and V's, spread over the banks.
template <typename T, int D>
static constexpr int RT_KP = D * sizeof(T) + 16;
template <typename T, int D>
static constexpr int RT_VP = sizeof(T) == 4 ? D * 4 + 32 : (D == 128 ? 320 : 192);
template <typename T, int D>
__host__ __device__ constexpr int rt_lds(int halves) {
    return 2 * rt_tokens(sizeof(T), halves) * (RT_KP<T, D> + RT_VP<T, D>);
}

// Workgroup wg of a part (EXTRA: which can be RT_OWN).
template <typename T, int D, int HALVES, bool EXTRA>
__device__ __forceinline__ void ranged_tiles_body(const RtArgs& ra, const RtPart pt, int wg, unsigned char* lds) {
    constexpr bool F32 = std::is_same<T, float>::value;
    constexpr bool BF16 = std::is_same<T, bf16_t>::value;
    constexpr int ES = sizeof(T), ROW = D * ES;       // bytes of a K / V row
    constexpr int COLS = rt_cols(HALVES);
    constexpr int TT = rt_tokens(ES, HALVES);         // positions of a tile
    constexpr int NB = TT / 32 / HALVES;              // the wave's blocks of 32
    constexpr int NO = D / 32;                        // 32-dim blocks of the output
    constexpr int KP = RT_KP<T, D>, VP = RT_VP<T, D>;
    constexpr int LPR = ROW / 16, RPP = 64 * RT_WAVES / LPR, NP = TT / RPP;  // staging: lanes a row, rows
                                                                            // and passes of 16 bytes a thread
    unsigned char (*const k_lds)[TT * KP] = reinterpret_cast<unsigned char (*)[TT * KP]>(lds);
    unsigned char (*const v_lds)[TT * VP] = reinterpret_cast<unsigned char (*)[TT * VP]>(lds + 2 * TT * KP);
    const RangedAttn& a = ra.a;
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, l32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n_rep = ra.n_rep;

    // ---- the item: (unit, column tile), kv head fastest (neighbouring workgroups, one an XCD, have
    // different heads, so each XCD's L2 holds its own heads' K/V)
    int piece = pt.by_items(wg);
    const int item = wg - piece * pt.items;
    int want = ra.by_kv_heads(item), g = item - want * a.kv_heads;
    const int units = pt.kind == RT_PREFIX ? a.num_groups : a.num_seqs;
    int unit = -1, ctile = 0, row0 = 0, rows = 0, kv = 0, seq = 0;
    // (what a prefix ends at, asked for beside the units)
    const RangedGroups groups = pt.kind == RT_OWN ? ranged_groups(a, 0) : RangedGroups{};
    const int extra = EXTRA && pt.extra > 0 ? wg - pt.items * pt.max_pieces : -1;
    if (extra < 0) {
        int before = 0;
        for (int u0 = 0; u0 < units; u0 += 64) {
            const int u = u0 + lane;
            int ur0 = 0, un = 0, ukv = 0, us = u;
            if (u < units) {
                if (pt.kind == RT_PREFIX) {
                    us = max(0, min(a.group_starts[u], a.num_seqs));
                    const int s1 = max(us, min(a.group_starts[u + 1], a.num_seqs));
                    ukv = max(0, min(a.shared_lens[u], a.max_shared));
                    ur0 = ranged_row(a, us);
                    un = ukv > 0 ? ranged_row(a, s1) - ur0 : 0;
                } else {
                    const RangedSeq q = ranged_seq(a, u);
                    ur0 = q.row0, un = q.rows, ukv = q.kv;
                }
            }
            const int nt = (un * n_rep + COLS - 1) / COLS;  // (rows * heads < 2^30)
            const int incl = wave_incl_sum(nt);
            const uint64_t hit = __ballot(before + incl > want);
            if (hit) {
                const int w = __builtin_ctzll(hit);
                unit = u0 + w;
                ctile = want - before - (__builtin_amdgcn_readlane(incl, w) - __builtin_amdgcn_readlane(nt, w));
                row0 = __builtin_amdgcn_readlane(ur0, w);
                rows = __builtin_amdgcn_readlane(un, w);
                kv = __builtin_amdgcn_readlane(ukv, w);
                seq = __builtin_amdgcn_readlane(us, w);  // (a group with rows starts before num_seqs)
                break;
            }
            before += __builtin_amdgcn_readlane(incl, 63);
        }
        if (unit < 0) return;
    }
    int own = 0;
    if (pt.kind == RT_OWN && extra < 0) own = __builtin_amdgcn_readfirstlane(ranged_shared_of(a, groups, seq));
    // ---- an extra workgroup, or an item of more tiles than planned: all such sequences' tiles say how many a piece
    // has, then the extra workgroup's piece is found by counting
    int over = 0;
    if (EXTRA && (extra >= 0 || rt_own_tiles(pt, kv, own) > rt_planned(pt))) {
        struct Beyond {
            RangedSeq q;
            int own, nt, tiles;  // tiles: 0 where they are not more than planned
        };
        auto beyond = [&](int u0) -> Beyond {
            Beyond x;
            x.own = ranged_shared_each(a, groups, u0 + lane);
            x.q = ranged_seq(a, min(u0 + lane, units - 1));
            x.nt = u0 + lane < units ? (x.q.rows * n_rep + COLS - 1) / COLS : 0;
            x.tiles = rt_own_tiles(pt, x.q.kv, x.own);
            if (x.tiles <= rt_planned(pt)) x.tiles = 0;
            return x;
        };
        double sum = 0.0;  // (whole numbers below 2^53: the same in every workgroup)
#pragma unroll 1
        for (int u0 = 0; u0 < units; u0 += 64) {
            const Beyond x = beyond(u0);
            sum += (double)x.nt * (double)x.tiles;
        }
        if (__ballot(sum > 0.0) == 0) return;
        for (int x = 32; x > 0; x >>= 1) sum += __shfl_xor(sum, x, 64);
        const double share = min(sum * a.kv_heads / pt.extra, (double)(1 << 30));
        over = __builtin_amdgcn_readfirstlane(max(pt.piece_tiles, (int)share + 1));
        if (extra == 0 && tid == 0) *rt_over(pt) = over;
        int before = 0;
#pragma unroll 1
        for (int u0 = 0; u0 < units && extra >= 0 && unit < 0; u0 += 64) {
            const Beyond x = beyond(u0);
            const int n = x.tiles > 0 ? (rt_over_pieces(pt, x.tiles, over) - pt.max_pieces) * x.nt * a.kv_heads : 0;
            const int incl = wave_incl_sum(n);
            const uint64_t hit = __ballot(before + incl > extra);
            if (hit) {
                const int w = __builtin_ctzll(hit), u_nt = __builtin_amdgcn_readlane(x.nt, w);
                const int k = extra - before - (__builtin_amdgcn_readlane(incl, w) - __builtin_amdgcn_readlane(n, w));
                const int by_head = ra.by_kv_heads(k), p = by_head / u_nt;
                g = k - by_head * a.kv_heads, ctile = by_head - p * u_nt, piece = pt.max_pieces + p;
                unit = seq = u0 + w;
                row0 = __builtin_amdgcn_readlane(x.q.row0, w);
                rows = __builtin_amdgcn_readlane(x.q.rows, w);
                kv = __builtin_amdgcn_readlane(x.q.kv, w);
                own = __builtin_amdgcn_readlane(x.own, w);
            }
            before += __builtin_amdgcn_readlane(incl, 63);
        }
        if (unit < 0) return;
    }
    const int ncols = rows * n_rep;
    const int32_t* bt = a.block_tables + (int64_t)seq * a.max_blocks;

    // ---- the positions
    const int sinks = pt.kind == RT_ROWS ? a.sinks : 0;
    const RtSpan sp = rt_span(ra, pt, rows, kv, ctile, own);
    const int front = sp.front, from = sp.from, to = sp.to, all_tiles = sp.tiles(TT);
    // Tiles from `plain` on hold consecutive positions, tok_off + TT t .. ; those before hold sinks.
    const int plain = (sp.front_runs + TT / 16 - 1) / (TT / 16), tok_off = sp.base - 16 * sp.front_runs;

    // ---- this workgroup's piece of the tiles
    const int pieces = over > 0 ? rt_over_pieces(pt, rt_own_tiles(pt, kv, own), over) : rt_pieces(all_tiles, pt);
    if (piece >= pieces) return;
    int t_begin = 0, t_end = all_tiles;
    if (pieces > 1) {
        const int share = all_tiles / pieces, more = all_tiles - share * pieces;  // (the first `more`: one more)
        t_begin = share * piece + min(piece, more), t_end = t_begin + share + (piece < more);
    }

    // ---- page slots of 16-position runs, 64 at a time, one a lane
    constexpr int UPT = TT / 16, WIN = 64 / UPT;  // runs a tile, tiles a refill
    const int max_id = ra.max_id;
    const int last_run = (to - 1) & ~15;
    auto load_slots = [&](int t0) -> uint32_t {  // byte offsets
        const int tok = min(sp.tok(min(t0 * UPT + lane, sp.runs - 1)), last_run);
        const int lb = ra.by_block(tok);
        int id = bt[lb];
        id = id < 0 ? 0 : (id > max_id ? max_id : id);  // a bad block id never leaves the pool
        return (uint32_t)(id * a.block_size + (tok - lb * a.block_size)) * (uint32_t)ROW;
    };

    const uint32_t head_bytes = (uint32_t)(a.num_slots * ROW);
    const __amdgpu_buffer_rsrc_t k_rsrc = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(static_cast<const char*>(a.k_pool) + (int64_t)g * a.num_slots * ROW), (short)0,
        (int)head_bytes, BUF_DWORD3);
    const __amdgpu_buffer_rsrc_t v_rsrc = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(static_cast<const char*>(a.v_pool) + (int64_t)g * a.num_slots * ROW), (short)0,
        (int)head_bytes, BUF_DWORD3);
    const int s_row = tid / LPR, s_col = (tid % LPR) * 16;  // staging: row of a pass, byte of the row
    const int w_row = wave * (64 / LPR);                    // the wave's first row of a pass
    u32x4 kreg[NP], vreg[NP];
    auto load_tile = [&](uint32_t slots, int t) __attribute__((always_inline)) {
        const int s0 = ((unsigned)(t - t_begin) % WIN) * UPT;
        uint32_t at[NP];
#pragma unroll
        for (int k = 0; k < NP; k++) at[k] = __builtin_amdgcn_readlane(slots, s0 + (k * RPP + w_row) / 16);
        __builtin_amdgcn_sched_barrier(0);  // (each load would wait for its readlane otherwise)
#pragma unroll
        for (int k = 0; k < NP; k++) {
            const uint32_t soff = at[k];
            const uint32_t voff = (uint32_t)(((k * RPP + s_row) & 15) * ROW + s_col);
            kreg[k] = __builtin_amdgcn_raw_buffer_load_b128(k_rsrc, voff, soff, 0);
            vreg[k] = __builtin_amdgcn_raw_buffer_load_b128(v_rsrc, voff, soff, 0);
        }
    };
    // positions of a loaded tile that no column sees: no bits of theirs
    auto cut_tile = [&](int t) __attribute__((always_inline)) {
        if (t > plain && t < all_tiles - 1) return;
#pragma unroll
        for (int k = 0; k < NP; k++) {
            const int tok = sp.tok(t * UPT + (k * RPP + w_row) / 16) + ((k * RPP + s_row) & 15);
            const bool keep = (tok < to) & ((tok >= from) | (tok < front));
#pragma unroll
            for (int e = 0; e < 4; e++) vreg[k][e] = keep ? vreg[k][e] : 0;
        }
    };
    auto stage_rows = [&](auto exact, int k, int buf) __attribute__((always_inline)) {
        const int r = k * RPP + s_row;
        *reinterpret_cast<u32x4*>(&k_lds[buf][r * KP + s_col]) = kreg[k];
        // (or the conversion moves up to the branch that compute() begins with, and with it the wait for the rows)
        if constexpr (!F32) asm volatile("" : "+v"(vreg[k]));
        u32x4 v = vreg[k];
        if constexpr (BF16 && !decltype(exact)::value)
#pragma unroll
            for (int e = 0; e < 4; e++)
                v[e] = pack2<f16_t>(lo_f32<bf16_t>(v[e]), hi_f32<bf16_t>(v[e]));
        *reinterpret_cast<u32x4*>(&v_lds[buf][r * VP + s_col]) = v;
    };

    // ---- the first tile is asked for before what the columns see, which can take a few reads
    uint32_t slots = 0, next = 0;
    auto begin = [&]() __attribute__((always_inline)) {
        if (t_begin >= t_end) return;
        slots = next = load_slots(t_begin);
        if (t_begin + WIN < t_end) next = load_slots(t_begin + WIN);
        load_tile(slots, t_begin);
    };
    begin();

    // ---- the lane's column, and which positions t it sees: t < hi and (t >= lo or t < sinks)
    const int col0 = ctile * COLS + 32 * (wave / HALVES);
    const int tok_half = 32 * NB * (wave % HALVES);  // of a tile, where the wave's positions start
    const bool live = col0 < ncols;  // (waves past the columns only stage)
    const int col = min(col0 + l32, ncols - 1);
    const bool real = col0 + l32 < ncols;
    const int row_i = ra.by_rep(col), head = g * n_rep + (col - row_i * n_rep);
    const int row = row0 + row_i;
    int hi, lo = 0;
    if (pt.kind == RT_PREFIX) {
        int s = row;
        if (a.cu) {  // the sequences from the wave's first row's to its last row's
            const int s0 = ranged_seq_of(a, __builtin_amdgcn_readfirstlane(row));
            const int s1 = ranged_seq_of(a, __builtin_amdgcn_readlane(row, 31));
            s = s0;
            for (int f = s0; f < s1; f += 64) {
                const int next = a.cu[min(f + 1 + lane, a.num_seqs)], n = min(64, s1 - f);
                for (int k = 0; k < n; k++) s += __builtin_amdgcn_readlane(next, k) <= row;
            }
        }
        const RangedSeq q = ranged_seq(a, s);
        hi = q.kv > 0 ? min(kv, q.kv - q.rows + (row - q.row0) + 1) : 0;
    } else {
        hi = kv > 0 ? kv - rows + row_i + 1 : 0;
        if (pt.kind == RT_ROWS)
            lo = max(0, hi - a.window);
        else
            lo = own;
    }
    // (lanes are columns in the order of their rows; a prefix's rows are of several sequences)
    int min_hi = __builtin_amdgcn_readfirstlane(hi), max_hi = __builtin_amdgcn_readlane(hi, 31);
    if (pt.kind == RT_PREFIX) {
        min_hi = __builtin_amdgcn_readfirstlane(wave_min_i32(hi));
        max_hi = __builtin_amdgcn_readfirstlane(wave_max_i32(hi));
    }
    const int min_lo = __builtin_amdgcn_readfirstlane(lo), max_lo = __builtin_amdgcn_readlane(lo, 31);

    // ---- Q^T as the B operand: dims 16 kk + 8 half .. + 7 for product kk; fp32: dims D/2 half + s for
    // product s
    constexpr int NQ = F32 ? D / 8 : D / 16;
    u32x4 qb[NQ];
    {
        const T* q = static_cast<const T*>(a.q) + (int64_t)row * a.q_st + (int64_t)head * a.q_sh;
#pragma unroll
        for (int kk = 0; kk < NQ; kk++)
            qb[kk] = live ? *reinterpret_cast<const u32x4*>(
                                q + (F32 ? D / 2 * half + 4 * kk : 16 * kk + 8 * half))
                          : u32x4{0, 0, 0, 0};
    }

    float m, l;
    f32x16 acc[NO];
    // Tile t, and meanwhile the next one's rows from registers to the other buffer, which frees the registers
    // for request().
    auto compute = [&](auto exact, int t, int buf, auto request) __attribute__((always_inline)) {
        int tok0 = tok_off + TT * t, tok_end = tok0 + TT;
        if (t < plain) {
            tok0 = sp.tok(t * UPT), tok_end = sp.tok(t * UPT + UPT - 1) + 16;
            asm volatile("" : "+s"(tok0), "+s"(tok_end));  // (a branch: every tile would compute both)
        }
        if (!live || tok0 >= max_hi || (tok_end <= min_lo && tok0 >= sinks)) {
#pragma unroll
            for (int k = 0; k < NP; k++) stage_rows(exact, k, buf ^ 1);
            request();
            return;
        }
        f32x16 s[NB];
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 16; e++) s[b][e] = 0.0f;
        const unsigned char* kr = &k_lds[buf][(tok_half + l32) * KP];
        if constexpr (F32) {
#pragma unroll
            for (int k = 0; k < NP; k++) stage_rows(exact, k, buf ^ 1);
            f32x16 s1 = s[0];
#pragma unroll
            for (int kk = 0; kk < NQ; kk++) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(kr + ROW / 2 * half + 16 * kk);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    f32x16& y = e & 1 ? s1 : s[0];
                    y = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], __uint_as_float(qb[kk][e]), y, 0, 0, 0);
                }
            }
            s[0] += s1;
        } else {
            // K fragments two steps ahead (left alone, the reads come right before their products)
            constexpr int AHEAD = 2;
            u32x4 kf[AHEAD][NB];
            auto read_k = [&](int kk) __attribute__((always_inline)) {
#pragma unroll
                for (int b = 0; b < NB; b++)
                    kf[kk % AHEAD][b] =
                        *reinterpret_cast<const u32x4*>(kr + 32 * b * KP + 32 * kk + 16 * half);
            };
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int kk = 0; kk < AHEAD; kk++) read_k(kk);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int kk = 0; kk < NQ; kk++) {
#pragma unroll
                for (int b = 0; b < NB; b++) s[b] = mfma32x32x16<T>(kf[kk % AHEAD][b], qb[kk], s[b]);
                if (kk + AHEAD < NQ) read_k(kk + AHEAD);
                if (kk & 1) stage_rows(exact, kk / 2, buf ^ 1);  // (beside the products)
                __builtin_amdgcn_sched_barrier(0);
            }
            static_assert(NP == NQ / 2, "rows staged under the score products");
            __builtin_amdgcn_s_setprio(0);
        }
        request();  // the tile after the next one
        const bool full = tok_end <= min_hi && (tok0 >= max_lo || tok_end <= sinks);
        // Masked scores are handed on whole: element by element, tiles without a mask would copy theirs too.
        auto masked = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int b = 0; b < NB; b++) asm volatile("" : "+v"(s[b]));
        };
        // (positions of a register are known up to where the tile and the lane's half start)
        if (!full && t >= plain) {
            const int at = tok0 + tok_half + 4 * half, r_hi = hi - at, r_lo = lo - at, r_sinks = sinks - at;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int x = 32 * b + 8 * (e >> 2) + (e & 3);
                    const bool sees = (x < r_hi) & ((x >= r_lo) | (x < r_sinks));
                    s[b][e] = sees ? s[b][e] : -INFINITY;
                }
            masked();
        } else if (!full) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int tok = sp.tok(t * UPT + tok_half / 16 + 2 * b + (e >> 3)) + 8 * ((e >> 2) & 1) +
                                    4 * half + (e & 3);
                    const bool sees = (tok < hi) & ((tok >= lo) | (tok < sinks));
                    s[b][e] = sees ? s[b][e] : -INFINITY;
                }
            masked();
        }
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                if (b + e > 0) top = vmax(top, s[b][e]);
        top = max_across_halves(top) * ra.scale_log2;
        constexpr float LAG = F32 ? 0.0f : 8.0f;
        const bool up = top > m + LAG;
        if (__builtin_amdgcn_ballot_w64(up) != 0) {
            const float m_new = up ? top : m, alpha = fast_exp2(m - m_new);
            m = m_new;
            l *= alpha;
#pragma unroll
            for (int o = 0; o < NO; o++) acc[o] *= alpha;
        }
        if constexpr (F32) {
            float p[16], x = 0.0f, y = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; e++) p[e] = fast_exp2(fmaf(s[0][e], ra.scale_log2, -m));
#pragma unroll
            for (int e = 0; e < 16; e += 2) x += p[e], y += p[e + 1];
            l += x + y;
#pragma unroll
            for (int o = 0; o < NO; o++) {
                // (the tile's sum by itself, then added: a long context's sum is one of sums)
                f32x16 z;
#pragma unroll
                for (int e = 0; e < 16; e++) z[e] = 0.0f;
#pragma unroll
                for (int e = 0; e < 16; e++)
                    z = __builtin_amdgcn_mfma_f32_32x32x2f32(
                        *reinterpret_cast<const float*>(
                            &v_lds[buf][(tok_half + 8 * (e >> 2) + 4 * half + (e & 3)) * VP +
                                        4 * (32 * o + l32)]),
                        p[e], z, 0, 0, 0);
                acc[o] += z;
            }
        } else {
            typedef typename std::conditional<BF16 && !decltype(exact)::value, f16_t, T>::type TP;
            constexpr bool SPLIT = BF16 && decltype(exact)::value;
            // V^T: 16 lanes read rows 4 half .. + 3 of 16 dims, and the rows 8 behind; fragment n is of
            // positions 16 (n / NO) .. + 15 and dims 32 (n % NO) .. + 31
            const unsigned char* vr = &v_lds[buf][(tok_half + 4 * half + ((lane >> 2) & 3)) * VP +
                                                  32 * ((lane >> 4) & 1) + 8 * (lane & 3)];
            constexpr int NF = 2 * NB * NO, AHEAD = 4;
            u32x4 vf[AHEAD];
            auto read_v = [&](int n) __attribute__((always_inline)) {
                const unsigned char* at = vr + 16 * (n / NO) * VP + 64 * (n % NO);
                const u32x2 v0 = lds_read_tr16(at), v1 = lds_read_tr16(at + 8 * VP);
                vf[n % AHEAD] = u32x4{v0[0], v0[1], v1[0], v1[1]};
            };
#pragma unroll
            for (int n = 0; n < AHEAD; n++) read_v(n);
            // weights 2 e and 2 e + 1 of the eight that the lane has of 16 positions
            u32x4 ph[2 * NB], pl[2 * NB];
            auto weigh = [&](int x, int e) __attribute__((always_inline)) {
                const int at = 8 * (x & 1) + 2 * e;
                const float p0 = fast_exp2(fmaf(s[x >> 1][at], ra.scale_log2, -m));
                const float p1 = fast_exp2(fmaf(s[x >> 1][at + 1], ra.scale_log2, -m));
                const uint32_t hi16 = pack2<TP>(p0, p1);
                ph[x][e] = hi16;
                if constexpr (SPLIT) {
                    pl[x][e] = pack2<TP>(p0 - lo_f32<TP>(hi16), p1 - hi_f32<TP>(hi16));
                    l += p0 + p1;
                } else {  // (the rounded weights that enter the product)
                    l = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, hi16), f16x2{1, 1}, l, false);
                }
            };
#pragma unroll
            for (int e = 0; e < 4; e++) weigh(0, e);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int n = 0; n < NF; n++) {
                f32x16& o = acc[n % NO];
                o = mfma32x32x16<TP>(vf[n % AHEAD], ph[n / NO], o);
                if constexpr (SPLIT) o = mfma32x32x16<TP>(vf[n % AHEAD], pl[n / NO], o);
                if (n + AHEAD < NF) read_v(n + AHEAD);
                if (n / NO + 1 < 2 * NB)  // the next 16 positions' weights beside the products
#pragma unroll
                    for (int e = n % NO * 4 / NO; e < (n % NO + 1) * 4 / NO; e++) weigh(n / NO + 1, e);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
        }
    };

    auto pass = [&](auto exact) __attribute__((always_inline)) {
        m = DEC_M0, l = 0.0f;
#pragma unroll
        for (int o = 0; o < NO; o++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[o][e] = 0.0f;
        if (t_begin >= t_end) return;
        cut_tile(t_begin);
#pragma unroll
        for (int k = 0; k < NP; k++) stage_rows(exact, k, 0);
        if (t_begin + 1 < t_end) load_tile(slots, t_begin + 1);
        __syncthreads();
        for (int t = t_begin; t < t_end; t++) {
            // (behind the last tile whatever the registers hold goes to a buffer that nobody reads)
            if (t + 1 < t_end) cut_tile(t + 1);
            compute(exact, t, (t - t_begin) & 1, [&]() __attribute__((always_inline)) {
                if (t + 2 >= t_end) return;
                if ((unsigned)(t + 2 - t_begin) % WIN == 0) {
                    slots = next;
                    if (t + 2 + WIN < t_end) next = load_slots(t + 2 + WIN);
                }
                load_tile(slots, t + 2);
            });
            __syncthreads();
        }
        l = sum_across_halves(l);
        if constexpr (HALVES == 2) {  // the second wave's state to the first, through LDS
            float* const st = reinterpret_cast<float*>(&v_lds[0][0]) + (wave / 2) * (64 * (16 * NO + 2));
            if (wave & 1) {
#pragma unroll
                for (int o = 0; o < NO; o++)
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        *reinterpret_cast<f32x4*>(st + (4 * o + e / 4) * 256 + 4 * lane) =
                            f32x4{acc[o][e], acc[o][e + 1], acc[o][e + 2], acc[o][e + 3]};
                st[16 * NO * 64 + lane] = m;
                st[16 * NO * 64 + 64 + lane] = l;
            }
            __syncthreads();
            if (!(wave & 1)) {
                const float m1 = st[16 * NO * 64 + lane], l1 = st[16 * NO * 64 + 64 + lane];
                const float mn = fmaxf(m, m1), w0 = fast_exp2(m - mn), w1 = fast_exp2(m1 - mn);
                l = l * w0 + l1 * w1;
                m = mn;
#pragma unroll
                for (int o = 0; o < NO; o++)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const f32x4 y = *reinterpret_cast<const f32x4*>(st + (4 * o + e / 4) * 256 + 4 * lane);
#pragma unroll
                        for (int x = 0; x < 4; x++) acc[o][e + x] = acc[o][e + x] * w0 + y[x] * w1;
                    }
            }
            __syncthreads();  // (another pass stages there)
        }
    };
    const bool owner = HALVES == 1 || !(wave & 1);  // of its columns' states
    using yes = std::integral_constant<bool, true>;
    using no = std::integral_constant<bool, false>;
    pass(no{});

    // ---- columns to compute again
    auto squares = [&]() -> float {
        float x[4] = {};
#pragma unroll
        for (int o = 0; o < NO; o++)
#pragma unroll
            for (int e = 0; e < 16; e++) x[e & 3] = fmaf(acc[o][e], acc[o][e], x[e & 3]);
        return (x[0] + x[1]) + (x[2] + x[3]);
    };
    // (sq: the lane's squares. They can overflow where the numbers do not.)
    auto finite = [&](float sq) -> bool {
        const bool good = sq - sq == 0.0f && l - l == 0.0f;
        if (__ballot(!good) == 0) return true;
        float x = l - l;  // 0, or NaN where it is not finite
#pragma unroll
        for (int o = 0; o < NO; o++)
#pragma unroll
            for (int e = 0; e < 16; e++) x = fmaf(acc[o][e], 0.0f, x);
        return x == 0.0f;
    };
    const bool mine = live && owner && real;
    float sq = squares();
    bool good = finite(sq);
    if constexpr (BF16) {
        const float least = 2.0f / (32768.0f * 1024.0f * 5e-4f * 2.0f);  // 2^-25 / 5e-4
        const bool again = mine && l != 0.0f && !(sum_across_halves(sq) >= D * least * least * l * l && good);
        int* const flags = reinterpret_cast<int*>(lds);  // (K's memory, which nobody reads any more)
        const bool any = __ballot(again) != 0;
        if (lane == 0) flags[wave] = any;
        __syncthreads();
        const u32x4 f = *reinterpret_cast<const u32x4*>(flags);
        if (__builtin_amdgcn_readfirstlane(f[0] | f[1] | f[2] | f[3]) != 0) {
            __syncthreads();  // (the pass stages there)
            begin();
            pass(yes{});
            sq = squares();
            good = finite(sq);
        }
    }

    // ---- out: a lane holds dims 32 o + 8 (e / 4) + 4 half + e % 4 of its column
    const bool final_out = pt.finals && pieces == 1;
    const int64_t slot = ((int64_t)row * a.num_heads + head) * pt.pitch + piece;
    const int64_t out_at = (int64_t)row * a.o_st + (int64_t)head * a.o_sh;
    const bool bad = mine && !good;
    auto emit = [&](float by, auto store) __attribute__((always_inline)) {
#pragma unroll
        for (int o = 0; o < NO; o++)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                store(32 * o + 2 * e, f32x4{acc[o][e] * by, acc[o][e + 1] * by, acc[o][e + 2] * by, acc[o][e + 3] * by});
    };
    // 16 bits: a lane and the one of the other half swap runs of 4 dims, so that each has 8 in a row
    auto emit16 = [&](auto type, float by) __attribute__((always_inline)) {
        using TO = decltype(type);
        TO* const to = static_cast<TO*>(a.out) + out_at + 8 * half;
#pragma unroll
        for (int o = 0; o < NO; o++)
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
                uint32_t w[4];
#pragma unroll
                for (int x = 0; x < 4; x++)
                    w[x] = pack2<TO>(acc[o][e + 2 * x] * by, acc[o][e + 2 * x + 1] * by);
                const auto a0 = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
                const auto a1 = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
                if (mine && !bad) *reinterpret_cast<u32x4*>(to + 32 * o + 2 * e) = u32x4{a0[0], a1[0], a0[1], a1[1]};
            }
    };
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (final_out && a.out_dtype != FLOUR_DTYPE_F32) {
        if (a.out_dtype == FLOUR_DTYPE_BF16)
            emit16(bf16_t{}, inv);
        else
            emit16(f16_t{}, inv);
    } else if (mine && !bad) {
        if (!final_out) {
            float* const to = pt.p_o + slot * D + 4 * half;
            emit(1.0f, [&](int d, f32x4 v) { *reinterpret_cast<f32x4*>(to + d) = v; });
            if (half == 0) *reinterpret_cast<f32x2*>(pt.p_ml + 2 * slot) = f32x2{m, l};
        } else {
            float* const to = static_cast<float*>(a.out) + out_at + 4 * half;
            emit(inv, [&](int d, f32x4 v) { *reinterpret_cast<f32x4*>(to + d) = v; });
        }
    }

    // ---- columns with numbers that are not finite, one at a time: 64 positions at once, one a lane, then
    // a lane's D / 64 dims over those that the column sees
    uint64_t todo = __ballot(bad);
    todo = (todo | (todo >> 32)) & 0xffffffffu;
    while (todo) {
        const int c = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int c_row = __builtin_amdgcn_readlane(row, c), c_head = __builtin_amdgcn_readlane(head, c);
        const int c_hi = __builtin_amdgcn_readlane(hi, c), c_lo = __builtin_amdgcn_readlane(lo, c);
        const T* q = static_cast<const T*>(a.q) + (int64_t)c_row * a.q_st + (int64_t)c_head * a.q_sh;
        const T* kp = static_cast<const T*>(a.k_pool) + (int64_t)g * a.num_slots * D;
        const T* vp = static_cast<const T*>(a.v_pool) + (int64_t)g * a.num_slots * D;
        float cm = DEC_M0, cl = 0.0f, co[D / 64] = {};
        for (int t = t_begin; t < t_end; t++) {
            const int tok = sp.tok(t * UPT + lane / 16) + lane % 16;
            const bool sees = lane < TT && tok < c_hi && (tok >= c_lo || tok < sinks);
            float sc = -INFINITY;
            int slot_j = 0;
            if (sees) {
                const int lb = ra.by_block(tok);
                int id = bt[lb];
                id = id < 0 ? 0 : (id > max_id ? max_id : id);
                slot_j = id * a.block_size + (tok - lb * a.block_size);
                float dot = 0.0f;
                for (int d = 0; d < D; d++) dot = fmaf(to_f32(q[d]), to_f32(kp[(int64_t)slot_j * D + d]), dot);
                sc = dot * ra.scale_log2;
            }
            const float m_new = fmaxf(cm, wave_max(sc)), alpha = fast_exp2(cm - m_new);
            const float p = sees ? fast_exp2(sc - m_new) : 0.0f;
            cl = cl * alpha + wave_sum(p);
#pragma unroll
            for (int x = 0; x < D / 64; x++) co[x] *= alpha;
            for (uint64_t left = __ballot(sees); left; left &= left - 1) {
                const int j = __builtin_ctzll(left);
                const float pj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(p), j));
                const int64_t v_at = (int64_t)__builtin_amdgcn_readlane(slot_j, j) * D + D / 64 * lane;
#pragma unroll
                for (int x = 0; x < D / 64; x++) co[x] = fmaf(pj, to_f32(vp[v_at + x]), co[x]);
            }
            cm = m_new;
        }
        const int64_t c_slot = ((int64_t)c_row * a.num_heads + c_head) * pt.pitch + piece;
        const float inv = cl == 0.0f ? 0.0f : 1.0f / cl;
#pragma unroll
        for (int x = 0; x < D / 64; x++) {
            const int d = D / 64 * lane + x;
            if (final_out) {
                const int64_t at = (int64_t)c_row * a.o_st + (int64_t)c_head * a.o_sh + d;
                const float y = cl == 0.0f ? 0.0f : co[x] * inv;
                store_1(a.out, a.out_dtype, at, y);
            } else {
                pt.p_o[c_slot * D + d] = co[x];
            }
        }
        if (!final_out && lane == 0) {
            pt.p_ml[2 * c_slot] = cm;
            pt.p_ml[2 * c_slot + 1] = cl;
        }
    }
}

template <typename T, int D, int HALVES, int LAST>
__global__ __launch_bounds__(64 * RT_WAVES, std::min(rt_workgroups(sizeof(T), D, HALVES),
                                                     rt_workgroups(sizeof(T), D, LAST))) void
ranged_tiles_kernel(RtArgs ra) {
    __shared__ __attribute__((aligned(16))) unsigned char
        lds[std::max(rt_lds<T, D>(HALVES), rt_lds<T, D>(LAST))];
    const int first = ra.part[0].items * ra.part[0].max_pieces;
    const bool second = blockIdx.x >= (unsigned)first;
    if (HALVES == LAST)
        ranged_tiles_body<T, D, HALVES, true>(ra, ra.part[second ? 1 : 0], (int)blockIdx.x - (second ? first : 0), lds);
    else if (second)
        ranged_tiles_body<T, D, LAST, true>(ra, ra.part[1], (int)blockIdx.x - first, lds);
    else
        ranged_tiles_body<T, D, HALVES, false>(ra, ra.part[0], (int)blockIdx.x, lds);
}

template <typename T, int D>
static int launch_ranged_tiles_d(const RtArgs& r, int halves, int last, hipStream_t stream) {
    auto kern = halves == 2 ? ranged_tiles_kernel<T, D, 2, 2> : ranged_tiles_kernel<T, D, 1, 1>;
    if constexpr (rt_mixes(sizeof(T), D))
        if (halves < last) kern = ranged_tiles_kernel<T, D, 1, 2>;
    int64_t grid = 0;
    for (int i = 0; i < r.parts; i++) grid += (int64_t)r.part[i].items * r.part[i].max_pieces + r.part[i].extra;
    kern<<<dim3((unsigned)grid), dim3(64 * RT_WAVES), 0, stream>>>(r);
    return check_hip(hipGetLastError(), "attention over ranges launch");
}

template <typename T>
static int launch_ranged_tiles(const RtArgs& r, int halves, int last, hipStream_t stream) {
    return r.a.head_dim == 64 ? launch_ranged_tiles_d<T, 64>(r, halves, last, stream)
                              : launch_ranged_tiles_d<T, 128>(r, halves, last, stream);
}

}  // namespace flour
