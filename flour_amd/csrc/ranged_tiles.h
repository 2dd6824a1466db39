// ranged_tiles.h — attention of many query columns over ranges of the cached positions, on the matrix
// cores: prompts with a sliding window, prefixes that sequences share. Instantiated per type in
// ranged_tiles_*.hip.
#pragma once

#include <math.h>

#include <type_traits>

#include "decode_ranges.h"
#include "ranged.h"

namespace flour {

// x / d of 0 <= x < 2^31 without a division: with 2^(s - 1) < d <= 2^s and mul = ceil(2^(31 + s) / d), mul * d is
// less than 2^s above 2^(31 + s), so mul * x / 2^(31 + s) is less than 1 / d above x / d. A workgroup has about
// eight to do before its first tile (compiled divisions: 150-1,000 cycles each).
struct RtDiv {
    uint32_t mul;
    int shift;  // 31 + s
    __device__ __forceinline__ int operator()(int x) const {
        return (int)(((uint64_t)(uint32_t)x * mul) >> shift);
    }
};
inline RtDiv rt_div(int64_t d) {
    int s = 0;
    while (((int64_t)1 << s) < d) s++;
    return RtDiv{(uint32_t)((((uint64_t)1 << (31 + s)) + d - 1) / d), 31 + s};
}

// What a launch attends: a unit's rows over a unit's positions.
enum RtKind {
    RT_ROWS,    // a unit is a sequence: its rows over what they see (window and sinks)
    RT_PREFIX,  // a unit is a group: its sequences' rows over the shared prefix
    RT_OWN,     // a unit is a sequence: its rows over the positions behind its group's prefix
};

// One kind's part of a launch: `items` (unit, column tile, kv head) triples at most, each of which has its
// tiles cut into up to max_pieces pieces of at least piece_tiles. A triple of one piece is written out
// where finals is set; otherwise piece k of packed row r, head h leaves its maximum and sum (exp2
// domain) and accumulator at slot (r * num_heads + h) * pitch + k.
//
// RT_OWN: a sequence of no group, or of one with a shorter prefix than another's, can have more tiles than its
// max_pieces pieces are planned for. It is cut into more, of as many tiles as it takes that `extra` workgroups behind
// the others are enough for them (left for the merge at rt_over, by the first of these).
struct RtPart {
    int kind, items, max_pieces, piece_tiles;
    RtDiv by_items, by_piece;
    int cols, tile;  // columns of an item, positions of a tile (rt_cols, rt_tokens)
    bool finals;
    uint16_t extra;
    int pitch;    // slots of a (row, head): pieces at most
    float* p_ml;  // [slot][2]
    float* p_o;   // [slot][D]
};
// (a launch's two parts at 96 bytes each: 0.3 us more of every call)
static_assert(sizeof(RtPart) == 64, "a part is one scalar load");
static constexpr int RT_OVER = 64;  // numbers before p_ml
__device__ __forceinline__ int* rt_over(const RtPart& pt) { return reinterpret_cast<int*>(pt.p_ml) - RT_OVER; }
__device__ __forceinline__ int rt_planned(const RtPart& pt) {
    return pt.extra > 0 ? pt.max_pieces * pt.piece_tiles : 0x7fffffff;
}
struct RtArgs {
    RangedAttn a;
    int n_rep, max_id;  // max_id: the last block
    RtDiv by_rep, by_heads, by_kv_heads, by_block;
    float scale_log2;
    int parts;
    RtPart part[2];  // the first one's workgroups come first
};

// Four waves a workgroup, of 32 columns = (row, query head of the kv head) pairs each. halves 2: two waves
// share 32 columns, each with every second block of 32 positions.
static constexpr int RT_WAVES = 4;
__host__ __device__ constexpr int rt_cols(int halves) { return 32 * RT_WAVES / halves; }
// Cached positions of a step: 64, but 32 of fp32 pools where a wave has all of a tile.
__host__ __device__ constexpr int rt_tokens(int elem_bytes, int halves) {
    return elem_bytes == 4 && halves == 1 ? 32 : 64;
}

// Workgroups of a CU. Three instead of two, 16-bit pools at head_dim 64: 16,384 tokens, window 2,048, 14 / 2
// heads 202 -> 179 us; four prompts of 2,000, 32 / 32 heads, 217 -> 194. At 128 the registers hold two.
__host__ __device__ constexpr int rt_workgroups(int elem_bytes, int head_dim, int halves) {
    const int row = elem_bytes * head_dim;
    return row == 128 ? 3 : row * halves > 512 ? 1 : 2;
}

// Whether a launch's parts may differ in their halves.
constexpr bool rt_mixes(int elem_bytes, int head_dim) {
    return rt_workgroups(elem_bytes, head_dim, 2) == rt_workgroups(elem_bytes, head_dim, 1);
}

__device__ __forceinline__ int rt_pieces(int tiles, const RtPart& pt) {
    return max(1, min(pt.by_piece(tiles + pt.piece_tiles - 1), pt.max_pieces));
}

// RT_OWN: the tiles of a sequence of kv positions, the first `own` of them its group's.
__device__ __forceinline__ int rt_own_tiles(const RtPart& pt, int kv, int own) {
    const int runs = (max(0, kv - (own & ~15)) + 15) >> 4;
    return (16 * runs + pt.tile - 1) >> (pt.tile == 64 ? 6 : 5);
}
// Pieces of the items of a sequence with more tiles than planned. (Theirs are cut alike, so those behind max_pieces
// are fewer than tiles / over an item, less than `extra` in all.)
__device__ __forceinline__ int rt_over_pieces(const RtPart& pt, int tiles, int over) {
    return max(pt.max_pieces, min((tiles + over - 1) / max(1, over), pt.pitch));
}

// The positions that a column tile of a unit goes through, in runs of 16: those of [0, front), then those of
// [from, to) from the last multiple of 16 on; a tile is as many of these runs as it has positions / 16.
struct RtSpan {
    int front, from, to, front_runs, base, runs;
    __device__ __forceinline__ int tok(int run) const {
        return run < front_runs ? 16 * run : base + 16 * (run - front_runs);
    }
    __device__ __forceinline__ int tiles(int tt) const { return (16 * runs + tt - 1) >> (tt == 64 ? 6 : 5); }
};
// rows and kv: the unit's. own: where the positions of RT_OWN start.
__device__ __forceinline__ RtSpan rt_span(const RtArgs& ra, const RtPart& pt, int rows, int kv, int ctile,
                                          int own) {
    RtSpan s;
    const int kind = pt.kind, sinks = kind == RT_ROWS ? ra.a.sinks : 0;
    s.from = 0, s.to = kv;
    if (kind != RT_PREFIX) {
        const int i0 = ra.by_rep(ctile * pt.cols);
        const int i1 = ra.by_rep(max(0, min(rows * ra.n_rep, ctile * pt.cols + pt.cols) - 1));
        s.to = kv > 0 ? kv - rows + i1 + 1 : 0;
        if (kind == RT_ROWS) {
            s.from = kv > 0 ? max(0, kv - rows + i0 + 1 - ra.a.window) : 0;
            if (s.from <= sinks) s.from = 0;
        } else {
            s.from = own;
            s.to = max(s.to, own);
        }
    }
    s.front = s.from > 0 ? min(sinks, s.to) : 0;
    s.front_runs = (s.front + 15) >> 4;
    s.base = max(s.from & ~15, 16 * s.front_runs);
    s.runs = s.front_runs + (s.to > s.base ? (s.to - s.base + 15) >> 4 : 0);
    return s;
}

// Joins the pieces of a launch's parts. Where the first part's finals is set, rows of one piece are left
// alone.
int launch_ranged_merge(const RtArgs& r, hipStream_t stream);

// halves: of the first part's items, last: of the last part's (the same, or 2 behind 1 where rt_mixes).
int launch_ranged_tiles_f32(const RtArgs& r, int halves, int last, hipStream_t stream);
int launch_ranged_tiles_bf16(const RtArgs& r, int halves, int last, hipStream_t stream);
int launch_ranged_tiles_f16(const RtArgs& r, int halves, int last, hipStream_t stream);

}  // namespace flour
