// ranged_tiles.h — attention of many query columns over ranges of the cached positions, on the matrix
// cores: prompts with a sliding window, prefixes that sequences share. Instantiated per type in
// ranged_tiles_*.hip.
#pragma once

#include <math.h>

#include <type_traits>

#include "decode_ranges.h"
#include "ranged.h"
#include "ranged_decode.h"

namespace flour {

// What a launch attends: a unit's rows over a unit's positions.
enum RtKind {
    RT_ROWS,    // a unit is a sequence: its rows over what they see (window and sinks)
    RT_PREFIX,  // a unit is a group: its sequences' rows over the shared prefix
    RT_OWN,     // a unit is a sequence: its rows over the positions behind its group's prefix
};

struct RtArgs {
    RangedAttn a;
    int kind;
    int n_rep;
    float scale_log2;
    // A pair's tiles are cut into up to max_pieces pieces of at least piece_tiles. A pair of one piece is
    // written out where finals is set; otherwise piece k of packed row r, head h leaves its maximum and
    // sum (exp2 domain) and accumulator at slot (r * num_heads + h) * max_pieces + k.
    int max_pieces, piece_tiles;
    bool finals;
    float* p_ml;  // [slot][2]
    float* p_o;   // [slot][D]
};

static constexpr int RT_WAVES = 4;              // waves of 32 columns each
static constexpr int RT_COLS = 32 * RT_WAVES;   // columns of a tile: (row, query head of the kv head)
// Cached positions of a step: 64 of a 16-bit pool, 32 of an fp32 one.
__host__ __device__ constexpr int rt_tokens(int elem_bytes) { return elem_bytes == 4 ? 32 : 64; }

__host__ __device__ __forceinline__ int rt_pieces(int tiles, int max_pieces, int piece_tiles) {
    const int n = (tiles + piece_tiles - 1) / piece_tiles;
    return n < 1 ? 1 : (n < max_pieces ? n : max_pieces);
}

// The positions that a column tile of a unit goes through: [0, front) and [from, to), the second behind the
// first, in tiles of tt positions (the second's start at a run of 16).
struct RtSpan {
    int front, from, to, ft, base, tiles;
    __device__ __forceinline__ int tok(int v, int tt) const {
        return v < ft ? v * tt : base + (v - ft) * tt;
    }
};
// rows and kv: the unit's. own: where the positions of RT_OWN start.
__device__ __forceinline__ RtSpan rt_span(const RtArgs& ra, int kind, int rows, int kv, int ctile,
                                          int own, int tt) {
    RtSpan s;
    const int sinks = kind == RT_ROWS ? ra.a.sinks : 0;
    s.from = 0, s.to = kv;
    if (kind != RT_PREFIX) {
        const int i0 = ctile * RT_COLS / ra.n_rep;
        const int i1 = min(rows * ra.n_rep - 1, ctile * RT_COLS + RT_COLS - 1) / ra.n_rep;
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
    s.ft = (s.front + tt - 1) / tt;
    s.base = max(s.from & ~15, s.ft * tt);
    s.tiles = s.ft + (s.to > s.base ? (s.to - s.base + tt - 1) / tt : 0);
    return s;
}

// Joins pieces: of `first`, and (or null) of `second`, whose launch had the same rows, or of a step's
// stream. Where first.finals is set, rows of one piece are left alone.
int launch_ranged_merge(const RtArgs& first, const RtArgs* second, const RangedStream* st,
                        hipStream_t stream);

int launch_ranged_tiles_f32(const RtArgs& r, int items, hipStream_t stream);
int launch_ranged_tiles_bf16(const RtArgs& r, int items, hipStream_t stream);
int launch_ranged_tiles_f16(const RtArgs& r, int items, hipStream_t stream);

}  // namespace flour
