// ranged_attn.cpp — C entries of the attention over a sliding window with sinks and over prefixes that
// sequences share: argument checks, workspaces and the choice of the kernel.
#include <math.h>

#include <algorithm>

#include "ranged_decode.h"
#include "ranged_tiles.h"

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

static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

// ---- the decode stream
static bool stream_fits(int batch, int num_heads, int kv_heads, int head_dim) {
    return (head_dim == 64 || head_dim == 128) && num_heads / kv_heads <= 16 &&
           batch <= DEC_MAX_BATCH && num_heads <= 65535;
}

static bool stream_takes(const RangedAttn& a) {
    const int es = elem_bytes(a.dtype);
    return stream_fits(a.num_seqs, a.num_heads, a.kv_heads, a.head_dim) && a.block_size % 16 == 0 &&
           a.num_slots * a.head_dim * es <= (int64_t)0x7fffffff &&
           (((uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)a.k_pool | (uintptr_t)a.v_pool) & 15) == 0;
}

static size_t stream_bytes(int batch, int num_heads, int kv_heads, int head_dim) {
    return decode_ws_bytes(decode_workgroups(FLOUR_DTYPE_F32), num_heads / kv_heads, head_dim, batch);
}

// Windows: whether each (sequence, kv head) is a workgroup of four waves with nothing to merge, rather than a
// part of the ranges of one wave each. A workgroup's time goes with its chunks (0.19-0.26 us each over 16-bit
// pools, 0.25 / 0.75 over fp32 ones of 64 / 128 dims), the ranges' with the bytes of all and a second launch.
// 32 / 8 heads of 128 in bf16, ranges / workgroups in us: 1 sequence, window 128 9.3 / 6.5, 1,024 10.6 / 13.8;
// 16, 1,024 20.1 / 20.1; 40, 128 14.7 / 9.9, 1,024 41.2 / 39.1. 8 / 8 of 64: 64, 1,024 34.5 / 27.0, 4 of 4,096
// 13.3 / 30.2.
static int g_window_pairs = -1;  // 1 always, 0 never, -1 by this (a test switch)
static bool prefer_pairs(int64_t pairs, int64_t chunks, int head_dim, int dtype) {
    if (pairs > 0x7fffffff || g_window_pairs >= 0) return pairs <= 0x7fffffff && g_window_pairs > 0;
    if (dtype == FLOUR_DTYPE_F32 && head_dim == 128) return chunks <= 8;
    const double per = dtype == FLOUR_DTYPE_F32 ? 0.25 : head_dim == 64 ? 0.19 : 0.26;
    const double bytes = 2.0 * dec_chunk(elem_bytes(dtype)) * head_dim * elem_bytes(dtype);
    return 5.0 + per * chunks <= 9.3 + pairs * chunks * bytes / 5.5e6;
}

static int launch_stream(const RangedAttn& a, void* workspace, hipStream_t stream) {
    const int nwg = decode_workgroups(a.dtype);
    RangedStream st{};
    st.ws = decode_ws_at(workspace, nwg, a.num_heads / a.kv_heads, a.head_dim);
    st.ws.rng = DecodeRange{a.window, a.sinks, a.out_dtype};
    // no more waves than ranges (range_count) for the longest visible parts
    const int64_t chunk = dec_chunk(elem_bytes(a.dtype));
    const int64_t span = std::min<int64_t>(a.max_kv, (int64_t)a.window + a.sinks + 2 * chunk);
    const int64_t half = (int64_t)a.num_seqs * a.kv_heads * ((span + chunk - 1) / chunk) / 2;
    st.grid = (int)std::max<int64_t>(1, std::min<int64_t>(half, nwg));
    const int64_t pairs = (int64_t)a.num_seqs * a.kv_heads;
    if (prefer_pairs(pairs, (span + chunk - 1) / chunk, a.head_dim, a.dtype))
        st.grid = (int)pairs, st.pairs = true;
    auto launch = a.dtype == FLOUR_DTYPE_F32    ? launch_ranged_decode_f32
                  : a.dtype == FLOUR_DTYPE_BF16 ? launch_ranged_decode_bf16
                                                : launch_ranged_decode_f16;
    return launch(a, st, stream);
}

// ---- the tile kernel
// What the shape says of it; a call's tensors can still refuse it (tiles_take).
static bool tiles_fit(int64_t rows, int num_heads, int kv_heads, int head_dim) {
    // (columns and items counted in 32 bits, a merge workgroup four (row, head) pairs)
    return (head_dim == 64 || head_dim == 128) && rows * num_heads < (int64_t)1 << 30 &&
           kv_heads <= 65535;
}

static bool tiles_take(const RangedAttn& a) {
    const int es = elem_bytes(a.dtype), oes = elem_bytes(a.out_dtype);
    return tiles_fit(a.rows, a.num_heads, a.kv_heads, a.head_dim) && a.block_size % 16 == 0 &&
           a.num_slots * a.head_dim * es <= (int64_t)0x7fffffff && a.scale > 0.0f &&
           isfinite(a.scale * 1.4426950408889634f) &&
           (((uint64_t)(uintptr_t)a.q | (uint64_t)(uintptr_t)a.out | (uint64_t)(uintptr_t)a.k_pool |
             (uint64_t)(uintptr_t)a.v_pool | (uint64_t)(a.q_st * es) | (uint64_t)(a.q_sh * es) |
             (uint64_t)(a.o_st * oes) | (uint64_t)(a.o_sh * oes)) & 15) == 0;
}

// A launch's items and the pieces that their tiles are cut into.
struct TilePlan {
    int items, max_pieces, piece_tiles, longest, halves;
    int extra, pitch;  // of RtPart
    size_t bytes;  // of the pieces
};
// Waves that share 32 columns: 1 or 2, 0 by the plans' rules, 3 one but two of own positions where the
// rules may say that (a test switch).
static int g_tile_halves = 0;
// Pieces have four tiles at least; five, and up to eight while that is one for a CU, where a launch could do
// without any (which saves the merge). 5 / 8 / 12 in us: 4 rows, window 2,000, 32 / 8 heads of 128 in bf16 16.1 /
// 18.7 / 21.4, in fp32 38.6 / 53.8 / 68.3; 100 rows (392 / 280 / 168 workgroups) 24.9 / 24.2 / 25.8 and 66.4 / 58.4 / 70.7.
static constexpr int LEAST_TILES = 4, LEAST_TILES_FINAL = 5, MOST_TILES_FINAL = 8;
// Units of up to unit_rows rows (rows in all), an item for each of their column tiles and kv heads.
static int64_t tile_items(int64_t units, int64_t unit_rows, int64_t rows, int64_t n_rep, int64_t kv_heads,
                          int64_t cols) {
    unit_rows = std::min(unit_rows, rows), units = std::min(units, rows);  // (of those that have rows)
    const int64_t tiles =
        std::min(rows * n_rep / cols + units, units * ((unit_rows * n_rep + cols - 1) / cols));
    return std::max<int64_t>(1, tiles * kv_heads);
}
// Tiles of a piece, so that `steps` of them come to seven workgroups for four CUs (fp32: eight), and `least` at
// least: more workgroups than are at work at once leave a last round of few and longer merges, fewer leave long
// pieces. 5 / 6 / 7 / 8 / 9 / 10 for four in us, 64 sequences of one prefix 4,096 + 64-1,024: bf16, 32 / 8 heads
// of 128 58.7 / 57.6 / 55.6 / 59.1 / 58.9 / 59.6, 28 / 4, eight rows each 69.5 / 67.1 / 65.3 / 76.8 / 77.0 / 76.8;
// the mean of 68 such batches 1 / 0.964 / 0.946 / 0.953 / 0.977 / 0.997, 35 of 14 / 2 heads of 64 1 / 0.975 / 0.956 /
// 0.964 / 0.955 / 0.953, 35 in fp32, 8 / 8 of 64, 1 / 0.929 / 0.889 / 0.868 / 0.861 / 0.865.
static int64_t tiles_of_piece(int64_t steps, int64_t least, int dtype) {
    const int64_t slots = (dtype == FLOUR_DTYPE_F32 ? 8 : 7) * device_cus() / 4;
    return std::max(least, (steps + slots - 1) / slots);
}
// A part's memory: RT_OVER numbers where it can have extra pieces, the pieces' maxima and sums, their accumulators.
struct PieceBytes {
    size_t over, ml, o;
};
static PieceBytes piece_bytes(int64_t rows, int num_heads, int pitch, int head_dim, int extra) {
    const size_t slots = (size_t)rows * num_heads * pitch;
    return PieceBytes{extra > 0 ? RT_OVER * sizeof(int) : 0, up256(slots * 2 * sizeof(float)),
                      up256(slots * head_dim * sizeof(float))};
}
// most: tiles of a unit, where it can have more than the longest that is planned for. A workgroup a CU for these: a
// call that has none takes 0-0.5 us of 15-46 more, as with one of them. 1 of 64 sequences with 16,640 positions
// to itself, the others behind a prefix of 16,384, takes 331 us without, 86 / 71 / 70 with 64 / 128 / 256 of them, 4
// of 64 with 8,000 (prefix 8,192) 176 and 108 / 79 / 66, 16 of 64 with up to 8,192 172 and 172 / 114 / 98.
static TilePlan tile_plan(int halves, int64_t items, int64_t longest, int64_t piece_tiles, int64_t rows,
                          int num_heads, int head_dim, bool finals, int64_t most = 0) {
    TilePlan p;
    p.halves = halves;
    p.items = (int)items;
    p.piece_tiles = (int)piece_tiles, p.longest = (int)longest;
    p.max_pieces = (int)((longest + piece_tiles - 1) / piece_tiles);
    const int cus = std::min(device_cus(), 0xffff);
    p.pitch = (int)std::max<int64_t>(p.max_pieces, std::min((most + piece_tiles - 1) / piece_tiles,
                                                            (int64_t)p.max_pieces + cus));
    p.extra = p.pitch > p.max_pieces ? cus : 0;
    const PieceBytes b = piece_bytes(rows, num_heads, p.pitch, head_dim, p.extra);
    p.bytes = finals && p.max_pieces == 1 ? 0 : b.over + b.ml + b.o;
    return p;
}

static RtArgs tile_args(const RangedAttn& a) {
    RtArgs r{};
    r.a = a, r.n_rep = a.num_heads / a.kv_heads;
    r.scale_log2 = a.scale * 1.4426950408889634f;
    r.max_id = (int)(a.num_slots / a.block_size - 1);
    r.by_rep = rt_div(r.n_rep), r.by_heads = rt_div(a.num_heads), r.by_kv_heads = rt_div(a.kv_heads);
    r.by_block = rt_div(a.block_size);
    return r;
}
static void add_part(RtArgs* r, int kind, const TilePlan& p, bool finals, char* ws) {
    RtPart& t = r->part[r->parts++];
    t.kind = kind, t.items = p.items, t.max_pieces = p.max_pieces, t.piece_tiles = p.piece_tiles;
    t.extra = (uint16_t)p.extra, t.pitch = p.pitch;
    t.cols = rt_cols(p.halves), t.tile = rt_tokens(elem_bytes(r->a.dtype), p.halves);
    t.by_items = rt_div(p.items), t.by_piece = rt_div(p.piece_tiles);
    t.finals = finals;
    const PieceBytes b = piece_bytes(r->a.rows, r->a.num_heads, p.pitch, r->a.head_dim, p.extra);
    t.p_ml = reinterpret_cast<float*>(ws + b.over);
    t.p_o = reinterpret_cast<float*>(ws + b.over + b.ml);
}

static int launch_tiles(const RtArgs& r, int halves, int last, hipStream_t stream) {
    auto launch = r.a.dtype == FLOUR_DTYPE_F32    ? launch_ranged_tiles_f32
                  : r.a.dtype == FLOUR_DTYPE_BF16 ? launch_ranged_tiles_bf16
                                                  : launch_ranged_tiles_f16;
    return launch(r, halves, last, stream);
}

// Rows over what they see: one launch, and a merge where items are cut.
static TilePlan rows_plan(int num_seqs, int max_rows, int rows, int num_heads, int kv_heads, int head_dim,
                          int max_kv, int window, int sinks, int dtype) {
    const int64_t n_rep = num_heads / kv_heads;
    // Two waves for 32 columns while that leaves the chip unfilled: half the time of an item, 1.3 times that of
    // all. Waves of 64 positions / half of them in us, by items (of 128 columns): bf16, 8 / 8 heads of 64,
    // window 512, 64 items 22.7 / 17.3, 384 30.0 / 25.1; 14 / 2, 352 22.9 / 21.3, 660 29.9 / 38.4; 32 / 8 of 128,
    // 80 23.5 / 21.2, 256 26.1 / 26.7; fp32, 8 / 8 of 64, 64 64.0 / 37.3, 384 107.2 / 108.0; 32 / 8 of 128,
    // 80 94.4 / 58.8, 224 86.1 / 91.6.
    const int64_t few = dtype == FLOUR_DTYPE_F32 ? (head_dim == 64 ? 384 : 128) : (head_dim == 64 ? 384 : 256);
    const int64_t cus = device_cus();
    int halves = 1;
    int64_t items = 0, longest = 0, piece = 0;
    // An item of several tiles is cut along the keys while the items leave CUs idle. Whole / cut in us, by items and
    // their tiles: bf16, 14 / 2 heads of 64, 44 items of 10 tiles 13.4 / 14.4, of 13 15.8 / 13.9, of 18 19.8 / 14.6;
    // 32 / 8 of 128, 8 of 13 18.3 / 14.8; fp32, 8 / 8 of 64, 16 of 10 32.9 / 24.7, of 18 55.1 / 24.9; many items: bf16,
    // 28 / 4 of 128, 220 of 34 59.6 / 67.4, of 130 133.9 / 120.1; 14 / 2 of 64, 352 of 130 113.6 / 140.9; fp32,
    // 32 / 8 of 128, 224 of 66 206 / 193.
    const int several = dtype == FLOUR_DTYPE_F32 ? 10 : 12;
    auto cut = [&](int h) {
        halves = h;
        const int cols = rt_cols(h);
        const int64_t tt = rt_tokens(elem_bytes(dtype), h);
        items = tile_items(num_seqs, max_rows, rows, n_rep, kv_heads, cols);
        const int64_t span = (int64_t)window + sinks + cols / n_rep + 2;
        longest = std::min<int64_t>(max_kv, span) / tt + 2;  // (ends that are not whole tiles)
        const bool idle = longest >= 64 ? items <= cus : longest >= several && 2 * items <= cus;
        const int64_t steps = items * longest, even = std::max<int64_t>(LEAST_TILES_FINAL, (steps + cus - 1) / cus);
        piece = idle ? tiles_of_piece(steps, std::min<int64_t>(even, MOST_TILES_FINAL), dtype) : longest;
    };
    cut(1);
    // (whole columns where the cut fills the chip: fp32, 32 / 8 of 128, 80 items of 258 tiles 258 / 277)
    const bool filled = longest >= 64 && 8 * items >= cus && 2 * items <= cus;
    if (g_tile_halves > 0 ? g_tile_halves == 2 : items <= few && !filled) cut(2);
    return tile_plan(halves, items, longest, piece, rows, num_heads, head_dim, true);
}

// Prefixes as a part of their own: 1 always, 0 never, -1 by prefer_shared (a test switch).
static int g_ranged_shared = -1;

// The prefixes by groups and each sequence's own positions, cut alike.
struct SharedPlan {
    TilePlan prefix, own;
};
static SharedPlan shared_plan(int num_seqs, int num_groups, int max_rows, int rows, int num_heads,
                              int kv_heads, int head_dim, int max_kv, int max_shared, int dtype) {
    const int64_t n_rep = num_heads / kv_heads;
    // Two waves for 32 columns, except at head_dim 128 in 16 bits, which they keep from two workgroups a CU, and
    // where large groups make the prefixes' products the most of the work. Waves of 64 positions / half of them
    // in us, 64 sequences: bf16, 32 / 8 heads of 128, one prefix 16,384 + 128 60.3 / 67.4, of eight 4,096 + 256
    // 59.5 / 67.7; of 64, 1,024 + 1,024 35.8 / 33.2; fp32, 8 / 8 of 64, 4,096 + 256 64.4 / 47.5; 64 / 8 of
    // 128, 16,384 418 / 499.
    const int64_t tiles_p = tile_items(num_groups, rows, rows, n_rep, kv_heads, rt_cols(1)) * (max_shared / 64);
    int halves = (dtype != FLOUR_DTYPE_F32 && head_dim == 128) ||
                         (rows * n_rep >= (int64_t)192 * num_groups && tiles_p >= 3000)
                     ? 1
                     : 2;
    if (g_tile_halves > 0) halves = g_tile_halves == 2 ? 2 : 1;
    // Own positions of up to 64 columns a sequence: two waves anyway, since items of 128 would be half empty, or
    // more. Prefixes and own positions by waves of 64 / the latter by half of them in us: 64 sequences of four
    // prefixes 4,096 + 64-1,024, eight rows each, bf16, 32 / 8 heads 99.1 / 91.2, one row 61.7 / 59.3; of one
    // 16,384 + 6-100, 64 / 8 heads, 72.1 / 68.9. (fp32 at 128 would keep one workgroup a CU for it.)
    const bool narrow = max_rows * n_rep <= rt_cols(2) && rt_mixes(elem_bytes(dtype), head_dim);
    const int own = narrow && (g_tile_halves == 0 || g_tile_halves == 3) ? 2 : halves;
    auto items = [&](int64_t units, int unit_rows, int h) {
        return tile_items(units, unit_rows, rows, n_rep, kv_heads, rt_cols(h));
    };
    const int es = elem_bytes(dtype), tt = rt_tokens(es, halves), tt_own = rt_tokens(es, own);
    const int64_t items_p = items(num_groups, rows, halves), items_o = items(num_seqs, max_rows, own);
    // (a sequence of no group, or of one with a shorter prefix, can have more of its own: RtPart's extra)
    const int64_t long_p = max_shared / tt + 1, long_o = std::max(0, max_kv - max_shared) / tt_own + 2;
    const int64_t piece = tiles_of_piece(items_p * long_p + items_o * long_o, LEAST_TILES, dtype);
    return SharedPlan{tile_plan(halves, items_p, long_p, piece, rows, num_heads, head_dim, false),
                      tile_plan(own, items_o, long_o, piece, rows, num_heads, head_dim, false, max_kv / tt_own + 2)};
}

// Whether prefixes are worth a part of their own, by an estimate of both ways in us from the host's bounds,
// fitted on 412 batches of up to 64 sequences (the rms of an estimate is 15%, the chosen way takes 1.006 times the
// better one in the mean). A step is 64 positions of 128 columns: `step` us of a CU; a piece's steps, one
// behind the other, take twice that, or a third where a prefix has its CU to itself, and pieces are written
// and read. Streamed decode steps are read at 5-6 TB/s, several times that where many sequences read the same.
// 32 / 8 heads of 128, bf16, prefix + own, us alone / shared: 64 sequences of one prefix 512 + 64 15.0 / 23.4,
// 2,048 + 256 39.6 / 32.6, 8,192 + 512 136 / 51; of eight, eight rows each, 512 + 64 25.9 / 41.1, 2,048 + 512
// 79.9 / 66.4; 2 of one 2,048 + 512, eight rows, 23.1 / 19.8; 16, 64 rows, 69.5 / 84.8. Packed batches of one row,
// 1-128 sequences: 1.002 times the better one in the mean of 204. Batches of 96-4,096 sequences, on which it was not
// fitted: 1.007 in the mean of 417, but where thousands have hundreds of short prefixes, since every workgroup walks all
// sequences (fp32, 4,096 of 512 prefixes 256 + 32: 504 alone, 1,460 shared and chosen). The bounds stand for every sequence, so own positions
// of thousands, or one such sequence, can still be judged too long: 64 over 8,192 + up to 8,192 370 / 289 (the other
// 63 up to 256: 202 / 180), chosen alone.
// as_step: the other way is the decode stream (a packed call of one row a sequence has row tiles).
static bool prefer_shared(bool as_step, int num_seqs, int num_groups, int max_rows, int rows, int num_heads,
                          int kv_heads, int head_dim, int max_kv, int max_shared, int dtype, const SharedPlan& p) {
    if (num_groups == 0 || max_shared == 0 || g_ranged_shared >= 0)
        return num_groups > 0 && max_shared > 0 && g_ranged_shared > 0;
    const int es = elem_bytes(dtype), n_rep = num_heads / kv_heads;
    const bool f32 = dtype == FLOUR_DTYPE_F32;
    const double step = f32 ? (head_dim == 64 ? 3.2 : 6.4) : (head_dim == 64 ? 0.7 : 1.15);
    auto chain = [&](const TilePlan& t) {
        return step * std::min(t.piece_tiles, t.longest) * rt_tokens(es, t.halves) / (64.0 * t.halves);
    };
    auto work = [&](const TilePlan& t) {
        return step * t.items * t.longest * rt_tokens(es, t.halves) / (64.0 * t.halves) / device_cus();
    };
    auto merge = [&](const TilePlan& t) { return 2.0 * t.max_pieces * rows * num_heads * (head_dim + 2) * 4 / 8e6; };
    const double shared_us = 12.5 + (f32 ? 1.2 : 0.34) * std::max(chain(p.prefix), chain(p.own)) + work(p.prefix) +
                             (f32 ? 0.87 : 1.85) * work(p.own) + 2.0 * (merge(p.prefix) + merge(p.own));
    double alone_us;
    if (as_step) {
        const double bytes = 2.0 * num_seqs * max_kv * kv_heads * head_dim * es;
        const double sharers = std::max(1.0, (double)num_seqs / num_groups);
        alone_us = 7.0 + bytes / ((f32 ? 5e6 : 6e6) * (1.0 + 0.25 * log2(sharers) * std::min(1.0, num_seqs / 64.0)));
    } else {
        const TilePlan t = rows_plan(num_seqs, max_rows, rows, num_heads, kv_heads, head_dim, max_kv, 0x7fffffff,
                                     0, dtype);
        alone_us = 6.5 + std::max(1.95 * chain(t), work(t)) + (t.max_pieces > 1 ? 6.5 + 4.2 * merge(t) : 0.0);
    }
    return shared_us < alone_us;
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
    size_t need = 0;
    int rc = shared ? flour_hip_shared_workspace_size(a.num_seqs, a.num_groups, a.max_rows, a.rows,
                                                      a.num_heads, a.kv_heads, a.head_dim, a.max_kv,
                                                      a.max_shared, a.dtype, &need)
                    : flour_hip_window_workspace_size(a.num_seqs, a.max_rows, a.rows, a.num_heads,
                                                      a.kv_heads, a.head_dim, a.max_kv, a.window, a.sinks,
                                                      a.dtype, &need);
    if (rc != FLOUR_OK) return rc;
    if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256 != 0)) {
        set_error("%s: workspace of %zu bytes (256-byte aligned) required, got %zu at %p", what, need,
                  workspace_bytes, workspace);
        return FLOUR_ERR_WORKSPACE;
    }
    char* ws = static_cast<char*>(workspace);
    const bool step = !a.cu && stream_takes(a), tiles = tiles_take(a);
    if (!step && !tiles) return launch_ranged_generic(a, stream);
    if (tiles && shared) {
        const SharedPlan p = shared_plan(a.num_seqs, a.num_groups, a.max_rows, a.rows, a.num_heads,
                                         a.kv_heads, a.head_dim, a.max_kv, a.max_shared, a.dtype);
        if (prefer_shared(step, a.num_seqs, a.num_groups, a.max_rows, a.rows, a.num_heads, a.kv_heads,
                          a.head_dim, a.max_kv, a.max_shared, a.dtype, p)) {
            RtArgs r = tile_args(a);
            add_part(&r, RT_PREFIX, p.prefix, false, ws);
            add_part(&r, RT_OWN, p.own, false, ws + p.prefix.bytes);
            rc = launch_tiles(r, p.prefix.halves, p.own.halves, stream);
            return rc != FLOUR_OK ? rc : launch_ranged_merge(r, stream);
        }
    }
    if (step) return launch_stream(a, ws, stream);
    const TilePlan p = rows_plan(a.num_seqs, a.max_rows, a.rows, a.num_heads, a.kv_heads, a.head_dim,
                                 a.max_kv, a.window, a.sinks, a.dtype);
    RtArgs r = tile_args(a);
    add_part(&r, RT_ROWS, p, true, ws);
    rc = launch_tiles(r, p.halves, p.halves, stream);
    return rc != FLOUR_OK || p.max_pieces == 1 ? rc : launch_ranged_merge(r, stream);
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
    size_t n = 0;
    if (tiles_fit(total_q, num_heads, kv_heads, head_dim))
        n = rows_plan(num_seqs, max_seqlen_q, total_q, num_heads, kv_heads, head_dim, max_kv_len, window,
                      sinks, dtype).bytes;
    if (total_q == num_seqs && stream_fits(num_seqs, num_heads, kv_heads, head_dim))  // a decode step
        n = std::max(n, stream_bytes(num_seqs, num_heads, kv_heads, head_dim));
    *bytes = n;
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
    // (whether it can be a decode step; if so a call of either form fits)
    const bool step = total_q == num_seqs && stream_fits(num_seqs, num_heads, kv_heads, head_dim);
    size_t n = 0;
    if (tiles_fit(total_q, num_heads, kv_heads, head_dim)) {
        const SharedPlan p = shared_plan(num_seqs, num_groups, max_seqlen_q, total_q, num_heads, kv_heads,
                                         head_dim, max_kv_len, max_shared_len, dtype);
        const auto prefer = [&](bool as_step) {
            return prefer_shared(as_step, num_seqs, num_groups, max_seqlen_q, total_q, num_heads, kv_heads,
                                 head_dim, max_kv_len, max_shared_len, dtype, p);
        };
        const bool rows = prefer(false);
        if (rows || (step && prefer(true))) n = p.prefix.bytes + p.own.bytes;
        if (!rows)
            n = std::max(n, rows_plan(num_seqs, max_seqlen_q, total_q, num_heads, kv_heads, head_dim, max_kv_len,
                                      0x7fffffff, 0, dtype).bytes);
    }
    if (step) n = std::max(n, stream_bytes(num_seqs, num_heads, kv_heads, head_dim));
    *bytes = n;
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

extern "C" int flour_hip_set_shared_prefix(int mode) {
    if (mode < -1 || mode > 1) return FLOUR_ERR_INVALID_ARGUMENT;
    g_ranged_shared = mode;
    switch_set();
    return FLOUR_OK;
}

extern "C" int flour_hip_set_window_pairs(int mode) {
    if (mode < -1 || mode > 1) return FLOUR_ERR_INVALID_ARGUMENT;
    g_window_pairs = mode;
    return FLOUR_OK;
}

extern "C" int flour_hip_set_tile_halves(int halves) {
    if (halves < 0 || halves > 3) return FLOUR_ERR_INVALID_ARGUMENT;
    g_tile_halves = halves;
    switch_set();
    return FLOUR_OK;
}
