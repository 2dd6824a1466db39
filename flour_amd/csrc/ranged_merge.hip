// ranged_merge.hip — joins the pieces of ranged_tiles.h: out = sum 2^(m_k - M) o_k / sum 2^(m_k - M) l_k over
// the pieces k of a (row, query head), M their largest maximum.
//
// A wave a (row, head), four to a workgroup; a lane holds the maximum and sum of one piece and D / 64
// dims of the output, over 8 pieces' rows at a time, all in flight together. It reads each piece once.
#include "ranged_tiles.h"

namespace flour {

static constexpr int RM_WAVES = 4;

// Piece k > 0 of a row is k steps behind ml and o, piece 0 has a place of its own.
struct RmPieces {
    int n;
    const float *ml0, *o0, *ml, *o;
    int64_t ml_step, o_step;
};

// The pieces of packed row `row`, head h in a tile launch; `shared`: the length of its group's prefix.
__device__ __forceinline__ RmPieces tile_pieces(const RtArgs& ra, const RangedSeq& q, int shared, int row,
                                                int h, int head_dim, int tt) {
    RmPieces p{};
    RtSpan sp;
    if (ra.kind == RT_PREFIX) {
        if (shared == 0) return p;
        sp = rt_span(ra, RT_PREFIX, 0, shared, 0, 0, tt);
    } else {
        const int col = (row - q.row0) * ra.n_rep + h % ra.n_rep;
        sp = rt_span(ra, ra.kind, q.rows, q.kv, col / RT_COLS, shared, tt);
    }
    p.n = rt_pieces(sp.tiles, ra.max_pieces, ra.piece_tiles);
    const int64_t slot = ((int64_t)row * ra.a.num_heads + h) * ra.max_pieces;
    p.ml0 = p.ml = ra.p_ml + 2 * slot;
    p.o0 = p.o = ra.p_o + slot * head_dim;
    p.ml_step = 2, p.o_step = head_dim;
    return p;
}

// The pieces of batch entry b, head h in a step's stream: of the wave ranges that its chunks lie in, two
// slots each, or the slot of its own where one wave has them all.
__device__ __forceinline__ RmPieces stream_pieces(const RangedStream& st, const RangedAttn& a, int b, int h,
                                                  int n_rep) {
    const DecodeWs& ws = st.ws;
    RmPieces p{};
    const int before = ws.pre[b], nch = ws.pre[b + 1] - before, all = ws.pre[a.num_seqs];
    if (nch == 0) return p;
    const int g = h / n_rep, hh = h - g * n_rep;
    const int64_t total = (int64_t)a.kv_heads * all, nwg = range_count(total, st.grid);
    const int64_t s = (int64_t)a.kv_heads * before + (int64_t)g * nch, e = s + nch;
    const bool narrow = ranges_narrow(total, nwg, ws.xcd_w);
    const WaveRanges<uint32_t> r32(narrow ? total : 1, nwg, ws.xcd_w);
    const WaveRanges<int64_t> r64(total, nwg, ws.xcd_w);
    const int64_t f = narrow ? (int64_t)r32.owner((uint32_t)s) : r64.owner(s);
    const int64_t l = narrow ? (int64_t)r32.owner((uint32_t)(e - 1)) : r64.owner(e - 1);
    const int D = a.head_dim;
    if (f == l) {
        const int64_t slot = (int64_t)b * a.num_heads + h;
        p.n = 1;
        p.ml0 = p.ml = ws.rng.pair_ml + 2 * slot;
        p.o0 = p.o = ws.rng.pair_o + slot * D;
        return p;
    }
    const bool f_first = s == (narrow ? (int64_t)r32.lo((uint32_t)f) : r64.lo(f));
    const int64_t slot = 2 * f * n_rep + hh, slot0 = slot + (f_first ? 0 : n_rep);
    p.n = (int)(l - f + 1);
    p.ml = ws.ml + 2 * slot, p.ml0 = ws.ml + 2 * slot0;
    p.o = ws.o + slot * D, p.o0 = ws.o + slot0 * D;
    p.ml_step = 4 * n_rep, p.o_step = (int64_t)2 * n_rep * D;
    return p;
}

template <int D>
__global__ __launch_bounds__(64 * RM_WAVES) void ranged_merge_kernel(RtArgs first, RtArgs second,
                                                                     bool two, RangedStream st, int tt) {
    constexpr int E = D / 64;
    typedef typename std::conditional<E == 2, f32x2, float>::type RowV;
    const RangedAttn& a = first.a;
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * RM_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= (int64_t)a.rows * a.num_heads) return;
    const int row = (int)(item / a.num_heads), h = (int)(item - (int64_t)row * a.num_heads);
    int s = row;
    if (a.cu) {
        int x = 0, y = a.num_seqs;
        while (y - x > 1) {
            const int mid = (x + y) >> 1;
            if (a.cu[mid] <= row)
                x = mid;
            else
                y = mid;
        }
        s = x;
    }
    const RangedSeq q = ranged_seq(a, s);
    if (row < q.row0 || row >= q.row0 + q.rows) return;  // (rows of no sequence)
    const int shared = a.num_groups > 0 ? ranged_shared_of(a, s) : 0;
    const RmPieces set[2] = {tile_pieces(first, q, shared, row, h, D, tt),
                             two           ? tile_pieces(second, q, shared, row, h, D, tt)
                             : st.grid > 0 ? stream_pieces(st, a, s, h, first.n_rep)
                                           : RmPieces{}};
    if (first.finals && set[0].n == 1) return;
    float M = DEC_M0, L = 0.0f, O[E] = {};
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const RmPieces& p = set[x];
        for (int p0 = 0; p0 < p.n; p0 += 64) {
            const bool on = p0 + lane < p.n;
            const float* ml = p0 + lane == 0 ? p.ml0 : p.ml + (int64_t)(p0 + lane) * p.ml_step;
            const float mx = on ? ml[0] : DEC_M0, lx = on ? ml[1] : 0.0f;
            const float Mn = fmaxf(M, wave_max(mx));
            const float w = on ? fast_exp2(mx - Mn) : 0.0f, old = fast_exp2(M - Mn);
            L = L * old + wave_sum(w * lx);
#pragma unroll
            for (int e = 0; e < E; e++) O[e] *= old;
            const int n = min(64, p.n - p0);
            for (int y0 = 0; y0 < n; y0 += 8) {
                RowV v[8];
#pragma unroll
                for (int y = 0; y < 8; y++) {  // (past the last one: that again, for nothing)
                    const int k = min(p0 + y0 + y, p.n - 1);
                    v[y] = *reinterpret_cast<const RowV*>((k == 0 ? p.o0 : p.o + k * p.o_step) + E * lane);
                }
#pragma unroll
                for (int y = 0; y < 8; y++) {
                    const float wy = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), (y0 + y) & 63));
                    if (y0 + y < n) {
                        if constexpr (E == 2) {
                            O[0] = fmaf(wy, v[y][0], O[0]);
                            O[1] = fmaf(wy, v[y][1], O[1]);
                        } else {
                            O[0] = fmaf(wy, v[y], O[0]);
                        }
                    }
                }
            }
            M = Mn;
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const int64_t at = (int64_t)row * a.o_st + (int64_t)h * a.o_sh + E * lane;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const float y = L == 0.0f ? 0.0f : O[e] * inv;
        store_1(a.out, a.out_dtype, at + e, y);
    }
}

int launch_ranged_merge(const RtArgs& first, const RtArgs* second, const RangedStream* st,
                        hipStream_t stream) {
    const int64_t items = (int64_t)first.a.rows * first.a.num_heads;
    const dim3 grid((unsigned)((items + RM_WAVES - 1) / RM_WAVES));
    const int tt = rt_tokens(elem_bytes(first.a.dtype));
    auto kern = first.a.head_dim == 64 ? ranged_merge_kernel<64> : ranged_merge_kernel<128>;
    kern<<<grid, dim3(64 * RM_WAVES), 0, stream>>>(first, second ? *second : first, second != nullptr,
                                                   st ? *st : RangedStream{}, tt);
    return check_hip(hipGetLastError(), "attention over ranges merge launch");
}

}  // namespace flour
