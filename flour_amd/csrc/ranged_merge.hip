// ranged_merge.hip — joins the pieces of ranged_tiles.h: out = sum 2^(m_k - M) o_k / sum 2^(m_k - M) l_k over
// the pieces k of a (row, query head), M their largest maximum.
//
// A wave a (row, head), four to a workgroup; a lane holds the maximum and sum of one piece and D / 64
// dims of the output, over 16 pieces' rows at a time, all in flight together. It reads each piece once. 64 rows of
// 32 heads of 128, nine pieces each: 5.1 us; 165 rows, five, 7.2; 16 rows of 8 heads of 64 4.0, which is its
// launch and its dependent reads (the row's sequence, its group, the pieces).
#include "ranged_tiles.h"

namespace flour {

static constexpr int RM_WAVES = 4, RM_ROWS = 16;

struct RmPieces {
    int n;
    const float *ml, *o;
};

// The pieces of packed row `row`, head h in a tile launch; `shared`: the length of its group's prefix. OWN: the part
// can be RT_OWN.
template <bool OWN>
__device__ __forceinline__ RmPieces tile_pieces(const RtArgs& ra, const RtPart& pt, const RangedSeq& q,
                                                int shared, int row, int h, int head_dim) {
    RmPieces p{};
    RtSpan sp;
    if (pt.kind == RT_PREFIX) {
        if (shared == 0) return p;
        sp = rt_span(ra, pt, 0, shared, 0, 0);
    } else {
        const int col = (row - q.row0) * ra.n_rep + h - ra.by_rep(h) * ra.n_rep;
        sp = rt_span(ra, pt, q.rows, q.kv, col >> (pt.cols == 128 ? 7 : 6), shared);
    }
    const int64_t slot = ((int64_t)row * ra.a.num_heads + h) * pt.pitch;
    p.n = rt_pieces(sp.tiles(pt.tile), pt);
    p.ml = pt.p_ml + 2 * slot;
    p.o = pt.p_o + slot * head_dim;
    if (OWN && __builtin_expect(rt_own_tiles(pt, q.kv, shared) > rt_planned(pt), 0))
        p.n = rt_over_pieces(pt, rt_own_tiles(pt, q.kv, shared), *rt_over(pt));
    return p;
}

template <int D>
__global__ __launch_bounds__(64 * RM_WAVES) void ranged_merge_kernel(RtArgs ra) {
    constexpr int E = D / 64;
    typedef typename std::conditional<E == 2, f32x2, float>::type RowV;
    const RangedAttn& a = ra.a;
    const int lane = threadIdx.x & 63;
    const int item = (int)blockIdx.x * RM_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= a.rows * a.num_heads) return;  // (rows * num_heads < 2^30)
    const int row = ra.by_heads(item), h = item - row * a.num_heads;
    const RangedGroups groups = ranged_groups(a, 0);  // (beside the sequence's search)
    const int s = a.cu ? ranged_seq_of(a, row) : row;
    const RangedSeq q = ranged_seq(a, s);
    if (row < q.row0 || row >= q.row0 + q.rows) return;  // (rows of no sequence)
    const int shared = ranged_shared_of(a, groups, s);
    const RmPieces p = tile_pieces<false>(ra, ra.part[0], q, shared, row, h, D);
    const RmPieces p2 = ra.parts > 1 ? tile_pieces<true>(ra, ra.part[1], q, shared, row, h, D) : RmPieces{};
    if (ra.part[0].finals && p.n == 1) return;
    const int all = p.n + p2.n;
    float M = DEC_M0, L = 0.0f, O[E] = {};
    for (int p0 = 0; p0 < all; p0 += 64) {  // piece p0 + lane, the second part's behind the first's
        const int n = min(64, all - p0), mine = min(p0 + lane, all - 1);
        const float* at = mine < p.n ? p.ml + 2 * mine : p2.ml + 2 * (mine - p.n);
        const float mx = at[0], lx = at[1];
        RowV v[RM_ROWS];
        auto request = [&](int y0) __attribute__((always_inline)) {
#pragma unroll
            for (int x = 0; x < RM_ROWS; x += 4)
                if (y0 + x < n)
#pragma unroll
                    for (int y = x; y < x + 4; y++) {  // (past the last one: that again, for nothing)
                        const int k = min(p0 + y0 + y, all - 1);
                        const float* o = k < p.n ? p.o + (int64_t)k * D : p2.o + (int64_t)(k - p.n) * D;
                        v[y] = *reinterpret_cast<const RowV*>(o + E * lane);
                    }
        };
        request(0);  // (beside the maxima)
        const bool on = lane < n;
        const float Mn = fmaxf(M, wave_max(on ? mx : DEC_M0));
        const float w = on ? fast_exp2(mx - Mn) : 0.0f, old = fast_exp2(M - Mn);
        L = L * old + wave_sum(on ? w * lx : 0.0f);
#pragma unroll
        for (int e = 0; e < E; e++) O[e] *= old;
        for (int y0 = 0; y0 < n; y0 += RM_ROWS) {
            if (y0 > 0) request(y0);
#pragma unroll
            for (int y = 0; y < RM_ROWS; y++) {
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
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const int64_t at = (int64_t)row * a.o_st + (int64_t)h * a.o_sh + E * lane;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const float y = L == 0.0f ? 0.0f : O[e] * inv;
        store_1(a.out, a.out_dtype, at + e, y);
    }
}

int launch_ranged_merge(const RtArgs& r, hipStream_t stream) {
    const int64_t items = (int64_t)r.a.rows * r.a.num_heads;
    const dim3 grid((unsigned)((items + RM_WAVES - 1) / RM_WAVES));
    auto kern = r.a.head_dim == 64 ? ranged_merge_kernel<64> : ranged_merge_kernel<128>;
    kern<<<grid, dim3(64 * RM_WAVES), 0, stream>>>(r);
    return check_hip(hipGetLastError(), "attention over ranges merge launch");
}

}  // namespace flour
