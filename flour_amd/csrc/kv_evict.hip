// kv_evict.hip — eviction by accumulated attention weight: each kv head of a sequence keeps its
// latest positions and the heaviest of the others, gathered into new blocks.
//
// Two kernels. Selection, a workgroup a (sequence, kv head): the weights become 32-bit keys, the m-th
// largest is found by counting, then one ordered pass writes the kept positions and their sums.
// Gather, a wave a (sequence, kv head, destination block): kept rows are copied (plain pools) or
// requantised under the destination block's own scale (8-bit pools).
//
// The gather of plain pools is bound by memory: 16 sequences' 1,000 positions of 8 bf16 heads of 128 (131
// MB) 22 us, 6.0 TB/s, from sources that the Infinity Cache holds, about 9 more from others. That of 8-bit
// pools is bound by vector issue (76% of its cycles: maxima and conversions): 4 x 4,096 in e4m3 (67 MB,
// rows of 128 bytes apart) 15 us, 4.5 TB/s. The selection is bound by what one CU does: 16 x 8 heads of
// 2-4K positions 10 us, 4 x 8 of 16-32K, on 32 CUs, 31 (load 3, range 3, digits 10, totals and kept
// positions 7, the latest and the zeros 4). One launch with no wait between workgroups is what this form
// has; several workgroups a head, in a few short launches, have not been measured.
#include <type_traits>

#include "cache8.h"

namespace flour {

static constexpr int EV_THREADS = 1024;
static constexpr int EV_WAVES = EV_THREADS / 64;
static_assert(EV_THREADS == 4 * 256, "a thread clears one bin of four histograms");

// Unsigned order of the keys = order of the weights, NaN (0) below all, -0 as +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (!(w == w)) return 0;
    if (w == 0.0f) w = 0.0f;
    const uint32_t u = __float_as_uint(w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_weight(uint32_t k) {
    return __uint_as_float(k == 0 ? 0x7fc00000u : k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// E: keys that a thread holds in registers, for up to 1,024 E positions; 0: any length, the weights
// read again for every count. Held / read again, in us: 16 x 8 heads of 8,000 positions 14 / 21, 4 x 8
// of 32,000 29 / 45, of 64,000 61 / 95; with 32 a thread instead of 8 16 x 8,000 take 22. A wave owns
// a run of consecutive positions, 64 at a step, so the ordered pass needs its predecessors' totals and
// no barrier a step.
//
// The m-th largest key is found eight bits at a time from the highest bit in which keys differ down: a
// histogram of the digit over the keys that share the digits found so far, in LDS, then the bin that the
// m-th falls into. After the first digit few keys take part, and a bin whose end is exactly the m-th ends the
// search. Counting one bit at a time (a compare and a popcount a key, a barrier a bit) took 46 us for
// 4 x 8 heads of 16-32K positions and 14 for 16 x 8 of 2-4K.
template <int E>
__global__ __launch_bounds__(EV_THREADS) void evict_select_kernel(
    const float* weights, float* weights_out, int64_t width, const int32_t* __restrict__ weight_rows,
    int num_rows, const int32_t* __restrict__ context_lens, const int32_t* __restrict__ keep_lens,
    int32_t* __restrict__ kept, int kv_heads, int max_ctx, int max_keep, int recent) {
    __shared__ int hist[4][256], tot_gt[EV_WAVES], tot_eq[EV_WAVES];
    __shared__ uint32_t range[2][EV_WAVES];
    const int g = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = weight_rows ? weight_rows[b] : b;
    const bool valid = r >= 0 && r < num_rows;
    const int L = valid ? max(min(context_lens[b], max_ctx), 0) : 0;
    const int n = max(min(min(keep_lens[b], max_keep), L), 0);
    const int late = min(recent, n), heavy = n - late, cand = L - late;
    int32_t* out = kept + ((int64_t)b * kv_heads + g) * max_keep;
    for (int i = n + tid; i < max_keep; i += EV_THREADS) out[i] = -1;
    if (!valid) return;
    const int64_t at = ((int64_t)r * kv_heads + g) * width;
    const float* w = weights + at;
    float* wo = weights_out + at;

    // ---- keys: the latest positions above every weight (so that n is the count to reach), positions
    // behind the end 0 like NaN
    constexpr uint32_t LATE = 0xffffffffu;
    const int steps = (L + EV_THREADS - 1) / EV_THREADS;  // of 64 positions, a wave
    const int j0 = wv * steps * 64 + lane;                // step i: position j0 + 64 i
    uint32_t k[E == 0 ? 8 : E];
    [[maybe_unused]] int first = 0;  // E == 0: the step of k[0]
    auto to_key = [&](int i, float x) -> uint32_t {
        const int j = j0 + 64 * i;
        return j >= L ? 0 : j >= cand ? LATE : weight_key(x);
    };
    if constexpr (E > 0) {
#pragma unroll
        for (int i = 0; i < E; i++)
            k[i] = i < steps && j0 + 64 * i < L ? __float_as_uint(w[j0 + 64 * i]) : 0;
#pragma unroll
        for (int i = 0; i < E; i++) k[i] = to_key(i, __uint_as_float(k[i]));
    }
    auto key = [&](int i) -> uint32_t {
        if constexpr (E > 0) return k[i];
        return k[i - first];
    };
    auto each = [&](auto f) __attribute__((always_inline)) {
        if constexpr (E > 0) {
#pragma unroll
            for (int i = 0; i < E; i++)
                if (i < steps) f(i);
        } else {
            for (first = 0; first < steps; first += 8) {  // (eight loads in flight)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int j = j0 + 64 * (first + i);
                    k[i] = first + i < steps && j < L ? __float_as_uint(w[j]) : 0;
                }
#pragma unroll
                for (int i = 0; i < 8; i++) k[i] = to_key(first + i, __uint_as_float(k[i]));
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (first + i < steps) f(first + i);
            }
        }
    };

    (&hist[0][0])[tid] = 0;  // one histogram a digit (a barrier stands between this and their use)

    // ---- T: keys above it are kept, and of those equal to it the first `ties`
    uint32_t T = 0;
    int ties = cand;  // (every candidate)
    if (heavy == 0) {
        T = LATE - 1;
        ties = 0;
    } else if (heavy < cand) {
        uint32_t lo = LATE, hi = 0;
        each([&](int i) {
            if (j0 + 64 * i < cand) {
                lo = min(lo, key(i));
                hi = max(hi, key(i));
            }
        });
        for (int o = 32; o > 0; o >>= 1) {
            lo = min(lo, (uint32_t)__shfl_xor((int)lo, o, 64));
            hi = max(hi, (uint32_t)__shfl_xor((int)hi, o, 64));
        }
        if (lane == 0) range[0][wv] = lo, range[1][wv] = hi;
        __syncthreads();
        for (int i = 0; i < EV_WAVES; i++) {
            lo = min(lo, range[0][i]);
            hi = max(hi, range[1][i]);
        }
        lo = __builtin_amdgcn_readfirstlane(lo);
        hi = __builtin_amdgcn_readfirstlane(hi);
        const uint32_t d = lo ^ hi;
        int top = d ? 32 - __builtin_clz(d) : 0;  // bits below `top` are open
        T = top == 32 ? 0 : hi & ~((1u << top) - 1);
        ties = heavy;  // wanted of the keys with T's bits from `top` up
        for (int digit = 0; top > 0; digit++) {
            const int b = max(top - 8, 0), bins = 1 << (top - b);
            each([&](int i) {
                const uint32_t x = key(i);
                if (x != LATE && (top == 32 || ((x ^ T) >> top) == 0))
                    atomicAdd(&hist[digit][(x >> b) & (bins - 1)], 1);
            });
            __syncthreads();
            // lane l: bins 4 l .. 4 l + 3, from the highest down
            int c[4], sum = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) sum += c[j] = hist[digit][255 - 4 * lane - j];
            int before = wave_incl_sum(sum) - sum;
            const int l = __builtin_amdgcn_readfirstlane(
                63 - __builtin_clzll(__ballot(before < ties) | 1));
            int bin = 255 - 4 * l;
            before = __builtin_amdgcn_readlane(before, l);
            int in = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int cj = __builtin_amdgcn_readlane(c[j], l);
                if (j == 0 || before + in < ties) {
                    if (j > 0) before += in, bin--;
                    in = cj;
                }
            }
            T |= (uint32_t)bin << b;
            ties -= before;
            top = b;
            if (in == ties) {  // all keys from T up: those above T - 1
                T -= 1;
                ties = 0;
                break;
            }
        }
    }

    // ---- totals of the waves before this one
    int n_gt = 0, n_eq = 0;
    auto is_eq = [&](int i) -> bool { return key(i) == T && j0 + 64 * i < cand; };
    each([&](int i) {
        n_gt += __popcll(__ballot(key(i) > T));
        n_eq += __popcll(__ballot(is_eq(i)));
    });
    if (lane == 0) tot_gt[wv] = n_gt, tot_eq[wv] = n_eq;
    __syncthreads();  // (E > 0: every candidate's weight has been read)
    int to = 0, eq = 0;
    for (int i = 0; i < wv; i++) {
        to += tot_gt[i] + min(max(ties - eq, 0), tot_eq[i]);
        eq += tot_eq[i];
    }
    to = __builtin_amdgcn_readfirstlane(to);
    eq = __builtin_amdgcn_readfirstlane(eq);
    const uint64_t below = (1ull << lane) - 1;
    each([&](int i) {
        const bool same = is_eq(i);
        const uint64_t beq = __ballot(same);
        const bool keep = key(i) > T || (same && eq + __popcll(beq & below) < ties);
        const uint64_t bk = __ballot(keep);
        if (keep) {
            const int x = to + __popcll(bk & below);
            out[x] = j0 + 64 * i;
            if (E > 0 && x < heavy) wo[x] = key_weight(key(i));
        }
        to += __popcll(bk);
        eq += __popcll(beq);
    });
    // Sums move to positions no later than their own: where weights_out is weights, in order, each
    // step's read before they are written. The latest positions' (a run, as a whole) always; all with
    // E == 0, by the positions just written. (Candidates' sums go below `heavy`, late ones lie behind.)
    __syncthreads();
    for (int i0 = E > 0 ? heavy : 0; i0 < n; i0 += EV_THREADS) {
        const int i = i0 + tid;
        const float x = i < n ? w[i < heavy ? out[i] : cand + (i - heavy)] : 0.0f;
        __syncthreads();
        if (i < n) wo[i] = x;
    }
    __syncthreads();
    for (int i = n + tid; i < L; i += EV_THREADS) wo[i] = 0.0f;
}

// What a wave's unit of the gather is: block lb of sequence b's destination, kv head g, and in lane i < rows
// the pool slot that row i comes from (-1 behind the last kept position).
struct EvUnit {
    int b, g, rows, slot, id;  // id: the source block of lane i's row
    int64_t to;                // destination block, -1: nothing to do
};
__device__ __forceinline__ EvUnit ev_unit(int64_t u, const int32_t* block_tables, int max_blocks,
                                          const int32_t* out_tables, int out_max_blocks,
                                          const int32_t* kept, int kv_heads, int block_size,
                                          int64_t num_slots, int max_keep, int row0) {
    const int lane = threadIdx.x & 63;
    const int per_seq = (max_keep + block_size - 1) / block_size;
    const int64_t bg = u / per_seq;
    const int lb = (int)(u - bg * per_seq);
    EvUnit x;
    x.b = (int)(bg / kv_heads);
    x.g = (int)(bg - (int64_t)x.b * kv_heads);
    const int64_t nb = num_slots / block_size;
    x.rows = min(block_size - row0, max_keep - lb * block_size - row0);
    const int64_t to = lb < out_max_blocks ? out_tables[(int64_t)x.b * out_max_blocks + lb] : -1;
    x.to = to >= 0 && to < nb ? to : -1;
    const int p = lane < x.rows ? kept[bg * max_keep + (int64_t)lb * block_size + row0 + lane] : -1;
    x.rows = __popcll(__ballot(p >= 0));  // (kept positions come first)
    const int pb = p / block_size;
    int id = p >= 0 ? block_tables[(int64_t)x.b * max_blocks + min(pb, max_blocks - 1)] : 0;
    x.id = id < 0 ? 0 : (id >= nb ? (int)nb - 1 : id);
    x.slot = x.id * block_size + (p - pb * block_size);
    return x;
}

// Rows of plain pools, in pieces of type V; up to 64 rows at a time, four loads of K and of V before their
// stores.
template <typename V>
__global__ __launch_bounds__(256) void evict_gather_kernel(
    char* k_pool, char* v_pool, const int32_t* __restrict__ block_tables, int max_blocks,
    const int32_t* __restrict__ out_tables, int out_max_blocks, const int32_t* __restrict__ kept,
    int kv_heads, int block_size, int64_t num_slots, int vecs, int max_keep, int64_t units) {
    const int lane = threadIdx.x & 63;
    const int64_t u = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (u >= units) return;
    for (int row0 = 0; row0 < block_size; row0 += 64) {
        const EvUnit x = ev_unit(u, block_tables, max_blocks, out_tables, out_max_blocks, kept, kv_heads,
                                 block_size, num_slots, max_keep, row0);
        if (x.to < 0 || x.rows <= 0) return;
        V* k = reinterpret_cast<V*>(k_pool) + (int64_t)x.g * num_slots * vecs;
        V* v = reinterpret_cast<V*>(v_pool) + (int64_t)x.g * num_slots * vecs;
        const int64_t dst = (x.to * block_size + row0) * vecs;
        const int all = x.rows * vecs;
        for (int e0 = 0; e0 < all; e0 += 256) {
            V kk[4], vv[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {  // (past the end: the last piece again)
                const int e = min(e0 + 64 * j + lane, all - 1), i = e / vecs;
                const int64_t from = (int64_t)__shfl(x.slot, i, 64) * vecs + (e - i * vecs);
                kk[j] = k[from];
                vv[j] = v[from];
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int e = e0 + 64 * j + lane;
                if (e < all) {
                    k[dst + e] = kk[j];
                    v[dst + e] = vv[j];
                }
            }
        }
    }
}

// The same over 8-bit pools: a wave a destination block, K and V, whose scale needs every row first. N
// elements a piece; up to EV_HELD pieces a lane stay in registers between the two walks, further
// ones (blocks of more than 64 x EV_HELD x N elements) are read again.
static constexpr int EV_HELD = 4;
template <typename TP, int N>
__global__ __launch_bounds__(256) void evict_gather8_kernel(
    uint8_t* k_pool, uint8_t* v_pool, float* k_scale, float* v_scale,
    const int32_t* __restrict__ block_tables, int max_blocks,
    const int32_t* __restrict__ out_tables, int out_max_blocks, const int32_t* __restrict__ kept,
    int kv_heads, int head_dim, int block_size, int64_t num_slots, int max_keep, int64_t units) {
    typedef typename std::conditional<N == 16, u32x4, uint8_t>::type Vt;
    const int lane = threadIdx.x & 63;
    const int64_t u = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (u >= units) return;
    const int64_t nb = num_slots / block_size;
    const int vecs = head_dim / N;  // pieces of a row
    // the largest magnitude of a piece (all of one row) under its row's scale
    auto amax_of = [&](Vt w, float S, uint32_t amax) -> uint32_t {
        if constexpr (N == 1) return max(amax, magnitude(Elem8<TP>::widen1(w) * S));
        else {
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) m = Elem8<TP>::max_halves(w[j], m);
            return max(amax, magnitude(Elem8<TP>::half_value(max(m & 0xffffu, m >> 16)) * S));
        }
    };
    // (0 for a block of zeros and for a poisoned one; bounded, since a row of zeros can have any scale)
    auto ratio = [](float S, float inv) { return inv > 0.0f ? fminf(S * inv, 0x1p100f) : 0.0f; };
    // f: the row's scale over the new one. Most rows come from blocks of the scale that theirs gets: where
    // all of a wave's do, the bits are copied.
    auto requantised = [&](Vt w, float f) -> Vt {
        if constexpr (N == 1) return Elem8<TP>::narrow1(Elem8<TP>::widen1(w) * f);
        else {
            if (__builtin_amdgcn_ballot_w64(f != 1.0f) == 0) return w;
            Vt z;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float y[4];
                Elem8<TP>::widen(w[j], y);
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] *= f;
                z[j] = Elem8<TP>::narrow(y);
            }
            return z;
        }
    };
    if (block_size <= 64) {  // the rows' slots and scales stay in lanes
        const EvUnit x = ev_unit(u, block_tables, max_blocks, out_tables, out_max_blocks, kept, kv_heads,
                                 block_size, num_slots, max_keep, 0);
        if (x.to < 0 || x.rows <= 0) return;
        Vt* k = reinterpret_cast<Vt*>(k_pool) + (int64_t)x.g * num_slots * vecs;
        Vt* v = reinterpret_cast<Vt*>(v_pool) + (int64_t)x.g * num_slots * vecs;
        const float ks = k_scale[x.g * nb + x.id], vs = v_scale[x.g * nb + x.id];
        const int64_t dst = x.to * block_size * vecs;
        const int all = x.rows * vecs;
        auto piece = [&](int e, int64_t& from, float& sk, float& sv) {
            const int i = e / vecs;
            from = (int64_t)__shfl(x.slot, i, 64) * vecs + (e - i * vecs);
            sk = __shfl(ks, i, 64);
            sv = __shfl(vs, i, 64);
        };
        Vt kh[EV_HELD], vh[EV_HELD];
        float skh[EV_HELD], svh[EV_HELD];
        uint32_t ka = 0, va = 0;
#pragma unroll
        for (int j = 0; j < EV_HELD; j++) {  // (past the end: the last piece again)
            if (64 * j >= all) break;
            int64_t from;
            piece(min(64 * j + lane, all - 1), from, skh[j], svh[j]);
            kh[j] = k[from];
            vh[j] = v[from];
        }
#pragma unroll
        for (int j = 0; j < EV_HELD; j++) {
            if (64 * j >= all) break;
            ka = amax_of(kh[j], skh[j], ka);
            va = amax_of(vh[j], svh[j], va);
        }
        for (int e0 = 64 * EV_HELD; e0 < all; e0 += 64) {
            int64_t from;
            float sk, sv;
            piece(min(e0 + lane, all - 1), from, sk, sv);
            ka = amax_of(k[from], sk, ka);
            va = amax_of(v[from], sv, va);
        }
        const float K = scale_for<TP>(wave_max_u32(ka)), V = scale_for<TP>(wave_max_u32(va));
        const float ki = inv_scale(K), vi = inv_scale(V);
#pragma unroll
        for (int j = 0; j < EV_HELD; j++) {
            const int e = 64 * j + lane;
            if (e < all) {
                k[dst + e] = requantised(kh[j], ratio(skh[j], ki));
                v[dst + e] = requantised(vh[j], ratio(svh[j], vi));
            }
        }
        for (int e0 = 64 * EV_HELD; e0 < all; e0 += 64) {
            int64_t from;
            float sk, sv;
            const int e = e0 + lane;
            piece(min(e, all - 1), from, sk, sv);
            if (e < all) {
                k[dst + e] = requantised(k[from], ratio(sk, ki));
                v[dst + e] = requantised(v[from], ratio(sv, vi));
            }
        }
        if (lane == 0) {
            k_scale[x.g * nb + x.to] = K;
            v_scale[x.g * nb + x.to] = V;
        }
        return;
    }
    // longer blocks: 64 rows at a time, all of them read twice
    float K = 0.0f, V = 0.0f;
    uint32_t ka = 0, va = 0;
    for (int pass = 0; pass < 2; pass++) {
        for (int row0 = 0; row0 < block_size; row0 += 64) {
            const EvUnit x = ev_unit(u, block_tables, max_blocks, out_tables, out_max_blocks, kept,
                                     kv_heads, block_size, num_slots, max_keep, row0);
            if (x.to < 0) return;
            if (x.rows <= 0) break;
            Vt* k = reinterpret_cast<Vt*>(k_pool) + (int64_t)x.g * num_slots * vecs;
            Vt* v = reinterpret_cast<Vt*>(v_pool) + (int64_t)x.g * num_slots * vecs;
            const float ks = k_scale[x.g * nb + x.id], vs = v_scale[x.g * nb + x.id];
            const int64_t dst = (x.to * block_size + row0) * vecs;
            const int all = x.rows * vecs;
            for (int e0 = 0; e0 < all; e0 += 64) {
                const int e = e0 + lane, i = min(e, all - 1) / vecs;
                const int64_t from =
                    (int64_t)__shfl(x.slot, i, 64) * vecs + (min(e, all - 1) - i * vecs);
                const float sk = __shfl(ks, i, 64), sv = __shfl(vs, i, 64);
                if (pass == 0) {
                    ka = amax_of(k[from], sk, ka);
                    va = amax_of(v[from], sv, va);
                } else if (e < all) {
                    k[dst + e] = requantised(k[from], ratio(sk, inv_scale(K)));
                    v[dst + e] = requantised(v[from], ratio(sv, inv_scale(V)));
                }
            }
            if (pass == 1 && row0 == 0 && lane == 0) {
                k_scale[x.g * nb + x.to] = K;
                v_scale[x.g * nb + x.to] = V;
            }
        }
        if (pass == 0) K = scale_for<TP>(wave_max_u32(ka)), V = scale_for<TP>(wave_max_u32(va));
    }
}

}  // namespace flour

using namespace flour;

extern "C" int flour_hip_kv_evict(void* k_pool, void* v_pool, float* k_scale, float* v_scale,
                                  int pool_dtype, const float* weights, float* weights_out,
                                  int64_t weights_width, const int32_t* weight_rows,
                                  int num_weight_rows, const int32_t* block_tables,
                                  int max_blocks_per_seq, const int32_t* context_lens,
                                  const int32_t* keep_lens, const int32_t* out_tables,
                                  int out_max_blocks, int32_t* kept, int batch, int kv_heads,
                                  int head_dim, int block_size, int64_t num_slots,
                                  int max_context_len, int max_keep_len, int recent,
                                  void* stream) {
    clear_error();
    const bool q8 = valid_pool8(pool_dtype);
    if (!q8 && !valid_dtype(pool_dtype)) {
        set_error("kv_evict: unknown pool dtype %d", pool_dtype);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    if (batch < 0 || kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || num_slots <= 0 ||
        num_slots > 0x7fffffff || num_slots % block_size != 0 || max_blocks_per_seq <= 0 ||
        out_max_blocks <= 0 || max_context_len < 0 || max_keep_len < 0 || recent < 0 ||
        num_weight_rows < 0 || (!weight_rows && num_weight_rows < batch) ||
        weights_width < max_context_len ||
        (int64_t)max_context_len > (int64_t)max_blocks_per_seq * block_size ||
        (int64_t)max_keep_len > (int64_t)out_max_blocks * block_size) {
        set_error("kv_evict: bad shape (batch=%d kv_heads=%d head_dim=%d bs=%d num_slots=%lld "
                  "max_blocks=%d out_blocks=%d max_ctx=%d max_keep=%d recent=%d weights %d x %lld)",
                  batch, kv_heads, head_dim, block_size, (long long)num_slots, max_blocks_per_seq,
                  out_max_blocks, max_context_len, max_keep_len, recent, num_weight_rows,
                  (long long)weights_width);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    if (batch == 0) return FLOUR_OK;
    if (!k_pool || !v_pool || !weights || !weights_out || !block_tables || !context_lens ||
        !keep_lens || !out_tables || (!kept && max_keep_len > 0)) {
        set_error("kv_evict: null pointer");
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    if (q8 != (k_scale != nullptr) || q8 != (v_scale != nullptr)) {
        set_error("kv_evict: scales go with 8-bit pools, and only with them");
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    const int64_t per_seq = ((int64_t)max_keep_len + block_size - 1) / block_size;
    const int64_t units = (int64_t)batch * kv_heads * per_seq, grid = (units + 3) / 4;
    if (batch > 65535 || grid > 0x7fffffff) {
        set_error("kv_evict: %d sequences of %d positions are too many for one call", batch,
                  max_keep_len);
        return FLOUR_ERR_UNSUPPORTED;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto select = max_context_len <= 8 * EV_THREADS    ? evict_select_kernel<8>
                  : max_context_len <= 32 * EV_THREADS ? evict_select_kernel<32>
                  : max_context_len <= 64 * EV_THREADS ? evict_select_kernel<64>
                                                       : evict_select_kernel<0>;
    select<<<dim3(kv_heads, batch), dim3(EV_THREADS), 0, s>>>(
        weights, weights_out, weights_width, weight_rows, num_weight_rows, context_lens, keep_lens,
        kept, kv_heads, max_context_len, max_keep_len, recent);
    int rc = check_hip(hipGetLastError(), "kv_evict selection launch");
    if (rc != FLOUR_OK || grid == 0) return rc;
    const uint64_t ptrs = (uint64_t)(uintptr_t)k_pool | (uint64_t)(uintptr_t)v_pool;
    if (q8) {
        const bool wide = head_dim % 16 == 0 && (ptrs & 15) == 0;
#define FLOUR_EV8(TP, N)                                                                          \
    evict_gather8_kernel<TP, N><<<dim3((unsigned)grid), dim3(256), 0, s>>>(                       \
        static_cast<uint8_t*>(k_pool), static_cast<uint8_t*>(v_pool), k_scale, v_scale,           \
        block_tables, max_blocks_per_seq, out_tables, out_max_blocks, kept, kv_heads, head_dim,   \
        block_size, num_slots, max_keep_len, units)
        if (pool_dtype == FLOUR_DTYPE_E4M3) {
            if (wide) FLOUR_EV8(e4m3_t, 16);
            else FLOUR_EV8(e4m3_t, 1);
        } else {
            if (wide) FLOUR_EV8(i8_t, 16);
            else FLOUR_EV8(i8_t, 1);
        }
#undef FLOUR_EV8
        return check_hip(hipGetLastError(), "kv_evict launch");
    }
    const int64_t row = (int64_t)head_dim * elem_bytes(pool_dtype);
    const uint64_t bits = (uint64_t)row | ptrs;
#define FLOUR_EV(V)                                                                               \
    evict_gather_kernel<V><<<dim3((unsigned)grid), dim3(256), 0, s>>>(                            \
        static_cast<char*>(k_pool), static_cast<char*>(v_pool), block_tables, max_blocks_per_seq, \
        out_tables, out_max_blocks, kept, kv_heads, block_size, num_slots,                        \
        (int)(row / (int64_t)sizeof(V)), max_keep_len, units)
    if ((bits & 15) == 0)
        FLOUR_EV(u32x4);
    else if ((bits & 3) == 0)
        FLOUR_EV(uint32_t);
    else
        FLOUR_EV(uint16_t);
#undef FLOUR_EV
    return check_hip(hipGetLastError(), "kv_evict launch");
}
