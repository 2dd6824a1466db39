// attn_pools.hip — attention over pools of any element type and shape, with the scores kept for the
// attention-weight sums where they are asked for.
//
// The kernels that every other one is checked against, and what runs where the streamed decode
// (decode_stream.h) does not take a shape: any head_dim up to 512, block size, group size,
// alignment. One workgroup a (row, query head): 256 positions at a time, a thread's whole dot
// product each, then a thread's output dims each over the 256 weights in LDS. Bound by the vector
// units and by reading K/V once a query head: 64 x 512-4,096 tokens of 32 / 8 heads of 128 in e4m3 take
// 807 us where the streamed kernel takes 58.
#include <math.h>

#include <algorithm>

#include "cache8.h"
#include "decode_pools.h"

namespace flour {

static constexpr int AP_THREADS = 256;
static constexpr int AP_MAX_D = 512;

template <typename T>
__device__ __forceinline__ float pool_f32(const T* p) {
    return to_f32(*p);
}
template <>
__device__ __forceinline__ float pool_f32<e4m3_t>(const e4m3_t* p) {
    return Elem8<e4m3_t>::widen1(p->bits);
}
template <>
__device__ __forceinline__ float pool_f32<i8_t>(const i8_t* p) {
    return (float)p->v;
}

template <typename F>
__device__ __forceinline__ float ap_reduce(float x, float* red, F op) {
    for (int o = 32; o > 0; o >>= 1) x = op(x, __shfl_xor(x, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    float r = red[0];
    for (int i = 1; i < AP_THREADS / 64; i++) r = op(r, red[i]);
    return r;
}

// Row r of q for query head h: row i of the q_len of sequence s. scores (or null): (batch, num_heads,
// score_stride) in the exp2 domain, ml (batch, num_heads, 2) their maximum and sum: decode steps only.
template <typename TQ, typename TP>
__device__ __forceinline__ void attn_row(const PoolAttn& a, int64_t r, int h, int s, int i, int q_len) {
    __shared__ float qs[AP_MAX_D];
    __shared__ float ps[AP_THREADS];
    __shared__ int64_t rows[AP_THREADS];
    __shared__ float red[AP_THREADS / 64];
    const TQ* __restrict__ q = static_cast<const TQ*>(a.q);
    const TP* __restrict__ k_pool = static_cast<const TP*>(a.k_pool);
    const TP* __restrict__ v_pool = static_cast<const TP*>(a.v_pool);
    const int tid = threadIdx.x, head_dim = a.head_dim, block_size = a.block_size;
    const float scale_log2 = a.scale * LOG2_E;
    const int kv_len =
        (int)min((int64_t)min(a.kv_lens[s], a.max_kv), (int64_t)a.max_blocks * block_size);
    const int64_t n_vis = kv_len >= q_len ? (int64_t)kv_len - q_len + i + 1 : 0;
    const int g = h / (a.num_heads / a.kv_heads);
    const int64_t nb = a.num_slots / block_size;
    const int32_t* bt = a.block_tables + (int64_t)s * a.max_blocks;
    for (int d = tid; d < head_dim; d += AP_THREADS) qs[d] = to_f32(q[r * a.q_st + h * a.q_sh + d]);
    __syncthreads();

    float m = -3.402823466e38f, l = 0.0f, acc[AP_MAX_D / AP_THREADS] = {};
    for (int64_t c0 = 0; c0 < n_vis; c0 += AP_THREADS) {
        const int64_t j = c0 + tid;
        float sc = -INFINITY, vs = 1.0f;
        int64_t row = 0;
        if (j < n_vis) {
            const int64_t lb = j / block_size;
            int64_t id = bt[lb];
            id = id < 0 ? 0 : (id >= nb ? nb - 1 : id);
            row = ((int64_t)g * a.num_slots + id * block_size + (j - lb * block_size)) * head_dim;
            float dot = 0.0f;
            for (int d = 0; d < head_dim; d++) dot = fmaf(qs[d], pool_f32(k_pool + row + d), dot);
            if (a.k_scale) {
                dot *= a.k_scale[g * nb + id];
                vs = a.v_scale[g * nb + id];
            }
            sc = dot * scale_log2;
            if (a.scores) a.scores[(r * a.num_heads + h) * a.score_stride + j] = sc;
        }
        rows[tid] = row;
        const float m_new =
            fmaxf(m, ap_reduce(sc, red, [](float a, float b) { return fmaxf(a, b); }));
        const float corr = fast_exp2(m - m_new);
        const float p = j < n_vis ? fast_exp2(sc - m_new) : 0.0f;
        ps[tid] = p * vs;
        // (its barriers also publish ps and rows)
        l = l * corr + ap_reduce(p, red, [](float a, float b) { return a + b; });
        const int nj = (int)min(n_vis - c0, (int64_t)AP_THREADS);
#pragma unroll
        for (int x = 0; x < AP_MAX_D / AP_THREADS; x++) {
            const int d = tid + x * AP_THREADS;
            if (d < head_dim) {
                float pv = 0.0f;
                for (int jj = 0; jj < nj; jj++)
                    pv = fmaf(ps[jj], pool_f32(v_pool + rows[jj] + d), pv);
                acc[x] = acc[x] * corr + pv;
            }
        }
        m = m_new;
        __syncthreads();  // ps and rows are written again by the next chunk
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (a NaN is handed on)
#pragma unroll
    for (int x = 0; x < AP_MAX_D / AP_THREADS; x++) {
        const int d = tid + x * AP_THREADS;
        if (d < head_dim) {
            const int64_t at = r * a.o_st + h * a.o_sh + d;
            const float y = l == 0.0f ? 0.0f : acc[x] * inv;
            if (a.out_dtype == FLOUR_DTYPE_F32)
                static_cast<float*>(a.out)[at] = y;
            else if (a.out_dtype == FLOUR_DTYPE_BF16)
                static_cast<bf16_t*>(a.out)[at] = from_f32<bf16_t>(y);
            else
                static_cast<f16_t*>(a.out)[at] = from_f32<f16_t>(y);
        }
    }
    if (a.scores && tid == 0) {
        a.ml[(r * a.num_heads + h) * 2] = m;
        a.ml[(r * a.num_heads + h) * 2 + 1] = l;
    }
}

template <typename TQ, typename TP>
__global__ __launch_bounds__(AP_THREADS) void attn_pools_kernel(PoolAttn a) {
    const int r = blockIdx.x;
    int s = r, i = 0, q_len = 1;
    if (a.cu) {
        int lo = 0, hi = a.batch;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.cu[mid] <= r)
                lo = mid;
            else
                hi = mid;
        }
        s = lo;
        i = r - a.cu[s];
        q_len = a.cu[s + 1] - a.cu[s];
        if (i < 0 || i >= q_len) return;  // (rows of no sequence)
    }
    attn_row<TQ, TP>(a, r, blockIdx.y, s, i, q_len);
}

// Prefill with f16 queries whose copy of the cache in f16 (kv_q8.hip) may have lost values: the rows of the
// (sequence, kv head) pairs that hold such a block, `share` workgroups each, from the 8 bits again. Other
// pairs' workgroups read the scales and end, so that a call without such blocks takes a launch more: 16 x
// 128-512 rows over 1,152-1,536 tokens of 28 / 4 heads of 128 125.5 -> 129 us, 4 x 256-512 over 512-1,024
// of 14 / 2 of 64 28 -> 31, 1,024 rows over 32,768 of 32 / 8 of 128 942 -> 952.
template <typename TP>
__global__ __launch_bounds__(AP_THREADS) void attn_beyond_f16_kernel(PoolAttn a, int share) {
    const int pair = blockIdx.x / share, part = blockIdx.x - pair * share;
    const int s = pair / a.kv_heads, g = pair - s * a.kv_heads, n_rep = a.num_heads / a.kv_heads;
    const int r0 = a.cu[s], q_len = a.cu[s + 1] - r0;
    if (q_len <= 0 || r0 < 0 || r0 + q_len > a.rows) return;
    const int64_t kv_len =
        min((int64_t)min(a.kv_lens[s], a.max_kv), (int64_t)a.max_blocks * a.block_size);
    const int64_t nb = a.num_slots / a.block_size;
    const int blocks = (int)((kv_len + a.block_size - 1) / a.block_size);
    bool beyond = false;
    for (int lb = threadIdx.x; lb < blocks; lb += AP_THREADS) {
        int64_t id = a.block_tables[(int64_t)s * a.max_blocks + lb];
        id = g * nb + (id < 0 ? 0 : (id >= nb ? nb - 1 : id));
        beyond |= beyond_f16<TP>(a.k_scale[id]) || beyond_f16<TP>(a.v_scale[id]);
    }
    if (!__syncthreads_or(beyond)) return;
    for (int64_t x = part; x < (int64_t)q_len * n_rep; x += share) {
        const int i = (int)(x / n_rep);
        attn_row<f16_t, TP>(a, r0 + i, g * n_rep + (int)(x - (int64_t)i * n_rep), s, i, q_len);
    }
}

// weights[r, g, j] += sum over kv head g's query heads of exp2(score - max) / sum, in their order. It moves
// 4 (n_rep + 2) bytes a position and kv head and computes little: a thread takes four consecutive
// positions, 16 bytes a load (rows of any width: the loads need 4-byte alignment only), the last of a
// row one at a time. 64 x 512-4,096 positions of 32 / 8 heads (26 MB): 8.5 us, 3 TB/s; with four positions
// AP_THREADS apart 13.6.
static constexpr int WA_POS = 4;
typedef f32x4 __attribute__((aligned(4))) f32x4_any;
__global__ __launch_bounds__(AP_THREADS) void weights_add_kernel(
    float* __restrict__ weights, int64_t width, const int32_t* __restrict__ weight_rows,
    int num_rows, const int32_t* __restrict__ context_lens, int max_ctx, int kv_heads, int n_rep,
    const float* __restrict__ scores, int64_t score_stride, const float* __restrict__ ml) {
    const int b = blockIdx.z, g = blockIdx.y;
    const int ctx = min(context_lens[b], max_ctx);
    const int j0 = (blockIdx.x * AP_THREADS + (int)threadIdx.x) * WA_POS;
    const int r = weight_rows ? weight_rows[b] : b;
    if (j0 >= ctx || r < 0 || r >= num_rows) return;
    const int64_t h0 = ((int64_t)b * kv_heads + g) * n_rep;
    float* w = weights + ((int64_t)r * kv_heads + g) * width + j0;
    scores += h0 * score_stride + j0;
    ml += 2 * h0;
    auto inv_of = [&](int i) { return ml[2 * i + 1] == 0.0f ? 0.0f : 1.0f / ml[2 * i + 1]; };
    if (j0 + WA_POS <= ctx) {
        const f32x4 old = *reinterpret_cast<const f32x4_any*>(w);
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int i = 0; i < n_rep; i++) {
            const f32x4 s = *reinterpret_cast<const f32x4_any*>(scores + i * score_stride);
            const float m = ml[2 * i], inv = inv_of(i);
#pragma unroll
            for (int x = 0; x < WA_POS; x++) sum[x] = fmaf(fast_exp2(s[x] - m), inv, sum[x]);
        }
        f32x4 y;
#pragma unroll
        for (int x = 0; x < WA_POS; x++) y[x] = old[x] + sum[x];
        *reinterpret_cast<f32x4_any*>(w) = y;
        return;
    }
    for (int x = 0; x < ctx - j0; x++) {
        float sum = 0.0f;
        for (int i = 0; i < n_rep; i++)
            sum = fmaf(fast_exp2(scores[i * score_stride + x] - ml[2 * i]), inv_of(i), sum);
        w[x] += sum;
    }
}

int launch_weights_add(float* weights, int64_t width, const int32_t* weight_rows, int num_rows,
                       const int32_t* context_lens, int max_ctx, int batch, int kv_heads,
                       int n_rep, const float* scores, int64_t score_stride, const float* ml,
                       hipStream_t stream) {
    if (max_ctx <= 0) return FLOUR_OK;
    const int per = AP_THREADS * WA_POS;
    weights_add_kernel<<<dim3((unsigned)(((int64_t)max_ctx + per - 1) / per), kv_heads, batch),
                         dim3(AP_THREADS), 0, stream>>>(weights, width, weight_rows, num_rows,
                                                        context_lens, max_ctx, kv_heads, n_rep,
                                                        scores, score_stride, ml);
    return check_hip(hipGetLastError(), "attention weights launch");
}

int launch_attn_pools(const PoolAttn& a, hipStream_t stream) {
    if (a.head_dim > AP_MAX_D) {
        set_error("attention over 8-bit pools or with weights: head_dim %d > %d is not supported",
                  a.head_dim, AP_MAX_D);
        return FLOUR_ERR_UNSUPPORTED;
    }
    if (a.num_heads > 65535) {
        set_error("attention: %d heads are too many", a.num_heads);
        return FLOUR_ERR_UNSUPPORTED;
    }
#define FLOUR_AP(TQ, TP)                                                                          \
    attn_pools_kernel<TQ, TP><<<dim3(a.rows, a.num_heads), dim3(AP_THREADS), 0, stream>>>(a)
#define FLOUR_AP_Q(TQ)                                                                            \
    do {                                                                                          \
        if (a.pool_dtype == FLOUR_DTYPE_E4M3) FLOUR_AP(TQ, e4m3_t);                               \
        else if (a.pool_dtype == FLOUR_DTYPE_I8) FLOUR_AP(TQ, i8_t);                              \
        else FLOUR_AP(TQ, TQ);                                                                    \
    } while (0)
    if (a.dtype == FLOUR_DTYPE_F32) FLOUR_AP_Q(float);
    else if (a.dtype == FLOUR_DTYPE_BF16) FLOUR_AP_Q(bf16_t);
    else FLOUR_AP_Q(f16_t);
#undef FLOUR_AP_Q
#undef FLOUR_AP
    return check_hip(hipGetLastError(), "attention (any pool) launch");
}

int launch_attn_beyond_f16(const PoolAttn& a, int max_rows, hipStream_t stream) {
    const int64_t pairs = (int64_t)a.batch * a.kv_heads;
    const int64_t work = (int64_t)max_rows * (a.num_heads / a.kv_heads);
    const int share = (int)std::max<int64_t>(1, std::min<int64_t>(1024 / pairs, work));
    if (pairs > 0x7fffffff / share) {
        set_error("attention: %d sequences of %d kv heads are too many", a.batch, a.kv_heads);
        return FLOUR_ERR_UNSUPPORTED;
    }
    auto kern = a.pool_dtype == FLOUR_DTYPE_E4M3 ? attn_beyond_f16_kernel<e4m3_t>
                                                 : attn_beyond_f16_kernel<i8_t>;
    kern<<<dim3((unsigned)(pairs * share)), dim3(AP_THREADS), 0, stream>>>(a, share);
    return check_hip(hipGetLastError(), "attention beyond f16 launch");
}

}  // namespace flour
