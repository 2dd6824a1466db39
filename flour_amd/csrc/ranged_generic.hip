// ranged_generic.hip — attention over a sliding window with sinks, or over everything, for every head_dim
// up to 512, page size, group size and alignment: what the faster kernels are checked against and
// what runs where they do not take a shape.
//
// A workgroup a (row, query head). Its visible positions are the sinks [0, a) and the window [b, p];
// it takes them 256 at a time: a thread's whole dot product each, one running maximum and sum, then a
// thread's output dims each over the 256 weights in LDS. Positions that the row does not see are
// never read, so their bits do not matter. A prefix that sequences share is read by each of its rows.
// Bound by the vector units and by reading K/V once a query head: decode, 64 x 512-4,096 tokens of 32 / 8
// heads of 128 in bf16 with a window of 1,024 takes 221 us.
#include <math.h>

#include "decode_ranges.h"
#include "ranged.h"

namespace flour {

static constexpr int RG_THREADS = 256;
static constexpr int RG_MAX_D = 512;

template <typename F>
__device__ __forceinline__ float rg_reduce(float x, float* red, F op) {
    for (int o = 32; o > 0; o >>= 1) x = op(x, __shfl_xor(x, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    float r = red[0];
    for (int i = 1; i < RG_THREADS / 64; i++) r = op(r, red[i]);
    return r;
}

template <typename T>
__global__ __launch_bounds__(RG_THREADS) void ranged_generic_kernel(RangedAttn a) {
    __shared__ float qs[RG_MAX_D];
    __shared__ float ps[RG_THREADS];
    __shared__ int64_t at[RG_THREADS];
    __shared__ float red[RG_THREADS / 64];
    const int r = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
    const int head_dim = a.head_dim, block_size = a.block_size;
    const int s = a.cu ? ranged_seq_of(a, r) : r;
    const RangedSeq sq = ranged_seq(a, s);
    const int i = r - sq.row0;
    if (i < 0 || i >= sq.rows) return;  // (rows of no sequence)
    const int p = sq.kv > 0 ? sq.kv - sq.rows + i : -1;  // the row's own position
    const int first = min(a.sinks, p + 1), from = max(first, p - a.window + 1);
    const int n_vis = first + (p + 1 - from);
    const int g = h / (a.num_heads / a.kv_heads);
    const int64_t max_id = a.num_slots / block_size - 1;
    const int32_t* bt = a.block_tables + (int64_t)s * a.max_blocks;
    const T* __restrict__ q = static_cast<const T*>(a.q) + r * a.q_st + h * a.q_sh;
    const T* __restrict__ k_pool = static_cast<const T*>(a.k_pool);
    const T* __restrict__ v_pool = static_cast<const T*>(a.v_pool);
    for (int d = tid; d < head_dim; d += RG_THREADS) qs[d] = to_f32(q[d]);
    __syncthreads();

    float m = DEC_M0, l = 0.0f, acc[RG_MAX_D / RG_THREADS] = {};
    for (int64_t c0 = 0; c0 < n_vis; c0 += RG_THREADS) {
        const int64_t x = c0 + tid;
        float sc = -INFINITY;
        int64_t row = 0;
        if (x < n_vis) {
            const int j = (int)(x < first ? x : x - first + from);
            const int lb = j / block_size;
            int64_t id = bt[lb];  // clamped: a bad block id never leaves the pool
            id = id < 0 ? 0 : (id > max_id ? max_id : id);
            row = ((int64_t)g * a.num_slots + id * block_size + (j - lb * block_size)) * head_dim;
            float dot = 0.0f;
            for (int d = 0; d < head_dim; d++) dot = fmaf(qs[d], to_f32(k_pool[row + d]), dot);
            sc = dot * a.scale;
        }
        at[tid] = row;
        const float m_new = fmaxf(m, rg_reduce(sc, red, [](float x, float y) { return fmaxf(x, y); }));
        const float corr = expf(m - m_new);
        const float w = x < n_vis ? expf(sc - m_new) : 0.0f;
        ps[tid] = w;
        // (its barriers also publish ps and at)
        l = l * corr + rg_reduce(w, red, [](float x, float y) { return x + y; });
        const int nj = (int)min((int64_t)n_vis - c0, (int64_t)RG_THREADS);
#pragma unroll
        for (int e = 0; e < RG_MAX_D / RG_THREADS; e++) {
            const int d = tid + e * RG_THREADS;
            if (d < head_dim) {
                float pv = 0.0f;
                for (int jj = 0; jj < nj; jj++) pv = fmaf(ps[jj], to_f32(v_pool[at[jj] + d]), pv);
                acc[e] = acc[e] * corr + pv;
            }
        }
        m = m_new;
        __syncthreads();  // ps and at are written again by the next chunk
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (a NaN is handed on)
#pragma unroll
    for (int e = 0; e < RG_MAX_D / RG_THREADS; e++) {
        const int d = tid + e * RG_THREADS;
        if (d < head_dim) {
            const int64_t to = r * a.o_st + h * a.o_sh + d;
            const float y = l == 0.0f ? 0.0f : acc[e] * inv;
            store_1(a.out, a.out_dtype, to, y);
        }
    }
}

int launch_ranged_generic(const RangedAttn& a, hipStream_t stream) {
    if (a.head_dim > RG_MAX_D) {
        set_error("attention over a window or a shared prefix: head_dim %d > %d is not supported",
                  a.head_dim, RG_MAX_D);
        return FLOUR_ERR_UNSUPPORTED;
    }
    if (a.num_heads > 65535) {
        set_error("attention: %d heads are too many", a.num_heads);
        return FLOUR_ERR_UNSUPPORTED;
    }
    auto kern = a.dtype == FLOUR_DTYPE_F32    ? ranged_generic_kernel<float>
                : a.dtype == FLOUR_DTYPE_BF16 ? ranged_generic_kernel<bf16_t>
                                              : ranged_generic_kernel<f16_t>;
    kern<<<dim3(a.rows, a.num_heads), dim3(RG_THREADS), 0, stream>>>(a);
    return check_hip(hipGetLastError(), "attention (window / shared prefix) launch");
}

}  // namespace flour
