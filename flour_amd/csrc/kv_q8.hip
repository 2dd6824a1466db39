// kv_q8.hip — new rows into an 8-bit cache, and the way back to a plain one.
//
// Write: a unit is one (block that the call writes, kv head, K or V). A block's scale depends on
// all of its new rows and on the scale that its kept rows have, so the unit finds the largest
// magnitude first (on the bit patterns, two 16-bit elements an instruction) and then rounds the rows to
// q = rne(x / S); they stay in registers in between. A wave takes a unit: the maximum is a wave
// reduction, no unit waits for another, nothing is atomic.
// Bound by memory for prompts: 7,547 rows of 8 heads of 128 from bf16 to int8 (46 MB) take 11 us, 4.2 TB/s
// (reading the rows twice 14.5), and by the launch and four dependent loads for decode steps: 64 rows 4.7.
// The units of a call are listed without a pass over it: sequence s owns the blocks from index
// cu[s] / bs + 2 s on, which leaves room for the n / bs + 2 blocks that n rows can touch.
#include "cache8.h"
#include "decode_pools.h"

namespace flour {

static constexpr int KQ_WAVES = 4;  // units of a workgroup, one a wave
static constexpr int KQ_HELD = 4;   // runs of a lane between the walks: 16 rows of 128 as 8-element runs

// N elements of a row, as they lie in memory. N is 8, or 1 where rows or pointers are not aligned.
template <typename T, int N>
struct Run {
    u32x4 w[sizeof(T) == 4 ? 2 : 1];
    __device__ __forceinline__ void clear() {
        for (auto& x : w) x = u32x4{0, 0, 0, 0};
    }
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(w) / 16); i++) w[i] = reinterpret_cast<const u32x4*>(p)[i];
    }
    // the largest magnitude, as an fp32 pattern (inf and NaN stay above the finite ones)
    __device__ __forceinline__ uint32_t amax() const {
        uint32_t m = 0;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; i++) m = max(m, w[i >> 2][i & 3] & 0x7fffffffu);
            return m;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) m = max_u16x2(m, w[0][i] & 0x7fff7fffu);
            m = max(m & 0xffffu, m >> 16);
            return __float_as_uint(to_f32(T{(uint16_t)m}));
        }
    }
    __device__ __forceinline__ void widen(float (&y)[N]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = __uint_as_float(w[i >> 2][i & 3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) y[2 * i] = lo_f32<T>(w[0][i]), y[2 * i + 1] = hi_f32<T>(w[0][i]);
        }
    }
};
template <typename T>
struct Run<T, 1> {
    float v;
    __device__ __forceinline__ void clear() { v = 0.0f; }
    __device__ __forceinline__ void load(const T* p) { v = to_f32(*p); }
    __device__ __forceinline__ uint32_t amax() const { return magnitude(v); }
    __device__ __forceinline__ void widen(float (&y)[1]) const { y[0] = v; }
};

// N elements q = rne(y * inv) at p.
template <typename TP, int N>
__device__ __forceinline__ void store_run8(uint8_t* p, const float (&y)[N], float inv) {
    if constexpr (N == 1) {
        *p = Elem8<TP>::narrow1(y[0] * inv);
    } else {
        const float a[4] = {y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv};
        const float b[4] = {y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv};
        *reinterpret_cast<u32x2*>(p) = u32x2{Elem8<TP>::narrow(a), Elem8<TP>::narrow(b)};
    }
}
template <int N>
using Raw8 = typename std::conditional<N == 1, uint8_t, u32x2>::type;  // N elements of a pool
template <typename TP, int N>
__device__ __forceinline__ void widen8(Raw8<N> w, float (&y)[N]) {
    if constexpr (N == 1) {
        y[0] = Elem8<TP>::widen1(w);
    } else {
        float a[4], b[4];
        Elem8<TP>::widen(w[0], a);
        Elem8<TP>::widen(w[1], b);
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = a[i], y[4 + i] = b[i];
    }
}

template <typename T, typename TP, int N>
__global__ __launch_bounds__(64 * KQ_WAVES) void kv_write_q8_kernel(
    const T* __restrict__ k, const T* __restrict__ v, int64_t st, int64_t sh,
    uint8_t* __restrict__ k_pool, uint8_t* __restrict__ v_pool, float* __restrict__ k_scale,
    float* __restrict__ v_scale, const int32_t* __restrict__ cu,
    const int32_t* __restrict__ kv_lens, const int32_t* __restrict__ block_tables, int max_blocks,
    int num_seqs, int total_q, int kv_heads, int head_dim, int block_size, int64_t num_slots,
    int64_t units) {
    const int lane = threadIdx.x & 63;
    const int64_t u = (int64_t)blockIdx.x * KQ_WAVES +
                      __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (u >= units) return;
    const int64_t item = u / (2 * kv_heads);
    const int rest = (int)(u - item * 2 * kv_heads), g = rest >> 1;
    const int s = wave_find_last(num_seqs, item, [&](int i) -> int64_t {
        return (int64_t)(cu[i] / block_size) + 2 * i;
    });
    const int r0 = cu[s], n = cu[s + 1] - r0, kv = kv_lens[s];
    if (n <= 0 || kv < n || r0 < 0 || r0 + n > total_q) return;
    const int p0 = kv - n;  // the first new position
    const int64_t nth = item - (r0 / block_size + 2 * s);  // of the sequence's blocks
    const int64_t lb = p0 / block_size + nth;
    const int64_t first = lb * block_size;  // the block's first position
    if (nth < 0 || first >= kv || lb >= max_blocks) return;
    const int64_t id = block_tables[(int64_t)s * max_blocks + lb];
    if (id < 0 || id >= num_slots / block_size) return;
    const int kept = (int)max((int64_t)p0 - first, (int64_t)0);
    const int end = (int)min(kv - first, (int64_t)block_size);  // rows kept .. end - 1 are new

    const bool is_v = rest & 1;
    // row i of the block, i >= kept, is packed row r0 + first + i - p0
    const T* src = (is_v ? v : k) + (r0 + first - p0) * st + g * sh;
    uint8_t* dst = (is_v ? v_pool : k_pool) + ((int64_t)g * num_slots + id * block_size) * head_dim;
    float* scale = (is_v ? v_scale : k_scale) + (int64_t)g * (num_slots / block_size) + id;
    const float old = kept > 0 ? *scale : 0.0f;
    const int runs = head_dim / N;  // of a row
    // a lane's runs: lane, lane + 64, .. of the new rows' (row i, run c), the first KQ_HELD of them held
    // between the two walks
    const int64_t step_i = 64 / runs * st;
    const int step_c = 64 % runs, all = (end - kept) * runs;
    int c = lane % runs;
    const T* row = src + (int64_t)(kept + lane / runs) * st;
    auto next = [&]() {
        c += step_c;
        row += step_i;
        if (c >= runs) c -= runs, row += st;
    };
    Run<T, N> held[KQ_HELD];
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < KQ_HELD; j++) {
        held[j].clear();
        if (64 * j + lane < all) held[j].load(row + c * N);
        next();
    }
    const int c1 = c;
    const T* row1 = row;
#pragma unroll
    for (int j = 0; j < KQ_HELD; j++) amax = max(amax, held[j].amax());
    for (int x = 64 * KQ_HELD + lane; x < all; x += 64) {
        Run<T, N> r;
        r.load(row + c * N);
        amax = max(amax, r.amax());
        next();
    }
    const float S = max_scale(pow2_scale(old), scale_for<TP>(wave_max_u32(amax)));
    const float inv = inv_scale(S);
    const bool poisoned = !(S >= 0.0f);  // (then zeros: only those that attend to the block see NaN)
    uint8_t* to = dst + (int64_t)kept * head_dim;
    auto store = [&](const Run<T, N>& r, int x) {
        float y[N];
        r.widen(y);
        if (poisoned)
#pragma unroll
            for (int e = 0; e < N; e++) y[e] = 0.0f;
        store_run8<TP, N>(to + (int64_t)x * N, y, inv);
    };
#pragma unroll
    for (int j = 0; j < KQ_HELD; j++)
        if (64 * j + lane < all) store(held[j], 64 * j + lane);
    c = c1;
    row = row1;
    for (int x = 64 * KQ_HELD + lane; x < all; x += 64) {
        Run<T, N> r;
        r.load(row + c * N);
        store(r, x);
        next();
    }
    if (S != old && S > 0.0f) {  // the kept rows, if the scale grew
        const float ratio = old * inv;
        for (int x = lane; x < kept * runs; x += 64) {
            float y[N];
            widen8<TP, N>(*reinterpret_cast<const Raw8<N>*>(dst + (int64_t)x * N), y);
            store_run8<TP, N>(dst + (int64_t)x * N, y, ratio);
        }
    }
    if (lane == 0) *scale = S;
}

// One wave a (sequence, block, kv head): rows of K and of V. STAGE: a copy for an attention kernel (out
// blocks by position, the table and lengths that go with them). What a block of scale NaN stands for
// must reach those that attend to it and nobody else, so it goes into the scores: K is NaN, V 0. It only
// moves bytes: four loads of K and of V a lane before their stores; 16,384 positions of 8 heads of 128 from
// e4m3 to bf16 (100 MB) take 17.5 us, 5.7 TB/s.
template <typename T, typename TP, int N, bool STAGE>
__global__ __launch_bounds__(64 * KQ_WAVES) void kv_dequant_kernel(
    T* __restrict__ k_out, T* __restrict__ v_out, const int32_t* __restrict__ out_tables,
    int out_max_blocks, int64_t out_slots, const uint8_t* __restrict__ k_pool,
    const uint8_t* __restrict__ v_pool, const float* __restrict__ k_scale,
    const float* __restrict__ v_scale, const int32_t* __restrict__ block_tables, int max_blocks,
    const int32_t* __restrict__ kv_lens, int num_seqs, int max_kv, int blocks_per_seq,
    int kv_heads, int head_dim, int block_size, int64_t num_slots, int32_t* __restrict__ staged_table,
    int32_t* __restrict__ staged_lens) {
    const int lane = threadIdx.x & 63;
    const int64_t u = (int64_t)blockIdx.x * KQ_WAVES +
                      __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t per_seq = (int64_t)blocks_per_seq * kv_heads;
    const int s = (int)(u / per_seq);
    if (s >= num_seqs) return;
    const int rest = (int)(u - s * per_seq), lb = rest / kv_heads, g = rest - lb * kv_heads;
    const int kv = min(kv_lens[s], max_kv);
    if constexpr (STAGE) {
        if (g == 0 && lane == 0) {
            staged_table[(int64_t)s * out_max_blocks + lb] = s * out_max_blocks + lb;
            if (lb == 0) staged_lens[s] = kv;
        }
    }
    const int64_t first = (int64_t)lb * block_size;
    if (first >= kv || lb >= max_blocks || lb >= out_max_blocks) return;
    const int64_t nb = num_slots / block_size;
    const int64_t raw = block_tables[(int64_t)s * max_blocks + lb];
    const int64_t id = raw < 0 ? 0 : (raw >= nb ? nb - 1 : raw);
    const int64_t to = STAGE ? (int64_t)s * out_max_blocks + lb
                             : (int64_t)out_tables[(int64_t)s * out_max_blocks + lb];
    if (to < 0 || to >= out_slots / block_size) return;
    const int rows = (int)min((int64_t)kv - first, (int64_t)block_size);
    const int64_t src = ((int64_t)g * num_slots + id * block_size) * head_dim;
    const int64_t dst = ((int64_t)g * out_slots + to * block_size) * head_dim;
    float ks = k_scale[g * nb + id], vs = v_scale[g * nb + id];
    if (STAGE && !(fabsf(vs) < INFINITY)) ks = __uint_as_float(0x7fc00000u), vs = 0.0f;
    auto put = [&](T* out, Raw8<N> w, float S) {
        float y[N];
        widen8<TP, N>(w, y);
#pragma unroll
        for (int j = 0; j < N; j++) {
            y[j] *= S;
            if constexpr (std::is_same<T, f16_t>::value)  // (a NaN stays one)
                y[j] = y[j] > 65504.0f ? 65504.0f : (y[j] < -65504.0f ? -65504.0f : y[j]);
        }
        if constexpr (N == 1) {
            *out = from_f32<T>(y[0]);
        } else if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<f32x4*>(out) = f32x4{y[0], y[1], y[2], y[3]};
            *reinterpret_cast<f32x4*>(out + 4) = f32x4{y[4], y[5], y[6], y[7]};
        } else {
            *reinterpret_cast<u32x4*>(out) = u32x4{pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]),
                                                   pack2<T>(y[4], y[5]), pack2<T>(y[6], y[7])};
        }
    };
    const int64_t all = (int64_t)rows * head_dim;
    for (int64_t x0 = (int64_t)lane * N; x0 < all; x0 += 64 * N * KQ_HELD) {
        Raw8<N> kw[KQ_HELD], vw[KQ_HELD];
#pragma unroll
        for (int j = 0; j < KQ_HELD; j++) {  // (past the end: the first again, for nothing)
            const int64_t x = x0 + 64 * N * j < all ? x0 + 64 * N * j : x0;
            kw[j] = *reinterpret_cast<const Raw8<N>*>(k_pool + src + x);
            vw[j] = *reinterpret_cast<const Raw8<N>*>(v_pool + src + x);
        }
#pragma unroll
        for (int j = 0; j < KQ_HELD; j++) {
            const int64_t x = x0 + 64 * N * j;
            if (x < all) {
                put(k_out + dst + x, kw[j], ks);
                put(v_out + dst + x, vw[j], vs);
            }
        }
    }
}

template <typename T, typename TP, int N>
static void launch_write_t(const void* k, const void* v, int64_t st, int64_t sh, void* k_pool,
                           void* v_pool, float* k_scale, float* v_scale, const int32_t* cu,
                           const int32_t* kv_lens, const int32_t* bt, int max_blocks, int num_seqs,
                           int total_q, int kv_heads, int head_dim, int block_size,
                           int64_t num_slots, int64_t units, hipStream_t s) {
    kv_write_q8_kernel<T, TP, N>
        <<<dim3((unsigned)((units + KQ_WAVES - 1) / KQ_WAVES)), dim3(64 * KQ_WAVES), 0, s>>>(
            static_cast<const T*>(k), static_cast<const T*>(v), st, sh,
            static_cast<uint8_t*>(k_pool), static_cast<uint8_t*>(v_pool), k_scale, v_scale, cu,
            kv_lens, bt, max_blocks, num_seqs, total_q, kv_heads, head_dim, block_size, num_slots,
            units);
}

bool check_pool8(const char* what, int pool_dtype, const void* k_pool, const void* v_pool,
                 const void* k_scale, const void* v_scale, int kv_heads, int head_dim,
                 int block_size, int64_t num_slots) {
    if (!valid_pool8(pool_dtype)) {
        set_error("%s: pool dtype %d is not an 8-bit one", what, pool_dtype);
        return false;
    }
    if (kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || num_slots <= 0 ||
        num_slots % block_size != 0 || num_slots > 0x7fffffff ||
        (int64_t)block_size * head_dim > 0x7fffffff) {
        set_error("%s: bad pool shape (kv_heads=%d head_dim=%d bs=%d num_slots=%lld)", what,
                  kv_heads, head_dim, block_size, (long long)num_slots);
        return false;
    }
    if (!k_pool || !v_pool || !k_scale || !v_scale) {
        set_error("%s: null pool or scale pointer", what);
        return false;
    }
    return true;
}

int launch_kv_dequant(void* k_out, void* v_out, int dtype, const int32_t* out_tables,
                      int out_max_blocks, int64_t out_slots, const void* k_pool,
                      const void* v_pool, const float* k_scale, const float* v_scale,
                      int pool_dtype, const int32_t* bt, int max_blocks, const int32_t* kv_lens,
                      int num_seqs, int max_kv, int kv_heads, int head_dim, int block_size,
                      int64_t num_slots, int32_t* staged_table, int32_t* staged_lens,
                      hipStream_t s) {
    const int per_seq = (int)(((int64_t)max_kv + block_size - 1) / block_size);
    const int64_t waves = (int64_t)num_seqs * per_seq * kv_heads;
    const int64_t grid = (waves + KQ_WAVES - 1) / KQ_WAVES;
    if (grid > 0x7fffffff) {
        set_error("kv_dequant: %lld blocks are too many for one call", (long long)waves);
        return FLOUR_ERR_UNSUPPORTED;
    }
    if (grid == 0) return FLOUR_OK;
    const bool wide = head_dim % 8 == 0 && (((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0 &&
                      (((uintptr_t)k_pool | (uintptr_t)v_pool) & 7) == 0;
#define FLOUR_DQ(T, TP, N)                                                                        \
    (staged_table ? kv_dequant_kernel<T, TP, N, true>                                             \
                  : kv_dequant_kernel<T, TP, N, false>)                                           \
        <<<dim3((unsigned)grid), dim3(64 * KQ_WAVES), 0, s>>>(                                    \
        static_cast<T*>(k_out), static_cast<T*>(v_out), out_tables, out_max_blocks, out_slots,    \
        static_cast<const uint8_t*>(k_pool), static_cast<const uint8_t*>(v_pool), k_scale,        \
        v_scale, bt, max_blocks, kv_lens, num_seqs, max_kv, per_seq, kv_heads, head_dim,          \
        block_size, num_slots, staged_table, staged_lens)
#define FLOUR_DQ_T(T)                                                                             \
    do {                                                                                          \
        if (pool_dtype == FLOUR_DTYPE_E4M3) {                                                     \
            if (wide) FLOUR_DQ(T, e4m3_t, 8);                                                     \
            else FLOUR_DQ(T, e4m3_t, 1);                                                          \
        } else {                                                                                  \
            if (wide) FLOUR_DQ(T, i8_t, 8);                                                       \
            else FLOUR_DQ(T, i8_t, 1);                                                            \
        }                                                                                         \
    } while (0)
    if (dtype == FLOUR_DTYPE_F32) FLOUR_DQ_T(float);
    else if (dtype == FLOUR_DTYPE_BF16) FLOUR_DQ_T(bf16_t);
    else FLOUR_DQ_T(f16_t);
#undef FLOUR_DQ_T
#undef FLOUR_DQ
    return check_hip(hipGetLastError(), "kv_dequant launch");
}

}  // namespace flour

using namespace flour;

extern "C" int flour_hip_kv_write_q8(const void* k, const void* v, int64_t stride_tok,
                                     int64_t stride_head, int dtype, void* k_pool, void* v_pool,
                                     float* k_scale, float* v_scale, int pool_dtype,
                                     const int32_t* cu_seqlens_q, const int32_t* kv_lens,
                                     const int32_t* block_tables, int max_blocks_per_seq,
                                     int num_seqs, int total_q, int kv_heads, int head_dim,
                                     int block_size, int64_t num_slots, void* stream) {
    clear_error();
    if (!valid_dtype(dtype)) {
        set_error("kv_write_q8: unknown dtype %d", dtype);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    if (!check_pool8("kv_write_q8", pool_dtype, k_pool, v_pool, k_scale, v_scale, kv_heads,
                     head_dim, block_size, num_slots))
        return FLOUR_ERR_INVALID_ARGUMENT;
    if (num_seqs < 0 || total_q < 0 || max_blocks_per_seq <= 0) {
        set_error("kv_write_q8: bad shape (seqs=%d total_q=%d max_blocks=%d)", num_seqs, total_q,
                  max_blocks_per_seq);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    if (num_seqs == 0 || total_q == 0) return FLOUR_OK;
    if (!k || !v || !cu_seqlens_q || !kv_lens || !block_tables) {
        set_error("kv_write_q8: null pointer");
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    const int64_t items = (int64_t)total_q / block_size + 2 * (int64_t)num_seqs;
    const int64_t units = items * 2 * kv_heads;
    if ((units + KQ_WAVES - 1) / KQ_WAVES > 0x7fffffff) {
        set_error("kv_write_q8: %d rows of %d sequences are too many for one call", total_q,
                  num_seqs);
        return FLOUR_ERR_UNSUPPORTED;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int es = elem_bytes(dtype);
    const bool wide =
        head_dim % 8 == 0 && ((stride_tok * es) | (stride_head * es)) % 16 == 0 &&
        (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && (((uintptr_t)k_pool | (uintptr_t)v_pool) & 7) == 0;
#define FLOUR_WQ(T, TP)                                                                           \
    (wide ? launch_write_t<T, TP, 8>(k, v, stride_tok, stride_head, k_pool, v_pool, k_scale,      \
                                     v_scale, cu_seqlens_q, kv_lens, block_tables,                \
                                     max_blocks_per_seq, num_seqs, total_q, kv_heads, head_dim,   \
                                     block_size, num_slots, units, s)                             \
          : launch_write_t<T, TP, 1>(k, v, stride_tok, stride_head, k_pool, v_pool, k_scale,      \
                                     v_scale, cu_seqlens_q, kv_lens, block_tables,                \
                                     max_blocks_per_seq, num_seqs, total_q, kv_heads, head_dim,   \
                                     block_size, num_slots, units, s))
    const bool f8 = pool_dtype == FLOUR_DTYPE_E4M3;
    if (dtype == FLOUR_DTYPE_F32) f8 ? FLOUR_WQ(float, e4m3_t) : FLOUR_WQ(float, i8_t);
    else if (dtype == FLOUR_DTYPE_BF16) f8 ? FLOUR_WQ(bf16_t, e4m3_t) : FLOUR_WQ(bf16_t, i8_t);
    else f8 ? FLOUR_WQ(f16_t, e4m3_t) : FLOUR_WQ(f16_t, i8_t);
#undef FLOUR_WQ
    return check_hip(hipGetLastError(), "kv_write_q8 launch");
}

extern "C" int flour_hip_kv_dequant(void* k_out, void* v_out, int dtype,
                                    const int32_t* out_tables, int out_max_blocks,
                                    int64_t out_slots, const void* k_pool, const void* v_pool,
                                    const float* k_scale, const float* v_scale, int pool_dtype,
                                    const int32_t* block_tables, int max_blocks_per_seq,
                                    const int32_t* kv_lens, int num_seqs, int max_kv_len,
                                    int kv_heads, int head_dim, int block_size, int64_t num_slots,
                                    void* stream) {
    clear_error();
    if (!valid_dtype(dtype)) {
        set_error("kv_dequant: unknown dtype %d", dtype);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    if (!check_pool8("kv_dequant", pool_dtype, k_pool, v_pool, k_scale, v_scale, kv_heads,
                     head_dim, block_size, num_slots))
        return FLOUR_ERR_INVALID_ARGUMENT;
    if (num_seqs < 0 || max_kv_len < 0 || max_blocks_per_seq <= 0 || out_max_blocks <= 0 ||
        out_slots <= 0 || out_slots % block_size != 0 ||
        (int64_t)max_kv_len > (int64_t)max_blocks_per_seq * block_size ||
        (int64_t)max_kv_len > (int64_t)out_max_blocks * block_size) {
        set_error("kv_dequant: bad shape (seqs=%d max_kv=%d max_blocks=%d out_blocks=%d "
                  "out_slots=%lld bs=%d)",
                  num_seqs, max_kv_len, max_blocks_per_seq, out_max_blocks, (long long)out_slots,
                  block_size);
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    if (num_seqs == 0 || max_kv_len == 0) return FLOUR_OK;
    if (!k_out || !v_out || !out_tables || !block_tables || !kv_lens) {
        set_error("kv_dequant: null pointer");
        return FLOUR_ERR_INVALID_ARGUMENT;
    }
    return launch_kv_dequant(k_out, v_out, dtype, out_tables, out_max_blocks, out_slots, k_pool,
                             v_pool, k_scale, v_scale, pool_dtype, block_tables,
                             max_blocks_per_seq, kv_lens, num_seqs, max_kv_len, kv_heads, head_dim,
                             block_size, num_slots, nullptr, nullptr,
                             static_cast<hipStream_t>(stream));
}
