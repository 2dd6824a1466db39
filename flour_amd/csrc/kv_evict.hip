// kv_evict.hip — eviction by accumulated attention weight: each kv head of a sequence keeps its
// latest positions and the heaviest of the others, gathered into new blocks.
//
// Two kernels. Selection, a workgroup a (sequence, kv head): the weights become 32-bit keys whose
// unsigned order is the weights' (NaN lowest, -0 as +0), the m-th largest key is found bit by bit
// by counting, then one ordered pass writes the kept positions and their sums. Gather, a wave a
// (sequence, destination block, kv head): kept rows are copied (plain pools) or requantised under
// the destination block's own scale (8-bit pools).
#include "cache8.h"
#include "decode_pools.h"

namespace flour {

static constexpr int EV_THREADS = 1024;
static constexpr int EV_WAVES = EV_THREADS / 64;

__device__ __forceinline__ uint32_t weight_key(float w) {
    if (!(w == w)) return 0;
    if (w == 0.0f) w = 0.0f;
    const uint32_t u = __float_as_uint(w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int ev_total(int x, int* red) {  // sum over the workgroup, in every thread
    const int w = wave_incl_sum(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = w;
    __syncthreads();
    int t = 0;
#pragma unroll
    for (int i = 0; i < EV_WAVES; i++) t += red[i];
    return t;
}

__global__ __launch_bounds__(EV_THREADS) void evict_select_kernel(
    const float* weights, float* weights_out, int64_t width, const int32_t* __restrict__ weight_rows,
    int num_rows, const int32_t* __restrict__ context_lens, const int32_t* __restrict__ keep_lens,
    int32_t* __restrict__ kept, int kv_heads, int max_ctx, int max_keep, int recent) {
    __shared__ int red[EV_WAVES], base_gt[EV_WAVES], base_eq[EV_WAVES];
    const int g = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
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

    // the largest T with at least `heavy` keys >= T
    uint32_t T = 0;
    if (heavy > 0 && heavy < cand)
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t t = T | (1u << bit);
            int c = 0;
            for (int j = tid; j < cand; j += EV_THREADS) c += weight_key(w[j]) >= t;
            if (ev_total(c, red) >= heavy) T = t;
        }
    int c = 0;
    for (int j = tid; j < cand; j += EV_THREADS) c += weight_key(w[j]) > T;
    const int above = heavy > 0 ? ev_total(c, red) : 0;
    const int ties = heavy < cand ? heavy - above : cand;  // of the keys equal to T, the first ones

    // in order: sums move towards the front, so that weights_out may be weights
    int n_gt = 0, n_eq = 0;  // kept so far, and keys equal to T so far
    for (int j0 = 0; j0 < L; j0 += EV_THREADS) {
        const int j = j0 + tid;
        const float x = j < L ? w[j] : 0.0f;
        const bool is_late = j >= cand && j < L;
        const uint32_t key = weight_key(x);
        const bool gt = j < L && (is_late || (heavy > 0 && key > T));
        const bool eq = j < cand && heavy > 0 && key == T;
        const uint64_t below = (1ull << lane) - 1;
        const uint64_t beq = __ballot(eq);
        __syncthreads();  // (also: every w[j] of this step is read before a sum is written)
        if (lane == 0) base_eq[wv] = __popcll(beq);
        __syncthreads();
        int before = n_eq, all = 0;
        for (int i = 0; i < EV_WAVES; i++) {
            if (i < wv) before += base_eq[i];
            all += base_eq[i];
        }
        n_eq += all;
        const bool keep = gt || (eq && before + __popcll(beq & below) < ties);
        const uint64_t bk = __ballot(keep);
        if (lane == 0) base_gt[wv] = __popcll(bk);
        __syncthreads();
        int to = n_gt + __popcll(bk & below);
        all = 0;
        for (int i = 0; i < EV_WAVES; i++) {
            if (i < wv) to += base_gt[i];
            all += base_gt[i];
        }
        n_gt += all;
        if (keep && to < n) {
            out[to] = j;
            wo[to] = x;
        }
    }
    __syncthreads();
    for (int i = n + tid; i < L; i += EV_THREADS) wo[i] = 0.0f;
}

// Rows of plain pools, in pieces of type V.
template <typename V>
__global__ __launch_bounds__(256) void evict_gather_kernel(
    char* k_pool, char* v_pool, const int32_t* __restrict__ block_tables, int max_blocks,
    const int32_t* __restrict__ out_tables, int out_max_blocks, const int32_t* __restrict__ kept,
    int kv_heads, int block_size, int64_t num_slots, int64_t row_bytes, int max_keep,
    int64_t units) {
    const int lane = threadIdx.x & 63;
    const int64_t u = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (u >= units) return;
    const int per_seq = (max_keep + block_size - 1) / block_size;
    const int64_t bg = u / per_seq;
    const int lb = (int)(u - bg * per_seq), b = (int)(bg / kv_heads), g = (int)(bg - (int64_t)b * kv_heads);
    const int64_t nb = num_slots / block_size;
    if (lb >= out_max_blocks) return;
    const int64_t to = out_tables[(int64_t)b * out_max_blocks + lb];
    if (to < 0 || to >= nb) return;
    const int32_t* pos = kept + bg * max_keep + (int64_t)lb * block_size;
    const int rows = min(block_size, max_keep - lb * block_size);
    const int64_t head = (int64_t)g * num_slots, vecs = row_bytes / (int64_t)sizeof(V);
    for (int64_t x = lane; x < rows * vecs; x += 64) {
        const int i = (int)(x / vecs);
        const int p = pos[i];
        if (p < 0) break;  // the rows behind it are too
        int64_t id = block_tables[(int64_t)b * max_blocks + min(p / block_size, max_blocks - 1)];
        id = id < 0 ? 0 : (id >= nb ? nb - 1 : id);
        const int64_t c = (x - i * vecs) * (int64_t)sizeof(V);
        const int64_t from = (head + id * block_size + p % block_size) * row_bytes + c;
        const int64_t dst = (head + to * block_size + i) * row_bytes + c;
        *reinterpret_cast<V*>(k_pool + dst) = *reinterpret_cast<const V*>(k_pool + from);
        *reinterpret_cast<V*>(v_pool + dst) = *reinterpret_cast<const V*>(v_pool + from);
    }
}

// The same over 8-bit pools; blockIdx.y: K or V.
template <typename TP>
__global__ __launch_bounds__(256) void evict_gather8_kernel(
    uint8_t* k_pool, uint8_t* v_pool, float* k_scale, float* v_scale,
    const int32_t* __restrict__ block_tables, int max_blocks,
    const int32_t* __restrict__ out_tables, int out_max_blocks, const int32_t* __restrict__ kept,
    int kv_heads, int head_dim, int block_size, int64_t num_slots, int max_keep, int64_t units) {
    const int lane = threadIdx.x & 63;
    const int64_t u = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (u >= units) return;
    const int per_seq = (max_keep + block_size - 1) / block_size;
    const int64_t bg = u / per_seq;
    const int lb = (int)(u - bg * per_seq), b = (int)(bg / kv_heads), g = (int)(bg - (int64_t)b * kv_heads);
    const int64_t nb = num_slots / block_size;
    if (lb >= out_max_blocks) return;
    const int64_t to = out_tables[(int64_t)b * out_max_blocks + lb];
    if (to < 0 || to >= nb) return;
    const int32_t* pos = kept + bg * max_keep + (int64_t)lb * block_size;
    const int rows = min(block_size, max_keep - lb * block_size);
    if (pos[0] < 0) return;
    uint8_t* pool = blockIdx.y ? v_pool : k_pool;
    float* scale = (blockIdx.y ? v_scale : k_scale) + g * nb;
    const int64_t head = (int64_t)g * num_slots;
    auto source = [&](int p, float& S) -> const uint8_t* {
        int64_t id = block_tables[(int64_t)b * max_blocks + min(p / block_size, max_blocks - 1)];
        id = id < 0 ? 0 : (id >= nb ? nb - 1 : id);
        S = scale[id];
        return pool + (head + id * block_size + p % block_size) * head_dim;
    };
    uint32_t amax = 0;
    for (int64_t x = lane; x < (int64_t)rows * head_dim; x += 64) {
        const int i = (int)(x / head_dim);
        if (pos[i] < 0) break;
        float S;
        const uint8_t* row = source(pos[i], S);
        amax = max(amax, magnitude(Elem8<TP>::widen1(row[x - (int64_t)i * head_dim]) * S));
    }
    const float T = scale_for<TP>(wave_max_u32(amax)), inv = inv_scale(T);
    uint8_t* dst = pool + (head + to * block_size) * head_dim;
    for (int64_t x = lane; x < (int64_t)rows * head_dim; x += 64) {
        const int i = (int)(x / head_dim);
        if (pos[i] < 0) break;
        float S;
        const uint8_t* row = source(pos[i], S);
        dst[x] = Elem8<TP>::narrow1(Elem8<TP>::widen1(row[x - (int64_t)i * head_dim]) * S * inv);
    }
    if (lane == 0) scale[to] = T;
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
    evict_select_kernel<<<dim3(kv_heads, batch), dim3(EV_THREADS), 0, s>>>(
        weights, weights_out, weights_width, weight_rows, num_weight_rows, context_lens, keep_lens,
        kept, kv_heads, max_context_len, max_keep_len, recent);
    int rc = check_hip(hipGetLastError(), "kv_evict selection launch");
    if (rc != FLOUR_OK || grid == 0) return rc;
    if (q8) {
#define FLOUR_EV8(TP)                                                                             \
    evict_gather8_kernel<TP><<<dim3((unsigned)grid, 2), dim3(256), 0, s>>>(                       \
        static_cast<uint8_t*>(k_pool), static_cast<uint8_t*>(v_pool), k_scale, v_scale,           \
        block_tables, max_blocks_per_seq, out_tables, out_max_blocks, kept, kv_heads, head_dim,   \
        block_size, num_slots, max_keep_len, units)
        if (pool_dtype == FLOUR_DTYPE_E4M3)
            FLOUR_EV8(e4m3_t);
        else
            FLOUR_EV8(i8_t);
#undef FLOUR_EV8
        return check_hip(hipGetLastError(), "kv_evict launch");
    }
    const int64_t row = (int64_t)head_dim * elem_bytes(pool_dtype);
    const uint64_t bits = (uint64_t)row | (uint64_t)(uintptr_t)k_pool | (uint64_t)(uintptr_t)v_pool;
#define FLOUR_EV(V)                                                                               \
    evict_gather_kernel<V><<<dim3((unsigned)grid), dim3(256), 0, s>>>(                            \
        static_cast<char*>(k_pool), static_cast<char*>(v_pool), block_tables, max_blocks_per_seq, \
        out_tables, out_max_blocks, kept, kv_heads, block_size, num_slots, row, max_keep_len,     \
        units)
    if ((bits & 15) == 0)
        FLOUR_EV(u32x4);
    else if ((bits & 3) == 0)
        FLOUR_EV(uint32_t);
    else
        FLOUR_EV(uint16_t);
#undef FLOUR_EV
    return check_hip(hipGetLastError(), "kv_evict launch");
}
