// decode_ranges.h — how the streamed decode kernels cut their list of chunks into wave ranges, and
// the running maximum that they start from.
#pragma once

#include "flour_common.h"

namespace flour {

// Wave ranges over the flattened chunk list. The dispatcher places workgroup i on XCD i % 8,
// and on this path the odd XCDs stream 6-9% slower than their even partners (per-workgroup
// clock stamps: every pair, three machines, both head shapes), so the launch would wait for the
// odd half. Even-indexed ranges therefore hold w/32 more chunks than the mean and odd ones w/32
// fewer: range i is [lo(i), lo(i + 1)) with lo(i) = floor(total (32 i + w (i & 1)) / W),
// W = 32 n + w (n & 1), so lo(0) = 0 and lo(n) = total. The split depends on the shapes alone,
// never on timing, so results stay deterministic. I is uint32_t when total * (W + 32) fits 32
// bits (a 64-bit division is a long instruction sequence), else int64_t.
template <typename I>
struct WaveRanges {
    I total, n, w, W;
    __device__ WaveRanges(int64_t total_, int64_t n_, int w_)
        : total((I)total_), n((I)n_), w((I)w_), W((I)(32 * n_ + w_ * (n_ & 1))) {}
    __device__ I lo(I i) const { return total * (32 * i + w * (i & 1)) / W; }
    // the range holding chunk x (0 <= x < total): the last i < n with lo(i) <= x (the estimate
    // is within a range or two of it, as no range differs from the mean by more than w/32)
    __device__ I owner(I x) const {
        I i = x * W / (32 * total);
        if (i > n - 1) i = n - 1;
        while (i + 1 < n && lo(i + 1) <= x) i++;
        while (i > 0 && lo(i) > x) i--;
        return i;
    }
};

// Whether every numerator of WaveRanges fits 32 bits: up to ~174,500 chunks on 768 waves (64 x 10.9K
// tokens over 8 kv heads of a 16-bit pool), ~131,000 on 1,024 (64 x 4.1K of an fp32 one).
__device__ __forceinline__ bool ranges_narrow(int64_t total, int64_t n, int w) {
    return (uint64_t)total * (uint64_t)(32 * n + w + 32) <= 0xffffffffull;
}

// Ranges that a list of `total` chunks is cut into by a grid of `cap` waves: at least two chunks
// each. Fewer, longer ranges leave fewer pieces to merge (one 2,000-token sequence of 8 kv heads,
// 504 chunks: 10.2 us on 252 waves, 10.9 on 504), a list of more than `cap` chunks has a range of
// two anyway, and no range is empty (the smallest share is (32 - w) / 32 >= 1/2 of the mean).
__device__ __forceinline__ int64_t range_count(int64_t total, int64_t cap) {
    const int64_t half = total >> 1;
    return half < 1 ? 1 : (half < cap ? half : cap);
}

// Running maxima start at the lowest finite value: with scores of -inf alone (K rows that hold -inf,
// products that overflow) the maximum stays finite, every weight is exp2(-inf) = 0 and no
// difference of infinities reaches the sums. It costs nothing where a select per chunk would.
static constexpr float DEC_M0 = -3.402823466e38f;

}  // namespace flour
