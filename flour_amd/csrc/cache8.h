// cache8.h — elements, scales and argument checks of the 8-bit KV pools.
//
// An element q of an 8-bit pool stands for q * S, S the fp32 scale of its (kv head, block). The
// write and the eviction choose S as a power of two, the smallest with which no element of the
// block exceeds QMAX (448 for e4m3, 127 for int8). With it q * S is exact in fp32 and bf16, x / S
// is an exact multiplication, a block whose scale grows is requantised by a change of exponent, and
// 64-bit and 32-bit arithmetic quantise to the same bits. What it costs is at most one bit of
// int8's seven; e4m3 has exponents of its own and loses none but at the bottom of its range.
#pragma once

#include "flour_common.h"

namespace flour {

struct e4m3_t {
    uint8_t bits;
};
struct i8_t {
    int8_t v;
};

inline bool valid_pool8(int dtype) {
    return dtype == FLOUR_DTYPE_E4M3 || dtype == FLOUR_DTYPE_I8;
}

// The larger of two dwords' 16-bit halves, as unsigned (magnitudes of 16-bit floats are ordered as their
// patterns, infinities and NaN above the finite ones).
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                  __builtin_bit_cast(u16x2, b)));
}

template <typename T>
struct Elem8;

template <>
struct Elem8<e4m3_t> {
    // amax = f 2^x, f in [1/2, 1): amax <= 448 2^e = 0.875 2^(9 + e)
    static constexpr float TOP = 0.875f;
    static constexpr int EXP = 9;
    static constexpr float QMAX = 448.0f;
    // the four elements of a dword
    static __device__ __forceinline__ void widen(uint32_t w, float (&y)[4]) {
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
        const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        y[0] = a[0], y[1] = a[1], y[2] = b[0], y[3] = b[1];
    }
    static __device__ __forceinline__ uint32_t narrow(const float (&y)[4]) {  // |y| <= 448
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        return __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
    }
    // m's halves: the larger of them and of the magnitudes (bit patterns) in w; what a half stands for
    static __device__ __forceinline__ uint32_t max_halves(uint32_t w, uint32_t m) {
        return max_u16x2(max_u16x2(m, w & 0x007f007fu), (w >> 8) & 0x007f007fu);
    }
    static __device__ __forceinline__ float half_value(uint32_t h) { return widen1((uint8_t)h); }
    static __device__ __forceinline__ float widen1(uint8_t b) {
        return __builtin_amdgcn_cvt_f32_fp8(b, 0);
    }
    static __device__ __forceinline__ uint8_t narrow1(float y) {
        return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false);
    }
};

template <>
struct Elem8<i8_t> {
    static constexpr float TOP = 0.9921875f;  // 127 / 128
    static constexpr int EXP = 7;
    static constexpr float QMAX = 127.0f;
    static __device__ __forceinline__ float widen1(uint8_t b) { return (float)(int8_t)b; }
    static __device__ __forceinline__ uint32_t max_halves(uint32_t w, uint32_t m) {
        typedef __attribute__((ext_vector_type(2))) int16_t i16x2;
        const i16x2 odd = __builtin_bit_cast(i16x2, w) >> (int16_t)8;
        const i16x2 even = __builtin_bit_cast(i16x2, w << 8) >> (int16_t)8;
        i16x2 x = __builtin_elementwise_max(__builtin_bit_cast(i16x2, m), odd);
        x = __builtin_elementwise_max(x, (i16x2)(-odd));
        x = __builtin_elementwise_max(x, even);
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(x, (i16x2)(-even)));
    }
    static __device__ __forceinline__ float half_value(uint32_t h) { return (float)h; }
    // |y| <= 127 (a NaN: some number). At 1.5 * 2^23 fp32 counts in ones: the sum rounds y to the nearest
    // even integer and its lowest byte is that in two's complement.
    static __device__ __forceinline__ uint32_t whole(float y) {
        return __float_as_uint(y + 12582912.0f);
    }
    static __device__ __forceinline__ uint8_t narrow1(float y) { return (uint8_t)whole(y); }
    static __device__ __forceinline__ void widen(uint32_t w, float (&y)[4]) {
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = (float)(int8_t)(w >> (8 * i));
    }
    static __device__ __forceinline__ uint32_t narrow(const float (&y)[4]) {
        return __builtin_amdgcn_perm(whole(y[1]), whole(y[0]), 0x0c0c0400u) |
               __builtin_amdgcn_perm(whole(y[3]), whole(y[2]), 0x04000c0cu);
    }
};

// The smallest power of two S >= 2^-126 with amax <= QMAX * S; 0 for 0, NaN for inf and NaN. amax is
// a magnitude's bit pattern, whose order as an unsigned integer is that of the magnitudes with
// inf and NaN last: maxima taken on patterns lose no NaN.
template <typename T>
__device__ __forceinline__ float scale_for(uint32_t amax) {
    if (amax == 0) return 0.0f;
    if (amax >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    int x;
    const float f = frexpf(__uint_as_float(amax), &x);
    const int e = max(x - Elem8<T>::EXP + (f > Elem8<T>::TOP ? 1 : 0), -126);
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// A stored scale as the write takes it: itself if it is a power of two from 2^-126 on or 0, the next one
// otherwise (scales that a caller chose), NaN if it is negative, inf, NaN or beyond 2^127.
__device__ __forceinline__ float pow2_scale(float s) {
    const uint32_t u = __float_as_uint(s + 0.0f);  // (-0 as 0)
    if (u > 0x7f000000u) return __uint_as_float(0x7fc00000u);  // (negative ones too: the sign bit)
    if (u == 0) return 0.0f;
    const uint32_t up = (u + 0x007fffffu) & 0xff800000u;
    return __uint_as_float(up < 0x00800000u ? 0x00800000u : up);
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t x) {  // of magnitudes: below 2^31
    return (uint32_t)wave_max_i32((int)x);
}

// The larger of two scales; NaN if either is.
__device__ __forceinline__ float max_scale(float a, float b) { return vmax(a, b); }

// Whether a copy of a block's values in f16 could lose what f16 has for them: its largest possible
// one, QMAX S, is beyond 65,504, or so small that f16's spacing near zero, 2^-24, rounds them by more than
// 2^-12 of QMAX S / 2 (a scale that the write chose is used to half at least). No for 0 and NaN.
template <typename T>
__device__ __forceinline__ bool beyond_f16(float s) {
    const float top = s * Elem8<T>::QMAX;
    return top > 65504.0f || (top > 0.0f && top < 0x1p-12f);
}

// What x is multiplied by for x / S (0 where the block has no scale).
__device__ __forceinline__ float inv_scale(float s) { return s > 0.0f ? 1.0f / s : 0.0f; }

// The last i < n with first(i) <= x, first rising and first(0) <= x: 64 samples a step, one a lane.
template <typename F>
__device__ __forceinline__ int wave_find_last(int n, int64_t x, F first) {
    const int lane = threadIdx.x & 63;
    int lo = 0, len = n;
    while (len > 1) {
        const int step = (len + 63) / 64;
        const int i = lo + lane * step;
        const bool le = lane * step < len && (lane == 0 || first(i) <= x);
        const int k = __popcll(__ballot(le)) - 1;
        const int end = lo + len;
        lo += k * step;
        len = min(step, end - lo);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

}  // namespace flour
