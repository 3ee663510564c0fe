// Values into e4m3 with a float32 scale for each block of 128: what the kernels that do so share.
//
//   a = max(amax of the block, 2^-100),  scale = a / 448,  code = e4m3 nearest to 448 x / a  (448 is the largest e4m3)
//
// 2^-100 keeps a block of zeros, or of nothing that counts, free of divisions by zero.  A block that holds a NaN has NaN as its scale and codes; one that holds an
// infinity an infinite scale and, there, a NaN.
//
// The quotient of two bfloat16 numbers often lies right between two e4m3 (2 to 3 of 1,000 codes), and p = x * fl(448 / a) is off by up to 2^-23 of it, to
// either side: p alone would take one code or the other by chance.  A point between two codes has five significant bits at most, and a quotient 7 X / A of
// integers of eight bits that is none of them is at least 2^-13 of it away.  So p rounded to 16 bits (off by 2^-17 at most) is that point where the quotient is,
// and stays on its side where it is not: for bfloat16 its e4m3 is the quotient's.  A float32 x may come closer: where the 16 bits may be such a point (one
// of 4,096), the sign of 448 x - p a says on which side of them the quotient lies (to_its_side).  (As divisions, all of them, the
// codes of 2,048 rows of 14,336 took 5 us more; two values at a time in an instruction 1.4 less than one by one: 16.6.)
#pragma once
#include "common.cuh"
#include <cuda_fp8.h>

namespace {
constexpr int QB = 128;                              // a block's edge
constexpr unsigned LEAST_BITS = 0x0D800000u;         // 2^-100
constexpr unsigned LARGE_BITS = 0x71800000u;         // 2^100
constexpr unsigned SMALL_BITS = 0x3c800000u;         // 2^-6

// What a block's values are turned to codes with.
struct Coding {
    float a, factor, scale;
};
__device__ __forceinline__ float least_of(unsigned amax_bits) { return __uint_as_float(max(amax_bits, LEAST_BITS)); }       // (a NaN's bits are above all others)
__device__ __forceinline__ Coding coding_of(unsigned amax_bits) {
    Coding c;
    c.a = least_of(amax_bits);
    c.factor = 448.f / c.a;
    c.scale = c.a / 448.f;
    return c;
}
// Two floats at a time, which takes as many instructions as one.
__device__ __forceinline__ unsigned long long pair_of(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ unsigned long long mul_pair(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long sub_pair(unsigned long long a, unsigned long long b) {        // a - b: b times -1 and a, rounded once
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(b), "l"(0xbf800000bf800000ull), "l"(a));
    return r;
}
// x * factor rounded to 16 significant bits (T. J. Dekker's splitting; a NaN stays one).
__device__ __forceinline__ void product_of_16_bits(float x0, float x1, unsigned long long factors, float& q0, float& q1) {
    const unsigned long long p = mul_pair(pair_of(x0, x1), factors), c = mul_pair(p, 0x4380800043808000ull /* 257 */), q = sub_pair(c, sub_pair(c, p));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(q0), "=f"(q1) : "l"(q));
}
__device__ __forceinline__ uint32_t pack_codes(const float* q) {
    const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3);
    const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(q[2], q[3]), __NV_SATFINITE, __NV_E4M3);
    return (uint32_t)lo | ((uint32_t)hi << 16);
}
// Eight consecutive values of a row of K as they lie in memory, zeros past the row's end.
template <typename T> struct Eight {
    static constexpr int WORDS = 2 * (int)sizeof(T);
    uint32_t w[WORDS];
};
template <typename T> __device__ __forceinline__ Eight<T> nothing8() {
    Eight<T> e;
#pragma unroll
    for (int i = 0; i < Eight<T>::WORDS; ++i) e.w[i] = 0u;
    return e;
}
template <typename T, bool VEC> __device__ __forceinline__ Eight<T> load8(const T* row, int k, int K) {
    Eight<T> e = nothing8<T>();
    if (VEC && k + 8 <= K) {
#pragma unroll
        for (int i = 0; i < Eight<T>::WORDS; i += 4) *reinterpret_cast<uint4*>(e.w + i) = *reinterpret_cast<const uint4*>(row + k + i * 4 / (int)sizeof(T));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (k + i < K) {
                if constexpr (sizeof(T) == 4) e.w[i] = reinterpret_cast<const uint32_t*>(row)[k + i];
                else e.w[i >> 1] |= (uint32_t) reinterpret_cast<const unsigned short*>(row)[k + i] << (i & 1) * 16;
            }
    }
    return e;
}
// The bits of the largest of their absolute values as a float (a NaN's are above all others).
template <typename T> __device__ __forceinline__ unsigned amax_bits(const Eight<T>& e) {
    unsigned m = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, e.w[i] & 0x7fffffffu);
        return m;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __vmaxu2(m, e.w[i] & 0x7fff7fffu);
        return max(m << 16, m & 0xffff0000u);
    }
}
template <typename T> __device__ __forceinline__ void widen(const Eight<T>& e, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(e.w[i]);
        else v[i] = __uint_as_float((i & 1) ? e.w[i >> 1] & 0xffff0000u : e.w[i >> 1] << 16);
    }
}
// q, to which p was rounded, goes a unit to the side of it on which 448 x / a lies, so that a q between two e4m3 takes the right one of them (any other stays between the
// same two).  448 x - q a is formed exactly for a q of five bits: each product is a float32 and what its rounding left (x and a have 24 bits, 448 three), the products lie
// next to each other, so their difference and that of the rests are numbers of a few bits.  `by` is 448, and beside an a above 2^100 both are 2^-20 of it.
__device__ __forceinline__ float to_its_side(float q, float x, float by, float a) {
    const float p = __fmul_rn(x, by), r = __fmul_rn(q, a);
    const float d = __fadd_rn(__fsub_rn(p, r), __fsub_rn(__fmaf_rn(x, by, -p), __fmaf_rn(q, a, -r)));
    const int unit = (__float_as_int(d) ^ __float_as_int(q)) >> 31 | 1;
    return __int_as_float(__float_as_int(q) + (fabsf(d) > 0.f ? unit : 0));         // (a NaN stays one)
}
template <typename T> __device__ __forceinline__ uint2 codes8(const Eight<T>& e, const Coding& c) {
    float v[8], q[8];
    widen(e, v);
    const unsigned long long factors = pair_of(c.factor, c.factor);
#pragma unroll
    for (int i = 0; i < 8; i += 2) product_of_16_bits(v[i], v[i + 1], factors, q[i], q[i + 1]);
    if (sizeof(T) == 4) {
        // a middle of two e4m3 has a one as its fifth bit and zeros behind it, or lies among those below 2^-6
        unsigned middle = ~0u, small = ~0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            middle = min(middle, (__float_as_uint(q[i]) & 0xfffffu) ^ 0x80000u);
            small = min(small, 2u * __float_as_uint(q[i]) - 2u);            // (a zero is none of them)
        }
        if (middle == 0u || small < 2u * SMALL_BITS - 2u) {
            const bool large = __float_as_uint(c.a) > LARGE_BITS;
            const float by = large ? 448.f * 0x1p-20f : 448.f, a = large ? c.a * 0x1p-20f : c.a;
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = to_its_side(q[i], v[i], by, a);
        }
    }
    return make_uint2(pack_codes(q), pack_codes(q + 4));
}

// Their codes, into a row that starts at a multiple of 16 bytes.
template <typename T> __device__ __forceinline__ void store8(unsigned char* row, int k, int K, const Eight<T>& e, const Coding& c) {
    if (k >= K) return;
    const uint2 v = codes8<T>(e, c);
    if (k + 8 <= K) {
        *reinterpret_cast<uint2*>(row + k) = v;
    } else {
        uint32_t w = v.x;
        row += k;
        int left = K - k;
        if (left >= 4) {
            *reinterpret_cast<uint32_t*>(row) = w;
            w = v.y, row += 4, left -= 4;
        }
#pragma unroll 1
        for (; left > 0; --left, ++row, w >>= 8) *row = (unsigned char)w;
    }
}
}  // namespace
