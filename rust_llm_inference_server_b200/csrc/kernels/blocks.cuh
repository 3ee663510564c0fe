// Values into e4m3 with a float32 scale for each block of 128: what the kernels that do so share.
//
//   a = max(amax of the block, 2^-100),  scale = a / 448,  code = e4m3 nearest to 448 x / a  (448 is the largest e4m3)
//
// The quotient is rounded once to float32 and once to e4m3: a quotient of two bfloat16 numbers often lies right between two e4m3, and a product with a
// rounded reciprocal would take one or the other by chance (2 to 3 of 1,000 codes).  2^-100 keeps a block of zeros, or of nothing that counts, free of
// divisions by zero.  A block that holds a NaN has NaN as its scale and codes; one that holds an infinity an infinite scale and, there, a NaN.
#pragma once
#include "common.cuh"
#include <cuda_fp8.h>

namespace {
constexpr int QB = 128;                              // a block's edge
constexpr unsigned LEAST_BITS = 0x0D800000u;         // 2^-100
constexpr unsigned LARGE_BITS = 0x71800000u;         // 2^100

// What a block's values are turned to codes with: x -> (x * mul) / div.  (Above 2^100 both by 2^-20 less, so that 448 x stays finite.)
struct Coding {
    float mul, div, scale;
};
__device__ __forceinline__ Coding coding_of(unsigned amax_bits) {
    const unsigned bits = max(amax_bits, LEAST_BITS);        // (a NaN's bits are above all others)
    const float a = __uint_as_float(bits);
    Coding c;
    c.mul = bits > LARGE_BITS ? 448.f * 0x1p-20f : 448.f;
    c.div = bits > LARGE_BITS ? a * 0x1p-20f : a;
    c.scale = a / 448.f;
    return c;
}
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t codes4(const float* v, const Coding& c) {
    const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(v[0] * c.mul, c.div), __fdiv_rn(v[1] * c.mul, c.div)), __NV_SATFINITE, __NV_E4M3);
    const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(v[2] * c.mul, c.div), __fdiv_rn(v[3] * c.mul, c.div)), __NV_SATFINITE, __NV_E4M3);
    return (uint32_t)lo | ((uint32_t)hi << 16);
}

// Eight consecutive values of a row of K, zeros past its end.
template <typename T, bool VEC> __device__ __forceinline__ void load8(const T* row, int k, int K, float (&v)[8]) {
    if (VEC && k + 8 <= K) {
#pragma unroll
        for (int i = 0; i < 8; i += Vec16<T>::N) load16<T>(row + k + i, v + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = k + i < K ? to_f<T>(row[k + i]) : 0.f;
    }
}
// Their codes, into a row that starts at a multiple of 16 bytes and has room for K rounded up to 16.
__device__ __forceinline__ void store8(unsigned char* row, int k, int K, const float (&v)[8], const Coding& c) {
    if (k < K) *reinterpret_cast<uint2*>(row + k) = make_uint2(codes4(v, c), codes4(v + 4, c));
}
}  // namespace
