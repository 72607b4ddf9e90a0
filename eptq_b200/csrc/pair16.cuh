// Two neighbouring fp16 or bf16 values in one 32-bit word, to and from fp32 (round to nearest even).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace eptq {

// Larger and smaller of two pairs of unsigned 16-bit numbers, which order 16-bit floats that are not negative as well.
__device__ __forceinline__ unsigned max2(unsigned a, unsigned b) {
    asm("max.u16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
    return a;
}
__device__ __forceinline__ unsigned min2(unsigned a, unsigned b) {
    asm("min.u16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
    return a;
}

template <typename T>
struct Pair16;

template <>
struct Pair16<__half> {
    static __device__ __forceinline__ float2 unpack(unsigned w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ unsigned pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const unsigned*>(&h);
    }
    // Weights a, b >= 0 as the sum of two 16-bit values each, the first cut off behind its last bit.  Neither is negative, and the second
    // is not zero where the first is not: an infinite factor of both stays infinite.
    static __device__ __forceinline__ uint2 split(float a, float b) {
        const float x = __uint_as_float(__float_as_uint(a) & 0xffffe000u), y = __uint_as_float(__float_as_uint(b) & 0xffffe000u);
        const unsigned high = pack(x, y);
        return make_uint2(high, max2(pack(a - x, b - y), min2(high, 0x00010001u)));      // 2^-24, the least above zero
    }
    // 0 * w + acc: NaN where w is not finite.
    static __device__ __forceinline__ unsigned zero_times(unsigned w, unsigned acc) {
        asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(w), "r"(0u));
        return acc;
    }
};

template <>
struct Pair16<__nv_bfloat16> {
    static __device__ __forceinline__ float2 unpack(unsigned w) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w)); }
    static __device__ __forceinline__ unsigned pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const unsigned*>(&h);
    }
    static __device__ __forceinline__ uint2 split(float a, float b) {
        const unsigned i = __float_as_uint(a), k = __float_as_uint(b), high = __byte_perm(i, k, 0x7632);
        const float x = __uint_as_float(i & 0xffff0000u), y = __uint_as_float(k & 0xffff0000u);
        return make_uint2(high, max2(pack(a - x, b - y), min2(high, 0x00800080u)));      // 2^-126, the least normal value
    }
    static __device__ __forceinline__ unsigned zero_times(unsigned w, unsigned acc) {
        asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(w), "r"(0u));
        return acc;
    }
};

}  // namespace eptq
