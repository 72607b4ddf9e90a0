// Two neighbouring fp16 or bf16 values in one 32-bit word, to and from fp32 (round to nearest even).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace eptq {

template <typename T>
struct Pair16;

template <>
struct Pair16<__half> {
    static __device__ __forceinline__ float2 unpack(unsigned w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ unsigned pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const unsigned*>(&h);
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
    static __device__ __forceinline__ unsigned zero_times(unsigned w, unsigned acc) {
        asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(w), "r"(0u));
        return acc;
    }
};

}  // namespace eptq
