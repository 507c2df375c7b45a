// Shared pieces of the products whose rows choose their own weights (lora.cu, moe.cu): two-byte element
// conversions and the host's pointer checks.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gemm_sm100.cuh"

namespace b200 {

struct Bf16 {
    static constexpr int kCode = B200_BF16;
    static constexpr float kMax = 3.38953139e38f;
    static constexpr bool kScaled = false;   // whether a pair (see split) loses what a float holds unless it is scaled
    static constexpr float kPairMin = 0x1p-100f;   // from here on a pair errs by 2^-16 at most, and what is smaller by 2^-17 of this
    // two packed elements -> two floats; element 0 sits in the low half
    __device__ static __forceinline__ float2 unpack(uint32_t v) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
    __device__ static __forceinline__ uint16_t round(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
    // v as the sum of two elements. The first one saturates, so that infinities (and what the pair cannot hold) arrive as
    // an infinity in the second one, not as infinity minus infinity.
    __device__ static __forceinline__ void split(float v, uint16_t &hi, uint16_t &lo) {
        hi = round(fminf(fmaxf(v, -kMax), kMax));
        lo = round(v - __uint_as_float(static_cast<uint32_t>(hi) << 16));
    }
};

struct Fp16 {
    static constexpr int kCode = B200_F16;
    static constexpr float kMax = 65504.0f;
    static constexpr bool kScaled = true;
    static constexpr float kPairMin = 0x1p-8f;     // 2^-25 / 2^-17
    __device__ static __forceinline__ float2 unpack(uint32_t v) {
        return __half22float2(*reinterpret_cast<const __half2 *>(&v));
    }
    __device__ static __forceinline__ uint16_t round(float v) { return __half_as_ushort(__float2half_rn(v)); }
    __device__ static __forceinline__ void split(float v, uint16_t &hi, uint16_t &lo) {
        hi = round(fminf(fmaxf(v, -kMax), kMax));
        lo = round(v - __half2float(__ushort_as_half(hi)));
    }
};

// fp32 dot product of eight packed elements on both sides, added to acc
template <typename T>
__device__ __forceinline__ float dot8(const uint4 &a, const uint4 &b, float acc) {
    const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = T::unpack(av[i]), y = T::unpack(bv[i]);
        acc = fmaf(x.x, y.x, acc);
        acc = fmaf(x.y, y.y, acc);
    }
    return acc;
}

// d += a * b on two pairs at once
__device__ __forceinline__ float2 fma2(const float2 &a, const float2 &b, const float2 &d) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t &>(r))
        : "l"(reinterpret_cast<const uint64_t &>(a)), "l"(reinterpret_cast<const uint64_t &>(b)), "l"(reinterpret_cast<const uint64_t &>(d)));
    return r;
}

// 32 bytes at a 32-byte aligned address
__device__ __forceinline__ void ld_32(const void *p, uint4 &a, uint4 &b) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
                 : "l"(p));
}

template <typename T>
__device__ __forceinline__ void store_four(uint16_t *p, const float4 &v) {   // 8-byte aligned
    *reinterpret_cast<uint2 *>(p) = make_uint2(T::round(v.x) | static_cast<uint32_t>(T::round(v.y)) << 16, T::round(v.z) | static_cast<uint32_t>(T::round(v.w)) << 16);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

inline bool misaligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

// whether [a, a + na) and [b, b + nb) share a byte
inline bool overlap(const void *a, int64_t na, const void *b, int64_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + static_cast<uintptr_t>(nb) && y < x + static_cast<uintptr_t>(na);
}

}  // namespace b200
