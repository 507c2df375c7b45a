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
    // two packed elements -> two floats; element 0 sits in the low half
    __device__ static __forceinline__ float2 unpack(uint32_t v) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
    __device__ static __forceinline__ uint16_t round(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
    // v as the sum of two elements. The first one saturates, so that infinities (and what the pair cannot hold) arrive as
    // an infinity in the second one, not as infinity minus infinity.
    __device__ static __forceinline__ void split(float v, uint16_t &hi, uint16_t &lo) {
        hi = round(fminf(fmaxf(v, -3.38953139e38f), 3.38953139e38f));
        lo = round(v - __uint_as_float(static_cast<uint32_t>(hi) << 16));
    }
};

struct Fp16 {
    static constexpr int kCode = B200_F16;
    __device__ static __forceinline__ float2 unpack(uint32_t v) {
        return __half22float2(*reinterpret_cast<const __half2 *>(&v));
    }
    __device__ static __forceinline__ uint16_t round(float v) { return __half_as_ushort(__float2half_rn(v)); }
    __device__ static __forceinline__ void split(float v, uint16_t &hi, uint16_t &lo) {
        hi = round(fminf(fmaxf(v, -65504.0f), 65504.0f));
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

// acc (16 x 8, fp32) += A (16 x 16) * B (16 x 8); lane = 4 * row + quad holds rows row and row + 8 of A, column row of B
template <typename T>
__device__ __forceinline__ void mma_16816(float (&acc)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (T::kCode == B200_BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(acc[0]), "+f"(acc[1]), "+f"(acc[2]), "+f"(acc[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(acc[0]), "+f"(acc[1]), "+f"(acc[2]), "+f"(acc[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 32 bytes at a 32-byte aligned address
__device__ __forceinline__ void ld_32(const void *p, uint4 &a, uint4 &b) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
                 : "l"(p));
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
