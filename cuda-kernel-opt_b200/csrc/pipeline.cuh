// What the warp-specialised kernels of lora.cu and moe.cu share: bounded waits that leave a record in the library's status
// word, and the few PTX forms that the GEMM does not need.
#pragma once

#include "../../include/b200_gemm.h"
#include "ptx_sm100.cuh"

namespace b200 {

// Where a bounded wait reports: the library's status record {code, block, wait id, detail}, a block-wide abort flag in
// shared memory that makes every role leave its loop, the budget in SM cycles.
struct WaitCtx {
    int *status;
    volatile int *abort_flag;
    long long budget;
};

static __device__ __noinline__ bool wait_slowly(uint32_t bar, uint32_t parity, const WaitCtx c, int wait_id) {
    const long long t0 = clock64();
    uint32_t spins = 0;
    for (;;) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((++spins & 31u) == 0) {
            if (*c.abort_flag) return false;
            if (clock64() - t0 > c.budget) {
                *c.abort_flag = 1;
                if (atomicCAS(&c.status[0], 0, B200_DEVICE_TIMEOUT) == 0) {
                    c.status[1] = static_cast<int>(blockIdx.x);
                    c.status[2] = wait_id;
                    c.status[3] = static_cast<int>(parity);
                }
                __threadfence();
                return false;
            }
        }
    }
}

// All lanes of a converged warp wait for the phase; false in every lane when the budget ran out here or elsewhere in the block.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, const WaitCtx &c, int wait_id) {
    bool ok = mbar_try_wait(bar, parity);
    if (__all_sync(0xffffffffu, ok)) return true;
    if (!ok) ok = wait_slowly(bar, parity, c, wait_id);
    return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ void mbar_arrive_many(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

// A bit set in a word of another CTA's shared memory (address from mapa_shared).
__device__ __forceinline__ void red_or_cluster(uint32_t cluster_addr, uint32_t bits) {
    asm volatile("red.shared::cluster.or.b32 [%0], %1;" ::"r"(cluster_addr), "r"(bits) : "memory");
}

// A word of another CTA's shared memory (address from mapa_shared).
__device__ __forceinline__ void st_cluster(uint32_t cluster_addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}

// Completes `bar` when the MMAs issued before have; for a pair (the two CTAs of a cluster) the barrier at this place in both.
template <int CG>
__device__ __forceinline__ void commit_cta(uint32_t bar) {
    if constexpr (CG == 1)
        umma_commit<1>(bar);
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                     "h"(static_cast<uint16_t>(3))
                     : "memory");
}

// Contiguous bytes global -> shared (both 16-byte aligned, a multiple of 16), counted by `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

// Contiguous bytes (16-byte aligned, a multiple of 16) on their way to the L2.
__device__ __forceinline__ void prefetch_l2(const void *src, uint32_t bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}

// 16 bytes global -> shared without passing through registers (L2 only); complete after cp_async_wait_all.
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ void st_shared_v4(uint32_t dst, const uint4 &v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

__device__ __forceinline__ void st_shared_v2(uint32_t dst, const uint2 &v) {
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(dst), "r"(v.x), "r"(v.y) : "memory");
}

// Byte offset of 16-byte chunk `chunk` of row `row` in a K block of 128-byte rows as TMA writes it with the 128-byte
// swizzle (the chunk index is exclusive-ored with the row's place in its group of eight).
__device__ __forceinline__ uint32_t swizzled(int row, int chunk) {
    return static_cast<uint32_t>(row * 128 + ((chunk ^ (row & 7)) << 4));
}

// How the K blocks of `units` tiles are dealt out: CTA c takes blocks
// [c * len, (c + 1) * len) of all of them in a row, wherever tiles begin and end. len is
// large enough for a tile to touch at most `parts` CTAs.
struct Cut {
    int kblocks, total, len;
    __device__ __forceinline__ Cut(int units, int kblocks_, int sms, int parts) : kblocks(kblocks_), total(units * kblocks_) {
        len = max(max((total + sms - 1) / sms, (kblocks - 1 + parts - 2) / (parts - 1)), 1);
    }
    __device__ __forceinline__ int first_cta(int unit) const { return unit * kblocks / len; }
    __device__ __forceinline__ int num_parts(int unit) const { return ((unit + 1) * kblocks - 1) / len - first_cta(unit) + 1; }
};

}  // namespace b200
