// A projection shared by all rows with low-rank adapters of many requests beside it:
//
//     D[i] = A[i] B^T + scale[s] (A[i] lora_a[s]^T) lora_b[s]^T,   s = row_adapter[i]
//
//   lora_shrink_*_kernel  u[i] = scale[s] (A[i] lora_a[s]^T), fp32, to the workspace
//   lora_product_kernel   the shared product on tcgen05 with B's rows on the 128-row side (D is computed transposed: a lane of
//                         tensor memory is a column of D, a column of tensor memory a row). Eight warps beside the
//                         pipeline compute (u lora_b[s]^T)[i][n] in fp32 while the tensor core is busy and hand it to
//                         the draining warps in pieces of 8 rows x 128 columns, which add it before the one rounding.
//
// The adapters' second product stays off the tensor core: a zero that stands for "not this row's adapter" does not mask an
// infinity or a NaN among an adapter's weights, so a row would see other requests' adapters; and a decode step in
// which every row has another adapter would feed it one useful row at a time. The fp32 units have the time: rows x N x rank
// multiply-adds against rows x N x K on the tensor core.
//
// Two forms of the product kernel, by the number of rows:
//   one CTA, up to 256 rows    B is read once and bounds it. The K blocks of all tiles (128 columns of D, all rows) are cut
//                              into one equal stretch per CTA (Cut); a tile that spans several CTAs leaves parts in the
//                              workspace, and the last of its CTAs to finish adds them in ascending order. No CTA waits
//                              for another.
//   CTA pair, more rows        256 x 256 tiles, the tensor core bounds it: whole tiles, dealt out in waves that share
//                              operand panels in L2, with K walked to and fro.
// The shrink kernel lets the product start at once; only the warps that need u wait for it.
#include <cuda_runtime.h>

#include "../../include/b200_gemm.h"
#include "gemm_sm100.cuh"
#include "pipeline.cuh"
#include "routed.cuh"

namespace b200 {
namespace {

constexpr int kLoraStages = 12;
constexpr int kDeltaWarps = 8;
constexpr int kLoraThreads = (2 + 4 + kDeltaWarps + 1) * 32;
constexpr int kChunkRows = 8;                              // rows of D in a piece of the adapters' product
constexpr int kChunks = 4;                                 // pieces on their way to the draining warps
constexpr int kAhead = 8;                                  // pieces whose adapters and u are on their way to the delta warps
constexpr int kChunkBytes = kChunkRows * 128 * 4;
constexpr int kOneCtaRows = 64;                            // most rows of the one-CTA form
constexpr int kFewRows = 256;                              // most rows that one tile takes
constexpr int kDotRows = 128;                              // most rows of the dot-product form of the shrink kernel
constexpr int kLoraBars = 2 * kLoraStages + 4 + 2 * kChunks + 2 * kAhead;
constexpr int kMaxLoraParts = 16;
constexpr int kMaxCtas = 256;
constexpr int kLoraGridSms = 148;                          // what the workspace is sized for
constexpr int kGroupRows = 16;                             // pair: row blocks that a wave walks together

struct alignas(64) LoraArgs {
    CUtensorMap map_b, map_a;      // B as {K, N}, A as {K, M}
    const uint16_t *A, *lora_a, *lora_b;
    uint16_t *D;
    const float *scale;
    const int *row_adapter;
    float *u;                      // [M][rank]
    float *o;                      // [part][M][N]: sums of tiles that span CTAs
    int *arrived;                  // per CTA: the warps that are done with the tile it began last
    int M, N, K, rank;
    int num_adapters;
    int wide_b;                    // rows of lora_b are whole 32-byte sectors
    int parts, sms;
    int rows;                      // of a tile: columns of an accumulator
    int a_bytes, stages, off_delta, off_u, off_ids, off_bars, off_misc;
    int tmem_cols;
    uint32_t idesc;
    int *status;
    long long budget;
};

// ---------------------------------------------------------------------------------------------- first product

// Few rows: a block takes four ranks of a row, its warps an eighth of K each. Bound by reading the adapters once (2 * rank * K bytes
// per adapter in use); a block has 40 loads of 16 bytes per lane in flight at K = 8192.
template <typename T>
__global__ void __launch_bounds__(256) lora_shrink_dot_kernel(const __grid_constant__ LoraArgs g) {
    __shared__ float sums[8][4];
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (blockIdx.x == 0) g.arrived[threadIdx.x] = 0;       // kMaxCtas of them
    const int quads = g.rank / 4;
    for (int64_t at = blockIdx.x; at < static_cast<int64_t>(g.M) * quads; at += gridDim.x) {
        const int m = static_cast<int>(at / quads), r0 = static_cast<int>(at - static_cast<int64_t>(m) * quads) * 4;
        const int s = __ldca(g.row_adapter + m);
        if (static_cast<unsigned>(s) >= static_cast<unsigned>(g.num_adapters)) continue;
        const uint16_t *const x = g.A + static_cast<int64_t>(m) * g.K;
        const uint16_t *const a = g.lora_a + (static_cast<int64_t>(s) * g.rank + r0) * g.K;
        float acc[4] = {};
#pragma unroll 4
        for (int k = threadIdx.x * 8; k < g.K; k += 2048) {
            const uint4 xv = __ldcg(reinterpret_cast<const uint4 *>(x + k));
            uint4 av[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) av[r] = __ldcg(reinterpret_cast<const uint4 *>(a + static_cast<int64_t>(r) * g.K + k));
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r] = dot8<T>(xv, av[r], acc[r]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] = warp_sum(acc[r]);
        __syncthreads();                                   // the sums of the turn before have been read
        if (lane == 0)
#pragma unroll
            for (int r = 0; r < 4; ++r) sums[warp][r] = acc[r];
        __syncthreads();
        if (threadIdx.x < 4) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) v += sums[w][threadIdx.x];
            g.u[static_cast<int64_t>(m) * g.rank + r0 + threadIdx.x] = (g.scale ? g.scale[s] : 1.0f) * v;
        }
    }
}

// Many rows: a block takes 16 rows and 8 * NT ranks, its warps an eighth of the K steps of 32 each, on mma.sync (the rows of an
// adapter are few and any; a 128-row tile of tcgen05 would be mostly other adapters' rows). One pass over K per adapter among
// the 16 rows; only its own rows keep the result. Within a step the four lanes of a quad hold 8 neighbouring elements each, of both
// operands alike: the order of K within a step is free.
template <typename T, int NT>
__global__ void __launch_bounds__(256) lora_shrink_mma_kernel(const __grid_constant__ LoraArgs g) {
    __shared__ float sums[8][16][8 * NT];
    __shared__ int ids[16];
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = lane >> 2, quad = lane & 3;
    if (blockIdx.x == 0 && blockIdx.y == 0) g.arrived[threadIdx.x] = 0;
    const int m0 = blockIdx.x * 16, r0 = blockIdx.y * 8 * NT;
    if (threadIdx.x < 16) {
        const int s = m0 + threadIdx.x < g.M ? __ldca(g.row_adapter + m0 + threadIdx.x) : -1;
        ids[threadIdx.x] = static_cast<unsigned>(s) < static_cast<unsigned>(g.num_adapters) ? s : -1;
    }
    __syncthreads();
    const uint16_t *const x0 = g.A + static_cast<int64_t>(m0 + row) * g.K + quad * 8;
    const bool in0 = m0 + row < g.M, in1 = m0 + row + 8 < g.M;
    for (int first = 0; first < 16; ++first) {
        const int s = ids[first];
        bool seen = s < 0;
        for (int i = 0; i < first; ++i) seen = seen || ids[i] == s;
        if (seen) continue;
        float acc[NT][4] = {};
        const uint16_t *const a0 = g.lora_a + (static_cast<int64_t>(s) * g.rank + r0 + row) * g.K + quad * 8;
#pragma unroll 2
        for (int k = warp * 32; k < g.K; k += 256) {
            const uint4 zero = make_uint4(0, 0, 0, 0);
            const bool in = k + quad * 8 < g.K;
            const uint4 p = in && in0 ? __ldcg(reinterpret_cast<const uint4 *>(x0 + k)) : zero;
            const uint4 q = in && in1 ? __ldcg(reinterpret_cast<const uint4 *>(x0 + 8 * static_cast<int64_t>(g.K) + k)) : zero;
            uint4 b[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t)
                b[t] = in && r0 + 8 * t + row < g.rank ? __ldcg(reinterpret_cast<const uint4 *>(a0 + static_cast<int64_t>(8 * t) * g.K + k)) : zero;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                mma_16816<T>(acc[t], p.x, q.x, p.y, q.y, b[t].x, b[t].y);
                mma_16816<T>(acc[t], p.z, q.z, p.w, q.w, b[t].z, b[t].w);
            }
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            *reinterpret_cast<float2 *>(&sums[warp][row][8 * t + 2 * quad]) = make_float2(acc[t][0], acc[t][1]);
            *reinterpret_cast<float2 *>(&sums[warp][row + 8][8 * t + 2 * quad]) = make_float2(acc[t][2], acc[t][3]);
        }
        __syncthreads();
        const float scale = g.scale ? g.scale[s] : 1.0f;
        for (int i = threadIdx.x; i < 16 * 8 * NT; i += 256) {
            const int m = i / (8 * NT), r = i % (8 * NT);
            if (ids[m] != s || r0 + r >= g.rank) continue;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) v += sums[w][m][r];
            g.u[static_cast<int64_t>(m0 + m) * g.rank + r0 + r] = scale * v;
        }
    }
}

// ---------------------------------------------------------------------------------------------- shared product

// K blocks [kb0, kb1) of the tile at row m0 and 128-column (pair: 256-column) tile `tile`, as part `part` of `parts`.
struct LoraSegment {
    int tile, m0, kb0, kb1, part, parts;
};

template <int CG, bool WAVES>
struct LoraWalker {
    int q, end, step, tiles_n, row_blocks, kblocks, rows, group;   // group: a CTA or a pair
    Cut cut;
    __device__ __forceinline__ LoraWalker(const LoraArgs &g)
        : tiles_n((g.N + 128 * CG - 1) / (128 * CG)), row_blocks((g.M + g.rows - 1) / g.rows), kblocks((g.K + 63) / 64), rows(g.rows),
          group(blockIdx.x / CG), cut(WAVES ? 0 : tiles_n, kblocks, gridDim.x / CG, g.parts) {
        if (WAVES) {
            q = group;
            step = gridDim.x / CG;
            end = tiles_n * row_blocks;
        } else {
            q = static_cast<int>(min(static_cast<long long>(group) * cut.len, static_cast<long long>(cut.total)));
            end = min(q + cut.len, cut.total);
        }
    }
    __device__ __forceinline__ bool next(LoraSegment &s) {
        if (q >= end) return false;
        if (!WAVES) {
            s.tile = q / kblocks;
            s.m0 = 0;
            s.kb0 = q - s.tile * kblocks;
            s.kb1 = min(kblocks, s.kb0 + end - q);
            s.part = group - cut.first_cta(s.tile);
            s.parts = cut.num_parts(s.tile);
            q += s.kb1 - s.kb0;
        } else {
            const int in_group = kGroupRows * tiles_n, first = q / in_group * kGroupRows;
            const int height = min(row_blocks - first, kGroupRows), i = q % in_group;
            s.m0 = (first + i % height) * rows;
            s.tile = i / height;
            s.kb0 = 0;
            s.kb1 = kblocks;
            s.part = 0;
            s.parts = 1;
            q += step;
        }
        return true;
    }
};

// One column n of D, four rows: sum over the ranks of u[j][r] * lora_b[s[j]][n][r], fp32, two ranks at a time. u lies in shared memory.
// Where the four rows have one adapter, its ranks are kept as floats from one call to the next (h.w, h.s: whose they
// are; up to 64 of them): a prompt's rows cost 32 packed multiply-adds each. Else every row's are read, 32 ranks at a
// time: 16 loads of 16 bytes in flight per lane, which is what reading each adapter once from memory takes.
struct Held {
    float2 w[32];
    int s;
};

template <typename T>
__device__ __forceinline__ void adapters_product(const LoraArgs &g, Held &h, const int (&s)[4], const float *u, int n, float (&d)[4]) {
    const int rank = g.rank;
    if (s[0] >= 0 && s[0] == s[1] && s[0] == s[2] && s[0] == s[3] && rank <= 64) {
        if (h.s != s[0]) {
            const uint4 *const b = reinterpret_cast<const uint4 *>(g.lora_b + (static_cast<int64_t>(s[0]) * g.N + n) * rank);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint4 v = i * 8 < rank ? __ldcg(b + i) : make_uint4(0, 0, 0, 0);
                h.w[4 * i] = T::unpack(v.x), h.w[4 * i + 1] = T::unpack(v.y), h.w[4 * i + 2] = T::unpack(v.z), h.w[4 * i + 3] = T::unpack(v.w);
            }
            h.s = s[0];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float4 *const uj = reinterpret_cast<const float4 *>(u + j * rank);
            float2 a = make_float2(0.0f, 0.0f), b = a;
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                if (i * 4 >= rank) break;
                const float4 f = uj[i], e = uj[i + 1];
                a = fma2(make_float2(f.x, f.y), h.w[2 * i], a);
                b = fma2(make_float2(f.z, f.w), h.w[2 * i + 1], b);
                a = fma2(make_float2(e.x, e.y), h.w[2 * i + 2], a);
                b = fma2(make_float2(e.z, e.w), h.w[2 * i + 3], b);
            }
            d[j] = (a.x + a.y) + (b.x + b.y);
        }
        return;
    }
    const bool wide = g.wide_b != 0;
    h.s = -1;                                              // its place takes the rows' elements as they were read
    float2 sum[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] = make_float2(0.0f, 0.0f);
    for (int r = 0; r < rank; r += 32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint4 *const b = reinterpret_cast<const uint4 *>(g.lora_b + (static_cast<int64_t>(s[j]) * g.N + n) * rank + r);
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                uint4 v = make_uint4(0, 0, 0, 0), w = v;
                if (s[j] >= 0 && r + 8 * i < rank) {
                    if (wide) ld_32(b + i, v, w);          // a whole sector per lane
                    else {
                        v = __ldcg(b + i);
                        if (r + 8 * i + 8 < rank) w = __ldcg(b + i + 1);
                    }
                }
                h.w[8 * j + 2 * i] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
                h.w[8 * j + 2 * i + 1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
                h.w[8 * j + 2 * i + 2] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
                h.w[8 * j + 2 * i + 3] = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (s[j] < 0) continue;
            const float4 *const uj = reinterpret_cast<const float4 *>(u + j * rank + r);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (r + 8 * i >= rank) break;
                const float4 f = uj[2 * i], e = uj[2 * i + 1];
                sum[j] = fma2(make_float2(f.x, f.y), T::unpack(__float_as_uint(h.w[8 * j + 2 * i].x)), sum[j]);
                sum[j] = fma2(make_float2(f.z, f.w), T::unpack(__float_as_uint(h.w[8 * j + 2 * i].y)), sum[j]);
                sum[j] = fma2(make_float2(e.x, e.y), T::unpack(__float_as_uint(h.w[8 * j + 2 * i + 1].x)), sum[j]);
                sum[j] = fma2(make_float2(e.z, e.w), T::unpack(__float_as_uint(h.w[8 * j + 2 * i + 1].y)), sum[j]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) d[j] = sum[j].x + sum[j].y;
}

// The pieces of one CTA's adapters' product in order: piece c of segment s, rows from s.m0 + c * kChunkRows on.
template <int CG, bool WAVES>
struct PieceWalker {
    LoraWalker<CG, WAVES> walk;
    LoraSegment s;
    int c, rows;
    __device__ __forceinline__ PieceWalker(const LoraWalker<CG, WAVES> &w) : walk(w) {
        c = rows = 0;
        s.parts = 0;
    }
    __device__ __forceinline__ bool next(const LoraArgs &g) {
        c += s.parts;
        while (c * kChunkRows >= rows) {
            if (!walk.next(s)) return false;
            rows = min(g.rows, g.M - s.m0);
            c = s.part;
        }
        return true;
    }
};

template <typename T, int CG, bool WAVES>
__global__ void __launch_bounds__(kLoraThreads, 1) lora_product_kernel(const __grid_constant__ LoraArgs g) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t ring = (raw + 1023u) & ~1023u;
    uint8_t *const sm = smem_raw + (ring - raw);
    float *const delta = reinterpret_cast<float *>(sm + g.off_delta);
    float *const u_s = reinterpret_cast<float *>(sm + g.off_u);
    int *const id_s = reinterpret_cast<int *>(sm + g.off_ids);
    const uint32_t full0 = ring + g.off_bars, empty0 = full0 + 8 * kLoraStages, acc_full0 = empty0 + 8 * kLoraStages, acc_empty0 = acc_full0 + 16,
                   delta_full0 = acc_empty0 + 16, delta_empty0 = delta_full0 + 8 * kChunks,
                   u_full0 = delta_empty0 + 8 * kChunks, u_empty0 = u_full0 + 8 * kAhead;
    volatile int *const misc = reinterpret_cast<volatile int *>(sm + g.off_misc);   // abort flag, tensor-memory base, two tiles whose parts this CTA adds
    const WaitCtx wait = {g.status, misc, g.budget};
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t rank = CG == 2 ? __shfl_sync(0xffffffffu, cluster_ctarank(), 0) : 0u;

    if (tid < kLoraBars) {
        // accumulators: full, empty (the draining warps of the pair); pieces: full (the delta warps), empty (the draining warps); u: full, empty
        const int j = tid - 2 * kLoraStages, i = j - 4 - 2 * kChunks;
        mbar_init(full0 + 8 * tid, j < 2 ? 1 : j < 4 ? 4 * CG : j < 4 + kChunks ? kDeltaWarps : i < 0 ? 4 : i < kAhead ? 1 : kDeltaWarps);
        fence_mbar_init();
    }
    if (tid == 0) misc[0] = 0, misc[2] = misc[3] = -1;
    if (tid == 32) tma_prefetch_desc(&g.map_b);
    if (tid == 64) tma_prefetch_desc(&g.map_a);
    if (warp == 1) {
        tmem_alloc<CG>(ring + g.off_misc + 4, g.tmem_cols);
        tmem_relinquish<CG>();
    }
    tc_fence_before_sync();
    __syncthreads();
    if (CG == 2) {
        cluster_arrive();
        cluster_wait();
    }
    tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, static_cast<uint32_t>(misc[1]), 0);
    // The shrink kernel waited for all work before the call and said so in every block before this kernel could start: operands
    // are complete here, u is not.
    griddep_launch_dependents();

    constexpr int kBBytes = 128 * 128;                     // 128 rows of B, 64 elements of K
    const uint32_t stage_bytes = kBBytes + g.a_bytes;
    const int stages = g.stages;
    LoraWalker<CG, WAVES> walk(g);
    LoraSegment s;
    int st = 0;
    uint32_t ph = 0;
    bool ok = true;

    if (warp == 0) {
        // -------------------------------------------------------------- operands: TMA
        const bool issuer = elect_one();
        const uint32_t full_leader = CG == 2 ? __shfl_sync(0xffffffffu, mapa_shared(full0, 0), 0) : full0;
        const uint64_t pol_b = l2_policy(WAVES ? 2 : 1), pol_a = l2_policy(2);
        for (int n = 0; ok && walk.next(s); ++n) {
            const int row_b = (s.tile * CG + static_cast<int>(rank)) * 128, row_a = s.m0 + static_cast<int>(rank) * (g.rows / CG);
            const bool down = WAVES && (n & 1);          // to and fro: the panel ends touched last are still in L2
            for (int i = s.kb0; i < s.kb1; ++i) {
                ok = wait_warp(empty0 + 8 * st, ph ^ 1u, wait, 2000 + st);
                if (!ok) break;
                const int k = (down ? s.kb1 - 1 - i : i) * 64;
                const uint32_t dst = ring + st * stage_bytes;
                if (issuer) {
                    if (rank == 0) mbar_arrive_expect_tx(full0 + 8 * st, CG * stage_bytes);
                    if constexpr (CG == 2) {
                        tma_load_2d_pair_hint(dst, &g.map_b, full_leader + 8 * st, k, row_b, pol_b);
                        tma_load_2d_pair_hint(dst + kBBytes, &g.map_a, full_leader + 8 * st, k, row_a, pol_a);
                    } else {
                        tma_load_2d_hint(dst, &g.map_b, full0 + 8 * st, k, row_b, pol_b);
                        tma_load_2d_hint(dst + kBBytes, &g.map_a, full0 + 8 * st, k, row_a, pol_a);
                    }
                }
                if (++st == stages) st = 0, ph ^= 1u;
            }
        }
    } else if (warp == 1) {
        // -------------------------------------------------------------- MMA
        if (rank == 0) {
            const bool issuer = elect_one();
            for (int n = 0; ok && walk.next(s); ++n) {
                const int acc = n & 1;
                ok = wait_warp(acc_empty0 + 8 * acc, ((n >> 1) & 1) ^ 1u, wait, 2100 + acc);
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t d = tmem + acc * g.rows;
                for (int kb = s.kb0; kb < s.kb1; ++kb) {
                    ok = wait_warp(full0 + 8 * st, ph, wait, 2200 + st);
                    if (!ok) break;
                    tc_fence_after_sync();
                    const uint32_t at = ring + st * stage_bytes;
                    const uint64_t b = umma_desc_sw128(at), a = umma_desc_sw128(at + kBBytes);
                    if (issuer) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) umma_f16<CG>(d, b + 2 * i, a + 2 * i, g.idesc, kb > s.kb0 || i > 0);
                        commit_cta<CG>(empty0 + 8 * st);
                    }
                    if (++st == stages) st = 0, ph ^= 1u;
                }
                if (ok && issuer) commit_cta<CG>(acc_full0 + 8 * acc);
            }
        }
        __syncwarp();
    } else if (warp < 6) {
        // -------------------------------------------------------------- accumulators (+ the adapters' product) -> D or parts
        const int quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t acc_empty_leader = CG == 2 ? mapa_shared(acc_empty0, 0) : acc_empty0;
        int piece = 0;
        griddep_wait();                                    // the counters below are zero
        for (int n = 0; ok && walk.next(s); ++n) {
            const int acc = n & 1, rows = min(g.rows, g.M - s.m0);
            const int col = (s.tile * CG + static_cast<int>(rank)) * 128 + r;
            const bool mine = col < g.N;
            ok = wait_warp(acc_full0 + 8 * acc, (n >> 1) & 1, wait, 2300 + acc);
            if (!ok) break;
            tc_fence_after_sync();
            for (int c = 0; c * kChunkRows < rows; ++c) {
                uint32_t v[8];
                tmem_ld_32x8(tmem + acc * g.rows + c * kChunkRows + (static_cast<uint32_t>(quarter * 32) << 16), v);
                tmem_ld_wait();
                if (c % s.parts == s.part) {               // the parts of a tile share its pieces
                    const int slot = piece % kChunks;
                    ok = wait_warp(delta_full0 + 8 * slot, (piece / kChunks) & 1, wait, 2400 + slot);
                    if (!ok) break;
#pragma unroll
                    for (int j = 0; j < kChunkRows; ++j)
                        v[j] = __float_as_uint(__uint_as_float(v[j]) + delta[(slot * kChunkRows + j) * 128 + r]);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(delta_empty0 + 8 * slot);
                    ++piece;
                }
                if (mine) {
                    const int64_t row = s.m0 + c * kChunkRows;
                    if (s.parts == 1) {
                        uint16_t *out = g.D + row * g.N + col;
#pragma unroll
                        for (int j = 0; j < kChunkRows; ++j, out += g.N)
                            if (c * kChunkRows + j < rows) *out = T::round(__uint_as_float(v[j]));
                    } else {
                        float *out = g.o + (static_cast<int64_t>(s.part) * g.M + row) * g.N + col;
#pragma unroll
                        for (int j = 0; j < kChunkRows; ++j, out += g.N)
                            if (c * kChunkRows + j < rows) *out = __uint_as_float(v[j]);
                    }
                }
                __syncwarp();
            }
            if (!ok) break;
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CG == 2) mbar_arrive_cluster(acc_empty_leader + 8 * acc);
                else mbar_arrive(acc_empty0 + 8 * acc);
            }
            if (!WAVES && s.parts > 1) {
                // Four warps of each CTA of the tile's columns count, under the number of the CTA that began them (no CTA begins
                // two tiles that it does not finish); the CTA whose warp is the last one adds the parts in the end.
                __threadfence();
                __syncwarp();
                if (lane == 0 && atomicAdd(g.arrived + blockIdx.x - CG * s.part, 1) == 4 * s.parts - 1) {
                    __threadfence();
                    misc[s.kb0 > 0 ? 2 : 3] = s.tile;
                }
            }
        }
    } else if (warp < 6 + kDeltaWarps) {
        // -------------------------------------------------------------- the adapters' product
        const int t = tid - 6 * 32, n = t & 127, half = (t >> 7) * 4;
        Held held;
        held.s = -1;
        int held_col = -1;
        PieceWalker<CG, WAVES> at(walk);
        griddep_wait();                                    // nothing that this SM's first-level cache may hold is older than the operands
        for (int piece = 0; ok && at.next(g); ++piece) {
            const int slot = piece % kChunks, from = piece % kAhead, col = (at.s.tile * CG + static_cast<int>(rank)) * 128 + n;
            if (col != held_col) held.s = -1, held_col = col;
            ok = wait_warp(u_full0 + 8 * from, (piece / kAhead) & 1, wait, 2600 + from);
            if (!ok) break;
            const int4 q = *reinterpret_cast<const int4 *>(id_s + from * kChunkRows + half);
            const int id[4] = {q.x, q.y, q.z, q.w};
            float d[4] = {};
            if (col < g.N) adapters_product<T>(g, held, id, u_s + (from * kChunkRows + half) * g.rank, col, d);
            __syncwarp();
            if (lane == 0) mbar_arrive(u_empty0 + 8 * from);
            ok = wait_warp(delta_empty0 + 8 * slot, ((piece / kChunks) & 1) ^ 1u, wait, 2500 + slot);
            if (!ok) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) delta[(slot * kChunkRows + half + j) * 128 + n] = d[j];
            __syncwarp();
            if (lane == 0) mbar_arrive(delta_full0 + 8 * slot);
        }
    } else {
        // -------------------------------------------------------------- u and the rows' adapters for the warps above
        PieceWalker<CG, WAVES> at(walk);
        griddep_wait();                                    // u; and in every CTA: this kernel must not complete before the shrink kernel
        for (int piece = 0; ok && at.next(g); ++piece) {
            const int from = piece % kAhead, m = at.s.m0 + at.c * kChunkRows;
            int id = -1;
            if (lane < kChunkRows && m + lane < g.M) id = __ldca(g.row_adapter + m + lane);
            ok = wait_warp(u_empty0 + 8 * from, ((piece / kAhead) & 1) ^ 1u, wait, 2700 + from);
            if (!ok) break;
            if (lane < kChunkRows) id_s[from * kChunkRows + lane] = static_cast<unsigned>(id) < static_cast<unsigned>(g.num_adapters) ? id : -1;
            __syncwarp();
            if (lane == 0) {
                const uint32_t bytes = static_cast<uint32_t>(min(kChunkRows, g.M - m) * g.rank * 4);
                mbar_arrive_expect_tx(u_full0 + 8 * from, bytes);
                bulk_load(smem_u32(u_s + from * kChunkRows * g.rank), g.u + static_cast<int64_t>(m) * g.rank, bytes, u_full0 + 8 * from);
            }
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    if (CG == 2) {
        cluster_arrive();
        cluster_wait();
    }
    if (!WAVES && !misc[0]) {
        for (int i = 2; i < 4; ++i) {
            const int tile = misc[i];
            if (tile < 0) continue;
            const int parts = walk.cut.num_parts(tile), col = (tile * CG + static_cast<int>(rank)) * 128 + lane * 4;
            if (col >= g.N) continue;
            const int64_t pitch = static_cast<int64_t>(g.M) * g.N;
            for (int m = warp; m < g.M; m += kLoraThreads / 32) {
                const float *o = g.o + static_cast<int64_t>(m) * g.N + col;
                float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                for (int p = 0; p < parts; ++p) {
                    const float4 v = __ldcg(reinterpret_cast<const float4 *>(o + p * pitch));
                    y.x += v.x, y.y += v.y, y.z += v.z, y.w += v.w;
                }
                *reinterpret_cast<uint2 *>(g.D + static_cast<int64_t>(m) * g.N + col) =
                    make_uint2(T::round(y.x) | static_cast<uint32_t>(T::round(y.y)) << 16, T::round(y.z) | static_cast<uint32_t>(T::round(y.w)) << 16);
            }
        }
    }
    if (warp == 1) {
        if (misc[0]) {   // aborted: give copies and MMAs in flight a bounded time to land before the memory goes
            const long long t0 = clock64();
            while (clock64() - t0 < 2000000) {
            }
        }
        tc_fence_after_sync();
        tmem_dealloc<CG>(tmem, g.tmem_cols);
    }
}

template <typename Kernel>
cudaError_t launch(Kernel *kernel, const LoraArgs &g, dim3 grid, int threads, int smem, int cluster, cudaStream_t stream) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, g);
}

template <typename T>
cudaError_t launch_lora(const LoraArgs &g, int smem, cudaStream_t stream) {
    cudaError_t e;
    if (g.M <= kDotRows) {
        const int blocks = g.M * (g.rank / 4);
        e = launch(lora_shrink_dot_kernel<T>, g, blocks < 8 * g.sms ? blocks : 8 * g.sms, 256, 0, 1, stream);
    } else {
        const int row_blocks = (g.M + 15) / 16;
        if (row_blocks * ((g.rank + 31) / 32) >= g.sms) e = launch(lora_shrink_mma_kernel<T, 4>, g, dim3(row_blocks, (g.rank + 31) / 32), 256, 0, 1, stream);
        else e = launch(lora_shrink_mma_kernel<T, 1>, g, dim3(row_blocks, g.rank / 8), 256, 0, 1, stream);
    }
    if (e != cudaSuccess) return e;
    if (g.M <= kOneCtaRows) return launch(lora_product_kernel<T, 1, false>, g, g.sms, kLoraThreads, smem, 1, stream);
    if (g.M <= kFewRows) return launch(lora_product_kernel<T, 2, false>, g, g.sms / 2 * 2, kLoraThreads, smem, 2, stream);
    return launch(lora_product_kernel<T, 2, true>, g, g.sms / 2 * 2, kLoraThreads, smem, 2, stream);
}

// CTAs that may share a tile, one more for stretches that do not start at a tile.
int most_parts(int64_t units, int64_t kblocks, int64_t groups) {
    const int64_t len = (units * kblocks + groups - 1) / groups;
    const int64_t parts = (kblocks - 1 + len - 1) / len + 1;
    return static_cast<int>(parts < 2 ? 2 : parts > kMaxLoraParts ? kMaxLoraParts : parts);
}

struct LoraLayout {
    int parts;
    int64_t off_u, off_o, bytes;
};

LoraLayout lora_layout(int64_t M, int64_t N, int64_t K, int rank) {
    LoraLayout l;
    l.parts = M > kFewRows ? 2 : M > kOneCtaRows ? most_parts((N + 255) / 256, (K + 63) / 64, kLoraGridSms / 2) : most_parts((N + 127) / 128, (K + 63) / 64, kLoraGridSms);
    l.off_u = kMaxCtas * 4;
    l.off_o = l.off_u + (M * rank * 4 + 255) / 256 * 256;
    l.bytes = l.off_o + (M <= kFewRows ? l.parts * M * N * 4 : 0);
    return l;
}

int check_lora(int64_t M, int64_t N, int64_t K, int64_t num_adapters, int rank) {
    if (M <= 0 || N <= 0 || K <= 0 || N % 8 || K % 8) return B200_INVALID_SHAPE;
    if (M > (int64_t(1) << 22) || N > (int64_t(1) << 30) || K > (int64_t(1) << 30)) return B200_INVALID_SHAPE;
    if (num_adapters < 1 || num_adapters > (int64_t(1) << 20)) return B200_INVALID_SHAPE;
    if (rank < 8 || rank > B200_LORA_MAX_RANK || rank % 8) return B200_INVALID_CONFIG;
    return B200_OK;
}

}  // namespace

int prepare_moe_kernels();
int prepare_routed_kernels() {
    void (*const kernels[])(LoraArgs) = {lora_product_kernel<Bf16, 1, false>, lora_product_kernel<Bf16, 2, false>, lora_product_kernel<Bf16, 2, true>,
                                         lora_product_kernel<Fp16, 1, false>, lora_product_kernel<Fp16, 2, false>, lora_product_kernel<Fp16, 2, true>};
    for (const auto k : kernels) {
        const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
        if (e != cudaSuccess) return static_cast<int>(e);
    }
    // An SM that runs the shrink kernel with little shared memory could not take a block of the product beside it.
    void (*const first[])(LoraArgs) = {lora_shrink_dot_kernel<Bf16>, lora_shrink_mma_kernel<Bf16, 1>, lora_shrink_mma_kernel<Bf16, 4>,
                                       lora_shrink_dot_kernel<Fp16>, lora_shrink_mma_kernel<Fp16, 1>, lora_shrink_mma_kernel<Fp16, 4>};
    for (const auto k : first) {
        const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        if (e != cudaSuccess) return static_cast<int>(e);
    }
    return prepare_moe_kernels();
}

}  // namespace b200

extern "C" int64_t b200_gemm_lora_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t num_adapters, int rank) {
    if (b200::check_lora(M, N, K, num_adapters, rank) != B200_OK) return -1;
    return b200::lora_layout(M, N, K, rank).bytes;
}

extern "C" int b200_gemm_lora(int dtype, const void *A, const void *Bt, void *D, int64_t M, int64_t N, int64_t K, const void *lora_a,
                              const void *lora_b, const float *lora_scale, const int *row_adapter, int64_t num_adapters, int rank,
                              void *workspace, size_t workspace_bytes, void *stream) {
    using namespace b200;
    if (dtype != B200_F16 && dtype != B200_BF16) return B200_INVALID_CONFIG;
    int st = check_lora(M, N, K, num_adapters, rank);
    if (st != B200_OK) return st;
    if (!A || !Bt || !D || !lora_a || !lora_b || !row_adapter) return B200_INVALID_POINTER;
    if (misaligned(A) || misaligned(Bt) || misaligned(D) || misaligned(lora_a) || misaligned(lora_b) || misaligned(workspace) ||
        (reinterpret_cast<uintptr_t>(row_adapter) & 3u) || (reinterpret_cast<uintptr_t>(lora_scale) & 3u))
        return B200_INVALID_POINTER;
    const int64_t need = b200_gemm_lora_workspace_bytes(M, N, K, num_adapters, rank);
    if (!workspace || workspace_bytes < static_cast<size_t>(need)) return B200_WORKSPACE_TOO_SMALL;
    const struct { const void *p; int64_t n; } in[] = {{A, M * K * 2}, {Bt, N * K * 2}, {lora_a, num_adapters * rank * K * 2},
                                                       {lora_b, num_adapters * rank * N * 2}, {lora_scale, num_adapters * 4}, {row_adapter, M * 4}};
    for (const auto &i : in)
        if (overlap(D, M * N * 2, i.p, i.n) || overlap(workspace, need, i.p, i.n)) return B200_INVALID_POINTER;
    if (overlap(D, M * N * 2, workspace, need)) return B200_INVALID_POINTER;
    LoraArgs g = {};
    st = current_device(&g.sms, &g.status);
    if (st != B200_OK) return st;
    if (g.sms > kMaxCtas) g.sms = kMaxCtas;
    const LoraLayout l = lora_layout(M, N, K, rank);
    g.A = static_cast<const uint16_t *>(A);
    g.lora_a = static_cast<const uint16_t *>(lora_a);
    g.lora_b = static_cast<const uint16_t *>(lora_b);
    g.D = static_cast<uint16_t *>(D);
    g.scale = lora_scale;
    g.row_adapter = row_adapter;
    uint8_t *const ws = static_cast<uint8_t *>(workspace);
    g.arrived = reinterpret_cast<int *>(ws);
    g.u = reinterpret_cast<float *>(ws + l.off_u);
    g.o = reinterpret_cast<float *>(ws + l.off_o);
    g.M = static_cast<int>(M);
    g.N = static_cast<int>(N);
    g.K = static_cast<int>(K);
    g.rank = rank;
    g.num_adapters = static_cast<int>(num_adapters);
    g.parts = l.parts;
    const int cg = M > kOneCtaRows ? 2 : 1;
    g.rows = M > kFewRows ? 256 : static_cast<int>((M + 16 * cg - 1) / (16 * cg) * (16 * cg));
    const int box_a = g.rows / cg;
    g.wide_b = rank % 16 == 0 && (reinterpret_cast<uintptr_t>(lora_b) & 31u) == 0;
    st = encode_operand_map(&g.map_b, dtype, Bt, K, N, 128);
    if (st == B200_OK) st = encode_operand_map(&g.map_a, dtype, A, K, M, box_a);
    if (st != B200_OK) return st;
    g.a_bytes = box_a * 128;
    const int u_bytes = kAhead * kChunkRows * rank * 4, rest = kChunks * kChunkBytes + u_bytes + kAhead * kChunkRows * 4 + kLoraBars * 8 + 16;
    // up to 256 rows 32 KB of the SM stay free for blocks of the shrink kernel
    g.stages = ((M > kFewRows ? kSmemLimit : 196 * 1024) - 1024 - rest) / (128 * 128 + g.a_bytes);
    if (g.stages > kLoraStages) g.stages = kLoraStages;
    g.off_delta = g.stages * (128 * 128 + g.a_bytes);
    g.off_u = g.off_delta + kChunks * kChunkBytes;
    g.off_ids = g.off_u + u_bytes;
    g.off_bars = g.off_ids + kAhead * kChunkRows * 4;
    g.off_misc = g.off_bars + kLoraBars * 8;
    const int smem = 1024 + g.off_delta + rest;
    g.tmem_cols = pow2_at_least(2 * g.rows);
    g.idesc = umma_idesc(128 * cg, g.rows, dtype == B200_BF16);
    g.budget = wait_budget_cycles();
    const cudaError_t e = dtype == B200_BF16 ? launch_lora<Bf16>(g, smem < kMinSmemRequest ? kMinSmemRequest : smem, static_cast<cudaStream_t>(stream))
                                             : launch_lora<Fp16>(g, smem < kMinSmemRequest ? kMinSmemRequest : smem, static_cast<cudaStream_t>(stream));
    return e != cudaSuccess ? record_cuda_error(e) : B200_OK;
}
