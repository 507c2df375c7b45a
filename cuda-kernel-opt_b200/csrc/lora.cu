// A projection shared by all rows with low-rank adapters of many requests beside it:
//
//     D[i] = A[i] B^T + u[i] lora_b[s]^T,   u[i] = scale[s] (A[i] lora_a[s]^T),   s = row_adapter[i]
//
// The product kernel has B's rows on the 128-row side of tcgen05.mma (D is computed transposed: a lane of tensor memory is a column
// of D, a column of tensor memory a row). Warps beside the pipeline compute u lora_b[s]^T in fp32 while the tensor core is
// busy ("delta warps") and hand it to the draining warps in pieces of 16 rows x 128 columns, which add it before the one
// rounding to 16 bits.
//
// Why not on the tensor core, as further columns of K: the zero that stands for "not this row's adapter" does not mask an infinity
// or a NaN among an adapter's weights, so a request would see other requests' adapters; and a decode step in which every
// row has another adapter would feed it one useful row at a time. (Columns of tensor memory of their own per adapter, of which
// only its rows are kept, as the first product does it, would need no zeros; there are none left beside two accumulators.) Only where 32 rows in a row have one adapter, as in a
// prompt, does the tensor core take them (u then as a pair of 16-bit numbers, value and remainder), as long as u fits those.
//
// Three forms, by the numbers of rows and columns (times: on the device, in a graph, SM clock 1965 MHz if nothing else is said):
//   up to 256     one CTA per tile of 128 columns, all rows. Reading B bounds it: 16 x 28672 x 8192, rank 16, takes 77 us, 6.3 TB/s; 128
//                 rows, rank 32, any of 64 adapters per row, 128 to 138 us, 4.4 to 4.8 TB/s. The K blocks of all tiles are cut into one equal
//                 stretch per CTA (Cut), so that every SM streams all the time; a tile that spans several leaves parts in the
//                 workspace, and the last of its CTAs to finish adds them in ascending order. No CTA waits for another,
//                 nothing is added atomically. (A CTA pair per 256 columns, which halves what the rows of A cost between L2 and
//                 SMs, measured the same within 1 % from 65 to 256 rows.)
//   few columns   the same with the rows in several blocks, each with its own stretches: more CTAs share the work, the rows' adapters
//                 above all. 225 x 672 x 3120, rank 72, any of 14 adapters per row: 107 -> 48 us, 25 x 384 x 744, rank 120: 39 ->
//                 18.6; beyond 256 rows while waves would have at most 18 tiles: 535 x 312 x 360, rank 72, 43 prompts: 134 ->
//                 39 us against waves, 1024 x 2048 x 2048 (32 tiles): 33 in waves, 45 in blocks. A kernel of its own, the
//                 general walk costs the form above 5 % of its smallest calls.
//   more          a CTA pair per 256 x 256 tile, whole tiles in waves, the tensor core bounds it: 4096 x 8192 x 8192, rank 64, eight
//                 prompts, takes 450 us call after call at the 1365 MHz that the power limit leaves, 1.25 PFLOP/s; the best of
//                 short runs 385 us. 512 rows of eight prompts take 78 us, two calls of 256 rows 120.
//
// u comes first, from lora_shrink_dot_kernel (few rows) or lora_list_kernel, lora_shrink_kernel and lora_join_kernel. They let the product
// start before they are done; only its warps that need u wait.
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
constexpr int kChunkRows = 16;                             // rows of D in a piece of the adapters' product
constexpr int kChunks = 8;                                 // pieces on their way to the draining warps
constexpr int kWaveChunks = 4;                             // the same in waves, whose ring needs the room (4096 x 8192 x 8192: 3 % over eight)
constexpr int kAhead = 4;                                  // pieces whose adapters and u are on their way to the delta warps
constexpr int kChunkBytes = kChunkRows * 128 * 4;
constexpr int kTileRows = 256;                             // most rows of a tile
constexpr int kLoraBars = 2 * kLoraStages + 4 + 2 * kChunks + 2 * kAhead;
constexpr int kNoRow = -2;                                 // in the place of an adapter: behind the last row
constexpr int kMaxLoraParts = 16;
constexpr int kMaxCtas = 256;
constexpr int kMaxBlocks = 256;                            // blocks of 256 rows of one pass; more rows are several passes
constexpr int kGroup = 32;                                 // rows that share a way of adding their adapters
constexpr int kLoraGridSms = 148;                          // what the workspace is sized for
constexpr int kGroupRows = 16;                             // row blocks that a wave walks together

struct alignas(64) LoraArgs {
    CUtensorMap map_b, map_a;      // B as {K, N}, A as {K, M}
    CUtensorMap map_s, map_la, map_lb, map_u;   // listed: A in boxes of 128 rows, lora_a as {K, adapters * rank}; many rows: lora_b as {rank, adapters * N}, u16 as {rank, 2 * M}
    const uint16_t *A, *lora_a, *lora_b;
    uint16_t *D;
    const float *scale;
    const int *row_adapter;
    float *u;                      // [M][rank]
    float *u_parts;                // [part][M][rank]
    uint16_t *u16;                 // [value, remainder][M][rank]
    struct {
        int *count, *adapter, *entry;   // per block of 256 rows: adapters that occur, and which; per row: which of them it has
        int *wide;                 // per 32 rows: u does not fit pairs of 16-bit numbers
    } list;
    int waves;                     // the form of the product: its own parameter, the last pass of many rows may be short
    int listed, parts_u, on_tensor;   // u by lists of adapters; its parts; whether the adapters' second product may use the tensor core
    uint32_t idesc_u, idesc_run;   // run: with N = 0
    float *o;                      // [part][M][N]: sums of tiles that span CTAs
    int *arrived;                  // per CTA: the warps that are done with the tile it began last
    int M, N, K, rank;
    int num_adapters;
    int wide_b;                    // rows of lora_b are whole 32-byte sectors
    int parts, sms;
    int rows;                      // of a tile: columns of an accumulator
    int u_pitch;                   // floats from row to row of u in shared memory
    int a_bytes, stages, off_delta, off_u, off_ids, off_bars, off_misc;
    int tmem_cols;
    uint32_t idesc;
    int *status;
    long long budget;
};

__device__ __forceinline__ int row_adapter(const LoraArgs &g, int m) {   // -1: none, kNoRow: no such row
    if (m >= g.M) return kNoRow;
    const int s = __ldca(g.row_adapter + m);
    return static_cast<unsigned>(s) < static_cast<unsigned>(g.num_adapters) ? s : -1;
}

// ---------------------------------------------------------------------------------------------- first product

// Few rows: a block takes four ranks of a row, its warps an eighth of K each. Bound by reading the adapters once (2 * rank * K bytes
// per adapter in use): 16 rows, rank 16, K = 8192 in 3 us, 128 rows, rank 32 (29 MB) in 8.5 us.
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
        const int s = row_adapter(g, m);
        if (s < 0) continue;
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

// More rows: lora_a's ranks on the 128-row side of tcgen05.mma, 256 rows of A as its columns, one product per block of rows and adapter
// that occurs among them; only the adapter's own rows are kept. The K blocks of all these products are cut into one
// stretch per CTA (Cut), the parts are joined by a kernel of their own, which also leaves u as a pair of 16-bit numbers.
// Bound by reading A once: 4096 rows, rank 64, K = 8192, eight adapters (67 MB of A) 30 us for the three kernels.

// The adapters that occur in a block of 256 rows, in the order of their first rows.
__global__ void __launch_bounds__(256) lora_list_kernel(const __grid_constant__ LoraArgs g) {
    __shared__ int lead_id[8][32], lead_row[8][32], leads[8], rank_of[256], firsts[8];
    griddep_wait();
    griddep_launch_dependents();
    const int i = threadIdx.x, m = blockIdx.x * 256 + i, warp = i >> 5, lane = i & 31;
    const int id = row_adapter(g, m);
    if (blockIdx.x == 0) g.arrived[i] = 0;                 // kMaxCtas of them
    // one row of the warp per adapter leads; it looks for its adapter among the leaders of the warps before
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    const int leader = __ffs(same) - 1;
    const uint32_t lead = __ballot_sync(0xffffffffu, id >= 0 && leader == lane);
    if (lead >> lane & 1u) {
        const int at = __popc(lead & ((1u << lane) - 1u));
        lead_id[warp][at] = id;
        lead_row[warp][at] = i;
    }
    if (lane == 0) leads[warp] = __popc(lead);
    __syncthreads();
    int first = i;
    if (lead >> lane & 1u)
        for (int w = 0; w < warp && first == i; ++w)
            for (int j = 0; j < leads[w] && first == i; ++j)
                if (lead_id[w][j] == id) first = lead_row[w][j];
    const uint32_t new_ones = __ballot_sync(0xffffffffu, (lead >> lane & 1u) && first == i);
    if (lane == 0) firsts[warp] = __popc(new_ones);
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        before += w < warp ? firsts[w] : 0;
        all += firsts[w];
    }
    if (new_ones >> lane & 1u) {
        rank_of[i] = before + __popc(new_ones & ((1u << lane) - 1u));
        g.list.adapter[blockIdx.x * 256 + rank_of[i]] = id;
    }
    __syncthreads();
    first = __shfl_sync(0xffffffffu, first, leader);
    if (m < g.M) g.list.entry[m] = id >= 0 ? rank_of[first] : -1;
    if (i == 0) g.list.count[blockIdx.x] = all;
}

// before[b] = adapters listed in the blocks before block b, before[blocks] = all; one warp.
__device__ __forceinline__ void scan_lists(const LoraArgs &g, int blocks, int lane, int *before) {
    int sum = 0;
    for (int b0 = 0; b0 < blocks; b0 += 32) {
        int v = b0 + lane < blocks ? __ldcg(g.list.count + b0 + lane) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int w = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += w;
        }
        if (b0 + lane < blocks) before[b0 + lane + 1] = sum + v;
        sum += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) before[0] = 0;
}

constexpr int kShrinkThreads = 192;                        // TMA, MMA and four draining warps
constexpr int kShrinkStages = 4;
constexpr int kShrinkStageBytes = (128 + 256) * 128;
constexpr int kShrinkSmem = 1024 + kShrinkStages * kShrinkStageBytes + (kMaxBlocks + 1) * 4 + 16 + (2 * kShrinkStages + 4) * 8 + 16;

struct ShrinkWalker {
    int q, end;
    Cut cut;
    __device__ __forceinline__ ShrinkWalker(const Cut &c) : cut(c) {
        q = static_cast<int>(min(static_cast<long long>(blockIdx.x) * c.len, static_cast<long long>(c.total)));
        end = min(q + c.len, c.total);
    }
    // block of rows, entry of its list, K blocks [kb0, kb1), part
    __device__ __forceinline__ bool next(const int *before, int blocks, int &block, int &entry, int &kb0, int &kb1, int &part) {
        if (q >= end) return false;
        const int unit = q / cut.kblocks;
        int lo = 0, hi = blocks - 1;                       // the last block whose list does not begin behind the unit
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (before[mid] <= unit) lo = mid;
            else hi = mid - 1;
        }
        block = lo;
        entry = unit - before[lo];
        kb0 = q - unit * cut.kblocks;
        kb1 = min(cut.kblocks, kb0 + end - q);
        part = static_cast<int>(blockIdx.x) - cut.first_cta(unit);
        q += kb1 - kb0;
        return true;
    }
};

__global__ void __launch_bounds__(kShrinkThreads, 1) lora_shrink_kernel(const __grid_constant__ LoraArgs g) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t ring = (raw + 1023u) & ~1023u;
    uint8_t *const sm = smem_raw + (ring - raw);
    constexpr int kOffBefore = kShrinkStages * kShrinkStageBytes, kOffBars = kOffBefore + ((kMaxBlocks + 1) * 4 + 15) / 16 * 16;
    int *const before = reinterpret_cast<int *>(sm + kOffBefore);
    const uint32_t full0 = ring + kOffBars, empty0 = full0 + 8 * kShrinkStages, acc_full0 = empty0 + 8 * kShrinkStages, acc_empty0 = acc_full0 + 16,
                   misc_at = acc_empty0 + 16;
    volatile int *const misc = reinterpret_cast<volatile int *>(sm + (misc_at - ring));
    const WaitCtx wait = {g.status, misc, g.budget};
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    if (tid < 2 * kShrinkStages + 4) {
        mbar_init(full0 + 8 * tid, tid < 2 * kShrinkStages + 2 ? 1 : 4);
        fence_mbar_init();
    }
    if (tid == 0) misc[0] = 0;
    if (warp == 1) {
        tmem_alloc<1>(misc_at + 4, 512);
        tmem_relinquish<1>();
    }
    griddep_wait();
    const int blocks = (g.M + 255) / 256;
    if (warp == 0) scan_lists(g, blocks, lane, before);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    griddep_launch_dependents();
    const uint32_t tmem = __shfl_sync(0xffffffffu, static_cast<uint32_t>(misc[1]), 0);
    ShrinkWalker walk(Cut(before[blocks], (g.K + 63) / 64, gridDim.x, g.parts_u));
    int block, entry, kb0, kb1, part, st = 0;
    uint32_t ph = 0;
    bool ok = true;
    if (warp == 0) {
        const bool issuer = elect_one();
        const uint64_t keep = l2_policy(2);                // A is read again by the product
        while (ok && walk.next(before, blocks, block, entry, kb0, kb1, part)) {
            const int row = __ldcg(g.list.adapter + block * 256 + entry) * g.rank;
            for (int kb = kb0; kb < kb1; ++kb) {
                ok = wait_warp(empty0 + 8 * st, ph ^ 1u, wait, 3000 + st);
                if (!ok) break;
                const uint32_t dst = ring + st * kShrinkStageBytes, bar = full0 + 8 * st;
                if (issuer) {
                    mbar_arrive_expect_tx(bar, (g.rank + 256) * 128);
                    tma_load_2d(dst, &g.map_la, bar, kb * 64, row);
                    tma_load_2d_hint(dst + 128 * 128, &g.map_s, bar, kb * 64, block * 256, keep);
                    tma_load_2d_hint(dst + 256 * 128, &g.map_s, bar, kb * 64, block * 256 + 128, keep);
                }
                if (++st == kShrinkStages) st = 0, ph ^= 1u;
            }
        }
    } else if (warp == 1) {
        const bool issuer = elect_one();
        for (int n = 0; ok && walk.next(before, blocks, block, entry, kb0, kb1, part); ++n) {
            const int acc = n & 1;
            ok = wait_warp(acc_empty0 + 8 * acc, ((n >> 1) & 1) ^ 1u, wait, 3100 + acc);
            if (!ok) break;
            tc_fence_after_sync();
            for (int kb = kb0; kb < kb1; ++kb) {
                ok = wait_warp(full0 + 8 * st, ph, wait, 3200 + st);
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t at = ring + st * kShrinkStageBytes;
                const uint64_t a = umma_desc_sw128(at), x = umma_desc_sw128(at + 128 * 128);
                if (issuer) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) umma_f16<1>(tmem + acc * 256, a + 2 * i, x + 2 * i, g.idesc_u, kb > kb0 || i > 0);
                    umma_commit<1>(empty0 + 8 * st);
                }
                if (++st == kShrinkStages) st = 0, ph ^= 1u;
            }
            if (ok && issuer) umma_commit<1>(acc_full0 + 8 * acc);
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, r = quarter * 32 + lane;   // a rank; ranks from g.rank on are other memory's
        for (int n = 0; ok && walk.next(before, blocks, block, entry, kb0, kb1, part); ++n) {
            const int acc = n & 1;
            uint32_t own = 0u;                             // lane i < 8: which rows of the i-th 32 have this adapter
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int m = block * 256 + 32 * i + lane;
                const uint32_t bits = __ballot_sync(0xffffffffu, m < g.M && __ldcg(g.list.entry + m) == entry);
                if (lane == i) own = bits;
            }
            ok = wait_warp(acc_full0 + 8 * acc, (n >> 1) & 1, wait, 3300 + acc);
            if (!ok) break;
            tc_fence_after_sync();
#pragma unroll 1
            for (int c = 0; c < 256; c += 16) {
                const uint32_t bits = __shfl_sync(0xffffffffu, own, c >> 5) >> (c & 16);
                if ((bits & 0xffffu) == 0u) continue;
                uint32_t v[16];
                tmem_ld_32x16(tmem + acc * 256 + c + (static_cast<uint32_t>(quarter * 32) << 16), v);
                tmem_ld_wait();
                float *const out = g.u_parts + (static_cast<int64_t>(part) * g.M + block * 256 + c) * g.rank + r;
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (r < g.rank && (bits >> j & 1u)) out[j * g.rank] = __uint_as_float(v[j]);
                __syncwarp();
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty0 + 8 * acc);
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        if (misc[0]) {   // aborted: give copies and MMAs in flight a bounded time to land before the memory goes
            const long long t0 = clock64();
            while (clock64() - t0 < 2000000) {
            }
        }
        tc_fence_after_sync();
        tmem_dealloc<1>(tmem, 512);
    }
}

// u from its parts, ascending: 32 rows per block, four ranks of one row per thread; as floats and as pairs of 16-bit numbers, and whether the
// rows' u fit those: no value beyond the type's range, and the largest of eight neighbouring ranks not so small that the pair's
// absolute error, half of the smallest step (fp16: 2^-25), is more than 2^-17 of it. Judging each value by itself would keep ordinary
// rows off the tensor core, in which some of the values are always small; judging whole rows would let adapters that are
// stacked along the rank hide one another. (4096 x 8192 x 8192, eight prompts, fp16, u of ordinary size against u of 10^-5: rank
// 64 some 410 and 650 us, rank 128 some 430 and 880.)
template <typename T>
__global__ void __launch_bounds__(1024) lora_join_kernel(const __grid_constant__ LoraArgs g) {
    __shared__ int before[kMaxBlocks + 1];
    griddep_launch_dependents();   // the product waits for this kernel where it reads u
    griddep_wait();
    const int blocks = (g.M + 255) / 256, quads = g.rank / 4;
    const int m = blockIdx.x * 32 + threadIdx.x / quads, r = threadIdx.x % quads * 4;
    const int entry = m < g.M ? __ldcg(g.list.entry + m) : -1;
    const float scale = entry >= 0 && g.scale ? g.scale[g.row_adapter[m]] : 1.0f;
    if (threadIdx.x < 32) scan_lists(g, blocks, threadIdx.x, before);
    __syncthreads();
    bool fits = true;
    float largest = 0.0f;
    if (entry >= 0) {
        const Cut cut(before[blocks], (g.K + 63) / 64, g.sms, g.parts_u);
        const int parts = cut.num_parts(before[m >> 8] + entry);
        const float *const src = g.u_parts + static_cast<int64_t>(m) * g.rank + r;
        const int64_t pitch = static_cast<int64_t>(g.M) * g.rank;
        float f[4] = {};
        for (int p0 = 0; p0 < parts; p0 += 8) {
            float4 w[8];
#pragma unroll
            for (int p = 0; p < 8; ++p) w[p] = p0 + p < parts ? __ldcg(reinterpret_cast<const float4 *>(src + (p0 + p) * pitch)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int p = 0; p < 8; ++p) f[0] += w[p].x, f[1] += w[p].y, f[2] += w[p].z, f[3] += w[p].w;
        }
        uint16_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[j] *= scale;
            T::split(f[j], hi[j], lo[j]);
            fits = fits && fabsf(f[j]) <= T::kMax;
            largest = fmaxf(largest, fabsf(f[j]));
        }
        *reinterpret_cast<float4 *>(g.u + static_cast<int64_t>(m) * g.rank + r) = make_float4(f[0], f[1], f[2], f[3]);
        if (g.waves) {
            *reinterpret_cast<uint2 *>(g.u16 + static_cast<int64_t>(m) * g.rank + r) = make_uint2(hi[0] | static_cast<uint32_t>(hi[1]) << 16, hi[2] | static_cast<uint32_t>(hi[3]) << 16);
            *reinterpret_cast<uint2 *>(g.u16 + (static_cast<int64_t>(g.M) + m) * g.rank + r) = make_uint2(lo[0] | static_cast<uint32_t>(lo[1]) << 16, lo[2] | static_cast<uint32_t>(lo[3]) << 16);
        }
    }
    largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));   // the neighbour has the same row: a row's threads are an even number
    fits = fits && (largest == 0.0f || largest >= T::kPairMin);
    const int all = __syncthreads_and(fits);
    if (g.waves && threadIdx.x == 0) g.list.wide[blockIdx.x] = !all;
}

// ---------------------------------------------------------------------------------------------- shared product

// K blocks [kb0, kb1) of the tile at row m0 and 128-column (waves: 256-column) tile `tile`, as part `part` of `parts`.
struct LoraSegment {
    int tile, m0, kb0, kb1, part, parts;
    int unit, own0, own1, row0, row1;   // stretches: number of the tile; the pieces that this part adds; their rows / 4, all but where there is one piece
};

enum Form { ONE, BLOCKS, WAVES };   // stretches with all rows in a tile; stretches with several blocks of rows; waves of whole tiles

template <Form F>
struct LoraWalker {
    static constexpr int CG = F == WAVES ? 2 : 1;
    int q, end, tiles_n, row_blocks;
    Cut cut;
    __device__ __forceinline__ LoraWalker(const LoraArgs &g)
        : tiles_n((g.N + 128 * CG - 1) / (128 * CG)), row_blocks(F == ONE ? 1 : (g.M + g.rows - 1) / g.rows), cut(F == WAVES ? 0 : tiles_n * row_blocks, (g.K + 63) / 64, gridDim.x, g.parts) {
        if (F == WAVES) {
            q = blockIdx.x / CG;
            end = tiles_n * row_blocks;
        } else {
            q = static_cast<int>(min(static_cast<long long>(blockIdx.x) * cut.len, static_cast<long long>(cut.total)));
            end = min(q + cut.len, cut.total);
        }
    }
    __device__ __forceinline__ bool next(const LoraArgs &g, LoraSegment &s) {
        if (q >= end) return false;
        const int rows = g.rows, kblocks = cut.kblocks;
        if (F != WAVES) {
            s.unit = q / kblocks;
            s.tile = F == ONE ? s.unit : s.unit / row_blocks;   // blocks of rows of the same columns behind one another
            s.m0 = F == ONE ? 0 : (s.unit - s.tile * row_blocks) * rows;
            s.kb0 = q - s.unit * kblocks;
            s.kb1 = min(kblocks, s.kb0 + end - q);
            s.part = static_cast<int>(blockIdx.x) - cut.first_cta(s.unit);
            s.parts = cut.num_parts(s.unit);
            q += s.kb1 - s.kb0;
            const int here = F == ONE ? g.M : min(rows, g.M - s.m0), pieces = (here + kChunkRows - 1) / kChunkRows;
            s.own0 = pieces * s.kb0 / kblocks;
            s.own1 = pieces * s.kb1 / kblocks;
            s.row0 = 0;
            s.row1 = kChunkRows / 4;
            if (pieces == 1) {
                const int fours = (here + 3) / 4;
                s.row0 = fours * s.kb0 / kblocks;
                s.row1 = fours * s.kb1 / kblocks;
                s.own0 = 0;
                s.own1 = s.row1 > s.row0;
            }
        } else {
            const int in_group = kGroupRows * tiles_n, first = q / in_group * kGroupRows;
            const int height = min(row_blocks - first, kGroupRows), i = q % in_group;
            s.m0 = (first + i % height) * rows;
            s.tile = i / height;
            s.kb0 = 0;
            s.kb1 = kblocks;
            s.part = 0;
            s.parts = 1;
            q += gridDim.x / CG;
        }
        return true;
    }
};

// Rows with adapters of their own: one column n per lane, four rows at a time, fp32 on pairs of ranks. The rows' adapters are read 32
// ranks at a time: 16 loads of 16 bytes (or 8 of a whole sector) in flight per lane.
template <typename T>
__device__ __forceinline__ void four_rows(const LoraArgs &g, const int4 id, const float *u, int pitch, int n, float *d) {
    const int rank = g.rank, s[4] = {id.x, id.y, id.z, id.w};
    const bool wide = g.wide_b != 0;
    float2 sum[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] = make_float2(0.0f, 0.0f);
    const int one = max(max(s[0], s[1]), max(s[2], s[3]));
    if (one < 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j * 128] = 0.0f;
        return;
    }
    if ((s[0] < 0 || s[0] == one) && (s[1] < 0 || s[1] == one) && (s[2] < 0 || s[2] == one) && (s[3] < 0 || s[3] == one)) {
        // one adapter among them, the usual case where requests bring several rows: read once, 64 ranks in one go
        const uint4 *const p = reinterpret_cast<const uint4 *>(g.lora_b + (static_cast<int64_t>(one) * g.N + n) * rank);
#pragma unroll 1
        for (int r = 0; r < rank; r += 64) {
            uint4 b[8];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                if (r + 8 * i >= rank) break;
                if (wide) ld_32(p + r / 8 + i, b[i], b[i + 1]);
                else {
                    b[i] = __ldcg(p + r / 8 + i);
                    b[i + 1] = r + 8 * i + 8 < rank ? __ldcg(p + r / 8 + i + 1) : make_uint4(0, 0, 0, 0);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (r + 8 * i >= rank) break;
                const float2 w0 = T::unpack(b[i].x), w1 = T::unpack(b[i].y), w2 = T::unpack(b[i].z), w3 = T::unpack(b[i].w);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 *const uj = reinterpret_cast<const float4 *>(u + j * pitch + r + 8 * i);
                    const float4 f = uj[0], e = uj[1];
                    sum[j] = fma2(make_float2(f.x, f.y), w0, sum[j]);
                    sum[j] = fma2(make_float2(f.z, f.w), w1, sum[j]);
                    sum[j] = fma2(make_float2(e.x, e.y), w2, sum[j]);
                    sum[j] = fma2(make_float2(e.z, e.w), w3, sum[j]);
                }
            }
        }
        // a row without an adapter has no u: what its place held is not its sum
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j * 128] = s[j] >= 0 ? sum[j].x + sum[j].y : 0.0f;
        return;
    }
    for (int r = 0; r < rank; r += 32) {
        uint4 b[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint4 *const p = reinterpret_cast<const uint4 *>(g.lora_b + (static_cast<int64_t>(s[j]) * g.N + n) * rank + r);
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                b[j][i] = b[j][i + 1] = make_uint4(0, 0, 0, 0);
                if (s[j] >= 0 && r + 8 * i < rank) {
                    if (wide) ld_32(p + i, b[j][i], b[j][i + 1]);
                    else {
                        b[j][i] = __ldcg(p + i);
                        if (r + 8 * i + 8 < rank) b[j][i + 1] = __ldcg(p + i + 1);
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (s[j] < 0) continue;
            const float4 *const uj = reinterpret_cast<const float4 *>(u + j * pitch + r);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (r + 8 * i >= rank) break;
                const float4 f = uj[2 * i], e = uj[2 * i + 1];
                sum[j] = fma2(make_float2(f.x, f.y), T::unpack(b[j][i].x), sum[j]);
                sum[j] = fma2(make_float2(f.z, f.w), T::unpack(b[j][i].y), sum[j]);
                sum[j] = fma2(make_float2(e.x, e.y), T::unpack(b[j][i].z), sum[j]);
                sum[j] = fma2(make_float2(e.z, e.w), T::unpack(b[j][i].w), sum[j]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) d[j * 128] = sum[j].x + sum[j].y;
}

// How the rows of a 256-row tile get their adapters, per group of 32: rows of one adapter whose u fits 16-bit pairs on the tensor core (its
// zeros would not keep another adapter's infinities out, but these groups have none), other rows with adapters in
// pieces. One warp; lane i < 8 holds the adapter of group i.
struct Groups {
    uint32_t run, piece;
    int adapter;
};

__device__ __forceinline__ Groups tile_groups(const LoraArgs &g, int m0, int lane) {
    Groups v = {0u, 0u, -1};
    int id[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) id[i] = row_adapter(g, m0 + kGroup * i + lane);
    const int wide = lane < 8 && m0 + kGroup * lane < g.M ? __ldcg(g.list.wide + m0 / kGroup + lane) : 0;
    const uint32_t no_run = __ballot_sync(0xffffffffu, wide != 0 || !g.on_tensor);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int first = __shfl_sync(0xffffffffu, id[i], 0);
        const bool one = __all_sync(0xffffffffu, id[i] == first || id[i] == kNoRow), some = __any_sync(0xffffffffu, id[i] >= 0);
        if (one && first >= 0 && !(no_run >> i & 1u)) v.run |= 1u << i;
        else if (some) v.piece |= 1u << i;
        if (lane == i) v.adapter = first;
    }
    return v;
}

// The next run of groups with one adapter from group `at` on: [from, at), its adapter; false when there is none.
__device__ __forceinline__ bool next_run(const Groups &v, int &at, int &from, int &adapter) {
    while (at < 8 && !(v.run >> at & 1u)) ++at;
    if (at >= 8) return false;
    from = at;
    adapter = __shfl_sync(0xffffffffu, v.adapter, at);
    do {
        ++at;
    } while (at < 8 && (v.run >> at & 1u) && __shfl_sync(0xffffffffu, v.adapter, at) == adapter);
    return true;
}

// Whether the delta warps compute something of piece c for this part of the tile. With few rows the parts of a tile share its pieces, and a
// single piece by its rows, four at a time: each as many as its share of the K blocks, so that every CTA has the same to do.
template <Form F>
__device__ __forceinline__ bool has_piece(const LoraSegment &s, const Groups &v, int c) {
    return F == WAVES ? (v.piece >> (c * kChunkRows / kGroup) & 1u) != 0u : c >= s.own0 && c < s.own1;
}

// The pieces of one CTA in order: piece c of segment s, rows from s.m0 + c * kChunkRows on.
template <Form F>
struct PieceWalker {
    LoraWalker<F> walk;
    LoraSegment s;
    Groups v;
    int c, rows;
    __device__ __forceinline__ PieceWalker(const LoraWalker<F> &w) : walk(w) { c = rows = 0; }
    __device__ __forceinline__ bool next(const LoraArgs &g, int lane) {
        ++c;
        for (;; ++c) {
            while (c * kChunkRows >= rows) {
                if (!walk.next(g, s)) return false;
                if (F == WAVES) v = tile_groups(g, s.m0, lane);
                rows = min(g.rows, g.M - s.m0);
                c = 0;
            }
            if (has_piece<F>(s, v, c)) return true;
        }
    }
};

template <typename T, Form F>
__global__ void __launch_bounds__(kLoraThreads, 1) lora_product_kernel(const __grid_constant__ LoraArgs g) {
    constexpr int CG = F == WAVES ? 2 : 1, kSlots = F == WAVES ? kWaveChunks : kChunks;
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
    LoraWalker<F> walk(g);
    LoraSegment s;
    int st = 0;
    uint32_t ph = 0;
    bool ok = true;

    if (warp == 0) {
        // -------------------------------------------------------------- operands: TMA
        const bool issuer = elect_one();
        const uint32_t full_leader = CG == 2 ? __shfl_sync(0xffffffffu, mapa_shared(full0, 0), 0) : full0;
        const uint64_t pol_b = l2_policy(walk.row_blocks > 1 ? 2 : 1), pol_a = l2_policy(2);
        for (int n = 0; ok && walk.next(g, s); ++n) {
            const int row_b = (s.tile * CG + static_cast<int>(rank)) * 128, row_a = s.m0 + static_cast<int>(rank) * (g.rows / CG);
            const bool down = F == WAVES && (n & 1);          // to and fro: the panel ends touched last are still in L2
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
            if constexpr (F == WAVES) {
                // then the adapters of whole groups: 64 ranks of lora_b and of u's values, the same ranks and u's remainders
                griddep_wait();
                const Groups v = tile_groups(g, s.m0, lane);
                int at = 0, from, adapter;
                while (ok && next_run(v, at, from, adapter)) {
                    const int row_u = s.m0 + kGroup * from + static_cast<int>(rank) * (kGroup * (at - from) / 2);
                    for (int i = 0; i < (g.rank + 63) / 64 * 2; ++i) {
                        ok = wait_warp(empty0 + 8 * st, ph ^ 1u, wait, 2000 + st);
                        if (!ok) break;
                        const uint32_t dst = ring + st * stage_bytes;
                        if (issuer) {
                            if (rank == 0) mbar_arrive_expect_tx(full0 + 8 * st, CG * stage_bytes);
                            tma_load_2d_pair(dst, &g.map_lb, full_leader + 8 * st, (i >> 1) * 64, adapter * g.N + row_b);
                            tma_load_2d_pair(dst + kBBytes, &g.map_u, full_leader + 8 * st, (i >> 1) * 64, (i & 1) * g.M + row_u);
                        }
                        if (++st == stages) st = 0, ph ^= 1u;
                    }
                }
            }
        }
    } else if (warp == 1) {
        // -------------------------------------------------------------- MMA
        if (rank == 0) {
            const bool issuer = elect_one();
            for (int n = 0; ok && walk.next(g, s); ++n) {
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
                if constexpr (F == WAVES) {
                    griddep_wait();
                    const Groups v = tile_groups(g, s.m0, lane);
                    int at = 0, from, adapter;
                    while (ok && next_run(v, at, from, adapter)) {
                        const uint32_t idesc = g.idesc_run | static_cast<uint32_t>(kGroup * (at - from) / 8) << 17;
                        for (int i = 0; i < (g.rank + 63) / 64 * 2; ++i) {
                            ok = wait_warp(full0 + 8 * st, ph, wait, 2200 + st);
                            if (!ok) break;
                            tc_fence_after_sync();
                            const uint32_t stage = ring + st * stage_bytes;
                            const uint64_t b = umma_desc_sw128(stage), a = umma_desc_sw128(stage + kBBytes);
                            const int steps = min(4, (g.rank - (i >> 1) * 64 + 15) / 16);
                            if (issuer) {
                                for (int j = 0; j < steps; ++j) umma_f16<CG>(d + kGroup * from, b + 2 * j, a + 2 * j, idesc, 1);
                                commit_cta<CG>(empty0 + 8 * st);
                            }
                            if (++st == stages) st = 0, ph ^= 1u;
                        }
                    }
                }
                if (ok && issuer) commit_cta<CG>(acc_full0 + 8 * acc);
            }
        }
        __syncwarp();
    } else if (warp < 6) {
        // -------------------------------------------------------------- accumulators (+ the adapters' product) -> D or parts
        const int quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t acc_empty_leader = CG == 2 ? mapa_shared(acc_empty0, 0) : acc_empty0;
        int slot = 0;
        uint32_t slot_ph = 0;
        griddep_wait();                                    // the counters below are zero
        for (int n = 0; ok && walk.next(g, s); ++n) {
            const int acc = n & 1, rows = min(g.rows, g.M - s.m0);
            const int col = (s.tile * CG + static_cast<int>(rank)) * 128 + r;
            const bool mine = col < g.N;
            Groups v_groups = {};
            if (F == WAVES) v_groups = tile_groups(g, s.m0, lane);
            ok = wait_warp(acc_full0 + 8 * acc, (n >> 1) & 1, wait, 2300 + acc);
            if (!ok) break;
            tc_fence_after_sync();
            for (int c = 0; c * kChunkRows < rows; ++c) {
                uint32_t v[16];
                tmem_ld_32x16(tmem + acc * g.rows + c * kChunkRows + (static_cast<uint32_t>(quarter * 32) << 16), v);
                const bool add = has_piece<F>(s, v_groups, c);
                if (add) ok = wait_warp(delta_full0 + 8 * slot, slot_ph, wait, 2400 + slot);
                tmem_ld_wait();
                if (!ok) break;
                if (add) {
#pragma unroll
                    for (int j = 0; j < kChunkRows; ++j)
                        v[j] = __float_as_uint(__uint_as_float(v[j]) + delta[(slot * kChunkRows + j) * 128 + r]);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(delta_empty0 + 8 * slot);
                    if (++slot == kSlots) slot = 0, slot_ph ^= 1u;
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
            if (F != WAVES && s.parts > 1) {
                // Four warps of each CTA of the tile's columns count, under the number of the CTA that began them (no CTA begins
                // two tiles that it does not finish); the CTA whose warp is the last one adds the parts in the end.
                __threadfence();
                __syncwarp();
                if (lane == 0 && atomicAdd(g.arrived + blockIdx.x - s.part, 1) == 4 * s.parts - 1) {
                    __threadfence();
                    misc[s.kb0 > 0 ? 2 : 3] = s.unit;
                }
            }
        }
    } else if (warp < 6 + kDeltaWarps) {
        // -------------------------------------------------------------- the adapters' product
        const int w = warp - 6, n = (w & 3) * 32 + lane, half = (w >> 2) * 8;
        int slot = 0, from = 0;
        uint32_t slot_ph = 1, from_ph = 0;
        PieceWalker<F> at(walk);
        griddep_wait();                                    // nothing that this SM's first-level cache may hold is older than the operands
        while (ok && at.next(g, lane)) {
            const int col0 = (at.s.tile * CG + static_cast<int>(rank)) * 128;
            ok = wait_warp(u_full0 + 8 * from, from_ph, wait, 2600 + from);
            if (!ok) break;
            const int *const id = id_s + from * kChunkRows;
            const float *const u = u_s + from * kChunkRows * g.u_pitch;
            float *const d = delta + slot * kChunkRows * 128;
            ok = wait_warp(delta_empty0 + 8 * slot, slot_ph, wait, 2500 + slot);
            if (!ok) break;
            if (col0 + n < g.N) {
#pragma unroll 1
                for (int j = half; j < half + 8; j += 4)
                    four_rows<T>(g, *reinterpret_cast<const int4 *>(id + j), u + j * g.u_pitch, g.u_pitch, col0 + n, d + j * 128 + n);
            }
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(u_empty0 + 8 * from);
                mbar_arrive(delta_full0 + 8 * slot);
            }
            if (++from == kAhead) from = 0, from_ph ^= 1u;
            if (++slot == kSlots) slot = 0, slot_ph ^= 1u;
        }
    } else {
        // -------------------------------------------------------------- u and the rows' adapters for the warps above
        PieceWalker<F> at(walk);
        int from = 0;
        uint32_t ph_from = 1;
        griddep_wait();                                    // u; and in every CTA: this kernel must not complete before the shrink kernel
        while (ok && at.next(g, lane)) {
            const int m = at.s.m0 + at.c * kChunkRows + lane;
            const bool there = lane < kChunkRows && m < g.M;
            int id = lane < kChunkRows ? row_adapter(g, m) : kNoRow;
            if (F != WAVES && (F == BLOCKS || g.M <= kChunkRows) && (lane < 4 * at.s.row0 || lane >= 4 * at.s.row1)) id = -1;
            if (id >= 0) {
                // what the piece will read of the adapter: 128 of its columns, which lie behind one another
                const int col = (at.s.tile * CG + static_cast<int>(rank)) * 128;
                if (col < g.N) prefetch_l2(g.lora_b + (static_cast<int64_t>(id) * g.N + col) * g.rank, static_cast<uint32_t>(min(128, g.N - col) * g.rank * 2));
            }
            ok = wait_warp(u_empty0 + 8 * from, ph_from, wait, 2700 + from);
            if (!ok) break;
            const int rows = __popc(__ballot_sync(0xffffffffu, there));
            if (lane < kChunkRows) id_s[from * kChunkRows + lane] = id;
            __syncwarp();
            if (lane == 0) mbar_arrive_expect_tx(u_full0 + 8 * from, static_cast<uint32_t>(rows * g.rank * 4));
            __syncwarp();
            if (there)
                bulk_load(smem_u32(u_s + (from * kChunkRows + lane) * g.u_pitch), g.u + static_cast<int64_t>(m) * g.rank, static_cast<uint32_t>(g.rank * 4), u_full0 + 8 * from);
            if (++from == kAhead) from = 0, ph_from ^= 1u;
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    if (CG == 2) {
        cluster_arrive();
        cluster_wait();
    }
    if (F != WAVES && !misc[0]) {
        for (int i = 2; i < 4; ++i) {
            const int unit = misc[i];
            if (unit < 0) continue;
            const int parts = walk.cut.num_parts(unit), tile = F == ONE ? unit : unit / walk.row_blocks, m0 = F == ONE ? 0 : (unit - tile * walk.row_blocks) * g.rows;
            const int col = tile * 128 + lane * 4, m1 = F == ONE ? g.M : min(m0 + g.rows, g.M);
            if (col >= g.N) continue;
            const int64_t pitch = static_cast<int64_t>(g.M) * g.N;
            constexpr int kWarps = kLoraThreads / 32;
            for (int m = m0 + warp; m < m1; m += 2 * kWarps) {  // two rows and four parts of each in flight
                const float *const o = g.o + static_cast<int64_t>(m) * g.N + col, *const o2 = o + static_cast<int64_t>(kWarps) * g.N;
                const bool two = m + kWarps < m1;
                float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f), y2 = y;
                for (int p0 = 0; p0 < parts; p0 += 4) {
                    float4 v[4], v2[4];
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        v[p] = v2[p] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (p0 + p < parts) v[p] = __ldcg(reinterpret_cast<const float4 *>(o + (p0 + p) * pitch));
                        if (p0 + p < parts && two) v2[p] = __ldcg(reinterpret_cast<const float4 *>(o2 + (p0 + p) * pitch));
                    }
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        y.x += v[p].x, y.y += v[p].y, y.z += v[p].z, y.w += v[p].w;
                        y2.x += v2[p].x, y2.y += v2[p].y, y2.z += v2[p].z, y2.w += v2[p].w;
                    }
                }
                store_four<T>(g.D + static_cast<int64_t>(m) * g.N + col, y);
                if (two) store_four<T>(g.D + static_cast<int64_t>(m + kWarps) * g.N + col, y2);
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
    if (!g.listed) {
        const int blocks = g.M * (g.rank / 4);
        e = launch(lora_shrink_dot_kernel<T>, g, blocks < 8 * g.sms ? blocks : 8 * g.sms, 256, 0, 1, stream);
    } else {
        e = launch(lora_list_kernel, g, (g.M + 255) / 256, 256, 0, 1, stream);
        if (e == cudaSuccess) e = launch(lora_shrink_kernel, g, g.sms, kShrinkThreads, kShrinkSmem, 1, stream);
        if (e == cudaSuccess) e = launch(lora_join_kernel<T>, g, (g.M + 31) / 32, 32 * (g.rank / 4), 0, 1, stream);
    }
    if (e != cudaSuccess) return e;
    if (!g.waves) return launch(g.rows < g.M ? lora_product_kernel<T, BLOCKS> : lora_product_kernel<T, ONE>, g, g.sms, kLoraThreads, smem, 1, stream);
    return launch(lora_product_kernel<T, WAVES>, g, g.sms / 2 * 2, kLoraThreads, smem, 2, stream);
}

// CTAs that may share a tile, one more for stretches that do not start at a tile.
int most_parts(int64_t units, int64_t kblocks, int64_t groups, int64_t most = kMaxLoraParts) {
    const int64_t len = (units * kblocks + groups - 1) / groups;
    const int64_t parts = (kblocks - 1 + len - 1) / len + 1;
    return static_cast<int>(parts < 2 ? 2 : parts > most ? most : parts);
}

struct LoraLayout {
    bool waves, listed;
    int rows, parts, parts_u;
    int64_t off_u, off_o, off_u16, off_u_parts, off_count, off_adapter, off_entry, off_wide, bytes;
};

LoraLayout lora_layout(int64_t M, int64_t N, int64_t K, int64_t num_adapters, int rank) {
    LoraLayout l = {};
    if (M > kMaxBlocks * 256) M = kMaxBlocks * 256;
    int64_t at = 0;
    auto take = [&at](int64_t bytes) {
        const int64_t from = at;
        at += (bytes + 255) / 256 * 256;
        return from;
    };
    take(kMaxCtas * 4);
    l.off_u = take(M * rank * 4);
    l.waves = M > kTileRows && (N + 255) / 256 * ((M + 255) / 256) > kLoraGridSms / 8;
    if (!l.waves) {
        const int64_t tiles_n = (N + 127) / 128, fewest = (M + kTileRows - 1) / kTileRows, most = (M + 15) / 16;
        // Blocks of rows: three parts per tile would fill the SMs, or two if a block keeps 96 rows or more, since every block reads B
        // again (77 x 4104 x 2056 with two blocks: 16.2 -> 20.3 us, 256 x 4096 x 4096, rank 64: 48 -> 41).
        const int64_t two_parts = kLoraGridSms / 2 / tiles_n, three_parts = kLoraGridSms / 3 / tiles_n;
        int64_t blocks = M / 96 < two_parts ? M / 96 : two_parts;
        blocks = blocks < three_parts ? three_parts : blocks;
        blocks = blocks < fewest ? fewest : blocks > most ? most : blocks;
        l.rows = static_cast<int>((M + 16 * blocks - 1) / (16 * blocks) * 16);
        blocks = (M + l.rows - 1) / l.rows;
        // More rows make a part dearer to write and add, the stretches are then kept longer (77 x 4104 x 2056: 16.2 us with
        // four parts, 22.9 with six).
        l.parts = most_parts(tiles_n * blocks, (K + 63) / 64, kLoraGridSms, l.rows > 64 ? 4 : kMaxLoraParts);
        l.off_o = take(l.parts * M * N * 4);
    } else {
        l.rows = 256;
        l.parts = 2;
        l.off_u16 = take(2 * M * rank * 2);
        l.off_wide = take((M + 31) / 32 * 4);
    }
    // Without waves u comes by dot products, which read an adapter for each of its rows, unless that is much more than the products by
    // lists read, which read the rows for each adapter, and enough to pay for two more kernels (256 x 8192 x 8192, rank 64, four
    // adapters: 73 -> 60 us). Beyond 256 rows requests bring many rows each, however many adapters there are to choose from.
    const bool few_adapters = M > kTileRows || M * rank > 2 * (num_adapters < M ? num_adapters : M) * (256 + rank);
    l.listed = l.waves || (few_adapters && M * rank * K * 2 > (int64_t(64) << 20));
    if (l.listed) {
        const int64_t blocks = (M + 255) / 256;
        l.parts_u = most_parts(blocks, (K + 63) / 64, kLoraGridSms);
        l.off_u_parts = take(l.parts_u * M * rank * 4);
        l.off_count = take(blocks * 4);
        l.off_adapter = take(blocks * 256 * 4);
        l.off_entry = take(M * 4);
    }
    l.bytes = at;
    return l;
}

int check_lora(int64_t M, int64_t N, int64_t K, int64_t num_adapters, int rank) {
    if (M <= 0 || N <= 0 || K <= 0 || N % 8 || K % 8) return B200_INVALID_SHAPE;
    if (M > (int64_t(1) << 24) || N > (int64_t(1) << 22) || K > (int64_t(1) << 18)) return B200_INVALID_SHAPE;   // K blocks are counted in 32 bits
    if (num_adapters < 1 || num_adapters > (int64_t(1) << 20)) return B200_INVALID_SHAPE;
    if (rank < 8 || rank > B200_LORA_MAX_RANK || rank % 8) return B200_INVALID_CONFIG;
    return B200_OK;
}

}  // namespace

int prepare_moe_kernels();
int prepare_routed_kernels() {
    void (*const kernels[])(LoraArgs) = {lora_product_kernel<Bf16, ONE>, lora_product_kernel<Bf16, BLOCKS>, lora_product_kernel<Bf16, WAVES>,
                                         lora_product_kernel<Fp16, ONE>, lora_product_kernel<Fp16, BLOCKS>, lora_product_kernel<Fp16, WAVES>};
    for (const auto k : kernels) {
        const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
        if (e != cudaSuccess) return static_cast<int>(e);
    }
    const cudaError_t e = cudaFuncSetAttribute(lora_shrink_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
    if (e != cudaSuccess) return static_cast<int>(e);
    return prepare_moe_kernels();
}

}  // namespace b200

extern "C" int64_t b200_gemm_lora_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t num_adapters, int rank) {
    if (b200::check_lora(M, N, K, num_adapters, rank) != B200_OK) return -1;
    return b200::lora_layout(M, N, K, num_adapters, rank).bytes;
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
    const LoraLayout l = lora_layout(M, N, K, num_adapters, rank);
    g.lora_a = static_cast<const uint16_t *>(lora_a);
    g.lora_b = static_cast<const uint16_t *>(lora_b);
    g.scale = lora_scale;
    uint8_t *const ws = static_cast<uint8_t *>(workspace);
    g.arrived = reinterpret_cast<int *>(ws);
    g.u = reinterpret_cast<float *>(ws + l.off_u);
    g.o = reinterpret_cast<float *>(ws + l.off_o);
    g.u16 = reinterpret_cast<uint16_t *>(ws + l.off_u16);
    g.u_parts = reinterpret_cast<float *>(ws + l.off_u_parts);
    g.list.count = reinterpret_cast<int *>(ws + l.off_count);
    g.list.adapter = reinterpret_cast<int *>(ws + l.off_adapter);
    g.list.entry = reinterpret_cast<int *>(ws + l.off_entry);
    g.list.wide = reinterpret_cast<int *>(ws + l.off_wide);
    g.N = static_cast<int>(N);
    g.K = static_cast<int>(K);
    g.rank = rank;
    g.num_adapters = static_cast<int>(num_adapters);
    g.parts = l.parts;
    g.parts_u = l.parts_u;
    g.listed = l.listed;
    g.waves = l.waves;
    const bool bf16 = dtype == B200_BF16;
    const int cg = g.waves ? 2 : 1;
    g.rows = l.rows;
    const int box_a = g.rows / cg;
    g.wide_b = rank % 16 == 0 && (reinterpret_cast<uintptr_t>(lora_b) & 31u) == 0;
    g.a_bytes = box_a * 128;
    g.u_pitch = rank + 4;   // rows of u start 16 bytes further each, modulo the banks
    const int u_bytes = kAhead * kChunkRows * g.u_pitch * 4, chunks = g.waves ? kWaveChunks : kChunks;
    const int rest = chunks * kChunkBytes + u_bytes + kAhead * kChunkRows * 4 + kLoraBars * 8 + 16;
    g.stages = (kSmemLimit - 1024 - rest) / (128 * 128 + g.a_bytes);
    if (g.stages > kLoraStages) g.stages = kLoraStages;
    g.off_delta = g.stages * (128 * 128 + g.a_bytes);
    g.off_u = g.off_delta + chunks * kChunkBytes;
    g.off_ids = g.off_u + u_bytes;
    g.off_bars = g.off_ids + kAhead * kChunkRows * 4;
    g.off_misc = g.off_bars + kLoraBars * 8;
    const int bytes = 1024 + g.off_delta + rest, smem = bytes < kMinSmemRequest ? kMinSmemRequest : bytes;
    g.tmem_cols = pow2_at_least(2 * g.rows);
    g.idesc = umma_idesc(128 * cg, g.rows, bf16);
    g.idesc_run = umma_idesc(256, 0, bf16);
    g.idesc_u = umma_idesc(128, 256, bf16);
    g.budget = wait_budget_cycles();
    st = encode_operand_map(&g.map_b, dtype, Bt, K, N, 128);
    if (st == B200_OK && l.listed) st = encode_operand_map(&g.map_la, dtype, lora_a, K, num_adapters * rank, rank);
    if (st == B200_OK && g.waves) {
        g.on_tensor = num_adapters * N < (int64_t(1) << 31) - 512;   // rows of lora_b as the copies count them
        if (g.on_tensor) st = encode_operand_map(&g.map_lb, dtype, lora_b, rank, num_adapters * N, 128);
    }
    for (int64_t m0 = 0; st == B200_OK && m0 < M; m0 += kMaxBlocks * 256) {
        const int64_t rows = M - m0 < kMaxBlocks * 256 ? M - m0 : kMaxBlocks * 256;
        g.A = static_cast<const uint16_t *>(A) + m0 * K;
        g.D = static_cast<uint16_t *>(D) + m0 * N;
        g.row_adapter = row_adapter + m0;
        g.M = static_cast<int>(rows);
        st = encode_operand_map(&g.map_a, dtype, g.A, K, rows, box_a);
        if (st == B200_OK && l.listed) st = encode_operand_map(&g.map_s, dtype, g.A, K, rows, 128);
        if (st == B200_OK && g.on_tensor) st = encode_operand_map(&g.map_u, dtype, g.u16, rank, 2 * rows, 128);
        if (st != B200_OK) break;
        const cudaError_t e = bf16 ? launch_lora<Bf16>(g, smem, static_cast<cudaStream_t>(stream)) : launch_lora<Fp16>(g, smem, static_cast<cudaStream_t>(stream));
        if (e != cudaSuccess) st = record_cuda_error(e);
    }
    return st;
}
