// A whole mixture-of-experts layer for a few tokens:
//
//     Y[t] = sum_j w[t][j] W2[e] (silu(G[e] X[t]) . (U[e] X[t])),   e = ids[t][j] = the j-th largest router logit of t
//
// What bounds it is reading the chosen experts' weights once (3 * inner * hidden two-byte values each): a token
// more per expert costs almost nothing. So the weights take the 128-row side of tcgen05.mma and the tokens of one expert
// its N side, and the work (chosen experts x row tiles x K blocks of 64) is cut into one equal, contiguous stretch of K
// blocks per CTA, wherever that falls: with 8 chosen experts of 96 tiles on 148 SMs whole tiles would leave a third of
// the SMs idle, and an SM streams at most some 45 GB/s. A tile whose K blocks end up in several CTAs leaves
// that many partial sums ("parts") in the workspace, which the next kernel adds in ascending order: no CTA waits for
// another, nothing is accumulated atomically, the same inputs give the same bits.
//
//   moe_route_kernel    one block: the choice per token (one warp each), the list of chosen experts with their tokens
//   moe_product_kernel  <UP>: a tile is 64 rows of G and the same 64 rows of U; parts of both (fp32) to the workspace
//   moe_product_kernel  <DOWN>: a tile is 128 rows of W2; the loader warps add the parts of a K block, apply silu and the
//                       gate, and hand the result to the tensor core as a pair of 16-bit numbers, value and remainder
//                       (two MMAs per K step: the tensor core idles here, and one 16-bit rounding of the gated value
//                       would cost as much accuracy as the rounding of the result)
//   moe_combine_kernel  adds the parts and the weighted choices of a token, one rounding
//
// The kernels are launched as programmatic dependents: UP lets DOWN start at once, so DOWN's CTAs (two CTAs fit an SM while
// the tokens are few) fill their ring with weights while UP still runs, and wait only before they read its sums.
#include <cuda_runtime.h>

#include <cfloat>
#include <cmath>

#include "../../include/b200_gemm.h"
#include "gemm_sm100.cuh"
#include "pipeline.cuh"
#include "routed.cuh"

namespace b200 {
namespace {

constexpr int kMoeStages = 16;      // most stages of the ring
constexpr int kMoeLoaders = 8;      // warps that bring the activations of a K block
constexpr int kMoeThreads = (2 + 4 + kMoeLoaders) * 32;
constexpr int kMaxParts = 16;
constexpr int kFewTokens = 16;      // up to here the loader warps of DOWN compute the gated values, beyond a kernel does
constexpr int kGridSms = 148;       // what the workspace is sized for; another count only changes how tiles are cut
constexpr int kBoxBytes = 16 * 128;      // 16 slots of 64 gated values
constexpr int kWeightBytes = 128 * 128;  // one K block of a weight tile: 128 rows of 64 elements

// What the route kernel leaves for the others, in the workspace.
struct Lists {
    int *header;     // [0] chosen experts, [1] most tokens of one
    int *expert;     // per chosen expert: its index, its number of tokens, the first of its slots
    int *count;
    int *base;
    int *token;      // per slot (sorted by expert, then token): its token
    int *slot;       // per (token, choice): its slot, -1 without one
    int *active;     // per (token, choice): the position of its expert in the list of chosen ones
    float *weight;   // per (token, choice)
};

struct alignas(64) MoeArgs {
    CUtensorMap map;          // of the product's weights
    CUtensorMap map_h;        // of h
    const uint16_t *X;
    const float *logits;
    uint16_t *Y;
    int *ids_out;
    float *weights_out;
    Lists list;
    float *z;                 // [part][slot][2 * inner]: sums of UP
    float *o;                 // [part][slot][hidden]: sums of DOWN
    uint16_t *h;              // [value, remainder][slot][inner]: gated values
    int tokens, hidden, inner, experts, top_k, normalise, slots;
    int parts_up, parts_down;
    int sms;
    int ring_bytes, off_token, off_expert, off_bars, off_misc;
    int tmem_cols, slot_cols;
    uint32_t idesc;           // with N = 0
    int *status;
    long long budget;
};

// How the K blocks of `units` tiles are dealt out: CTA c takes blocks [c * len, (c + 1) * len) of all of them in a row. len is
// large enough for a tile to touch at most `parts` CTAs.
struct Cut {
    int kblocks, total, len;
    __device__ __forceinline__ Cut(int units, int kblocks_, int sms, int parts) : kblocks(kblocks_), total(units * kblocks_) {
        len = max(max((total + sms - 1) / sms, (kblocks - 1 + parts - 2) / (parts - 1)), 1);
    }
    __device__ __forceinline__ int first_cta(int unit) const { return unit * kblocks / len; }
    __device__ __forceinline__ int num_parts(int unit) const { return ((unit + 1) * kblocks - 1) / len - first_cta(unit) + 1; }
};

// Order-preserving map of a logit to an unsigned key; 0 = never chosen (-infinity, NaN). Equal floats (+-0 among
// them) get equal keys; +infinity counts as the largest finite value.
__device__ __forceinline__ uint32_t logit_key(float v) {
    if (!(v > -INFINITY)) return 0u;
    v = fminf(v, FLT_MAX) + 0.0f;
    const uint32_t u = __float_as_uint(v);
    return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) { return __uint_as_float((k >> 31) ? k ^ 0x80000000u : ~k); }

// One warp, one token, up to 32 * PER experts: the top_k largest keys in descending order, ties to the lower index; lane
// j < top_k returns choice j (id -1, weight 0 where no expert is left). A lane keeps its own largest key, so a step is
// two warp reductions and only the winning lane looks through its keys again.
template <int PER>
__device__ __forceinline__ void choose_experts(const float *logits, int experts, int top_k, int normalise, int lane, int &id, float &weight) {
    uint32_t key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane + 32 * i;
        key[i] = e < experts ? logit_key(__ldcg(logits + e)) : 0u;
    }
    uint32_t best = 0u;
    int best_i = 0;
    auto look = [&] {
        best = 0u;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (key[i] > best) best = key[i], best_i = i;
    };
    look();
    const float top = key_logit(__reduce_max_sync(0xffffffffu, best));
    float sum = 0.0f;
    if (!normalise) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (key[i]) sum += expf(key_logit(key[i]) - top);
        sum = warp_sum(sum);
    }
    id = -1;
    uint32_t chosen = 0u;
    for (int j = 0; j < top_k; ++j) {
        const uint32_t most = __reduce_max_sync(0xffffffffu, best);
        if (most == 0u) break;
        const uint32_t e = __reduce_min_sync(0xffffffffu, best == most ? static_cast<uint32_t>(lane + 32 * best_i) : 0xffffffffu);
        if (lane == static_cast<int>(e & 31u)) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (i == best_i) key[i] = 0u;
            look();
        }
        if (lane == j) id = static_cast<int>(e), chosen = most;
    }
    weight = id >= 0 ? expf(key_logit(chosen) - top) : 0.0f;
    if (normalise) sum = warp_sum(weight);
    if (id >= 0) weight /= sum;
}

// One cluster of up to eight blocks, a warp per token; its first block then lists the chosen experts and their tokens.
__global__ void __launch_bounds__(1024) moe_route_kernel(const __grid_constant__ MoeArgs g) {
    __shared__ uint32_t mask[B200_MOE_MAX_EXPERTS][B200_MOE_MAX_TOKENS / 32];   // the tokens of an expert (of the first block)
    __shared__ short place[B200_MOE_MAX_EXPERTS];                               // its position among the chosen
    __shared__ int first[B200_MOE_MAX_EXPERTS];                                 // its first slot
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int words = (g.tokens + 31) / 32;
    if (blockIdx.x == 0)
        for (int i = tid; i < g.experts * words; i += 1024) mask[i / words][i % words] = 0u;
    cluster_arrive();
    griddep_wait();
    griddep_launch_dependents();
    const int t = blockIdx.x * 32 + warp;
    int id = -1;
    float w = 0.0f;
    if (t < g.tokens) {
        const float *const row = g.logits + static_cast<int64_t>(t) * g.experts;
        if (g.experts <= 32) choose_experts<1>(row, g.experts, g.top_k, g.normalise, lane, id, w);
        else if (g.experts <= 64) choose_experts<2>(row, g.experts, g.top_k, g.normalise, lane, id, w);
        else if (g.experts <= 128) choose_experts<4>(row, g.experts, g.top_k, g.normalise, lane, id, w);
        else if (g.experts <= 256) choose_experts<8>(row, g.experts, g.top_k, g.normalise, lane, id, w);
        else choose_experts<16>(row, g.experts, g.top_k, g.normalise, lane, id, w);
    }
    cluster_wait();                                         // the first block's masks are zero
    if (t < g.tokens && lane < g.top_k) {
        const int at = t * g.top_k + lane;
        g.list.slot[at] = id;                               // the expert for now
        g.list.weight[at] = w;
        if (g.ids_out) g.ids_out[at] = id;
        if (g.weights_out) g.weights_out[at] = w;
        if (id >= 0) red_or_cluster(mapa_shared(smem_u32(&mask[id][t >> 5]), 0), 1u << (t & 31));
    }
    cluster_arrive();
    cluster_wait();
    if (blockIdx.x != 0) return;
    if (warp == 0) {
        int chosen = 0, slots = 0, most = 0;
        for (int e0 = 0; e0 < g.experts; e0 += 32) {
            const int e = e0 + lane;
            int n = 0;
            if (e < g.experts)
                for (int i = 0; i < words; ++i) n += __popc(mask[e][i]);
            const uint32_t ballot = __ballot_sync(0xffffffffu, n > 0);
            int before = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= o) before += v;
            }
            if (n > 0) {
                const int at = chosen + __popc(ballot & ((1u << lane) - 1u));
                g.list.expert[at] = e;
                g.list.count[at] = n;
                g.list.base[at] = slots + before - n;
                place[e] = static_cast<short>(at);
                first[e] = slots + before - n;
            }
            chosen += __popc(ballot);
            slots += __shfl_sync(0xffffffffu, before, 31);
            most = max(most, static_cast<int>(__reduce_max_sync(0xffffffffu, static_cast<uint32_t>(n))));
        }
        if (lane == 0) {
            g.list.header[0] = chosen;
            g.list.header[1] = most;
        }
    }
    __syncthreads();
    for (int at = tid; at < g.slots; at += 1024) {
        const int t = at / g.top_k, e = __ldcg(g.list.slot + at);
        if (e < 0) continue;
        int slot = first[e] + __popc(mask[e][t >> 5] & ((1u << (t & 31)) - 1u));
        for (int i = 0; i < (t >> 5); ++i) slot += __popc(mask[e][i]);
        g.list.token[slot] = t;
        g.list.slot[at] = slot;
        g.list.active[at] = place[e];
    }
}

// The stretch of one CTA, cut at tile borders: K blocks [kb0, kb1) of tile `tile` of chosen expert `ai`.
struct Segment {
    int ai, tile, kb0, kb1, part;
};

struct Walker {
    int q, end, tiles, cta;
    Cut cut;
    __device__ __forceinline__ Walker(const Cut &c, int tiles_, int cta_) : tiles(tiles_), cta(cta_), cut(c) {
        q = min(static_cast<long long>(cta) * c.len, static_cast<long long>(c.total));
        end = min(q + c.len, c.total);
    }
    __device__ __forceinline__ bool next(Segment &s) {
        if (q >= end) return false;
        const int unit = q / cut.kblocks;
        s.ai = unit / tiles;
        s.tile = unit - s.ai * tiles;
        s.kb0 = q - unit * cut.kblocks;
        s.kb1 = min(cut.kblocks, s.kb0 + end - q);
        s.part = cta - cut.first_cta(unit);
        q += s.kb1 - s.kb0;
        return true;
    }
};

enum Product {
    UP,           // gate and up rows times the tokens of X, gathered by the loader warps
    DOWN_INLINE,  // W2 times the gated values, which the loader warps compute from UP's parts
    DOWN          // W2 times the gated values that moe_gate_kernel has left in the workspace, by TMA
};

// The gated value of eight neighbouring inner rows of one slot from UP's parts (ascending), as pairs of 16-bit numbers.
// The exponential and the quotient err by 2^-21 together: a 128th of what the pair keeps of a bf16, an 8th of an fp16.
template <typename T>
__device__ __forceinline__ void gated_values(const float *z, int inner, int parts, int64_t part_pitch, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
    float gate[8] = {}, up[8] = {};
    for (int p = 0; p < parts; ++p, z += part_pitch) {
        const float4 a = __ldcg(reinterpret_cast<const float4 *>(z)), b = __ldcg(reinterpret_cast<const float4 *>(z + 4));
        const float4 c = __ldcg(reinterpret_cast<const float4 *>(z + inner)), d = __ldcg(reinterpret_cast<const float4 *>(z + inner + 4));
        gate[0] += a.x, gate[1] += a.y, gate[2] += a.z, gate[3] += a.w, gate[4] += b.x, gate[5] += b.y, gate[6] += b.z, gate[7] += b.w;
        up[0] += c.x, up[1] += c.y, up[2] += c.z, up[3] += c.w, up[4] += d.x, up[5] += d.y, up[6] += d.z, up[7] += d.w;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint16_t h0, h1, l0, l1;
        T::split(__fdividef(gate[2 * i], 1.0f + __expf(-gate[2 * i])) * up[2 * i], h0, l0);
        T::split(__fdividef(gate[2 * i + 1], 1.0f + __expf(-gate[2 * i + 1])) * up[2 * i + 1], h1, l1);
        hi[i] = h0 | static_cast<uint32_t>(h1) << 16;
        lo[i] = l0 | static_cast<uint32_t>(l1) << 16;
    }
}

template <typename T, Product P>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_product_kernel(const __grid_constant__ MoeArgs g) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t ring = (raw + 1023u) & ~1023u;
    uint8_t *const sm = smem_raw + (ring - raw);
    uint16_t *const token_s = reinterpret_cast<uint16_t *>(sm + g.off_token);
    int *const expert_s = reinterpret_cast<int *>(sm + g.off_expert);
    int *const count_s = expert_s + g.experts, *const base_s = count_s + g.experts;
    const uint32_t full0 = ring + g.off_bars, empty0 = full0 + 8 * kMoeStages, acc_full0 = empty0 + 8 * kMoeStages, acc_empty0 = acc_full0 + 16;
    volatile int *const misc = reinterpret_cast<volatile int *>(sm + g.off_misc);   // [0] abort flag, [1] tensor-memory base
    const WaitCtx wait = {g.status, misc, g.budget};
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);

    if (tid < 2 * kMoeStages + 4) {
        // full: the producer's byte count and four arrivals of the loader warps; accumulator empty: the four draining warps
        mbar_init(full0 + 8 * tid, tid < kMoeStages ? (P == DOWN ? 1 : 5) : tid < 2 * kMoeStages + 2 ? 1 : 4);
        fence_mbar_init();
    }
    if (tid == 0) misc[0] = 0;
    if (tid == 32) tma_prefetch_desc(&g.map);
    if (P == DOWN && tid == 64) tma_prefetch_desc(&g.map_h);
    if (warp == 1) {
        tmem_alloc<1>(ring + g.off_misc + 4, g.tmem_cols);
        tmem_relinquish<1>();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    // UP waits for the route kernel; every CTA of UP says so before DOWN may start, so DOWN finds the lists (and all that came
    // before the call) complete without a wait of its own, and waits later for UP's sums.
    if (P == UP) griddep_wait();
    griddep_launch_dependents();
    const int chosen = __ldcg(g.list.header), most = __ldcg(g.list.header + 1);
    for (int i = tid; i < chosen; i += kMoeThreads) {
        expert_s[i] = __ldcg(g.list.expert + i);
        count_s[i] = __ldcg(g.list.count + i);
        base_s[i] = __ldcg(g.list.base + i);
    }
    if (P == UP)
        for (int i = tid; i < g.slots; i += kMoeThreads) token_s[i] = static_cast<uint16_t>(__ldcg(g.list.token + i));
    __syncthreads();
    const uint32_t tmem = __shfl_sync(0xffffffffu, static_cast<uint32_t>(misc[1]), 0);

    const int tiles_up = (g.inner + 63) / 64, kb_up = (g.hidden + 63) / 64;
    const int tiles = P != UP ? (g.hidden + 127) / 128 : tiles_up;
    const Cut cut(chosen * tiles, P != UP ? tiles_up : kb_up, g.sms, P != UP ? g.parts_down : g.parts_up);
    const uint32_t rows_bytes = static_cast<uint32_t>((most + 15) / 16 * 16 * 128);   // the activations of a K block (16-bit values)
    const uint32_t stage_bytes = kWeightBytes + rows_bytes * (P != UP ? 2 : 1);
    const int stages = min(kMoeStages, static_cast<int>(g.ring_bytes / stage_bytes));
    Walker walk(cut, tiles, blockIdx.x);
    Segment s;
    int st = 0;
    uint32_t ph = 0;

    if (warp == 0) {
        // -------------------------------------------------------------- weights: TMA
        const bool issuer = elect_one();
        const uint64_t once = l2_policy(1);
        bool ok = true;
        Walker ahead = walk;
        Segment f;
        int fst = 0, fkb = 0, filled = 0;
        if (P == DOWN) {
            // the weights of the first stages do not depend on the kernels before: on their way before the wait
            while (filled < stages && ahead.next(f)) {
                const int row = expert_s[f.ai] * g.hidden + f.tile * 128;
                for (fkb = f.kb0; fkb < f.kb1 && filled < stages; ++fkb, ++filled, ++fst)
                    if (issuer) {
                        mbar_arrive_expect_tx(full0 + 8 * fst, kWeightBytes + (count_s[f.ai] + 15) / 16 * 2 * kBoxBytes);
                        tma_load_2d_hint(ring + fst * stage_bytes, &g.map, full0 + 8 * fst, fkb * 64, row, once);
                    }
            }
            griddep_wait();
        }
        while (ok && walk.next(s)) {
            const int e = expert_s[s.ai];
            const int boxes = (count_s[s.ai] + 15) / 16;
            const int row = P != UP ? e * g.hidden + s.tile * 128 : e * 2 * g.inner + s.tile * 64;
            for (int kb = s.kb0; kb < s.kb1; ++kb) {
                if (P == DOWN && filled > 0) {
                    --filled;                              // its weights are on their way
                } else {
                    ok = wait_warp(empty0 + 8 * st, ph ^ 1u, wait, 1000 + st);
                    if (!ok) break;
                    if (issuer) {
                        const uint32_t bar = full0 + 8 * st, dst = ring + st * stage_bytes;
                        mbar_arrive_expect_tx(bar, kWeightBytes + (P == DOWN ? boxes * 2 * kBoxBytes : 0));
                        tma_load_2d_hint(dst, &g.map, bar, kb * 64, row, once);
                        if (P == UP) tma_load_2d_hint(dst + kWeightBytes / 2, &g.map, bar, kb * 64, row + g.inner, once);
                    }
                }
                if (P == DOWN && issuer) {
                    const uint32_t bar = full0 + 8 * st, dst = ring + st * stage_bytes + kWeightBytes;
                    for (int b = 0; b < boxes; ++b) {
                        tma_load_2d(dst + b * kBoxBytes, &g.map_h, bar, kb * 64, base_s[s.ai] + 16 * b);
                        tma_load_2d(dst + rows_bytes + b * kBoxBytes, &g.map_h, bar, kb * 64, g.slots + base_s[s.ai] + 16 * b);
                    }
                }
                if (++st == stages) st = 0, ph ^= 1u;
            }
        }
    } else if (warp == 1) {
        // -------------------------------------------------------------- MMA
        const bool issuer = elect_one();
        bool ok = true;
        for (int n = 0; ok && walk.next(s); ++n) {
            const int acc = n & 1;
            ok = wait_warp(acc_empty0 + 8 * acc, ((n >> 1) & 1) ^ 1u, wait, 1100 + acc);
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t d = tmem + acc * g.slot_cols;
            const uint32_t idesc = g.idesc | static_cast<uint32_t>((count_s[s.ai] + 15) / 16 * 2) << 17;
            for (int kb = s.kb0; kb < s.kb1; ++kb) {
                ok = wait_warp(full0 + 8 * st, ph, wait, 1200 + st);
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t at = ring + st * stage_bytes;
                const uint64_t a = umma_desc_sw128(at), b = umma_desc_sw128(at + kWeightBytes), lo = umma_desc_sw128(at + kWeightBytes + rows_bytes);
                if (issuer) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        umma_f16<1>(d, a + 2 * i, b + 2 * i, idesc, kb > s.kb0 || i > 0);
                        if (P != UP) umma_f16<1>(d, a + 2 * i, lo + 2 * i, idesc, 1);
                    }
                    umma_commit<1>(empty0 + 8 * st);
                }
                if (++st == stages) st = 0, ph ^= 1u;
            }
            if (ok && issuer) umma_commit<1>(acc_full0 + 8 * acc);
        }
        __syncwarp();
    } else if (warp < 6) {
        // -------------------------------------------------------------- accumulators -> parts in the workspace
        const int quarter = warp & 3;
        const int r = quarter * 32 + lane;                 // row of the tile
        bool ok = true;
        if (P != UP) griddep_wait();                          // in every CTA, with work or without: DOWN must not complete before UP
        for (int n = 0; ok && walk.next(s); ++n) {
            const int acc = n & 1, count = count_s[s.ai];
            const int64_t slot = static_cast<int64_t>(s.part) * g.slots + base_s[s.ai];
            float *out;
            int pitch;
            bool mine;
            if (P != UP) {
                mine = s.tile * 128 + r < g.hidden;
                pitch = g.hidden;
                out = g.o + slot * pitch + s.tile * 128 + r;
            } else {
                const int i = s.tile * 64 + (r & 63);
                mine = i < g.inner;
                pitch = 2 * g.inner;
                out = g.z + slot * pitch + (r < 64 ? i : g.inner + i);
            }
            ok = wait_warp(acc_full0 + 8 * acc, (n >> 1) & 1, wait, 1300 + acc);
            if (!ok) break;
            tc_fence_after_sync();
            for (int c = 0; c < count; c += 16) {
                uint32_t v[16];
                tmem_ld_32x16(tmem + acc * g.slot_cols + c + (static_cast<uint32_t>(quarter * 32) << 16), v);
                tmem_ld_wait();
                if (mine) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (c + j < count) out[static_cast<int64_t>(c + j) * pitch] = __uint_as_float(v[j]);
                }
                __syncwarp();
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty0 + 8 * acc);
        }
    } else if (P != DOWN) {
        // -------------------------------------------------------------- activations
        // The loader warps form groups that take the K blocks in turn, so that the latency of a block's loads is spread over
        // several blocks. A group looks at a stage only when its own turn comes; the phase it waits for cannot be
        // mistaken for the one two before it as long as there are no more groups than stages.
        const int group_warps = stages >= 8 ? 1 : stages >= 4 ? 2 : 4, groups = kMoeLoaders / group_warps;
        const int mine = (warp - 6) / group_warps, chunk = lane & 7;
        const int row0 = (warp - 6) % group_warps * 4 + (lane >> 3), row_step = 4 * group_warps;
        const Cut up(chosen * tiles_up, kb_up, g.sms, g.parts_up);
        const int64_t part_pitch = static_cast<int64_t>(g.slots) * 2 * g.inner;
        int turn = 0;
        bool ok = true;
        if (P != UP) griddep_wait();
        while (ok && walk.next(s)) {
            const int count = count_s[s.ai], base = base_s[s.ai];
            for (int kb = s.kb0; kb < s.kb1; ++kb) {
                if (turn == mine) {
                    ok = wait_warp(empty0 + 8 * st, ph ^ 1u, wait, 1400 + st);
                    if (!ok) break;
                    const uint32_t dst = ring + st * stage_bytes + kWeightBytes;
                    const int k = kb * 64 + chunk * 8;
                    if (P == UP) {
                        for (int r = row0; r < count; r += row_step) {
                            if (k < g.hidden) cp_async_16(dst + swizzled(r, chunk), g.X + static_cast<int64_t>(token_s[base + r]) * g.hidden + k);
                            else st_shared_v4(dst + swizzled(r, chunk), make_uint4(0, 0, 0, 0));
                        }
                        cp_async_wait_all();
                    } else {
                        const int unit = s.ai * tiles_up + kb, parts = up.num_parts(unit);
                        for (int r = row0; r < count; r += row_step) {
                            uint32_t hi[4] = {}, lo[4] = {};
                            if (k < g.inner) gated_values<T>(g.z + static_cast<int64_t>(base + r) * 2 * g.inner + k, g.inner, parts, part_pitch, hi, lo);
                            st_shared_v4(dst + swizzled(r, chunk), make_uint4(hi[0], hi[1], hi[2], hi[3]));
                            st_shared_v4(dst + rows_bytes + swizzled(r, chunk), make_uint4(lo[0], lo[1], lo[2], lo[3]));
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_many(full0 + 8 * st, 4 / group_warps);
                }
                if (++turn == groups) turn = 0;
                if (++st == stages) st = 0, ph ^= 1u;
            }
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
        tmem_dealloc<1>(tmem, g.tmem_cols);
    }
}

// The gated values for DOWN: eight inner rows of one slot per thread.
template <typename T>
__global__ void __launch_bounds__(256) moe_gate_kernel(const __grid_constant__ MoeArgs g) {
    griddep_launch_dependents();   // DOWN reads nothing of this kernel before its own wait
    griddep_wait();
    const int chunks = g.inner / 8, tiles = (g.inner + 63) / 64;
    const int at = blockIdx.x * 256 + threadIdx.x, slot = at / chunks, k = (at - slot * chunks) * 8;
    const int chosen = __ldcg(g.list.header);
    if (slot >= g.slots || chosen == 0) return;
    // the expert of a slot: the last one whose first slot is not behind it
    int lo_ai = 0, hi_ai = chosen - 1;
    while (lo_ai < hi_ai) {
        const int mid = (lo_ai + hi_ai + 1) >> 1;
        if (__ldcg(g.list.base + mid) <= slot) lo_ai = mid;
        else hi_ai = mid - 1;
    }
    if (slot >= __ldcg(g.list.base + lo_ai) + __ldcg(g.list.count + lo_ai)) return;
    const Cut up(chosen * tiles, (g.hidden + 63) / 64, g.sms, g.parts_up);
    uint32_t hi[4], lo[4];
    gated_values<T>(g.z + static_cast<int64_t>(slot) * 2 * g.inner + k, g.inner, up.num_parts(lo_ai * tiles + k / 64),
                    static_cast<int64_t>(g.slots) * 2 * g.inner, hi, lo);
    *reinterpret_cast<uint4 *>(g.h + static_cast<int64_t>(slot) * g.inner + k) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4 *>(g.h + (static_cast<int64_t>(g.slots) + slot) * g.inner + k) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

// One warp per 128 columns of one token, four per lane: the weighted parts, in ascending order within a choice, choices in
// descending order of their logits. The warp first lists where they are, so that eight loads are in flight at a time.
template <typename T>
__global__ void __launch_bounds__(128) moe_combine_kernel(const __grid_constant__ MoeArgs g) {
    __shared__ int2 entry[4][B200_MOE_MAX_TOP_K * kMaxParts];
    const int t = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tile = blockIdx.x * 4 + warp, n = tile * 128 + lane * 4;
    const int tiles = (g.hidden + 127) / 128;
    griddep_wait();
    griddep_launch_dependents();
    int slot = -1, parts = 0;
    float w = 0.0f;
    if (lane < g.top_k) {
        const Cut cut(__ldcg(g.list.header) * tiles, (g.inner + 63) / 64, g.sms, g.parts_down);
        const int at = t * g.top_k + lane;
        slot = __ldcg(g.list.slot + at);
        w = __ldcg(g.list.weight + at);
        if (slot >= 0 && tile < tiles) parts = cut.num_parts(__ldcg(g.list.active + at) * tiles + tile);
    }
    int before = parts;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    const int total = __shfl_sync(0xffffffffu, before, 31);
    for (int p = 0; p < parts; ++p) entry[warp][before - parts + p] = make_int2(p * g.slots + slot, __float_as_int(w));
    __syncwarp();
    if (n >= g.hidden) return;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i0 = 0; i0 < total; i0 += 8) {
        float4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i0 + i < total) v[i] = __ldcg(reinterpret_cast<const float4 *>(g.o + static_cast<int64_t>(entry[warp][i0 + i].x) * g.hidden + n));
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i0 + i < total) {
                const float f = __int_as_float(entry[warp][i0 + i].y);
                y.x = fmaf(f, v[i].x, y.x), y.y = fmaf(f, v[i].y, y.y), y.z = fmaf(f, v[i].z, y.z), y.w = fmaf(f, v[i].w, y.w);
            }
    }
    uint2 out;
    out.x = T::round(y.x) | static_cast<uint32_t>(T::round(y.y)) << 16;
    out.y = T::round(y.z) | static_cast<uint32_t>(T::round(y.w)) << 16;
    *reinterpret_cast<uint2 *>(g.Y + static_cast<int64_t>(t) * g.hidden + n) = out;
}

int check_moe(int64_t tokens, int64_t hidden, int64_t inner, int64_t experts, int top_k) {
    if (tokens <= 0 || tokens > B200_MOE_MAX_TOKENS || hidden <= 0 || inner <= 0 || hidden % 8 || inner % 8) return B200_INVALID_SHAPE;
    if (hidden > 65536 || inner > 65536 || experts <= 0 || experts > B200_MOE_MAX_EXPERTS) return B200_INVALID_SHAPE;
    if (top_k < 1 || top_k > B200_MOE_MAX_TOP_K || top_k > experts) return B200_INVALID_CONFIG;
    return B200_OK;
}

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

// CTAs that may share a tile: what the cut needs when every token chooses the same experts, and one more for stretches that
// do not start at a tile. Fewer experts than that (masked logits) are cut more coarsely than they could be.
int most_parts(int64_t units, int64_t kblocks) {
    const int64_t len = (units * kblocks + kGridSms - 1) / kGridSms;
    const int64_t parts = (kblocks - 1 + len - 1) / len + 1;
    return static_cast<int>(parts < 2 ? 2 : parts > kMaxParts ? kMaxParts : parts);
}

struct MoeLayout {
    int parts_up, parts_down;
    bool gate_kernel;
    int64_t off_list, off_z, off_o, off_h, bytes;
};

MoeLayout moe_layout(int64_t tokens, int64_t hidden, int64_t inner, int64_t experts, int top_k) {
    MoeLayout l;
    const int64_t slots = tokens * top_k, up_tiles = (inner + 63) / 64;
    l.parts_up = most_parts(top_k * up_tiles, (hidden + 63) / 64);
    l.parts_down = most_parts(top_k * ((hidden + 127) / 128), up_tiles);
    l.off_list = 0;
    l.off_z = up256((2 + 3 * experts + 4 * slots) * 4);
    l.off_o = l.off_z + up256(l.parts_up * slots * 2 * inner * 4);
    l.off_h = l.off_o + up256(l.parts_down * slots * hidden * 4);
    l.gate_kernel = tokens > kFewTokens;
    l.bytes = l.off_h + (l.gate_kernel ? up256(2 * slots * inner * 2) : 0);
    return l;
}

template <typename T>
cudaError_t launch_moe(MoeArgs &g, const CUtensorMap &up, const CUtensorMap &down, bool gate_kernel, int smem, cudaStream_t stream) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cfg.gridDim = dim3((g.tokens + 31) / 32);
    cfg.blockDim = dim3(1024);
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cfg.gridDim.x;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, moe_route_kernel, g);
    cfg.numAttrs = 1;
    cfg.gridDim = dim3(g.sms);
    cfg.blockDim = dim3(kMoeThreads);
    cfg.dynamicSmemBytes = smem;
    g.map = up;
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, moe_product_kernel<T, UP>, g);
    if (gate_kernel) {
        cfg.gridDim = dim3(static_cast<unsigned>((static_cast<int64_t>(g.slots) * (g.inner / 8) + 255) / 256));
        cfg.blockDim = dim3(256);
        cfg.dynamicSmemBytes = 0;
        if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, moe_gate_kernel<T>, g);
    }
    cfg.gridDim = dim3(g.sms);
    cfg.blockDim = dim3(kMoeThreads);
    cfg.dynamicSmemBytes = smem;
    g.map = down;
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, gate_kernel ? moe_product_kernel<T, DOWN> : moe_product_kernel<T, DOWN_INLINE>, g);
    cfg.gridDim = dim3((g.hidden + 511) / 512, g.tokens);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = 0;
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, moe_combine_kernel<T>, g);
    return e;
}

}  // namespace

int prepare_moe_kernels() {
    void (*const kernels[])(MoeArgs) = {moe_product_kernel<Bf16, UP>, moe_product_kernel<Bf16, DOWN_INLINE>, moe_product_kernel<Bf16, DOWN>,
                                        moe_product_kernel<Fp16, UP>, moe_product_kernel<Fp16, DOWN_INLINE>, moe_product_kernel<Fp16, DOWN>};
    for (const auto k : kernels) {
        const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
        if (e != cudaSuccess) return static_cast<int>(e);
    }
    return 0;
}

}  // namespace b200

extern "C" int64_t b200_moe_workspace_bytes(int64_t tokens, int64_t hidden, int64_t inner, int64_t experts, int top_k) {
    if (b200::check_moe(tokens, hidden, inner, experts, top_k) != B200_OK) return -1;
    return b200::moe_layout(tokens, hidden, inner, experts, top_k).bytes;
}
extern "C" int b200_moe(int dtype, const void *X, const float *logits, const void *W13, const void *W2, void *Y, int *ids, float *weights,
                        int64_t tokens, int64_t hidden, int64_t inner, int64_t experts, int top_k, int normalise, void *workspace,
                        size_t workspace_bytes, void *stream) {
    using namespace b200;
    if (dtype != B200_F16 && dtype != B200_BF16) return B200_INVALID_CONFIG;
    if (normalise != 0 && normalise != 1) return B200_INVALID_CONFIG;
    int st = check_moe(tokens, hidden, inner, experts, top_k);
    if (st != B200_OK) return st;
    if (!X || !logits || !W13 || !W2 || !Y) return B200_INVALID_POINTER;
    if (misaligned(X) || misaligned(W13) || misaligned(W2) || misaligned(Y) || misaligned(workspace) ||
        ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(ids) | reinterpret_cast<uintptr_t>(weights)) & 3u))
        return B200_INVALID_POINTER;
    const int64_t need = b200_moe_workspace_bytes(tokens, hidden, inner, experts, top_k);
    if (!workspace || workspace_bytes < static_cast<size_t>(need)) return B200_WORKSPACE_TOO_SMALL;
    const struct { const void *p; int64_t n; } in[] = {{X, tokens * hidden * 2}, {logits, tokens * experts * 4}, {W13, experts * 2 * inner * hidden * 2},
                                                       {W2, experts * hidden * inner * 2}};
    const struct { const void *p; int64_t n; } out[] = {{Y, tokens * hidden * 2}, {ids, tokens * top_k * 4}, {weights, tokens * top_k * 4}, {workspace, need}};
    for (int o = 0; o < 4; ++o) {
        for (const auto &i : in)
            if (overlap(out[o].p, out[o].n, i.p, i.n)) return B200_INVALID_POINTER;
        for (int p = 0; p < o; ++p)
            if (overlap(out[o].p, out[o].n, out[p].p, out[p].n)) return B200_INVALID_POINTER;
    }
    MoeArgs g = {};
    st = current_device(&g.sms, &g.status);
    if (st != B200_OK) return st;
    CUtensorMap up, down;
    st = encode_operand_map(&up, dtype, W13, hidden, experts * 2 * inner, 64);
    if (st == B200_OK) st = encode_operand_map(&down, dtype, W2, inner, experts * hidden, 128);
    const MoeLayout l = moe_layout(tokens, hidden, inner, experts, top_k);
    uint8_t *const ws = static_cast<uint8_t *>(workspace);
    const int64_t slots = tokens * top_k;
    g.h = reinterpret_cast<uint16_t *>(ws + l.off_h);
    if (st == B200_OK && l.gate_kernel) st = encode_operand_map(&g.map_h, dtype, g.h, inner, 2 * slots, 16);
    if (st != B200_OK) return st;
    int *const list = reinterpret_cast<int *>(ws + l.off_list);
    g.list.header = list;
    g.list.expert = list + 2;
    g.list.count = g.list.expert + experts;
    g.list.base = g.list.count + experts;
    g.list.token = g.list.base + experts;
    g.list.slot = g.list.token + slots;
    g.list.active = g.list.slot + slots;
    g.list.weight = reinterpret_cast<float *>(g.list.active + slots);
    g.z = reinterpret_cast<float *>(ws + l.off_z);
    g.o = reinterpret_cast<float *>(ws + l.off_o);
    g.X = static_cast<const uint16_t *>(X);
    g.logits = logits;
    g.Y = static_cast<uint16_t *>(Y);
    g.ids_out = ids;
    g.weights_out = weights;
    g.tokens = static_cast<int>(tokens);
    g.hidden = static_cast<int>(hidden);
    g.inner = static_cast<int>(inner);
    g.experts = static_cast<int>(experts);
    g.top_k = top_k;
    g.normalise = normalise;
    g.slots = static_cast<int>(slots);
    g.parts_up = l.parts_up;
    g.parts_down = l.parts_down;
    // Two accumulators of up to `tokens` columns. While the tokens are few a CTA takes less than half of an SM's shared memory,
    // so that DOWN can start beside UP; more tokens need the larger ring (a K block of DOWN is up to 80 KB then).
    g.slot_cols = static_cast<int>((tokens + 15) / 16 * 16);
    g.tmem_cols = pow2_at_least(2 * g.slot_cols);
    const int lists = static_cast<int>(up256(slots * 2) + up256(experts * 12));
    const int smem = tokens <= kFewTokens ? 113 * 1024 : kSmemLimit;
    g.ring_bytes = (smem - 1024 - lists - 512) / 1024 * 1024;
    g.off_token = g.ring_bytes;
    g.off_expert = g.off_token + static_cast<int>(up256(slots * 2));
    g.off_bars = g.ring_bytes + lists;
    g.off_misc = g.off_bars + (2 * kMoeStages + 4) * 8;
    g.idesc = umma_idesc(128, 0, dtype == B200_BF16);
    g.budget = wait_budget_cycles();
    const cudaError_t e = dtype == B200_BF16 ? launch_moe<Bf16>(g, up, down, l.gate_kernel, smem, static_cast<cudaStream_t>(stream))
                                             : launch_moe<Fp16>(g, up, down, l.gate_kernel, smem, static_cast<cudaStream_t>(stream));
    return e != cudaSuccess ? record_cuda_error(e) : B200_OK;
}
