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
// Up to 128 (token, choice) pairs, two kernels (three with fp16):
//   moe_product_kernel<UP_FEW>    every CTA makes the router's choice for itself (the logits are few), then its stretch of G and U: a tile
//                                 is 64 rows of G and the same 64 rows of U; sums (fp32) to the workspace
//   moe_product_kernel<DOWN_FEW>  a tile is 128 rows of W2; loader warps add the parts of a K block, apply silu and the gate, and hand the
//                                 result to the tensor core as a pair of 16-bit numbers, value and remainder (two MMAs per
//                                 K step: the tensor core idles here, and one 16-bit rounding of the gated value would
//                                 cost as much accuracy as the rounding of the result); the last CTA of a tile of Y adds
//                                 its parts and the weighted choices. With fp16 the pairs have to be scaled, for which a
//                                 slot's largest value has to be known: moe_gate_kernel makes them in between, at the price of
//                                 a kernel in the chain (2 tokens, 8 experts of 1024 x 512, top 2: 15.5 us with bf16, 20.0 with
//                                 fp16; one token, 8 of 128 experts of 2048 x 768: 28.6 and 33.1; 16 tokens, 64 experts of 4096 x
//                                 2048, top 6: 398 and 406)
// beyond that five, because each CTA would spend too long on the choice, the gated values and the last sums (48 tokens, 32 experts
// of 1024 x 512, top 4: 38 against 41 us; 256 tokens, 128 experts of 2048 x 768, top 8: 230 against 404):
//   moe_route_kernel              a cluster of up to eight blocks: the choice per token (one warp each), the chosen experts' tokens
//   moe_product_kernel<UP>        as above, with two 64 + 64 row atoms per tile
//   moe_gate_kernel               the gated values of all slots, as pairs, scaled with fp16
//   moe_product_kernel<DOWN>      as above, the pairs by TMA, two 128-row atoms per tile
//   moe_combine_kernel            parts and weighted choices of a token, one rounding
//
// All are launched as programmatic dependents: DOWN_FEW starts as soon as UP_FEW runs (two CTAs fit an SM), fills its ring with weights and
// waits only before it reads UP's sums. Measured as device time in a graph, bf16: 16 tokens, 64 experts of 4096 x 2048, top 6, 398 us:
// 6.4 TB/s, 98 % of the copy rate; 64 tokens, experts of 4096 x 1408, 354 us, 95 %; 256 tokens as above 229 us, 80 %: the
// activations and sums of 2048 slots cross the L2 beside the weights; one token, 8 of 128 experts of 2048 x 768, 28.6 us, 40 %:
// the choice, two starts and two joins frame 11 us of reading.
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
constexpr int kMaxHidden = 65536;
constexpr int kTileWords = kMaxHidden / 128 / 32;   // a bit per tile of Y
constexpr int kFewSlots = 128;      // (token, choice) pairs and tokens up to which two kernels do all of it; the tokens also
constexpr int kFewTokens = 64;      // bound a stage of the smaller ring, which must hold two
constexpr int kGridSms = 148;       // what the workspace is sized for; another count only changes how tiles are cut
constexpr int kGateThreads = 256;   // most threads of a block of moe_gate_kernel, most blocks of a slot, quads that a thread keeps
constexpr int kGateBlocks = 8;
constexpr int kGateQuads = 2;
constexpr int kBoxBytes = 16 * 128;      // 16 slots of 64 gated values
constexpr int kWeightBytes = 128 * 128;  // one K block of a weight tile: 128 rows of 64 elements

// What the route kernel leaves for the others, in the workspace.
struct Lists {
    int *header;     // [0] chosen experts, [1] most tokens of one, [2] slots
    int *expert;     // per chosen expert: its index, its number of tokens, the first of its slots
    int *count;
    int *base;
    int *token;      // per slot (sorted by expert, then token): its token
    int *owner;      // per slot: the position of its expert in the list of chosen ones
    int *slot;       // per (token, choice): its slot, -1 without one
    int *active;     // per (token, choice): the position of its expert in the list of chosen ones
    float *weight;   // per (token, choice)
    float *unscale;  // per slot, fp16: the power of two that its gated values, as DOWN sees them, have to be multiplied with
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
    uint16_t *h;              // [value, remainder][slot][inner]: gated values, scaled
    int tokens, hidden, inner, experts, top_k, normalise, slots;
    int parts_up, parts_down;
    int sms;
    int ring_bytes, off_slots, off_experts, off_bars, off_misc;
    int tmem_cols, slot_cols;
    uint32_t idesc;           // with N = 0
    int *arrived;             // few: per tile of Y, the warps that are done with it
    int *status;
    long long budget;
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
        int e = lane + 32 * best_i, winner = best == most;
        const uint32_t equal = __ballot_sync(0xffffffffu, winner);
        int from = __ffs(equal) - 1;
        if (equal & (equal - 1u)) {   // several lanes: the lowest index wins
            const int low = static_cast<int>(__reduce_min_sync(0xffffffffu, winner ? static_cast<uint32_t>(e) : 0xffffffffu));
            from = low & 31;
            winner = lane == from;
        }
        e = __shfl_sync(0xffffffffu, e, from);
        if (lane == j) id = e, chosen = most;
        if (winner) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (i == best_i) key[i] = 0u;
            look();
        }
        __syncwarp();
    }
    weight = id >= 0 ? expf(key_logit(chosen) - top) : 0.0f;
    if (normalise) sum = warp_sum(weight);
    if (id >= 0) weight /= sum;
}

__device__ __forceinline__ void choose(const MoeArgs &g, int t, int lane, int &id, float &weight) {
    const float *const row = g.logits + static_cast<int64_t>(t) * g.experts;
    if (g.experts <= 32) choose_experts<1>(row, g.experts, g.top_k, g.normalise, lane, id, weight);
    else if (g.experts <= 64) choose_experts<2>(row, g.experts, g.top_k, g.normalise, lane, id, weight);
    else if (g.experts <= 128) choose_experts<4>(row, g.experts, g.top_k, g.normalise, lane, id, weight);
    else if (g.experts <= 256) choose_experts<8>(row, g.experts, g.top_k, g.normalise, lane, id, weight);
    else choose_experts<16>(row, g.experts, g.top_k, g.normalise, lane, id, weight);
}

// One warp: emit(position among the chosen, expert, tokens, first slot) for every expert that a token chose, in ascending order;
// mask[e * words ..] holds the tokens of expert e as bits. Returns how many are chosen, the most tokens of one, and the slots.
template <typename Emit>
__device__ __forceinline__ int3 list_experts(const uint32_t *mask, int words, int experts, int lane, Emit emit) {
    int chosen = 0, slots = 0, most = 0;
    for (int e0 = 0; e0 < experts; e0 += 32) {
        const int e = e0 + lane;
        int n = 0;
        if (e < experts)
            for (int i = 0; i < words; ++i) n += __popc(mask[e * words + i]);
        const uint32_t ballot = __ballot_sync(0xffffffffu, n > 0);
        if (ballot == 0u) continue;
        int before = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += v;
        }
        if (n > 0) emit(chosen + __popc(ballot & ((1u << lane) - 1u)), e, n, slots + before - n);
        chosen += __popc(ballot);
        slots += __shfl_sync(0xffffffffu, before, 31);
        most = max(most, static_cast<int>(__reduce_max_sync(0xffffffffu, static_cast<uint32_t>(n))));
    }
    return make_int3(chosen, most, slots);
}

// The place of token t among the tokens of its expert.
__device__ __forceinline__ int rank_of(const uint32_t *mask, int words, int e, int t) {
    int r = __popc(mask[e * words + (t >> 5)] & ((1u << (t & 31)) - 1u));
    for (int i = 0; i < (t >> 5); ++i) r += __popc(mask[e * words + i]);
    return r;
}

// One cluster of up to eight blocks, a warp per token; its first block then lists the chosen experts and their tokens.
__global__ void __launch_bounds__(1024) moe_route_kernel(const __grid_constant__ MoeArgs g) {
    __shared__ uint32_t mask[B200_MOE_MAX_EXPERTS * (B200_MOE_MAX_TOKENS / 32)];   // the tokens of an expert (of the first block)
    __shared__ short place[B200_MOE_MAX_EXPERTS];                                  // its position among the chosen
    __shared__ int first[B200_MOE_MAX_EXPERTS];                                    // its first slot
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int words = (g.tokens + 31) / 32;
    if (blockIdx.x == 0)
        for (int i = tid; i < g.experts * words; i += 1024) mask[i] = 0u;
    cluster_arrive();
    griddep_wait();
    griddep_launch_dependents();
    const int t = blockIdx.x * 32 + warp;
    int id = -1;
    float w = 0.0f;
    if (t < g.tokens) choose(g, t, lane, id, w);
    cluster_wait();                                         // the first block's masks are zero
    if (t < g.tokens && lane < g.top_k) {
        const int at = t * g.top_k + lane;
        g.list.slot[at] = id;                               // the expert for now
        g.list.weight[at] = w;
        if (g.ids_out) g.ids_out[at] = id;
        if (g.weights_out) g.weights_out[at] = w;
        if (id >= 0) red_or_cluster(mapa_shared(smem_u32(&mask[id * words + (t >> 5)]), 0), 1u << (t & 31));
    }
    cluster_arrive();
    cluster_wait();
    if (blockIdx.x != 0) return;
    if (warp == 0) {
        const int3 n = list_experts(mask, words, g.experts, lane, [&](int at, int e, int count, int base) {
            g.list.expert[at] = e;
            g.list.count[at] = count;
            g.list.base[at] = base;
            place[e] = static_cast<short>(at);
            first[e] = base;
        });
        if (lane == 0) {
            g.list.header[0] = n.x;
            g.list.header[1] = n.y;
            g.list.header[2] = n.z;
        }
    }
    __syncthreads();
    for (int at = tid; at < g.slots; at += 1024) {
        const int t = at / g.top_k, e = __ldcg(g.list.slot + at);
        if (e < 0) continue;
        const int slot = first[e] + rank_of(mask, words, e, t);
        g.list.token[slot] = t;
        g.list.owner[slot] = place[e];
        g.list.slot[at] = slot;
        g.list.active[at] = place[e];
    }
}

// The stretch of one CTA, cut at tile borders: K blocks [kb0, kb1) of tile `tile` of chosen expert `ai`.
struct Segment {
    int ai, tile, kb0, kb1, part;
};

// Tiles in a row are those of one expert, or with BY_TILE the experts of one tile.
template <bool BY_TILE>
struct Walker {
    int q, end, tiles, chosen, cta;
    Cut cut;
    __device__ __forceinline__ Walker(const Cut &c, int tiles_, int chosen_, int cta_) : tiles(tiles_), chosen(chosen_), cta(cta_), cut(c) {
        q = min(static_cast<long long>(cta) * c.len, static_cast<long long>(c.total));
        end = min(q + c.len, c.total);
    }
    __device__ __forceinline__ bool next(Segment &s) {
        if (q >= end) return false;
        const int unit = q / cut.kblocks;
        if (BY_TILE) {
            s.tile = unit / chosen;
            s.ai = unit - s.tile * chosen;
        } else {
            s.ai = unit / tiles;
            s.tile = unit - s.ai * tiles;
        }
        s.kb0 = q - unit * cut.kblocks;
        s.kb1 = min(cut.kblocks, s.kb0 + end - q);
        s.part = cta - cut.first_cta(unit);
        q += s.kb1 - s.kb0;
        return true;
    }
};

// 128-row atoms of the weights per tile. With more than a few tokens two share the activations of a K block, which halves what those
// cost between L2 and SM (256 tokens, 128 experts of 2048 x 768: 0.44 GB of activations beside 0.41 GB of W2), as long as
// two accumulators of both fit the tensor memory.
__device__ __forceinline__ int tile_atoms(const MoeArgs &g, int most) { return 4 * ((most + 15) / 16 * 16) <= g.tmem_cols ? 2 : 1; }

enum Product {
    UP,        // gate and up rows times the tokens of X, gathered by the loader warps
    DOWN,      // W2 times the gated values that moe_gate_kernel has left in the workspace, by TMA
    UP_FEW,    // UP where every CTA makes the router's choice for itself
    DOWN_FEW   // so does this one; its loader warps compute the gated values from UP's parts, and the last CTA to finish a tile
               // of Y adds the tile's parts
};

// The gated values of four neighbouring inner rows of one slot from UP's parts (ascending, BATCH of them in flight). The quick exponential
// errs by up to 2 + |1.173 gate| units of 2^-23, where the gate is negative undiminished in silu too: 2^-21 near zero, 2^-19 at
// -10, 2^-17 at -46; the quick quotient by two units, and it is zero for gates below -87.3. That is a 64th of what fp16's rounding
// of the result costs at -46, a 512th of bf16's, and more than the pair of an fp16 loses (2^-22). expf and a rounded quotient measured
// 29.2 -> 30.4 us (64 tokens, 8 experts of 1024 x 512, top 2), 398 -> 401 (16 tokens, 64 experts of 4096 x 2048, top 6).
template <int BATCH>
__device__ __forceinline__ float4 gated_values(const float *z, int inner, int parts, int64_t part_pitch) {
    float4 gate = make_float4(0.0f, 0.0f, 0.0f, 0.0f), up = gate;
    for (int p0 = 0; p0 < parts; p0 += BATCH, z += BATCH * part_pitch) {
        float4 a[BATCH], b[BATCH];
#pragma unroll
        for (int p = 0; p < BATCH; ++p)
            if (p0 + p < parts) {
                a[p] = __ldcg(reinterpret_cast<const float4 *>(z + p * part_pitch));
                b[p] = __ldcg(reinterpret_cast<const float4 *>(z + p * part_pitch + inner));
            }
#pragma unroll
        for (int p = 0; p < BATCH; ++p)
            if (p0 + p < parts) {
                gate.x += a[p].x, gate.y += a[p].y, gate.z += a[p].z, gate.w += a[p].w;
                up.x += b[p].x, up.y += b[p].y, up.z += b[p].z, up.w += b[p].w;
            }
    }
    const auto gated = [](float g, float u) { return __fdividef(g, 1.0f + __expf(-g)) * u; };
    return make_float4(gated(gate.x, up.x), gated(gate.y, up.y), gated(gate.z, up.z), gated(gate.w, up.w));
}

template <typename T>
__device__ __forceinline__ void split_four(const float4 &v, uint2 &hi, uint2 &lo) {   // as pairs of 16-bit numbers
    uint16_t h[4], l[4];
    T::split(v.x, h[0], l[0]);
    T::split(v.y, h[1], l[1]);
    T::split(v.z, h[2], l[2]);
    T::split(v.w, h[3], l[3]);
    hi = make_uint2(h[0] | static_cast<uint32_t>(h[1]) << 16, h[2] | static_cast<uint32_t>(h[3]) << 16);
    lo = make_uint2(l[0] | static_cast<uint32_t>(l[1]) << 16, l[2] | static_cast<uint32_t>(l[3]) << 16);
}

// One warp, 128 columns of one token, four per lane from n on: the weighted parts, in ascending order within a choice, choices in
// descending order of their logits. Lane j < top_k brings choice j: its slot, the number of its parts in these
// columns, its weight. The warp first lists where the parts are, so that four loads are in flight at a time; eight, and
// with them a longer stretch of code that runs once per launch and has to be fetched for that, measured slower
// (one token, 8 of 128 experts of 2048 x 768: 28.7 against 34.4 us for the layer).
template <typename T>
__device__ __forceinline__ void combine(const MoeArgs &g, int2 *entry, int t, int n, int lane, int slot, int parts, float w) {
    constexpr int kBatch = 4;
    int before = parts;
#pragma unroll 1
    for (int o = 1; o < B200_MOE_MAX_TOP_K; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    const int total = __shfl_sync(0xffffffffu, before, B200_MOE_MAX_TOP_K - 1);
    __syncwarp();
    for (int p = 0; p < parts; ++p) entry[before - parts + p] = make_int2(p * g.slots + slot, __float_as_int(w));
    __syncwarp();
    if (n >= g.hidden) return;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i0 = 0; i0 < total; i0 += kBatch) {
        float4 v[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (i0 + i < total) v[i] = __ldcg(reinterpret_cast<const float4 *>(g.o + static_cast<int64_t>(entry[i0 + i].x) * g.hidden + n));
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (i0 + i < total) {
                const float f = __int_as_float(entry[i0 + i].y);
                y.x = fmaf(f, v[i].x, y.x), y.y = fmaf(f, v[i].y, y.y), y.z = fmaf(f, v[i].z, y.z), y.w = fmaf(f, v[i].w, y.w);
            }
    }
    store_four<T>(g.Y + static_cast<int64_t>(t) * g.hidden + n, y);
}

template <typename T, Product P>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_product_kernel(const __grid_constant__ MoeArgs g) {
    constexpr bool kUp = P == UP || P == UP_FEW, kFew = P == UP_FEW || P == DOWN_FEW;
    constexpr bool kGated = P == DOWN || (P == DOWN_FEW && T::kScaled);   // moe_gate_kernel has left the gated values
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t ring = (raw + 1023u) & ~1023u;
    uint8_t *const sm = smem_raw + (ring - raw);
    float *const weight_s = reinterpret_cast<float *>(sm + g.off_slots);                    // few: per (token, choice)
    uint16_t *const token_s = reinterpret_cast<uint16_t *>(weight_s + (kFew ? g.slots : 0));   // per slot
    int16_t *const slot_s = reinterpret_cast<int16_t *>(token_s + g.slots);                 // few: per (token, choice), -1 without an expert
    int16_t *const active_s = slot_s + g.slots;                                             // few: per (token, choice)
    int *const expert_s = reinterpret_cast<int *>(sm + g.off_experts);
    int *const count_s = expert_s + g.experts, *const base_s = count_s + g.experts;
    uint32_t *const mask_s = reinterpret_cast<uint32_t *>(base_s + g.experts);              // few
    const int words = (g.tokens + 31) / 32;
    int16_t *const place_s = reinterpret_cast<int16_t *>(mask_s + g.experts * words);       // few
    const uint32_t full0 = ring + g.off_bars, empty0 = full0 + 8 * kMoeStages, acc_full0 = empty0 + 8 * kMoeStages, acc_empty0 = acc_full0 + 16;
    volatile int *const misc = reinterpret_cast<volatile int *>(sm + g.off_misc);   // abort flag, tensor-memory base, chosen experts, most tokens; few: tiles to add
    const WaitCtx wait = {g.status, misc, g.budget};
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);

    if (tid < 2 * kMoeStages + 4) {
        // full: the producer's byte count and four arrivals of the loader warps; accumulator empty: the four draining warps
        mbar_init(full0 + 8 * tid, tid < kMoeStages ? (kGated ? 1 : 5) : tid < 2 * kMoeStages + 2 ? 1 : 4);
        fence_mbar_init();
    }
    if (tid == 0) misc[0] = 0;
    if (P == DOWN_FEW && tid >= 64 && tid < 64 + kTileWords) misc[4 + tid - 64] = 0;
    if (kFew)
        for (int i = tid; i < g.experts * words; i += kMoeThreads) mask_s[i] = 0u;
    if (tid == 32) tma_prefetch_desc(&g.map);
    if (kGated && tid == 64) tma_prefetch_desc(&g.map_h);
    if (warp == 1) {
        tmem_alloc<1>(ring + g.off_misc + 4, g.tmem_cols);
        tmem_relinquish<1>();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    // UP waits for what came before (the route kernel, or with few tokens all work before the call); every CTA of UP says so
    // before DOWN may start, so DOWN finds lists, logits and weights complete without a wait of its own, and waits later for
    // UP's sums.
    if (kUp) griddep_wait();
    griddep_launch_dependents();
    if (kUp && kFew && blockIdx.x == 0)
        for (int i = tid; i < (g.hidden + 127) / 128; i += kMoeThreads) g.arrived[i] = 0;
    if (kFew && g.tokens == 1) {
        // one token: its choices are the list
        if (warp == 0) {
            int id;
            float w;
            choose(g, 0, lane, id, w);
            const int n = __popc(__ballot_sync(0xffffffffu, id >= 0));
            if (lane < g.top_k) {
                expert_s[lane] = id;
                count_s[lane] = 1;
                base_s[lane] = lane;
                token_s[lane] = 0;
                slot_s[lane] = static_cast<int16_t>(id >= 0 ? lane : -1);
                active_s[lane] = static_cast<int16_t>(lane);
                weight_s[lane] = w;
                if (kUp && blockIdx.x == 0) {
                    if (g.ids_out) g.ids_out[lane] = id;
                    if (g.weights_out) g.weights_out[lane] = w;
                    if (T::kScaled) {
                        g.list.owner[lane] = lane;
                        if (lane == 0) g.list.header[0] = g.list.header[2] = n;
                    }
                }
            }
            if (lane == 0) misc[2] = n, misc[3] = n > 0;
        }
    } else if (kFew) {
        for (int t = warp; t < g.tokens; t += kMoeThreads / 32) {
            int id;
            float w;
            choose(g, t, lane, id, w);
            if (lane < g.top_k) {
                const int at = t * g.top_k + lane;
                slot_s[at] = static_cast<int16_t>(id);         // the expert for now
                weight_s[at] = w;
                if (id >= 0) atomicOr(&mask_s[id * words + (t >> 5)], 1u << (t & 31));
                if (kUp && blockIdx.x == 0) {
                    if (g.ids_out) g.ids_out[at] = id;
                    if (g.weights_out) g.weights_out[at] = w;
                }
            }
        }
        __syncthreads();
        if (warp == 0) {
            const int3 n = list_experts(mask_s, words, g.experts, lane, [&](int at, int e, int count, int base) {
                expert_s[at] = e;
                count_s[at] = count;
                base_s[at] = base;
                place_s[e] = static_cast<int16_t>(at);
            });
            if (lane == 0) {
                misc[2] = n.x, misc[3] = n.y;
                if (kUp && T::kScaled && blockIdx.x == 0) g.list.header[0] = n.x, g.list.header[2] = n.z;
            }
        }
        __syncthreads();
        for (int at = tid; at < g.slots; at += kMoeThreads) {
            const int t = at / g.top_k, e = slot_s[at];
            if (e < 0) continue;
            const int slot = base_s[place_s[e]] + rank_of(mask_s, words, e, t);
            token_s[slot] = static_cast<uint16_t>(t);
            slot_s[at] = static_cast<int16_t>(slot);
            active_s[at] = place_s[e];
            if (kUp && T::kScaled && blockIdx.x == 0) g.list.owner[slot] = place_s[e];
        }
    } else {
        const int n = __ldcg(g.list.header);
        if (tid == 0) misc[2] = n, misc[3] = __ldcg(g.list.header + 1);
        for (int i = tid; i < n; i += kMoeThreads) {
            expert_s[i] = __ldcg(g.list.expert + i);
            count_s[i] = __ldcg(g.list.count + i);
            base_s[i] = __ldcg(g.list.base + i);
        }
        if (kUp)
            for (int i = tid; i < g.slots; i += kMoeThreads) token_s[i] = static_cast<uint16_t>(__ldcg(g.list.token + i));
    }
    __syncthreads();
    const int chosen = __shfl_sync(0xffffffffu, misc[2], 0), most = __shfl_sync(0xffffffffu, misc[3], 0);
    const uint32_t tmem = __shfl_sync(0xffffffffu, static_cast<uint32_t>(misc[1]), 0);

    const int atoms = kFew ? 1 : tile_atoms(g, most);
    const int blocks_up = (g.inner + 63) / 64, kb_up = (g.hidden + 63) / 64, tiles_up = (blocks_up + atoms - 1) / atoms;   // blocks: of one atom
    const int blocks = kUp ? blocks_up : (g.hidden + 127) / 128, tiles = (blocks + atoms - 1) / atoms;
    const Cut cut(chosen * tiles, kUp ? kb_up : blocks_up, g.sms, kUp ? g.parts_up : g.parts_down);
    const uint32_t columns = static_cast<uint32_t>((most + 15) / 16 * 16), acc_cols = kFew ? static_cast<uint32_t>(g.slot_cols) : atoms * columns;
    const uint32_t rows_bytes = columns * 128;             // the activations of a K block (16-bit values)
    const uint32_t rows_at = kWeightBytes * atoms, stage_bytes = rows_at + rows_bytes * (kUp ? 1 : 2);
    const int stages = min(kMoeStages, static_cast<int>(g.ring_bytes / stage_bytes));
    Walker<P == DOWN_FEW> walk(cut, tiles, chosen, blockIdx.x);
    Segment s;
    int st = 0;
    uint32_t ph = 0;

    if (warp == 0) {
        // -------------------------------------------------------------- weights: TMA
        const bool issuer = elect_one();
        const uint64_t once = l2_policy(1);
        bool ok = true;
        Walker<P == DOWN_FEW> ahead = walk;
        Segment f;
        int fst = 0, fkb = 0, filled = 0;
        if (kGated) {
            // the weights of the first stages do not depend on the kernels before: on their way before the wait
            while (filled < stages && ahead.next(f)) {
                const int row = expert_s[f.ai] * g.hidden + f.tile * atoms * 128, na = min(atoms, blocks - f.tile * atoms);
                for (fkb = f.kb0; fkb < f.kb1 && filled < stages; ++fkb, ++filled, ++fst)
                    if (issuer) {
                        mbar_arrive_expect_tx(full0 + 8 * fst, kWeightBytes * na + (count_s[f.ai] + 15) / 16 * 2 * kBoxBytes);
                        for (int a = 0; a < na; ++a) tma_load_2d_hint(ring + fst * stage_bytes + a * kWeightBytes, &g.map, full0 + 8 * fst, fkb * 64, row + a * 128, once);
                    }
            }
            griddep_wait();
        }
        while (ok && walk.next(s)) {
            const int e = expert_s[s.ai];
            const int boxes = (count_s[s.ai] + 15) / 16;
            const int row = kUp ? e * 2 * g.inner + s.tile * atoms * 64 : e * g.hidden + s.tile * atoms * 128;
            const int na = min(atoms, blocks - s.tile * atoms);
            for (int kb = s.kb0; kb < s.kb1; ++kb) {
                if (kGated && filled > 0) {
                    --filled;                              // its weights are on their way
                } else {
                    ok = wait_warp(empty0 + 8 * st, ph ^ 1u, wait, 1000 + st);
                    if (!ok) break;
                    if (issuer) {
                        const uint32_t bar = full0 + 8 * st, dst = ring + st * stage_bytes;
                        mbar_arrive_expect_tx(bar, kWeightBytes * na + (kGated ? boxes * 2 * kBoxBytes : 0));
                        for (int a = 0; a < na; ++a) {
                            const uint32_t to = dst + a * kWeightBytes;
                            tma_load_2d_hint(to, &g.map, bar, kb * 64, row + a * (kUp ? 64 : 128), once);
                            if (kUp) tma_load_2d_hint(to + kWeightBytes / 2, &g.map, bar, kb * 64, row + a * 64 + g.inner, once);
                        }
                    }
                }
                if (kGated && issuer) {
                    const uint32_t bar = full0 + 8 * st, dst = ring + st * stage_bytes + rows_at;
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
            const uint32_t d = tmem + acc * acc_cols;
            const int na = min(atoms, blocks - s.tile * atoms);
            const uint32_t idesc = g.idesc | static_cast<uint32_t>((count_s[s.ai] + 15) / 16 * 2) << 17;
            for (int kb = s.kb0; kb < s.kb1; ++kb) {
                ok = wait_warp(full0 + 8 * st, ph, wait, 1200 + st);
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t at = ring + st * stage_bytes;
                const uint64_t w = umma_desc_sw128(at), b = umma_desc_sw128(at + rows_at), lo = umma_desc_sw128(at + rows_at + rows_bytes);
                if (issuer) {
                    for (int a = 0; a < na; ++a) {
                        const uint64_t wa = w + a * (kWeightBytes >> 4);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            umma_f16<1>(d + a * columns, wa + 2 * i, b + 2 * i, idesc, kb > s.kb0 || i > 0);
                            if (!kUp) umma_f16<1>(d + a * columns, wa + 2 * i, lo + 2 * i, idesc, 1);
                        }
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
        if (!kUp) griddep_wait();                          // in every CTA, with work or without: DOWN must not complete before UP
        for (int n = 0; ok && walk.next(s); ++n) {
            const int acc = n & 1, count = count_s[s.ai];
            const int64_t slot = static_cast<int64_t>(s.part) * g.slots + base_s[s.ai];
            const int na = min(atoms, blocks - s.tile * atoms);
            ok = wait_warp(acc_full0 + 8 * acc, (n >> 1) & 1, wait, 1300 + acc);
            if (!ok) break;
            tc_fence_after_sync();
            for (int a = 0; a < na; ++a) {
                const int block = s.tile * atoms + a;
                float *out;
                int pitch;
                bool mine;
                if (kUp) {
                    const int i = block * 64 + (r & 63);
                    mine = i < g.inner;
                    pitch = 2 * g.inner;
                    out = g.z + slot * pitch + (r < 64 ? i : g.inner + i);
                } else {
                    mine = block * 128 + r < g.hidden;
                    pitch = g.hidden;
                    out = g.o + slot * pitch + block * 128 + r;
                }
                for (int c = 0; c < count; c += 16) {
                    uint32_t v[16];
                    tmem_ld_32x16(tmem + acc * acc_cols + a * columns + c + (static_cast<uint32_t>(quarter * 32) << 16), v);
                    tmem_ld_wait();
                    if (mine) {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (c + j < count) out[static_cast<int64_t>(c + j) * pitch] = __uint_as_float(v[j]);
                    }
                    __syncwarp();
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty0 + 8 * acc);
            if constexpr (P == DOWN_FEW) {
                // With the last of its experts this CTA is done with the tile. Four warps of each of its CTAs count; the CTA
                // whose warp is the last one adds the parts, when its own stretch is done.
                auto rest = walk;
                Segment after;
                if (rest.next(after) && after.tile == s.tile) continue;
                const int q0 = s.tile * chosen * cut.kblocks, ctas = (q0 + chosen * cut.kblocks - 1) / cut.len - q0 / cut.len + 1;
                __threadfence();
                __syncwarp();
                if (lane == 0 && atomicAdd(g.arrived + s.tile, 1) == 4 * ctas - 1) {
                    __threadfence();
                    atomicOr(const_cast<int *>(misc) + 4 + (s.tile >> 5), 1 << (s.tile & 31));
                }
            }
        }
        if (P == DOWN_FEW && chosen == 0)
            for (int i = blockIdx.x * 128 + r; i < g.tokens * g.hidden; i += gridDim.x * 128) g.Y[i] = 0;
    } else if (!kGated) {
        // -------------------------------------------------------------- activations
        // The loader warps form groups that take the K blocks in turn, so that the latency of a block's loads is spread over
        // several blocks. A group looks at a stage only when its own turn comes; the phase it waits for cannot be
        // mistaken for the one two before it as long as there are no more groups than stages.
        const int group_warps = stages >= 8 ? 1 : stages >= 4 ? 2 : 4, groups = kMoeLoaders / group_warps;
        const int mine = (warp - 6) / group_warps, chunk = lane & 7;
        constexpr int kRows = kUp ? 4 : 2;              // rows that a warp takes at a time
        const int row0 = (warp - 6) % group_warps * kRows + lane / (32 / kRows), row_step = kRows * group_warps;
        const Cut up(chosen * tiles_up, kb_up, g.sms, g.parts_up);
        const int64_t part_pitch = static_cast<int64_t>(g.slots) * 2 * g.inner;
        int turn = 0;
        bool ok = true;
        if (!kUp) griddep_wait();
        while (ok && walk.next(s)) {
            const int count = count_s[s.ai], base = base_s[s.ai];
            for (int kb = s.kb0; kb < s.kb1; ++kb) {
                if (turn == mine) {
                    ok = wait_warp(empty0 + 8 * st, ph ^ 1u, wait, 1400 + st);
                    if (!ok) break;
                    const uint32_t dst = ring + st * stage_bytes + rows_at;
                    const int k = kb * 64 + chunk * 8;
                    if (kUp) {
                        for (int r = row0; r < count; r += row_step) {
                            if (k < g.hidden) cp_async_16(dst + swizzled(r, chunk), g.X + static_cast<int64_t>(token_s[base + r]) * g.hidden + k);
                            else st_shared_v4(dst + swizzled(r, chunk), make_uint4(0, 0, 0, 0));
                        }
                        cp_async_wait_all();
                    } else {
                        // sixteen lanes to a row, four values each: half a 16-byte chunk of the swizzled row
                        const int parts = up.num_parts(s.ai * tiles_up + kb), k4 = kb * 64 + (lane & 15) * 4;
                        for (int r = row0; r < count; r += row_step) {
                            uint2 hi = make_uint2(0, 0), lo = hi;
                            if (k4 < g.inner) split_four<T>(gated_values<4>(g.z + static_cast<int64_t>(base + r) * 2 * g.inner + k4, g.inner, parts, part_pitch), hi, lo);
                            const uint32_t at = dst + swizzled(r, (lane & 15) >> 1) + (lane & 1) * 8;
                            st_shared_v2(at, hi);
                            st_shared_v2(at + rows_bytes, lo);
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
    if (P == DOWN_FEW && !misc[0]) {
        // the ring is free now: each warp lists parts in its own corner of it
        int2 *const entry = reinterpret_cast<int2 *>(sm) + warp * (B200_MOE_MAX_TOP_K * kMaxParts);
        for (int tile = 0; tile < tiles; ++tile) {
            if (!(misc[4 + (tile >> 5)] >> (tile & 31) & 1)) continue;
            for (int t = warp; t < g.tokens; t += kMoeThreads / 32) {
                int slot = -1, parts = 0;
                float w = 0.0f;
                if (lane < g.top_k) {
                    slot = slot_s[t * g.top_k + lane];
                    w = weight_s[t * g.top_k + lane];
                    if (slot >= 0) parts = cut.num_parts(tile * chosen + active_s[t * g.top_k + lane]);
                    if (T::kScaled && slot >= 0) w *= __ldcg(g.list.unscale + slot);
                }
                combine<T>(g, entry, t, tile * 128 + lane * 4, lane, slot, parts, w);
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
        tmem_dealloc<1>(tmem, g.tmem_cols);
    }
}

// The gated values for DOWN, up to eight blocks per slot. A pair of fp16 numbers keeps an absolute 2^-25 and holds nothing beyond 2 *
// 65504, so with fp16 the blocks of a slot, a cluster, first find its largest finite value and scale by the power of two that
// brings it to 2^14 .. 2^15: each value then errs by 2^-22 of itself and 2^-39 of the largest. The sums of DOWN, which are kept
// per slot, are multiplied back exactly with the choice's weight (factors beyond 2^100 would leave the range of fp32 there).
// A pair of bf16 numbers keeps 2^-16 of any value as it is.
// A slot's values come in one or two parts where there is much to do, so more threads per SM serve better than more parts in
// flight (256 tokens, 128 experts of 2048 x 768, top 8: 232 us for the layer with four, 228 with two). What a thread computes
// for the maximum it keeps, as long as that is kGateQuads quads.
template <typename T, bool FEW>
__global__ void __launch_bounds__(kGateThreads, 4) moe_gate_kernel(const __grid_constant__ MoeArgs g) {
    __shared__ uint32_t largest_s[kGateBlocks * kGateThreads / 32];
    const bool cluster = T::kScaled && gridDim.x > 1;
    griddep_launch_dependents();   // DOWN reads nothing of this kernel before its own wait
    if (cluster) cluster_arrive();
    griddep_wait();
    if (cluster) cluster_wait();   // every block runs: its shared memory may be written
    const int slot = blockIdx.y, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int chosen = __ldcg(g.list.header), most = FEW ? 0 : __ldcg(g.list.header + 1), slots = __ldcg(g.list.header + 2), owner = __ldcg(g.list.owner + slot);
    if (slot >= slots) return;     // nobody's: its entries are what the workspace held
    const int atoms = FEW ? 1 : tile_atoms(g, most), tiles = ((g.inner + 63) / 64 + atoms - 1) / atoms;
    const Cut up(chosen * tiles, (g.hidden + 63) / 64, g.sms, g.parts_up);
    const auto values = [&](int k) {
        return gated_values<2>(g.z + static_cast<int64_t>(slot) * 2 * g.inner + k, g.inner, up.num_parts(owner * tiles + k / 64 / atoms),
                               static_cast<int64_t>(g.slots) * 2 * g.inner);
    };
    const int first = (blockIdx.x * blockDim.x + threadIdx.x) * 4, step = gridDim.x * blockDim.x * 4, span = step * kGateQuads;
    float4 v[kGateQuads];
    float scale = 1.0f;
    if constexpr (T::kScaled) {
        const auto size = [](float f) {   // of a finite number, as bits that compare like it
            const uint32_t b = __float_as_uint(f) & 0x7fffffffu;
            return b < 0x7f800000u ? b : 0u;
        };
        uint32_t largest = 0u;
        for (int k0 = first; k0 < g.inner; k0 += span)
#pragma unroll
            for (int i = 0; i < kGateQuads; ++i)
                if (k0 + i * step < g.inner) {
                    v[i] = values(k0 + i * step);
                    largest = max(max(max(largest, size(v[i].x)), max(size(v[i].y), size(v[i].z))), size(v[i].w));
                }
        largest = __reduce_max_sync(0xffffffffu, largest);
        if (cluster) {   // every warp tells every block
            if (lane < gridDim.x) st_cluster(mapa_shared(smem_u32(&largest_s[blockIdx.x * warps + (threadIdx.x >> 5)]), lane), largest);
            cluster_arrive();
            cluster_wait();
        } else {
            if (lane == 0) largest_s[threadIdx.x >> 5] = largest;
            __syncthreads();
        }
        largest = 0u;
        for (int w = lane; w < gridDim.x * warps; w += 32) largest = max(largest, largest_s[w]);
        largest = __reduce_max_sync(0xffffffffu, largest);
        const int shift = min(max(127 + 14 - static_cast<int>(largest >> 23), -100), 100);
        scale = __uint_as_float(static_cast<uint32_t>(127 + shift) << 23);
        if (blockIdx.x == 0 && threadIdx.x == 0) g.list.unscale[slot] = __uint_as_float(static_cast<uint32_t>(127 - shift) << 23);
    }
    for (int k0 = first; k0 < g.inner; k0 += span)
#pragma unroll
        for (int i = 0; i < kGateQuads; ++i) {
            const int k = k0 + i * step;
            if (k >= g.inner) continue;
            if (!T::kScaled || g.inner > span) v[i] = values(k);
            uint2 hi, lo;
            split_four<T>(make_float4(v[i].x * scale, v[i].y * scale, v[i].z * scale, v[i].w * scale), hi, lo);
            *reinterpret_cast<uint2 *>(g.h + static_cast<int64_t>(slot) * g.inner + k) = hi;
            *reinterpret_cast<uint2 *>(g.h + (static_cast<int64_t>(g.slots) + slot) * g.inner + k) = lo;
        }
}

template <typename T>
__global__ void __launch_bounds__(128) moe_combine_kernel(const __grid_constant__ MoeArgs g) {
    __shared__ int2 entry[4][B200_MOE_MAX_TOP_K * kMaxParts];
    const int t = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int block = blockIdx.x * 4 + warp, blocks = (g.hidden + 127) / 128;
    griddep_wait();
    griddep_launch_dependents();
    int slot = -1, parts = 0;
    float w = 0.0f;
    if (lane < g.top_k) {
        const int atoms = tile_atoms(g, __ldcg(g.list.header + 1)), tiles = (blocks + atoms - 1) / atoms;
        const Cut cut(__ldcg(g.list.header) * tiles, (g.inner + 63) / 64, g.sms, g.parts_down);
        const int at = t * g.top_k + lane;
        slot = __ldcg(g.list.slot + at);
        w = __ldcg(g.list.weight + at);
        if (T::kScaled && slot >= 0) w *= __ldcg(g.list.unscale + slot);
        if (slot >= 0 && block < blocks) parts = cut.num_parts(__ldcg(g.list.active + at) * tiles + block / atoms);
    }
    combine<T>(g, entry[warp], t, block * 128 + lane * 4, lane, slot, parts, w);
}

int check_moe(int64_t tokens, int64_t hidden, int64_t inner, int64_t experts, int top_k) {
    if (tokens <= 0 || tokens > B200_MOE_MAX_TOKENS || hidden <= 0 || inner <= 0 || hidden % 8 || inner % 8) return B200_INVALID_SHAPE;
    if (hidden > kMaxHidden || inner > kMaxHidden || experts <= 0 || experts > B200_MOE_MAX_EXPERTS) return B200_INVALID_SHAPE;
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
    bool few;
    int64_t off_list, off_z, off_o, off_h, bytes;   // few: the counters of the tiles before the list
};

MoeLayout moe_layout(int64_t tokens, int64_t hidden, int64_t inner, int64_t experts, int top_k) {
    MoeLayout l;
    const int64_t slots = tokens * top_k, up_tiles = (inner + 63) / 64;
    l.parts_up = most_parts(top_k * up_tiles, (hidden + 63) / 64);
    l.parts_down = most_parts(top_k * ((hidden + 127) / 128), up_tiles);
    l.few = slots <= kFewSlots && tokens <= kFewTokens;
    l.off_list = l.few ? up256((hidden + 127) / 128 * 4) : 0;
    l.off_z = l.off_list + up256((3 + 3 * experts + 6 * slots) * 4);
    l.off_o = l.off_z + up256(l.parts_up * slots * 2 * inner * 4);
    l.off_h = l.off_o + up256(l.parts_down * slots * hidden * 4);
    l.bytes = l.off_h + up256(2 * slots * inner * 2);
    return l;
}

template <typename Kernel>
cudaError_t launch(Kernel *kernel, const MoeArgs &g, dim3 grid, int threads, int smem, int cluster, cudaStream_t stream) {
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
    cfg.numAttrs = cluster > 0 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, g);
}

template <typename Kernel>
cudaError_t launch_gate(Kernel *kernel, const MoeArgs &g, cudaStream_t stream) {
    const int quads = g.inner / 4, threads = quads >= kGateThreads ? kGateThreads : (quads + 31) / 32 * 32;
    int blocks = 1;
    while (blocks < kGateBlocks && blocks * threads * kGateQuads < quads) blocks *= 2;
    return launch(kernel, g, dim3(blocks, g.slots), threads, 0, blocks, stream);
}

template <typename T>
cudaError_t launch_moe(MoeArgs &g, const CUtensorMap &up, const CUtensorMap &down, bool few, int smem, cudaStream_t stream) {
    g.map = up;
    if (few) {
        const cudaError_t e = launch(moe_product_kernel<T, UP_FEW>, g, g.sms, kMoeThreads, smem, 0, stream);
        if (e != cudaSuccess) return e;
        if constexpr (T::kScaled) {
            const cudaError_t gate = launch_gate(moe_gate_kernel<T, true>, g, stream);
            if (gate != cudaSuccess) return gate;
        }
        g.map = down;
        return launch(moe_product_kernel<T, DOWN_FEW>, g, g.sms, kMoeThreads, smem, 0, stream);
    }
    const int blocks = (g.tokens + 31) / 32;
    cudaError_t e = launch(moe_route_kernel, g, blocks, 1024, 0, blocks, stream);
    if (e == cudaSuccess) e = launch(moe_product_kernel<T, UP>, g, g.sms, kMoeThreads, smem, 0, stream);
    if (e == cudaSuccess) e = launch_gate(moe_gate_kernel<T, false>, g, stream);
    g.map = down;
    if (e == cudaSuccess) e = launch(moe_product_kernel<T, DOWN>, g, g.sms, kMoeThreads, smem, 0, stream);
    if (e == cudaSuccess) e = launch(moe_combine_kernel<T>, g, dim3((g.hidden + 511) / 512, g.tokens), 128, 0, 0, stream);
    return e;
}

}  // namespace

int prepare_moe_kernels() {
    void (*const kernels[])(MoeArgs) = {moe_product_kernel<Bf16, UP>, moe_product_kernel<Bf16, DOWN>, moe_product_kernel<Bf16, UP_FEW>, moe_product_kernel<Bf16, DOWN_FEW>,
                                        moe_product_kernel<Fp16, UP>, moe_product_kernel<Fp16, DOWN>, moe_product_kernel<Fp16, UP_FEW>, moe_product_kernel<Fp16, DOWN_FEW>};
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
    if (st == B200_OK && (!l.few || dtype == B200_F16)) st = encode_operand_map(&g.map_h, dtype, g.h, inner, 2 * slots, 16);
    if (st != B200_OK) return st;
    int *const list = reinterpret_cast<int *>(ws + l.off_list);
    g.arrived = reinterpret_cast<int *>(ws);
    g.list.header = list;
    g.list.expert = list + 3;
    g.list.count = g.list.expert + experts;
    g.list.base = g.list.count + experts;
    g.list.token = g.list.base + experts;
    g.list.owner = g.list.token + slots;
    g.list.slot = g.list.owner + slots;
    g.list.active = g.list.slot + slots;
    g.list.weight = reinterpret_cast<float *>(g.list.active + slots);
    g.list.unscale = g.list.weight + slots;
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
    g.tmem_cols = pow2_at_least((l.few ? 2 : 4) * g.slot_cols);
    if (g.tmem_cols > kTmemColumns) g.tmem_cols = kTmemColumns;
    const int slot_lists = static_cast<int>(up256(slots * (l.few ? 10 : 2)));
    const int expert_lists = static_cast<int>(up256(experts * (12 + (l.few ? (tokens + 31) / 32 * 4 + 2 : 0))));
    // Two blocks and the KB that the hardware takes for each fit an SM's 228; with fp16 a block of the gate kernel fits beside them (37 tokens,
    // 20 experts of 1000 x 360, top 3: 31.0 us, 32.5 where it does not).
    const int smem = l.few ? (dtype == B200_F16 ? 112 : 113) * 1024 : kSmemLimit;
    g.ring_bytes = (smem - 1024 - slot_lists - expert_lists - 512) / 1024 * 1024;
    g.off_slots = g.ring_bytes;
    g.off_experts = g.off_slots + slot_lists;
    g.off_bars = g.off_experts + expert_lists;
    g.off_misc = g.off_bars + (2 * kMoeStages + 4) * 8;
    g.idesc = umma_idesc(128, 0, dtype == B200_BF16);
    g.budget = wait_budget_cycles();
    const cudaError_t e = dtype == B200_BF16 ? launch_moe<Bf16>(g, up, down, l.few, smem, static_cast<cudaStream_t>(stream))
                                             : launch_moe<Fp16>(g, up, down, l.few, smem, static_cast<cudaStream_t>(stream));
    return e != cudaSuccess ? record_cuda_error(e) : B200_OK;
}
