// A whole mixture-of-experts layer for a few tokens:
//
//     Y[t] = sum_j w[t][j] W2[e] (silu(G[e] X[t]) . (U[e] X[t])),   e = ids[t][j] = the j-th largest router logit of t
//
// Three kernels: the router's choice, the gated product of every (token, choice) slot, the second product
// with the weighted sum over a token's choices.
#include <cuda_runtime.h>

#include <cfloat>
#include <cmath>

#include "../../include/b200_gemm.h"
#include "gemm_sm100.cuh"
#include "routed.cuh"

namespace b200 {
namespace {

struct MoeArgs {
    const uint16_t *X, *W13, *W2;
    const float *logits;
    uint16_t *Y;
    int *ids_out;
    float *weights_out;
    int *ids;        // tokens x top_k, workspace
    float *weights;  // tokens x top_k, workspace
    float *h;        // tokens x top_k x inner, workspace
    int tokens, hidden, inner, experts, top_k, normalise;
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

// One warp, one token: the top_k largest keys in descending order, ties to the lower index; lane j < top_k returns
// choice j (id -1, weight 0 where no expert is left).
__device__ __forceinline__ void choose_experts(const float *logits, int experts, int top_k, int normalise, int lane, int &id, float &weight) {
    constexpr int kPer = B200_MOE_MAX_EXPERTS / 32;
    uint32_t key[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = lane + 32 * i;
        key[i] = e < experts ? logit_key(__ldcg(logits + e)) : 0u;
    }
    uint32_t best = 0u;
#pragma unroll
    for (int i = 0; i < kPer; ++i) best = max(best, key[i]);
    const float top = key_logit(__reduce_max_sync(0xffffffffu, best));
    float sum = 0.0f;
    if (!normalise) {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (key[i]) sum += expf(key_logit(key[i]) - top);
        sum = warp_sum(sum);
    }
    id = -1;
    weight = 0.0f;
    for (int j = 0; j < top_k; ++j) {
        uint32_t k = 0u;
        int at = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (key[i] > k) {
                k = key[i];
                at = lane + 32 * i;
            }
        const uint32_t most = __reduce_max_sync(0xffffffffu, k);
        if (most == 0u) break;
        const int e = static_cast<int>(__reduce_min_sync(0xffffffffu, static_cast<uint32_t>(k == most ? at : 0x7fffffff)));
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (e == lane + 32 * i) key[i] = 0u;
        const float w = expf(key_logit(most) - top);
        if (normalise) sum += w;
        if (lane == j) {
            id = e;
            weight = w;
        }
    }
    if (id >= 0) weight /= sum;
}

__global__ void __launch_bounds__(32) moe_route_kernel(const MoeArgs g) {
    const int t = blockIdx.x, lane = threadIdx.x;
    int id;
    float w;
    choose_experts(g.logits + static_cast<int64_t>(t) * g.experts, g.experts, g.top_k, g.normalise, lane, id, w);
    if (lane < g.top_k) {
        const int at = t * g.top_k + lane;
        g.ids[at] = id;
        g.weights[at] = w;
        if (g.ids_out) g.ids_out[at] = id;
        if (g.weights_out) g.weights_out[at] = w;
    }
}

// One warp per (slot, inner row): both halves' dot products.
template <typename T>
__global__ void __launch_bounds__(256) moe_up_kernel(const MoeArgs g) {
    const int slot = blockIdx.x, lane = threadIdx.x & 31, e = g.ids[slot];
    if (e < 0) return;
    const uint4 *x = reinterpret_cast<const uint4 *>(g.X + static_cast<int64_t>(slot / g.top_k) * g.hidden);
    for (int i = blockIdx.y * 8 + (threadIdx.x >> 5); i < g.inner; i += gridDim.y * 8) {
        const uint4 *wg = reinterpret_cast<const uint4 *>(g.W13 + (static_cast<int64_t>(e) * 2 * g.inner + i) * g.hidden);
        const uint4 *wu = reinterpret_cast<const uint4 *>(g.W13 + (static_cast<int64_t>(e) * 2 * g.inner + g.inner + i) * g.hidden);
        float a = 0.0f, b = 0.0f;
        for (int k = lane; k < g.hidden / 8; k += 32) {
            a = dot8<T>(x[k], wg[k], a);
            b = dot8<T>(x[k], wu[k], b);
        }
        a = warp_sum(a);
        b = warp_sum(b);
        if (lane == 0) g.h[static_cast<int64_t>(slot) * g.inner + i] = a / (1.0f + expf(-a)) * b;
    }
}

// One warp per (token, hidden row): the choices in order.
template <typename T>
__global__ void __launch_bounds__(256) moe_down_kernel(const MoeArgs g) {
    const int t = blockIdx.x, lane = threadIdx.x & 31;
    for (int n = blockIdx.y * 8 + (threadIdx.x >> 5); n < g.hidden; n += gridDim.y * 8) {
        float y = 0.0f;
        for (int j = 0; j < g.top_k; ++j) {
            const int slot = t * g.top_k + j, e = g.ids[slot];
            if (e < 0) continue;
            const uint4 *w = reinterpret_cast<const uint4 *>(g.W2 + (static_cast<int64_t>(e) * g.hidden + n) * g.inner);
            const float4 *h = reinterpret_cast<const float4 *>(g.h + static_cast<int64_t>(slot) * g.inner);
            float acc = 0.0f;
            for (int k = lane; k < g.inner / 8; k += 32) {
                const uint4 q = w[k];
                const float4 h0 = h[2 * k], h1 = h[2 * k + 1];
                const float2 w0 = T::unpack(q.x), w1 = T::unpack(q.y), w2 = T::unpack(q.z), w3 = T::unpack(q.w);
                acc = fmaf(h0.x, w0.x, fmaf(h0.y, w0.y, fmaf(h0.z, w1.x, fmaf(h0.w, w1.y, acc))));
                acc = fmaf(h1.x, w2.x, fmaf(h1.y, w2.y, fmaf(h1.z, w3.x, fmaf(h1.w, w3.y, acc))));
            }
            y = fmaf(g.weights[slot], warp_sum(acc), y);
        }
        if (lane == 0) g.Y[static_cast<int64_t>(t) * g.hidden + n] = T::round(y);
    }
}

template <typename T>
int launch_moe(const MoeArgs &g, cudaStream_t stream) {
    moe_route_kernel<<<g.tokens, 32, 0, stream>>>(g);
    moe_up_kernel<T><<<dim3(g.tokens * g.top_k, (g.inner + 31) / 32), 256, 0, stream>>>(g);
    moe_down_kernel<T><<<dim3(g.tokens, (g.hidden + 31) / 32), 256, 0, stream>>>(g);
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess ? record_cuda_error(e) : B200_OK;
}

int check_moe(int64_t tokens, int64_t hidden, int64_t inner, int64_t experts, int top_k) {
    if (tokens <= 0 || tokens > B200_MOE_MAX_TOKENS || hidden <= 0 || inner <= 0 || hidden % 8 || inner % 8) return B200_INVALID_SHAPE;
    if (hidden > (1 << 20) || inner > (1 << 20) || experts <= 0 || experts > B200_MOE_MAX_EXPERTS) return B200_INVALID_SHAPE;
    if (top_k < 1 || top_k > B200_MOE_MAX_TOP_K || top_k > experts) return B200_INVALID_CONFIG;
    return B200_OK;
}

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

}  // namespace
}  // namespace b200

extern "C" int64_t b200_moe_workspace_bytes(int64_t tokens, int64_t hidden, int64_t inner, int64_t experts, int top_k) {
    if (b200::check_moe(tokens, hidden, inner, experts, top_k) != B200_OK) return -1;
    return 2 * b200::up256(tokens * top_k * 4) + tokens * top_k * inner * 4;
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
    st = current_device(nullptr);
    if (st != B200_OK) return st;
    MoeArgs g = {};
    g.X = static_cast<const uint16_t *>(X);
    g.W13 = static_cast<const uint16_t *>(W13);
    g.W2 = static_cast<const uint16_t *>(W2);
    g.logits = logits;
    g.Y = static_cast<uint16_t *>(Y);
    g.ids_out = ids;
    g.weights_out = weights;
    uint8_t *const ws = static_cast<uint8_t *>(workspace);
    const int64_t slot_bytes = up256(tokens * top_k * 4);
    g.ids = reinterpret_cast<int *>(ws);
    g.weights = reinterpret_cast<float *>(ws + slot_bytes);
    g.h = reinterpret_cast<float *>(ws + 2 * slot_bytes);
    g.tokens = static_cast<int>(tokens);
    g.hidden = static_cast<int>(hidden);
    g.inner = static_cast<int>(inner);
    g.experts = static_cast<int>(experts);
    g.top_k = top_k;
    g.normalise = normalise;
    return dtype == B200_BF16 ? launch_moe<Bf16>(g, static_cast<cudaStream_t>(stream)) : launch_moe<Fp16>(g, static_cast<cudaStream_t>(stream));
}
