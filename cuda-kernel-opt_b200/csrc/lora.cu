// A projection shared by all rows with low-rank adapters of many requests beside it:
//
//     D[i] = A[i] B^T + scale[s] (A[i] lora_a[s]^T) lora_b[s]^T,   s = row_adapter[i]
//
// Two kernels: the first projects every row into its adapter's rank (u, fp32, in the workspace), the second
// computes the shared product and adds u lora_b[s]^T before the one rounding.
#include <cuda_runtime.h>

#include "../../include/b200_gemm.h"
#include "gemm_sm100.cuh"
#include "routed.cuh"

namespace b200 {
namespace {

struct LoraArgs {
    const uint16_t *A, *Bt, *lora_a, *lora_b;
    uint16_t *D;
    const float *scale;
    const int *row_adapter;
    float *u;  // M x rank
    int M, N, K, rank;
    int64_t num_adapters;
};

// One block per row, one warp per rank: u[i][r] = scale * <A[i], lora_a[s][r]>.
template <typename T>
__global__ void __launch_bounds__(256) lora_shrink_kernel(const LoraArgs g) {
    const int lane = threadIdx.x & 31;
    for (int64_t m = blockIdx.x; m < g.M; m += gridDim.x) {
        const int64_t s = g.row_adapter[m];
        if (s < 0 || s >= g.num_adapters) continue;
        const float scale = g.scale ? g.scale[s] : 1.0f;
        const uint4 *x = reinterpret_cast<const uint4 *>(g.A + m * g.K);
        for (int r = threadIdx.x >> 5; r < g.rank; r += blockDim.x >> 5) {
            const uint4 *a = reinterpret_cast<const uint4 *>(g.lora_a + (s * g.rank + r) * g.K);
            float acc = 0.0f;
            for (int k = lane; k < g.K / 8; k += 32) acc = dot8<T>(x[k], a[k], acc);
            acc = warp_sum(acc);
            if (lane == 0) g.u[m * g.rank + r] = scale * acc;
        }
    }
}

// 64 x 64 tiles of D, 4 x 4 values per thread, operands as fp32 in shared memory.
template <typename T>
__global__ void __launch_bounds__(256) lora_product_kernel(const LoraArgs g) {
    __shared__ float xs[32][65], ws[32][65];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * 64, n0 = static_cast<int64_t>(blockIdx.x) * 64;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < g.K; k0 += 32) {
        // 64 rows x 32 elements of either operand: one 16-byte load per thread
        const int row = threadIdx.x >> 2, kk = (threadIdx.x & 3) * 8;
        uint4 a = make_uint4(0, 0, 0, 0), b = a;
        if (k0 + kk < g.K) {
            if (m0 + row < g.M) a = *reinterpret_cast<const uint4 *>(g.A + (m0 + row) * g.K + k0 + kk);
            if (n0 + row < g.N) b = *reinterpret_cast<const uint4 *>(g.Bt + (n0 + row) * g.K + k0 + kk);
        }
        const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 x = T::unpack(av[i]), w = T::unpack(bv[i]);
            xs[kk + 2 * i][row] = x.x;
            xs[kk + 2 * i + 1][row] = x.y;
            ws[kk + 2 * i][row] = w.x;
            ws[kk + 2 * i + 1][row] = w.y;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 32; ++k) {
            float x[4], w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = xs[k][ty + 16 * i];
                w[i] = ws[k][tx + 16 * i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x[i], w[j], acc[i][j]);
        }
    }
    for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + ty + 16 * i;
        if (m >= g.M) continue;
        const int64_t s = g.row_adapter[m];
        const bool has = s >= 0 && s < g.num_adapters;
        for (int j = 0; j < 4; ++j) {
            const int64_t n = n0 + tx + 16 * j;
            if (n >= g.N) continue;
            float v = acc[i][j];
            if (has) {
                const uint4 *b = reinterpret_cast<const uint4 *>(g.lora_b + (s * g.N + n) * g.rank);
                const float *u = g.u + m * g.rank;
                for (int r = 0; r < g.rank; r += 8) {
                    const uint4 q = b[r / 8];
                    const uint32_t qv[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        const float2 w = T::unpack(qv[p]);
                        v = fmaf(u[r + 2 * p], w.x, v);
                        v = fmaf(u[r + 2 * p + 1], w.y, v);
                    }
                }
            }
            g.D[m * g.N + n] = T::round(v);
        }
    }
}

template <typename T>
int launch_lora(const LoraArgs &g, cudaStream_t stream) {
    lora_shrink_kernel<T><<<g.M < 4096 ? g.M : 4096, 256, 0, stream>>>(g);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return record_cuda_error(e);
    lora_product_kernel<T><<<dim3((g.N + 63) / 64, (g.M + 63) / 64), 256, 0, stream>>>(g);
    e = cudaGetLastError();
    return e != cudaSuccess ? record_cuda_error(e) : B200_OK;
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
int prepare_routed_kernels() { return prepare_moe_kernels(); }

}  // namespace b200

extern "C" int64_t b200_gemm_lora_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t num_adapters, int rank) {
    if (b200::check_lora(M, N, K, num_adapters, rank) != B200_OK) return -1;
    return M * rank * 4;
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
    st = current_device(nullptr, nullptr);
    if (st != B200_OK) return st;
    LoraArgs g = {};
    g.A = static_cast<const uint16_t *>(A);
    g.Bt = static_cast<const uint16_t *>(Bt);
    g.lora_a = static_cast<const uint16_t *>(lora_a);
    g.lora_b = static_cast<const uint16_t *>(lora_b);
    g.D = static_cast<uint16_t *>(D);
    g.scale = lora_scale;
    g.row_adapter = row_adapter;
    g.u = static_cast<float *>(workspace);
    g.M = static_cast<int>(M);
    g.N = static_cast<int>(N);
    g.K = static_cast<int>(K);
    g.rank = rank;
    g.num_adapters = num_adapters;
    return dtype == B200_BF16 ? launch_lora<Bf16>(g, static_cast<cudaStream_t>(stream)) : launch_lora<Fp16>(g, static_cast<cudaStream_t>(stream));
}
