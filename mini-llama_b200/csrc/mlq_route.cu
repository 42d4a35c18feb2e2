// mlq_route.cu -- the router of a mixture-of-experts layer.
//
// logits = x Wr^T in 64 bits, then per row the scores, the top_k choice and
// its weights.  64 bits because the choice is discrete: two experts whose logits
// differ by less than an fp32 sum's error would be swapped against the exact
// result; a product of two fp32 values is exact in fp64, and its sum is off
// by ~1e-15.
#include <limits.h>
#include <math.h>

#include "mlq_device.cuh"
#include "mlq_kernels.h"

namespace mlq {
namespace {

struct RouteArgs {
    const float* w;
    const float* bias;
    const float* x;
    int rows, in, n_experts, top_k, scoring, renorm;
    float scale;
    double* l;  // [rows][n_experts]
    int32_t* ids;
    float* weights;
    float* logits;
};

constexpr int kRowsPerWarp = 4;

// One warp: one expert against 4 rows of x.
__global__ void __launch_bounds__(256) route_logits_kernel(const RouteArgs a) {
    launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const int e = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int r0 = blockIdx.y * kRowsPerWarp;
    if (e >= a.n_experts) return;
    const float* w = a.w + (size_t)e * a.in;
    double acc[kRowsPerWarp] = {};
    for (int i = lane; i < a.in; i += 32) {
        const double wv = (double)w[i];
#pragma unroll
        for (int k = 0; k < kRowsPerWarp; ++k)
            if (r0 + k < a.rows) acc[k] = fma(wv, (double)a.x[(size_t)(r0 + k) * a.in + i], acc[k]);
    }
#pragma unroll
    for (int k = 0; k < kRowsPerWarp; ++k) {
        for (int o = 16; o > 0; o >>= 1) acc[k] += __shfl_xor_sync(0xffffffffu, acc[k], o);
        if (lane == 0 && r0 + k < a.rows) {
            a.l[(size_t)(r0 + k) * a.n_experts + e] = acc[k];
            if (a.logits) a.logits[(size_t)(r0 + k) * a.n_experts + e] = (float)acc[k];
        }
    }
}

// (a, i) ranks before (b, j): NaN first, then the larger, then the lower index.
__device__ __forceinline__ bool ranks_before(double a, int i, double b, int j) {
    const bool an = a != a, bn = b != b;
    if (an != bn) return an;
    if (!an && a != b) return a > b;
    return i < j;
}

constexpr int kTopkWarps = 4;

// One warp per row.
__global__ void __launch_bounds__(32 * kTopkWarps) route_topk_kernel(const RouteArgs a) {
    __shared__ double s_choice[kTopkWarps][MLQ_MOE_MAX_EXPERTS];
    launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = blockIdx.x * kTopkWarps + warp;
    if (r >= a.rows) return;
    const double* l = a.l + (size_t)r * a.n_experts;
    double* c = s_choice[warp];
    double top = -INFINITY, sum = 0.0;
    if (a.scoring == MLQ_SCORE_SOFTMAX) {
        bool nan = false;
        for (int e = lane; e < a.n_experts; e += 32) {
            const double v = l[e];
            nan |= v != v;
            top = v > top ? v : top;
        }
        for (int o = 16; o > 0; o >>= 1) {
            const double v = __shfl_xor_sync(0xffffffffu, top, o);
            top = v > top ? v : top;
        }
        if (__any_sync(0xffffffffu, nan)) top = NAN;
        for (int e = lane; e < a.n_experts; e += 32) sum += exp(l[e] - top);
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    auto score = [&](int e) { return a.scoring == MLQ_SCORE_SOFTMAX ? exp(l[e] - top) / sum : 1.0 / (1.0 + exp(-l[e])); };
    for (int e = lane; e < a.n_experts; e += 32) c[e] = a.bias ? score(e) + (double)a.bias[e] : score(e);
    __syncwarp();
    double picked_sum = 0.0, mine[2] = {0.0, 0.0};  // lane j keeps slots j and j + 32
    int my_id[2] = {-1, -1};
    for (int j = 0; j < a.top_k; ++j) {
        double best = -INFINITY;
        int at = INT_MAX;
        for (int e = lane; e < a.n_experts; e += 32)
            if (ranks_before(c[e], e, best, at)) best = c[e], at = e;
        for (int o = 16; o > 0; o >>= 1) {
            const double v = __shfl_xor_sync(0xffffffffu, best, o);
            const int i = __shfl_xor_sync(0xffffffffu, at, o);
            if (ranks_before(v, i, best, at)) best = v, at = i;
        }
        if (best == -INFINITY) break;  // only masked experts are left
        const double s = score(at);
        picked_sum += s;
        if (lane == (j & 31)) mine[j >> 5] = s, my_id[j >> 5] = at;
        if (lane == (at & 31)) c[at] = -INFINITY;
        __syncwarp();
    }
    for (int q = 0; q < 2; ++q) {
        const int j = lane + 32 * q;
        if (j >= a.top_k) break;
        double v = mine[q];
        if (a.renorm) v = picked_sum == 0.0 ? 0.0 : v / picked_sum;
        a.ids[(size_t)r * a.top_k + j] = my_id[q];
        a.weights[(size_t)r * a.top_k + j] = my_id[q] < 0 ? 0.0f : (float)(v * (double)a.scale);
    }
}

constexpr int kPassRows = 4096;

template <typename... Params, typename... Args>
cudaError_t launch_pdl(void (*kernel)(Params...), dim3 grid, int block, cudaStream_t stream, Args&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

}  // namespace

size_t route_workspace_bytes(int n_experts, int rows) {
    const size_t n = rows < kPassRows ? rows : kPassRows;
    return (n * n_experts * sizeof(double) + 255) & ~(size_t)255;
}

cudaError_t launch_route(const mlq_router& r, const float* x, int rows, int32_t* ids, float* weights, float* logits,
                         void* ws, cudaStream_t stream) {
    for (int r0 = 0; r0 < rows; r0 += kPassRows) {
        RouteArgs a{};
        a.w = r.w, a.bias = r.bias;
        a.x = x + (size_t)r0 * r.in_features;
        a.rows = rows - r0 < kPassRows ? rows - r0 : kPassRows;
        a.in = r.in_features, a.n_experts = r.n_experts, a.top_k = r.top_k;
        a.scoring = r.scoring, a.renorm = r.renormalize, a.scale = r.scale;
        a.l = static_cast<double*>(ws);
        a.ids = ids + (size_t)r0 * r.top_k;
        a.weights = weights + (size_t)r0 * r.top_k;
        a.logits = logits ? logits + (size_t)r0 * r.n_experts : nullptr;
        cudaError_t e = launch_pdl(route_logits_kernel,
                                   dim3((r.n_experts + 7) / 8, (a.rows + kRowsPerWarp - 1) / kRowsPerWarp), 256, stream, a);
        if (e != cudaSuccess) return e;
        e = launch_pdl(route_topk_kernel, dim3((a.rows + kTopkWarps - 1) / kTopkWarps), 32 * kTopkWarps, stream, a);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace mlq
