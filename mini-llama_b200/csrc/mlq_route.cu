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

// Sums N values over the warp's lanes; lane l < N gets value l (N a power of
// two, at most 32): half of the values change hands at each step.
template <int N>
__device__ __forceinline__ double warp_sums(double (&v)[N], int lane) {
    int o = 16;
#pragma unroll
    for (int n = N / 2; n >= 1; n /= 2, o /= 2)
#pragma unroll
        for (int k = 0; k < n; ++k) {
            const bool up = lane & o;
            const double give = up ? v[k] : v[n + k], keep = up ? v[n + k] : v[k];
            v[k] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    for (; o >= 1; o /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    // the lane bits 16, 8, .. hold the value's index from its highest bit: bring value l to lane l
    int from = 0;
#pragma unroll
    for (int n = N / 2, bit = 16; n >= 1; n /= 2, bit /= 2)
        if (lane & n) from |= bit;
    return __shfl_sync(0xffffffffu, v[0], from);
}

// One CTA: E experts against R rows of x, the K axis split over 8 warps.  A
// decode step's router reads a few 100 KB: latency decides, so every load of a
// thread is independent and the grid is as wide as the experts.
template <int E, int R>
__global__ void __launch_bounds__(256) route_logits_kernel(const RouteArgs a, int vec) {
    __shared__ double part[8][E * R];
    launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int e0 = blockIdx.x * E, r0 = blockIdx.y * R;
    double acc[E * R] = {};
    grid_dependency_wait();
    if (vec) {
#pragma unroll 2
        for (int i = threadIdx.x * 4; i < a.in; i += 1024) {
            float4 w[E], x[R];
#pragma unroll
            for (int e = 0; e < E; ++e)
                w[e] = *reinterpret_cast<const float4*>(a.w + (size_t)min(e0 + e, a.n_experts - 1) * a.in + i);
#pragma unroll
            for (int r = 0; r < R; ++r)
                x[r] = *reinterpret_cast<const float4*>(a.x + (size_t)min(r0 + r, a.rows - 1) * a.in + i);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const double x0 = x[r].x, x1 = x[r].y, x2 = x[r].z, x3 = x[r].w;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    double& s = acc[e * R + r];
                    s = fma((double)w[e].x, x0, s);
                    s = fma((double)w[e].y, x1, s);
                    s = fma((double)w[e].z, x2, s);
                    s = fma((double)w[e].w, x3, s);
                }
            }
        }
    } else {
        for (int i = threadIdx.x; i < a.in; i += 256)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const double x = (double)a.x[(size_t)min(r0 + r, a.rows - 1) * a.in + i];
#pragma unroll
                for (int e = 0; e < E; ++e)
                    acc[e * R + r] = fma((double)a.w[(size_t)min(e0 + e, a.n_experts - 1) * a.in + i], x, acc[e * R + r]);
            }
    }
    const double v = warp_sums(acc, lane);
    if (lane < E * R) part[warp][lane] = v;
    __syncthreads();
    if (threadIdx.x < E * R) {
        double sum = 0.0;
        for (int w = 0; w < 8; ++w) sum += part[w][threadIdx.x];
        const int e = e0 + threadIdx.x / R, r = r0 + threadIdx.x % R;
        if (e < a.n_experts && r < a.rows) {
            a.l[(size_t)r * a.n_experts + e] = sum;
            if (a.logits) a.logits[(size_t)r * a.n_experts + e] = (float)sum;
        }
    }
}

// Many rows: 64 rows x 64 experts per CTA on the fp64 matrix instructions, K
// in steps of 32 through shared memory (fp32 there, converted in registers;
// a pitch of 36 words keeps the 8 rows x 4 columns of a fragment in 32 banks).
// Warp w: rows 16 (w % 4) .., experts 32 (w / 4) ..
constexpr int kTile = 64, kTileK = 32, kTilePitch = kTileK + 4;

__device__ __forceinline__ void mma_f64(double (&c)[4], const double (&a)[8], const double (&b)[4]) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f64.f64.f64.f64 {%0,%1,%2,%3}, {%4,%5,%6,%7,%8,%9,%10,%11}, "
        "{%12,%13,%14,%15}, {%0,%1,%2,%3};"
        : "+d"(c[0]), "+d"(c[1]), "+d"(c[2]), "+d"(c[3])
        : "d"(a[0]), "d"(a[1]), "d"(a[2]), "d"(a[3]), "d"(a[4]), "d"(a[5]), "d"(a[6]), "d"(a[7]), "d"(b[0]), "d"(b[1]),
          "d"(b[2]), "d"(b[3]));
}

__global__ void __launch_bounds__(256) route_tile_kernel(const RouteArgs a, int vec) {
    __shared__ __align__(16) float tile[2][2][kTile * kTilePitch];  // [buffer][x, w]
    launch_dependents();
    grid_dependency_wait();
    const int r0 = blockIdx.x * kTile, e0 = blockIdx.y * kTile;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int rw = 16 * (warp & 3), ew = 32 * (warp >> 2);
    // a thread fetches 4 columns of rows threadIdx / 8 and 32 more on, of x and of w
    auto fetch = [&](int k0, int buf) {
        const int c = (threadIdx.x & 7) * 4, k = k0 + c;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = (threadIdx.x >> 3) + 32 * (i & 1);
            const float* src = (i < 2 ? a.x + (size_t)min(r0 + row, a.rows - 1) * a.in
                                      : a.w + (size_t)min(e0 + row, a.n_experts - 1) * a.in);
            float* dst = tile[buf][i >> 1] + row * kTilePitch + c;
            if (vec) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)),
                             "l"(src + (k < a.in ? k : 0)), "r"(k < a.in ? 16 : 0)
                             : "memory");
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) dst[q] = k + q < a.in ? src[k + q] : 0.0f;
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    double acc[4][4] = {};
    fetch(0, 0);
    for (int k0 = 0, buf = 0; k0 < a.in; k0 += kTileK, buf ^= 1) {
        if (k0 + kTileK < a.in) {
            fetch(k0 + kTileK, buf ^ 1);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncthreads();
        const float *xt = tile[buf][0] + (rw + g) * kTilePitch + t, *wt = tile[buf][1] + (ew + g) * kTilePitch + t;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            double x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (double)xt[(i & 1) * 8 * kTilePitch + 16 * h + 4 * (i >> 1)];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                double w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = (double)wt[n * 8 * kTilePitch + 16 * h + 4 * i];
                mma_f64(acc[n], x, w);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + rw + g + 8 * (i >> 1), e = e0 + ew + 8 * n + 2 * t + (i & 1);
            if (r < a.rows && e < a.n_experts) {
                a.l[(size_t)r * a.n_experts + e] = acc[n][i];
                if (a.logits) a.logits[(size_t)r * a.n_experts + e] = (float)acc[n][i];
            }
        }
}

// Order of the choice as a number: NaN greatest, then by value; 0 only for -inf.
__device__ __forceinline__ unsigned long long rank_key(double v) {
    if (v != v) return ~0ull;
    const long long b = __double_as_longlong(v + 0.0);  // -0 ranks as 0
    return b < 0 ? (unsigned long long)(~b) - 0x000fffffffffffffull : (unsigned long long)b | 0x8000000000000000ull;
}

constexpr int kTopkWarps = 4;

// One warp per row.
__global__ void __launch_bounds__(32 * kTopkWarps) route_topk_kernel(const RouteArgs a) {
    extern __shared__ unsigned long long s_keys[];  // per warp: [n_experts] keys of the choice, [n_experts] scores
    launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = blockIdx.x * kTopkWarps + warp;
    if (r >= a.rows) return;
    const double* l = a.l + (size_t)r * a.n_experts;
    unsigned long long* key = s_keys + (size_t)warp * 2 * a.n_experts;
    double* score = reinterpret_cast<double*>(key + a.n_experts);
    double sum = 1.0;
    if (a.scoring == MLQ_SCORE_SOFTMAX) {
        double top = -INFINITY;
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
        sum = 0.0;
        for (int e = lane; e < a.n_experts; e += 32) {
            const double v = exp(l[e] - top);
            score[e] = v;
            sum += v;
        }
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    } else {
        for (int e = lane; e < a.n_experts; e += 32) score[e] = 1.0 / (1.0 + exp(-l[e]));
    }
    for (int e = lane; e < a.n_experts; e += 32) {
        const double v = score[e] / sum;
        score[e] = v;
        key[e] = rank_key(a.bias ? v + (double)a.bias[e] : v);
    }
    __syncwarp();
    double picked_sum = 0.0, mine[2] = {0.0, 0.0};  // lane j keeps slots j and j + 32
    int my_id[2] = {-1, -1};
    for (int j = 0; j < a.top_k; ++j) {
        unsigned long long best = 0;
        int at = 0;
        for (int e = lane; e < a.n_experts; e += 32)
            if (key[e] > best) best = key[e], at = e;  // the first of equals in this lane
        const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(best >> 32));
        const bool h = (unsigned)(best >> 32) == hi;
        const unsigned lo = __reduce_max_sync(0xffffffffu, h ? (unsigned)best : 0u);
        if (hi == 0 && lo == 0) break;  // only masked experts are left
        at = (int)__reduce_min_sync(0xffffffffu, h && (unsigned)best == lo ? (unsigned)at : 0xffffffffu);
        const double s = score[at];
        picked_sum += s;
        if (lane == (j & 31)) mine[j >> 5] = s, my_id[j >> 5] = at;
        if (lane == (at & 31)) key[at] = 0;
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
// rows x experts from which the tiled logits are faster (K = 3584: 127 x 256 takes 33 us there and 150 us tiled, where a
// tile's K steps take that long however few the tiles; 2048 x 256 takes ~600 us there and ~300 us tiled)
constexpr long long kTileWork = 280 * 1024;

template <typename... Params, typename... Args>
cudaError_t launch_pdl(void (*kernel)(Params...), dim3 grid, int block, size_t smem, cudaStream_t stream, Args&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
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
        const int vec = a.in % 4 == 0 && reinterpret_cast<uintptr_t>(a.w) % 16 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0;
        auto up = [](int n, int d) { return (unsigned)((n + d - 1) / d); };
        cudaError_t e;
        if (a.rows == 1)
            e = launch_pdl(route_logits_kernel<2, 1>, dim3(up(a.n_experts, 2)), 256, 0, stream, a, vec);
        else if ((long long)a.rows * a.n_experts < kTileWork)
            e = launch_pdl(route_logits_kernel<4, 4>, dim3(up(a.n_experts, 4), up(a.rows, 4)), 256, 0, stream, a, vec);
        else
            e = launch_pdl(route_tile_kernel, dim3(up(a.rows, kTile), up(a.n_experts, kTile)), 256, 0, stream, a, vec);
        if (e != cudaSuccess) return e;
        // at most 64 KB (1024 experts); the default limit of 48 KB is raised only for calls that need it
        const size_t smem = (size_t)kTopkWarps * 2 * a.n_experts * sizeof(double);
        if (smem > 48 * 1024) {
            e = cudaFuncSetAttribute(route_topk_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)(kTopkWarps * 2 * MLQ_MOE_MAX_EXPERTS * sizeof(double)));
            if (e != cudaSuccess) return e;
        }
        e = launch_pdl(route_topk_kernel, dim3(up(a.rows, kTopkWarps)), 32 * kTopkWarps, smem, stream, a);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace mlq
