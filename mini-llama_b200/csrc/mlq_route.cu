// mlq_route.cu -- the router of a mixture-of-experts layer.
//
// logits = x Wr^T, then per row the scores, the top_k choice and its weights.
// The choice is discrete: two experts whose logits differ by less than an fp32
// sum's error would be swapped against the exact result.  So
// * few rows: fp64 sums (a product of two fp32 values is exact in fp64, its sum
//   off by ~1e-15);
// * many rows, where fp64 would take most of the time (8 TMAC/s at best): rows of x and of w
//   as 31-bit fixed point, each with its own power-of-two scale, in four signed
//   base-256 digits; the products of digits i and j meet in int8 matrix
//   instructions with int32 sums, one sum for each i + j <= 4 (13 of the 16 products;
//   all sums exact).  What rounding to 31 bits and the three left-out
//   products can change in a logit has a bound (error_bound below).  A row two of
//   whose candidates are closer than that, or whose bound is large (an outlier),
//   or not finite, goes on a list and is computed again in fp64: the choice is the fp64 one
//   in every case.
#include <limits.h>
#include <math.h>

#include <type_traits>

#include "mlq_device.cuh"
#include "mlq_kernels.h"
#include "mlq_tc.cuh"

namespace mlq {
namespace {

struct RouteArgs {
    const float* w;
    const float* bias;
    const float* x;
    int rows, in, n_experts, top_k, scoring, renorm;
    float scale;
    double* l;  // [rows][n_experts]; by digits: [rows on the list][n_experts]
    int32_t* ids;
    float* weights;
    float* logits;
    // by digits:
    uint8_t* xd;        // digits of x, an image of shared memory per 128 rows and K step
    uint8_t* wd;        // the same of w, per `tile` experts
    float2* xs;         // [rows]: what a unit of the row's last digit is worth, the row's sum of magnitudes
    float2* ws;         // [n_experts]
    long long* sums;    // [splits][row tiles * 128][expert tiles * tile]: products in units of 2^16 last digits
    int* list;          // [rows] rows to compute in fp64
    int* n_list;
    int* err;
    int steps, splits, row_tiles, expert_tiles, tile;
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
// Row r0 of x has its logits in row l0 of a.l.
template <int E, int R>
__device__ __forceinline__ void logits_of(const RouteArgs& a, int vec, int e0, int r0, int l0) {
    __shared__ double part[8][E * R];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double acc[E * R] = {};
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
            a.l[(size_t)(l0 + r - r0) * a.n_experts + e] = sum;
            if (a.logits) a.logits[(size_t)r * a.n_experts + e] = (float)sum;
        }
    }
}

template <int E, int R>
__global__ void __launch_bounds__(256) route_logits_kernel(const RouteArgs a, int vec) {
    launch_dependents();
    grid_dependency_wait();
    logits_of<E, R>(a, vec, blockIdx.x * E, blockIdx.y * R, blockIdx.y * R);
}

// The rows on the list, 4 experts at a time (mostly there are none).  x and w are
// read again for every 4 logits: 2048 x 256 x 4096 takes 49 us without such rows, 108 us with 64 of them, and
// 1.75 ms where every row has an element of 1e5 times the others.
__global__ void __launch_bounds__(256) route_again_kernel(const RouteArgs a, int vec) {
    launch_dependents();
    grid_dependency_wait();
    const int groups = (a.n_experts + 3) / 4;
    const long long n = (long long)*a.n_list * groups;
    for (long long i = blockIdx.x; i < n; i += gridDim.x) {
        const int at = (int)(i / groups);
        logits_of<4, 1>(a, vec, (int)(i % groups) * 4, a.list[at], at);
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// Many rows, by digits
// ---------------------------------------------------------------------------
constexpr int kRowTile = 128;     // rows of x per product: the lanes of tensor memory
constexpr int kExpertTile = 64;   // at most: all 4 digits of w are one operand of up to 256 columns
constexpr int kStepBytes = 128;   // values per K step: a row of the swizzled operand
constexpr int kStages = 2;        // a stage is 4 digits of 128 + 64 rows: 96 KB
constexpr int kXStage = 4 * kRowTile * kStepBytes, kWStage = 4 * kExpertTile * kStepBytes;
constexpr int kDigitSmem = 1024 + kStages * (kXStage + kWStage);
constexpr int kMaxSplits = 8;
constexpr int kSplitSteps = 128;  // 16384 values: an int32 sum takes 4 * 2^14 each, up to 32767 of them

// A row of x (or of w) per CTA, 16 values per thread and 4096 columns: the
// largest magnitude and the sum of magnitudes, then 16 bytes of each digit's
// image: a row's 128 bytes of a K step, 16-byte pieces exchanged as the 128-byte
// swizzle wants them.  Up to 4096 columns the values wait in registers.
__global__ void __launch_bounds__(256) route_digits_kernel(const RouteArgs a, int vec) {
    __shared__ float s_max[8], s_sum[8];
    launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool of_x = (int)blockIdx.x < a.rows;
    const int row = of_x ? blockIdx.x : blockIdx.x - a.rows;
    const float* src = (of_x ? a.x : a.w) + (size_t)row * a.in;
    grid_dependency_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.n_list = 0;
    const int k_end = a.steps * kStepBytes;
    float v[16];
    auto load = [&](int k0) {
        if (vec) {
#pragma unroll
            for (int k = 0; k < 16; k += 4) {
                const float4 q = k0 + k < a.in ? *reinterpret_cast<const float4*>(src + k0 + k) : make_float4(0, 0, 0, 0);
                v[k] = q.x, v[k + 1] = q.y, v[k + 2] = q.z, v[k + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) v[k] = k0 + k < a.in ? src[k0 + k] : 0.0f;
        }
    };
    float amax = 0.0f, sum = 0.0f;
    bool bad = false;
    for (int k0 = threadIdx.x * 16; k0 < k_end; k0 += 4096) {
        load(k0);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const float q = fabsf(v[k]);
            amax = fmaxf(amax, q), sum += q, bad |= !(q <= 3.402823466e38f);
        }
    }
    for (int o = 16; o > 0; o >>= 1) {
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (__any_sync(0xffffffffu, bad)) amax = NAN;
    if (lane == 0) s_max[warp] = amax, s_sum[warp] = sum;
    __syncthreads();
    amax = sum = 0.0f, bad = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = s_max[i];
        bad |= q != q, amax = fmaxf(amax, q), sum += s_sum[i];
    }
    if (bad) amax = 0.0f;
    // the power of two whose product with amax is in (limit / 2, limit]: four signed digits hold +-limit
    constexpr float kLimit = 2139062016.0f;  // below 127 * (2^24 + 2^16 + 2^8 + 1)
    int e = 254 + 30 - ((int)(__float_as_uint(amax) >> 23) & 0xff);
    if (e > 253) e = 253;
    if (amax * __uint_as_float((uint32_t)e << 23) > kLimit) --e;
    const float up = __uint_as_float((uint32_t)e << 23);
    if (threadIdx.x == 0)
        (of_x ? a.xs : a.ws)[row] =
            make_float2(bad ? NAN : amax == 0.0f ? 0.0f : __uint_as_float((254u << 23) - ((uint32_t)e << 23)), sum);
    const int tile = of_x ? kRowTile : a.tile, in_tile = row % tile;
    uint8_t* image = (of_x ? a.xd : a.wd) + (size_t)(row / tile) * a.steps * 4 * tile * kStepBytes + in_tile * kStepBytes;
    for (int k0 = threadIdx.x * 16; k0 < k_end; k0 += 4096) {
        if (k_end > 4096) load(k0);
        uint32_t digit[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t q[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // the signed digits of n are the bytes of n + 0x80808080, each less 128
                const int n = bad ? 0 : __float2int_rn(v[4 * k + j] * up);
                q[j] = ((uint32_t)n + 0x80808080u) ^ 0x80808080u;
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {  // 0: the highest
                const uint32_t sel = (uint32_t)(3 - d) | (uint32_t)(7 - d) << 4;
                digit[d][k] = __byte_perm(__byte_perm(q[0], q[1], sel), __byte_perm(q[2], q[3], sel), 0x5410);
            }
        }
        uint8_t* to = image + (size_t)(k0 / kStepBytes) * 4 * tile * kStepBytes + ((k0 / 16 & 7) ^ (in_tile & 7)) * 16;
#pragma unroll
        for (int d = 0; d < 4; ++d)
            *reinterpret_cast<uint4*>(to + (size_t)d * tile * kStepBytes) =
                make_uint4(digit[d][0], digit[d][1], digit[d][2], digit[d][3]);
    }
}

// One CTA: 128 rows x `tile` experts over one range of K steps.  Warp 0 fetches
// (a stage is two copies: the images are laid out for it), warp 1 issues the
// products, all four then add up the five sums of an element as one 64-bit number.
// 2048 x 256 x 4096: 24 us, 1.2 Pmac/s of int8 over its 28 Tmac; the matrix unit is
// busy for 64 % of that, the rest is the first loads, the last stage and the sums' way
// out.  With the digits' kernel (13 us, 76 MB in and out), the choice (12 us) and two
// nearly empty launches 52 us, where fp64 matrix instructions took 316.
__global__ void __launch_bounds__(128) route_product_kernel(const RouteArgs a) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(8) uint64_t s_full[kStages], s_empty[kStages], s_done;
    __shared__ uint32_t s_tmem;
    const uint32_t base = (smem_u32(smem) + 1023u) & ~1023u;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rt = blockIdx.x, et = blockIdx.y, split = blockIdx.z;
    const int k0 = (int)((long long)a.steps * split / a.splits), k1 = (int)((long long)a.steps * (split + 1) / a.splits);
    launch_dependents();
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(smem_u32(&s_full[i]), 1), mbar_init(smem_u32(&s_empty[i]), 1);
        mbar_init(smem_u32(&s_done), 1);
        fence_mbar_init();
    }
    if (warp == 1) tmem_alloc(smem_u32(&s_tmem), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    grid_dependency_wait();
    const uint32_t w_step = 4u * a.tile * kStepBytes;
    if (threadIdx.x == 0) {
        const uint8_t* x = a.xd + (size_t)rt * a.steps * kXStage;
        const uint8_t* w = a.wd + (size_t)et * a.steps * w_step;
        int k = k0;
        for (; k < k1; ++k) {
            const int s = (k - k0) % kStages;
            if (!mbar_wait(smem_u32(&s_empty[s]), ((k - k0) / kStages & 1) ^ 1)) {
                report_error(a.err, 34);
                break;
            }
            const uint32_t to = base + s * (kXStage + kWStage), bar = smem_u32(&s_full[s]);
            mbar_arrive_expect_tx(bar, kXStage + w_step);
            bulk_g2s(to, x + (size_t)k * kXStage, kXStage, bar);
            bulk_g2s(to + kXStage, w + (size_t)k * w_step, w_step, bar);
        }
        if (k < k1)  // gave up: the copies under way end before shared memory is given back
            for (int j = k > k0 + kStages ? k - kStages : k0; j < k; ++j)
                mbar_wait(smem_u32(&s_full[(j - k0) % kStages]), (j - k0) / kStages & 1);
    } else if (threadIdx.x == 32) {
        // D int32, A and B int8, both K-major, 128 rows; the columns are added below
        constexpr uint32_t idesc = 2u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(kRowTile >> 4) << 24;
        for (int k = k0; k < k1; ++k) {
            const int s = (k - k0) % kStages;
            if (!mbar_wait(smem_u32(&s_full[s]), (k - k0) / kStages & 1)) {
                report_error(a.err, 35);
                break;
            }
            tc_fence_after();
            const uint32_t at = base + s * (kXStage + kWStage);
            const uint64_t xd = sw128_desc(at), wd = sw128_desc(at + kXStage);
            const uint64_t x_digit = kRowTile * kStepBytes >> 4, w_digit = (uint64_t)a.tile * kStepBytes >> 4;
            // digit i of x against the first n digits of w, side by side, is one product: sum i + j stands next to
            // sum i + j - 1, and a digit of x is read once for all
#pragma unroll
            for (int q = 0; q < kStepBytes / 32; ++q) {
                auto product = [&](int i, int j, int n, bool add) {
                    mma_i8kind(tmem + (i + j) * a.tile, xd + i * x_digit + 2 * q, wd + j * w_digit + 2 * q,
                               idesc + ((uint32_t)(n * a.tile >> 3) << 17), add);
                };
                const bool more = k > k0 || q > 0;
                product(0, 0, 4, more);
                if (more) {
                    product(1, 0, 4, true);
                } else {
                    product(1, 0, 3, true);
                    product(1, 3, 1, false);  // the first into the last sum
                }
                product(2, 0, 3, true);
                product(3, 0, 2, true);
            }
            mma_commit(smem_u32(&s_empty[s]));
        }
        mma_commit(smem_u32(&s_done));
    }
    __syncwarp();
    if (!mbar_wait(smem_u32(&s_done), 0) && lane == 0) report_error(a.err, 36);
    tc_fence_after();
    // a thread has a row, but a warp writes a row at a time: through shared memory, which the products are done with
    const uint32_t pitch = a.tile * 8 + 16, rows = base + warp * 32 * pitch;
    for (int c = 0; c < a.tile; c += 16) {
        uint32_t v[5][16];
#pragma unroll
        for (int l = 0; l < 5; ++l) tmem_ld16_issue(tmem + ((uint32_t)(warp * 32) << 16) + l * a.tile + c, v[l]);
#pragma unroll
        for (int l = 0; l < 5; ++l) tmem_wait_ld(v[l]);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            long long n[2] = {(int)v[0][i], (int)v[0][i + 1]};
#pragma unroll
            for (int l = 1; l < 5; ++l) n[0] = n[0] * 256 + (int)v[l][i], n[1] = n[1] * 256 + (int)v[l][i + 1];
            asm volatile("st.shared.v2.b64 [%0], {%1, %2};" ::"r"(rows + lane * pitch + (c + i) * 8), "l"(n[0]), "l"(n[1])
                         : "memory");
        }
    }
    __syncwarp();
    long long* out = a.sums + (((size_t)split * a.row_tiles + rt) * kRowTile + warp * 32) * (a.expert_tiles * a.tile) +
                     et * a.tile;
    const int pairs = a.tile / 2;
#pragma unroll 4
    for (int i = lane; i < 32 * pairs; i += 32) {
        const int r = i / pairs, c = i % pairs * 2;
        long long n[2];
        asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(n[0]), "=l"(n[1]) : "r"(rows + r * pitch + c * 8));
        *reinterpret_cast<longlong2*>(out + (size_t)r * (a.expert_tiles * a.tile) + c) = make_longlong2(n[0], n[1]);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, 512);
}

// Order of the choice as a number: NaN greatest, then by value; 0 only for -inf.
__device__ __forceinline__ unsigned long long rank_key(double v) {
    if (v != v) return ~0ull;
    const long long b = __double_as_longlong(v + 0.0);  // -0 ranks as 0
    return b < 0 ? (unsigned long long)(~b) - 0x000fffffffffffffull : (unsigned long long)b | 0x8000000000000000ull;
}

constexpr int kTopkWarps = 4;

// Rows whose logits may be off by more than this are computed again.  (The bound adds up the worst case of every
// element; what is seen is about a hundredth of it.)
constexpr double kLogitError = 1.0 / (1 << 15);

// How far a logit by digits can be from the exact one: half a unit of the last
// digit in x, against the magnitudes of w, and the other way round; the three
// left-out products (digits 2 and 3: 2 * 2^14 * 2^8; 3 and 3: 2^14) and both
// halves' product.  1.01: the sums of magnitudes are fp32 sums.
__device__ __forceinline__ double error_bound(float2 x, float2 w, int in) {
    return 1.01 * (0.5 * x.x * w.y + 0.5 * w.x * x.y + (double)x.x * w.x * in * (8388608.0 + 16384.0 + 0.25));
}

enum { kRowsExact, kRowsByDigits, kRowsListed };

// Row r; its fp64 logits are row `at` of a.l.
template <int FROM>
__device__ __forceinline__ void choose(const RouteArgs& a, int r, int at_l) {
    extern __shared__ unsigned long long s_keys[];  // per warp: [n_experts] keys of the choice, [n_experts] scores
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long* key = s_keys + (size_t)warp * 2 * a.n_experts;
    double* score = reinterpret_cast<double*>(key + a.n_experts);
    double sum = 1.0, off = 0.0;
    // four experts of a lane at a time: a load, an exp or a division is a long chain of dependent steps
    constexpr int U = 4;
    if constexpr (FROM == kRowsByDigits) {
        const float2 xs = a.xs[r];
        const int pitch = a.expert_tiles * a.tile;
        const size_t plane = (size_t)a.row_tiles * kRowTile * pitch;
        float2 most = make_float2(0.0f, 0.0f);  // the bound grows with both
        bool bad = false;
        for (int e0 = lane; e0 < a.n_experts; e0 += 32 * U) {
            long long n[U] = {};
            float2 ws[U];
#pragma unroll
            for (int u = 0; u < U; ++u) ws[u] = a.ws[min(e0 + 32 * u, a.n_experts - 1)];
            const long long* from[U];
#pragma unroll
            for (int u = 0; u < U; ++u) from[u] = a.sums + (size_t)r * pitch + min(e0 + 32 * u, a.n_experts - 1);
#pragma unroll 4
            for (int i = 0; i < a.splits; ++i)
#pragma unroll
                for (int u = 0; u < U; ++u) n[u] += *from[u], from[u] += plane;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                bad |= ws[u].x != ws[u].x;
                most.x = fmaxf(most.x, ws[u].x), most.y = fmaxf(most.y, ws[u].y);
                const int e = e0 + 32 * u;
                const double v = (double)n[u] * 65536.0 * ((double)xs.x * ws[u].x);
                if (e < a.n_experts) {
                    score[e] = v;
                    if (a.logits) a.logits[(size_t)r * a.n_experts + e] = (float)v;
                }
            }
        }
        for (int o = 16; o > 0; o >>= 1) {
            most.x = fmaxf(most.x, __shfl_xor_sync(0xffffffffu, most.x, o));
            most.y = fmaxf(most.y, __shfl_xor_sync(0xffffffffu, most.y, o));
        }
        off = __any_sync(0xffffffffu, bad) ? NAN : error_bound(xs, most, a.in);
    } else {
#pragma unroll 4
        for (int e = lane; e < a.n_experts; e += 32) score[e] = a.l[(size_t)at_l * a.n_experts + e];
    }
    const bool softmax = a.scoring == MLQ_SCORE_SOFTMAX;
    double top = 0.0;
    if (softmax) {
        top = -INFINITY;
        bool nan = false;
        for (int e = lane; e < a.n_experts; e += 32) {
            const double v = score[e];
            nan |= v != v;
            top = v > top ? v : top;
        }
        for (int o = 16; o > 0; o >>= 1) {
            const double v = __shfl_xor_sync(0xffffffffu, top, o);
            top = v > top ? v : top;
        }
        if (__any_sync(0xffffffffu, nan)) top = NAN;
        sum = 0.0;
    }
    for (int e0 = lane; e0 < a.n_experts; e0 += 32 * U) {
        double v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = score[min(e0 + 32 * u, a.n_experts - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = exp(softmax ? v[u] - top : -v[u]);
        if (!softmax)
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = 1.0 / (1.0 + v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (e0 + 32 * u < a.n_experts) {
                score[e0 + 32 * u] = v[u];
                sum += v[u];
            }
    }
    if (softmax) {
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    } else {
        sum = 1.0;
    }
    const double of_sum = 1.0 / sum;
#pragma unroll 4
    for (int e = lane; e < a.n_experts; e += 32) {
        const double v = score[e] * of_sum;
        score[e] = v;
        key[e] = rank_key(a.bias ? v + (double)a.bias[e] : v);
    }
    __syncwarp();
    double picked_sum = 0.0, mine[2] = {0.0, 0.0};  // lane j keeps slots j and j + 32
    int my_id[2] = {-1, -1};
    // by digits one more than is asked for: is the last choice certain?
    const int picks = FROM == kRowsByDigits ? a.top_k + 1 : a.top_k;
    double extra = NAN;  // the score of that one
    int extra_id = -1;
    for (int j = 0; j < picks; ++j) {
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
        if (FROM == kRowsByDigits && j == a.top_k) {
            extra = s, extra_id = at;
            break;
        }
        picked_sum += s;
        if (lane == (j & 31)) mine[j >> 5] = s, my_id[j >> 5] = at;
        if (lane == (at & 31)) key[at] = 0;
        __syncwarp();
    }
    if constexpr (FROM == kRowsByDigits) {
        // lane j: is its slots' lead over the next ones larger than what both may be off by?
        bool certain = true;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            double next = __shfl_down_sync(0xffffffffu, mine[q], 1);
            int next_id = __shfl_down_sync(0xffffffffu, my_id[q], 1);
            const double wrap = __shfl_sync(0xffffffffu, mine[1], 0);
            const int wrap_id = __shfl_sync(0xffffffffu, my_id[1], 0);
            if (lane == 31) next = wrap, next_id = q == 0 ? wrap_id : -1;
            if (lane + 32 * q == a.top_k - 1) next = extra, next_id = extra_id;
            if (my_id[q] < 0 || next_id < 0 || lane + 32 * q >= a.top_k) continue;
            const double high = a.bias ? mine[q] + (double)a.bias[my_id[q]] : mine[q];
            const double low = a.bias ? next + (double)a.bias[next_id] : next;
            // d sigmoid <= 1/4 d logit; d softmax <= p (exp(2 d logit) - 1): with a bias every expert's p matters, not
            // the two's (without one the order of the scores is that of the logits)
            const double may = a.scoring == MLQ_SCORE_SIGMOID ? 0.5 * off
                               : a.bias                       ? 4.2 * off * of_sum
                                                              : 2.1 * off * (mine[q] + next);
            certain &= high - low > may + 4.5e-16 * (fabs(high) + fabs(low) + 1.0);
        }
        // (no bound at all: a row of zeros, whose logits are exact)
        if (off != 0.0 && (!__all_sync(0xffffffffu, certain) || !(off <= kLogitError))) {
            if (lane == 0) a.list[atomicAdd(a.n_list, 1)] = r;
            return;
        }
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

// One warp per row: logits from fp64 sums, from the products by digits (then
// the row goes on the list if its choice is not certain), or of the rows on that list.
template <int FROM>
__global__ void __launch_bounds__(32 * kTopkWarps) route_topk_kernel(const RouteArgs a) {
    launch_dependents();
    grid_dependency_wait();
    const int first = blockIdx.x * kTopkWarps + (threadIdx.x >> 5);
    if constexpr (FROM == kRowsListed) {
        for (int i = first; i < *a.n_list; i += gridDim.x * kTopkWarps) {
            choose<FROM>(a, a.list[i], i);
            __syncwarp();
        }
    } else {
        if (first < a.rows) choose<FROM>(a, first, first);
    }
}

constexpr int kPassRows = 2048;
constexpr int kCtas = 148;  // one per multiprocessor
// rows x experts x in_features from which the products go by digits (256 x 3584: 64 rows 21.5 us in fp64 and 24 us by
// digits, 127 rows 36 and 25, 2048 rows 590 and 50; 64 x 2048: 1024 rows 54 and 21; 8 x 4096: 2048 rows 26 and 31)
constexpr long long kDigitWork = 64ll << 20;

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// a product of two 31-bit values is below 2^62, in units of 2^16 2^46: the 64-bit sum takes 2^17 of them
constexpr int kDigitFeatures = 1 << 17;

bool by_digits(int n_experts, int in, int rows) {
    return rows >= 32 && in <= kDigitFeatures && (long long)rows * n_experts * in >= kDigitWork;
}

// The digits' part of the arguments, with the arrays at `ws`; their bytes.
size_t lay_out(RouteArgs& a, char* ws) {
    size_t n = 0;
    auto take = [&](auto*& p, size_t count) {
        p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(ws + n);
        n += up256(count * sizeof(*p));
    };
    if (!by_digits(a.n_experts, a.in, a.rows)) {
        take(a.l, (size_t)a.rows * a.n_experts);
        return n;
    }
    a.steps = (a.in + kStepBytes - 1) / kStepBytes;
    a.row_tiles = (a.rows + kRowTile - 1) / kRowTile;
    a.expert_tiles = (a.n_experts + kExpertTile - 1) / kExpertTile;
    a.tile = ((a.n_experts + a.expert_tiles - 1) / a.expert_tiles + 15) / 16 * 16;
    // one CTA each as far as they go; a range of K steps no longer than an int32 sum takes
    a.splits = kCtas / (a.row_tiles * a.expert_tiles);
    if (a.splits > kMaxSplits) a.splits = kMaxSplits;
    if (a.splits > a.steps) a.splits = a.steps;
    const int least = (a.steps + kSplitSteps - 1) / kSplitSteps;
    if (a.splits < least) a.splits = least;
    take(a.xd, (size_t)a.row_tiles * a.steps * kXStage);
    take(a.wd, (size_t)a.expert_tiles * a.steps * 4 * a.tile * kStepBytes);
    take(a.xs, a.rows);
    take(a.ws, a.n_experts);
    // for any number of splits, so that the workspace of more rows holds that of fewer
    const int tiles = a.row_tiles * a.expert_tiles * least;
    take(a.sums, (size_t)(tiles > kCtas ? tiles : kCtas) * kRowTile * a.tile);
    take(a.l, (size_t)a.rows * a.n_experts);
    take(a.list, a.rows);
    take(a.n_list, 1);
    return n;
}

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

size_t route_workspace_bytes(int n_experts, int in, int rows) {
    RouteArgs a{};
    a.n_experts = n_experts, a.in = in, a.rows = rows < kPassRows ? rows : kPassRows;
    return lay_out(a, nullptr);
}

cudaError_t launch_route(const mlq_router& r, const float* x, int rows, int32_t* ids, float* weights, float* logits,
                         void* ws, size_t ws_bytes, int* err, cudaStream_t stream) {
    for (int r0 = 0; r0 < rows; r0 += kPassRows) {
        RouteArgs a{};
        a.w = r.w, a.bias = r.bias;
        a.x = x + (size_t)r0 * r.in_features;
        a.rows = rows - r0 < kPassRows ? rows - r0 : kPassRows;
        a.in = r.in_features, a.n_experts = r.n_experts, a.top_k = r.top_k;
        a.scoring = r.scoring, a.renorm = r.renormalize, a.scale = r.scale;
        a.ids = ids + (size_t)r0 * r.top_k;
        a.weights = weights + (size_t)r0 * r.top_k;
        a.logits = logits ? logits + (size_t)r0 * r.n_experts : nullptr;
        a.err = err;
        if (lay_out(a, static_cast<char*>(ws)) > ws_bytes) return cudaErrorInvalidValue;
        const int vec = a.in % 4 == 0 && reinterpret_cast<uintptr_t>(a.w) % 16 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0;
        auto up = [](int n, int d) { return (unsigned)((n + d - 1) / d); };
        // at most 64 KB (1024 experts); the default limit of 48 KB is raised only for calls that need it
        const size_t smem = (size_t)kTopkWarps * 2 * a.n_experts * sizeof(double);
        auto topk = [&](auto kernel, unsigned grid) {
            if (smem > 48 * 1024) {
                const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                           (int)(kTopkWarps * 2 * MLQ_MOE_MAX_EXPERTS * sizeof(double)));
                if (e != cudaSuccess) return e;
            }
            return launch_pdl(kernel, dim3(grid), 32 * kTopkWarps, smem, stream, a);
        };
        cudaError_t e;
        if (!a.xd) {
            e = a.rows == 1
                    ? launch_pdl(route_logits_kernel<2, 1>, dim3(up(a.n_experts, 2)), 256, 0, stream, a, vec)
                    : launch_pdl(route_logits_kernel<4, 4>, dim3(up(a.n_experts, 4), up(a.rows, 4)), 256, 0, stream, a, vec);
            if (e == cudaSuccess) e = topk(route_topk_kernel<kRowsExact>, up(a.rows, kTopkWarps));
            if (e != cudaSuccess) return e;
            continue;
        }
        e = launch_pdl(route_digits_kernel, dim3(a.rows + a.n_experts), 256, 0, stream, a, vec);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(route_product_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kDigitSmem);
        if (e == cudaSuccess)
            e = launch_pdl(route_product_kernel, dim3(a.row_tiles, a.expert_tiles, a.splits), 128, kDigitSmem, stream, a);
        if (e == cudaSuccess) e = topk(route_topk_kernel<kRowsByDigits>, up(a.rows, kTopkWarps));
        if (e == cudaSuccess) e = launch_pdl(route_again_kernel, dim3(2 * kCtas), 256, 0, stream, a, vec);
        if (e == cudaSuccess) e = topk(route_topk_kernel<kRowsListed>, kCtas);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace mlq
