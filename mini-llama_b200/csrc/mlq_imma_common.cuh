// mlq_imma_common.cuh -- what the two streaming kernels share: activations,
// asynchronous copies, and how work is dealt out.
#pragma once

#include <atomic>
#include <type_traits>

#include "mlq_imma_args.cuh"
#include "mlq_tmap.h"

namespace mlq {
namespace {

// f(integral_constant 0), .., f(integral_constant N - 1)
template <int N, int I = 0, class Fn>
__device__ __forceinline__ void static_for(Fn f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        static_for<N, I + 1>(f);
    }
}

// Two fp32 values in one instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

__device__ __forceinline__ float activate(float v, int act) {
    switch (act) {
        case MLQ_ACT_SILU: return v / (1.0f + expf(-v));
        // v * Phi(v), by the complementary error function: no cancellation for negative v
        case MLQ_ACT_GELU: return 0.5f * v * erfcf(-0.70710678118654752f * v);
        // 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u)), u = sqrt(2 / pi) (v + 0.044715 v^3)
        case MLQ_ACT_GELU_TANH: return v / (1.0f + expf(-1.5957691216057308f * v * (1.0f + 0.044715f * v * v)));
        case MLQ_ACT_RELU: return v < 0.0f ? 0.0f : v;
        case MLQ_ACT_SIGMOID: return 1.0f / (1.0f + expf(-v));
        default: return v;
    }
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// This thread's arrival at an mbarrier once its copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// How a launch's units, of `per` rounds each, are dealt out.  Every team takes
// `each` whole units; the units left over are spread by rounds, a contiguous
// range per team, when that saves more than `join` rounds, which the adding up
// costs whoever finishes a shared unit, else one unit each to as many teams.
struct Deal {
    int teams, per, each, rest;  // rest: units left over
    long long rounds;            // theirs, dealt by rounds to the first `sharers` teams; 0: dealt whole
    int sharers;                 // each has a round at least: who shares a unit follows from its ends
    __device__ __forceinline__ Deal(int units, int per_, int teams_, int join) : teams(teams_), per(per_) {
        each = units / teams;
        rest = units - each * teams;
        const long long all = (long long)rest * per;
        rounds = (all + teams - 1) / teams + join < per ? all : 0;
        sharers = rounds < teams ? (int)rounds : teams;
    }
    // first round (among the left-over units') of team i, and the team that has round t
    __device__ __forceinline__ long long begin(int i) const { return i < sharers ? rounds * i / sharers : rounds; }
    __device__ __forceinline__ int owner(long long t) const { return (int)(((t + 1) * sharers - 1) / rounds); }
};

// A team's work, piece by piece: rounds [r0, r1) of unit u.
struct Work {
    int u, r0, r1, n;    // the piece, and how many there were
    long long t, t_end;  // rounds of left-over units still to come
    int left;            // whole units still to come
    __device__ __forceinline__ Work(const Deal& d, int id) : u(0), r0(0), r1(0), n(0) {
        left = d.each + (d.rounds == 0 && id < d.rest ? 1 : 0);
        t = d.rounds ? d.begin(id) : 0;
        t_end = d.rounds ? d.begin(id + 1) : 0;
    }
    // whole units lie `teams` apart, so that the teams work on neighbours
    __device__ __forceinline__ bool next(const Deal& d, int id) {
        if (left > 0) {
            u = n * d.teams + id, r0 = 0, r1 = d.per;
            --left, ++n;
            return true;
        }
        if (t >= t_end) return false;
        const int k = (int)(t / d.per);
        u = d.each * d.teams + k;
        r0 = (int)(t - (long long)k * d.per);
        r1 = t_end - t < d.per - r0 ? r0 + (int)(t_end - t) : d.per;
        t += r1 - r0;
        return true;
    }
};

inline bool aligned_rows(int fmt, const void* w, int bpr) {
    return reinterpret_cast<uintptr_t>(w) % 16 == 0 && (long long)bpr * block_bytes(fmt) % 16 == 0 &&
           encode_fn() != nullptr;
}

// Tensor maps of a launch's matrices: boxes of 16 rows (kPair: 8 of each) x 8
// blocks (q4_1: 4), in 16-bit elements.
inline bool make_weight_maps(ImmaMaps* maps, const ImmaArgs& a, bool pair, int box_bytes) {
    for (int i = 0; i < (pair ? 2 : 1); ++i)
        if (!make_map_2d(&maps->m[i], CU_TENSOR_MAP_DATA_TYPE_UINT16, const_cast<uint8_t*>(a.w[i]),
                         (uint64_t)a.row_bytes / 2, (uint64_t)a.total_rows, (uint64_t)a.row_bytes, box_bytes / 2,
                         pair ? 8 : 16, CU_TENSOR_MAP_SWIZZLE_NONE))
            return false;
    return true;
}

// Once per kernel and device (`done`: a bit per device): the kernel may use
// all the shared memory there is, and was built with the registers that its split
// between producers and computing warps counts on (with fewer, the computing
// warps would wait for more for ever).
template <class Kernel>
cudaError_t ready_kernel(Kernel k, int regs, std::atomic<uint64_t>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    cudaFuncAttributes fa{};
    e = cudaFuncGetAttributes(&fa, k);
    if (e != cudaSuccess) return e;
    if (fa.numRegs < regs) return cudaErrorInvalidConfiguration;
    int most = 0;
    e = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, most - (int)fa.sharedSizeBytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
}

}  // namespace
}  // namespace mlq
