// mlq_imma_many.cuh -- the streaming kernel for many rows of x per matrix
// (tcgen05 with fp16 operands; mathematics: mlq_imma.cuh; the launches around
// it: mlq_imma.cu).
//
// One CTA per SM.  A unit is a tile of 128 rows of one matrix (kPair: 64 gate
// and 64 up rows) against one segment of up to 128 rows of x; a stage is 64
// values of K (2 blocks), a round 4 stages.  Weights arrive as packed blocks
// (TMA, or 16-byte pieces where rows are not aligned) and go through the registers
// into tensor memory as the A operand: shared memory holds each only once, packed.
// x (hi and lo, fp16) comes by TMA as the B operand.  12 products of 16 values
// per stage (lo hi and hi lo first, then hi hi: the sum has its full size in 4
// only), and a stage's sums are drained into fp32 registers with the power-of-two scales
// of its weight row and its row of x.
//
//   warps 0-7    decode: warp w row 32 (w mod 4) + lane, block w / 4 of a stage
//   warps 8-15   drain: the same rows, half of the segment's columns; the end of a unit
//   warp 16, 19  weights; 17: x; 18: products
//
// Tensor memory: 2 sums of 128 columns (4 of 64 where a segment has no more), 4 operands of 64 (hi 32, lo 32).
// Rounds are dealt out evenly as in mlq_imma_few.cuh.
//
// 18944 x 16384, q4_0: 16 rows 134 us, 64 rows 159 us (250 TFLOP/s), 128 rows
// 234 us (340).  A stage takes ~1200 cycles at 64 rows, of which the products are
// 400 to 550; decoding (~500 and ~300 of handing over) and draining (~650) run beside
// them but on the same schedulers, which issue 0.55 instructions a cycle, and each
// stage passes three barriers.  Twice the decoding warps, two stages at a time and more
// sums in tensor memory changed nothing.  The int8 and fp16 instructions of
// a warp (mma.sync) did the same work at 85 TFLOP/s.
#pragma once

#include <cuda_fp16.h>

#include "mlq_imma_common.cuh"
#include "mlq_tc.cuh"

namespace mlq {
namespace {

constexpr int kUnitRows = 128;
constexpr int kRoleWarps = 8;                    // that decode, and that drain
constexpr int kManyThreads = 32 * (2 * kRoleWarps + 4);
constexpr int kDrainThreads = 32 * kRoleWarps;
constexpr int kOperands = 4, kScaleRing = 8, kXRing = 16, kDone = 8;
constexpr int kMaxBStages = 6;                   // + 4 sums: scales of x outlive the operand by as many products
constexpr int kXchPitch = kUnitRows + 4;         // exchange of a unit's results: [32 rows of x][128 rows + 4]
constexpr int kXchBytes = 32 * kXchPitch * 4;
constexpr int kManyJoin = 2;                     // rounds
// registers at launch, and after the split
constexpr int kManyLaunchRegs = 96, kDecodeRegs = 88, kDrainRegs = 136, kOtherRegs = 32;
static_assert((kRoleWarps * (kDecodeRegs + kDrainRegs) + 4 * kOtherRegs) * 32 <= kManyThreads * kManyLaunchRegs,
              "the shares must not exceed the launch's registers, or setmaxnreg would wait for ever");

// Tensor maps: weights ([1]: the up projections of kPair), x in boxes of 32,
// 64, 96 and 128 rows, hi and lo in one.
struct ManyMaps {
    CUtensorMap w[2], x[4];
};

// Packed blocks of 128 rows, one round.  Aligned: as TMA boxes (q4_1: two of 4
// blocks, so that 8 rows' 16-byte pieces lie in different banks); else the 16-byte
// windows that hold a row's blocks.
template <int F, bool ALN>
struct RawSlot {
    static constexpr int kChunk = 8 * (F == kQ8_0 ? 34 : F == kQ4_0 ? 18 : 20);
    static constexpr int kBoxes = ALN && F == kQ4_1 ? 2 : 1;
    static constexpr int kPitch = ALN ? kChunk / kBoxes : (kChunk + 15 + 15) / 16 * 16;
    static constexpr int kBytes = kUnitRows * kPitch * kBoxes;
};

__device__ __forceinline__ void drain_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kDrainThreads) : "memory"); }

// Whether `p` holds for any draining thread.
__device__ __forceinline__ bool drain_any(bool p) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r)
                 : "r"((uint32_t)p), "n"(kDrainThreads)
                 : "memory");
    return r;
}

__device__ __forceinline__ uint32_t h2(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 as_h2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

// A block's codes: W words of them, and its d (q4_1: d, m) as they are stored.
template <int F>
struct Block {
    static constexpr int W = F == kQ8_0 ? 8 : 4;
    uint32_t qs[W], dm;
};

// Block h of pair j of a round, and the d (q4_1: d, m) of the pair's other one;
// at: the lane's row in the slot (unaligned: its first byte).
template <int F, bool ALN>
__device__ __forceinline__ void load_block(uint32_t at, int j, int h, Block<F>& b, uint32_t& other) {
    constexpr int W = Block<F>::W, BB = F == kQ8_0 ? 34 : F == kQ4_0 ? 18 : 20;
    if constexpr (ALN) {
        const uint32_t pair = at + (F == kQ4_1 ? (j >> 1) * kUnitRows * 80 + (j & 1) * 40 : j * 2 * BB);
        if constexpr (F == kQ4_1) {
            const uint32_t from = pair + BB * h;
            b.dm = lds_u32(from);
#pragma unroll
            for (int k = 0; k < W; ++k) b.qs[k] = lds_u32(from + 4 + 4 * k);
            other = lds_u32(pair + BB * (1 - h));
        } else {
            // starts at a word, for h = 1 two bytes later
            const uint32_t from = pair + (BB - 2) * h;
            uint32_t w[W + 1];
#pragma unroll
            for (int k = 0; k <= W; ++k) w[k] = lds_u32(from + 4 * k);
            b.dm = (w[0] >> (16 * h)) & 0xffffu;
#pragma unroll
            for (int k = 0; k < W; ++k) b.qs[k] = __funnelshift_rc(w[k], w[k + 1], 16 + 16 * h);
            other = lds_u16(pair + BB * (1 - h));
        }
    } else {
        auto word = [](uint32_t at, uint32_t lo, uint32_t hi) { return __funnelshift_r(lo, hi, 8 * (at & 3)); };
        const uint32_t from = at + (2 * j + h) * BB, to = at + (2 * j + 1 - h) * BB;
        b.dm = word(from, lds_u32(from & ~3u), lds_u32((from & ~3u) + 4));
        other = word(to, lds_u32(to & ~3u), lds_u32((to & ~3u) + 4));
        const uint32_t qs = from + (F == kQ4_1 ? 4 : 2);
        uint32_t last = lds_u32(qs & ~3u);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const uint32_t next = lds_u32((qs & ~3u) + 4 * k + 4);
            b.qs[k] = word(qs, last, next);
            last = next;
        }
    }
}

// The power of two that brings the larger of two blocks' weights to 2^13 .. 2^14
// (q4_1: 2^15), as float bits; *inverse undoes it.
template <int F>
__device__ __forceinline__ float weight_scale(uint32_t dm0, uint32_t dm1, float* inverse) {
    uint32_t most = max(dm0 & 0x7fffu, dm1 & 0x7fffu);
    float v = __half2float(__ushort_as_half((unsigned short)most));
    int top = 260;  // 127 * 2^6 below 2^13, codes up to 128
    if (F == kQ4_1) {
        most = max((dm0 >> 16) & 0x7fffu, (dm1 >> 16) & 0x7fffu);
        v = fmaxf(16.0f * v, __half2float(__ushort_as_half((unsigned short)most)));
        if (most > 0x7c00u) v = NAN;
        top = 267;
    }
    int f = top - (int)(__float_as_uint(v) >> 23);
    if (f > 253) f = 253;
    *inverse = __uint_as_float((uint32_t)(254 - f) << 23);
    return __uint_as_float((uint32_t)f << 23);
}

// A block's weights times `scale`, as fp16 pairs hi and lo.  d * c has at most
// 19 bits, so hi + lo is exact (q4_1: d * c + m is rounded once in fp32, and
// hi + lo keeps 22 bits of it).
template <int F>
__device__ __forceinline__ void to_halves(const Block<F>& b, float scale, uint32_t (&hi)[16], uint32_t (&lo)[16]) {
    const float d = __half2float(__ushort_as_half((unsigned short)(b.dm & 0xffffu))) * scale;
    const float m = F == kQ4_1 ? __half2float(__ushort_as_half((unsigned short)(b.dm >> 16))) * scale : 0.0f;
    const __half2 d2 = __float2half2_rn(d);
    auto put = [&](int i, __half2 c) {
        if constexpr (F == kQ4_1) {
            const float2 q = __half22float2(c);
            const float w0 = fmaf(q.x, d, m), w1 = fmaf(q.y, d, m);
            const __half2 h = __floats2half2_rn(w0, w1);
            const float2 r = __half22float2(h);
            hi[i] = h2(h), lo[i] = h2(__floats2half2_rn(w0 - r.x, w1 - r.y));
        } else {
            const __half2 h = __hmul2(c, d2);
            hi[i] = h2(h), lo[i] = h2(__hfma2(c, d2, __hneg2(h)));
        }
    };
    if constexpr (F == kQ8_0) {
        // signed bytes u - 128 as the low bits of 1024 + u
        const __half2 off = __float2half2_rn(-1152.0f);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t u = b.qs[k] ^ 0x80808080u;
            put(2 * k, __hadd2(as_h2(__byte_perm(u, 0x64646464u, 0x4140)), off));
            put(2 * k + 1, __hadd2(as_h2(__byte_perm(u, 0x64646464u, 0x4342)), off));
        }
    } else {
        // 1024 + c from low nibbles; 1024 + 16 c from high ones, times 1 / 16
        constexpr float zero = F == kQ4_0 ? 8.0f : 0.0f;
        const __half2 low = __float2half2_rn(-1024.0f - zero), high = __float2half2_rn(-64.0f - zero),
                      sixteenth = __float2half2_rn(0.0625f);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint32_t q = b.qs[k] >> (8 * s);
                put(4 * k + 2 * s, __hadd2(as_h2((q & 0x000f000fu) | 0x64006400u), low));
                put(4 * k + 2 * s + 1, __hfma2(as_h2((q & 0x00f000f0u) | 0x64006400u), sixteenth, high));
            }
    }
}

template <int F, int MODE, bool ALN>
__global__ void __launch_bounds__(kManyThreads, 1)
    imma_many_kernel(const __grid_constant__ ManyMaps maps, const __grid_constant__ ImmaArgs a) {
    extern __shared__ __align__(1024) uint8_t smem[];
    using S = RawSlot<F, ALN>;
    __shared__ int s_last, s_dead, s_raw_issued, s_b_issued;
    __shared__ uint32_t s_tmem;
    __shared__ __align__(16) float s_w[kScaleRing][kUnitRows], s_x[kXRing][128];
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int steps = (a.bpr + kChunkBlocks - 1) / kChunkBlocks;
    const uint32_t xrows = (a.seg_cap + 31) / 32 * 32;  // of a stage of x
    // shared memory: x, weights, (not kDown) exchange, barriers
    const uint32_t b_bytes = 256u * xrows;
    const uint32_t b_ring = (smem_u32(smem) + 1023u) & ~1023u, raw_ring = b_ring + a.x_slots * b_bytes;
    const uint32_t xch = raw_ring + a.slots * S::kBytes;
    const uint32_t bars = xch + (MODE == kDown ? 0 : kXchBytes);
    // done: a stage's products; it frees x and the operand too
    const uint32_t raw_full = bars, raw_empty = raw_full + 64, b_full = raw_empty + 64, done = b_full + 64,
                   a_full = done + 8 * (kDone + 1), d_free = a_full + 32;
    if (threadIdx.x == 0) {
        s_dead = 0;
        for (int i = 0; i < 8; ++i) {
            mbar_init(raw_full + 8 * i, ALN ? 1 : 64);
            mbar_init(raw_empty + 8 * i, kRoleWarps);
            mbar_init(b_full + 8 * i, 1);
        }
        for (int i = 0; i <= kDone; ++i) mbar_init(done + 8 * i, 1);
        for (int i = 0; i < kOperands; ++i) mbar_init(a_full + 8 * i, kRoleWarps);
        for (int i = 0; i < 4; ++i) mbar_init(d_free + 8 * i, kRoleWarps);
        fence_mbar_init();
    }
    if (warp == 18) tmem_alloc(smem_u32(&s_tmem), 512);
    tc_fence_before();
    // Segments: as in mlq_imma_few.cuh.
    if (MODE == kPair) grid_dependency_wait();
    if (MODE != kDown) launch_dependents();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    const int nseg = MODE == kPlain ? (a.rows + a.seg_cap - 1) / a.seg_cap : __shfl_sync(0xffffffffu, __ldcg(a.nseg), 0);
    const int id = blockIdx.x;
    const Deal deal(nseg * a.tiles, steps, gridDim.x, kManyJoin);
    Work work(deal, id);
    constexpr int tile_rows = MODE == kPair ? kUnitRows / 2 : kUnitRows;
    auto segment = [&](int seg, int& e, int& first, int& count) {
        e = MODE == kPlain ? 0 : __ldcg(&a.segs[seg].expert);
        first = MODE == kPlain ? seg * a.seg_cap : __ldcg(&a.segs[seg].start);
        count = MODE == kPlain ? min(a.rows - first, a.seg_cap) : __ldcg(&a.segs[seg].count);
    };
    // sums in tensor memory: 4 of 64 columns or 2 of 128
    const uint32_t sums = xrows <= 64 ? 4 : 2, sum_shift = xrows <= 64 ? 2 : 1, sum_cols = 256 / sums;
    auto stages = [&](int c) { return min(4, (a.bpr - c * kChunkBlocks + 1) / 2); };
    // (whoever gives up lets the others run into their own limits)
    auto wait = [&](uint32_t bar, uint32_t parity, int code) {
        if (mbar_wait(bar, parity)) return true;
        report_error(a.err, code);
        *(volatile int*)&s_dead = 1;
        return false;
    };
    bool alive = true;

    if (warp < kRoleWarps) {
        // ---- decode ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kDecodeRegs));
        const int row = 32 * (warp & 3) + lane, h = warp >> 2;
        int slot = 0;
        uint32_t slot_phase = 0, n = 0;  // n: stages so far
        bool behind = false;             // the last one is on its way to tensor memory
        auto hand_over = [&] {
            if (!behind) return;
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(a_full + 8 * ((n - 1) % kOperands));
            behind = false;
        };
        while (alive && work.next(deal, id)) {
            int e, first, count;
            segment(work.u % nseg, e, first, count);
            [[maybe_unused]] uint32_t window = 0;
            if constexpr (!ALN) {
                // where the row starts in its 16-byte window
                const bool up = MODE == kPair && row >= 64;
                const long long at = (long long)e * a.out + work.u / nseg * tile_rows + (MODE == kPair ? row & 63 : row);
                window = (uint32_t)(reinterpret_cast<uintptr_t>(a.w[up ? 1 : 0]) + at * a.row_bytes) & 15;
            }
            for (int c = work.r0; alive && c < work.r1; ++c) {
                if (!__all_sync(0xffffffffu, wait(raw_full + 8 * slot, slot_phase, 44))) {
                    alive = false;
                    break;
                }
                uint32_t at = raw_ring + slot * S::kBytes + row * S::kPitch;
                if constexpr (!ALN) at += (window + (uint32_t)c * (S::kChunk & 15)) & 15;
                const int valid = a.bpr - c * kChunkBlocks;
#pragma unroll 1
                for (int j = 0; j < 4 && 2 * j < valid; ++j) {
                    Block<F> b;
                    uint32_t other;
                    load_block<F, ALN>(at, j, h, b, other);
                    if (2 * j + 1 >= valid) {  // the row ends with the first block of this pair
                        if (h == 0)
                            other = 0;
                        else
                            b.dm = 0;
                    }
                    float inverse;
                    const float scale = weight_scale<F>(b.dm, other, &inverse);
                    uint32_t hi[16], lo[16];
                    to_halves<F>(b, scale, hi, lo);
                    hand_over();  // a store takes as long as a stage's conversion
                    const int k = n % kOperands;
                    const uint32_t before = n - kOperands;  // had this place
                    if (n >= kOperands &&
                        !__all_sync(0xffffffffu, wait(done + 8 * (before % kDone), before / kDone & 1, 45))) {
                        alive = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t to = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + 256 + 64 * k + 16 * h;
                    tmem_st16(to, hi);
                    tmem_st16(to + 32, lo);
                    if (h == 0) s_w[n % kScaleRing][row] = inverse;
                    ++n, behind = true;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(raw_empty + 8 * slot);
                if (++slot == a.slots) slot = 0, slot_phase ^= 1;
            }
            hand_over();
        }
    } else if (warp < 2 * kRoleWarps) {
        // ---- drain ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kDrainRegs));
        if (MODE != kPair) grid_dependency_wait();
        if (MODE == kDown) launch_dependents();
        const int dw = warp - kRoleWarps, row = 32 * (dw & 3) + lane, half = dw >> 2;
        uint32_t n = 0;
        while (alive && work.next(deal, id)) {
            const int tile = work.u / nseg;
            int e, first, count;
            segment(work.u % nseg, e, first, count);
            const int cols = (count + 15) / 16 * 8;  // of this half
            // for the end of the unit: lane l has rows of x l and l + 32 of this half
            [[maybe_unused]] int pair[2];
            if (MODE == kDown)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int tok = half * cols + lane + 32 * k;
                    pair[k] = tok < count ? __ldcg(a.order + first + tok) : 0;
                }
            uint64_t acc2[32];  // pairs of columns
#pragma unroll
            for (int i = 0; i < 32; ++i) acc2[i] = 0;
            int todo = 0;
            for (int c = work.r0; c < work.r1; ++c) todo += stages(c);
            for (; todo > 0; --todo, ++n) {
                const uint32_t s = n & (sums - 1);
                if (!__all_sync(0xffffffffu, wait(done + 8 * (n % kDone), n / kDone & 1, 46))) {
                    alive = false;
                    break;
                }
                tc_fence_after();
                const uint32_t from = tmem + ((uint32_t)(32 * (dw & 3)) << 16) + sum_cols * s + half * cols;
                const float sw = s_w[n % kScaleRing][row];
                const float* sx = &s_x[n % kXRing][half * cols];
                const uint64_t sw2 = pack2(sw, sw);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (16 * q >= cols) break;
                    uint32_t v[16];
                    tmem_ld16_issue(from + 16 * q, v);
                    uint64_t f[8];
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const float4 x = *reinterpret_cast<const float4*>(sx + 16 * q + i);
                        f[i / 2] = mul2(pack2(x.x, x.y), sw2), f[i / 2 + 1] = mul2(pack2(x.z, x.w), sw2);
                    }
                    tmem_wait_ld(v);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        acc2[8 * q + i] = fma2(pack2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), f[i],
                                               acc2[8 * q + i]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(d_free + 8 * s);
            }
            float acc[64];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float2 p = unpack2(acc2[i]);
                acc[2 * i] = p.x, acc[2 * i + 1] = p.y;
            }
            // together, or some would wait below for others that have gone
            if (drain_any(!alive)) break;
            // a unit that several CTAs share: each leaves its sums in a slot (head: the unit started before its range,
            // tail: in it), and whoever comes last adds them up in order
            if (work.r1 - work.r0 != deal.per) {
                auto slot_of = [&](int c, bool tail) {
                    return a.split + ((size_t)2 * c + (tail ? 1 : 0)) * a.split_size + (size_t)(half * cols) * kUnitRows + row;
                };
                const long long r = (long long)(work.u - deal.each * deal.teams) * deal.per;
                const int j0 = deal.owner(r), j1 = deal.owner(r + deal.per - 1);
                float* mine = slot_of(id, id == j0);
#pragma unroll
                for (int i = 0; i < 64; ++i)
                    if (i < cols) mine[i * kUnitRows] = acc[i];
                __threadfence();
                drain_sync();
                if (dw == 0 && lane == 0) {
                    s_last = atomicAdd(a.split_done + j0, 1u) == (unsigned)(j1 - j0);
                    __threadfence();
                }
                drain_sync();
                if (!s_last) continue;
#pragma unroll
                for (int q = 0; q < 64; q += 8) {
                    if (q >= cols) break;
#pragma unroll
                    for (int i = q; i < q + 8; ++i) acc[i] = __ldcg(slot_of(j0, true) + i * kUnitRows);
#pragma unroll 4
                    for (int c = j0 + 1; c <= j1; ++c) {
                        const float* from = slot_of(c, false);
#pragma unroll
                        for (int i = q; i < q + 8; ++i) acc[i] += __ldcg(from + i * kUnitRows);
                    }
                }
            }
            const int tok0 = half * cols;
            if constexpr (MODE == kPair) {
                // 32 rows of x at a time through shared memory (16 of each half): a warp takes the 64 hidden values of a
                // row, in the order of the next product, to hi and lo
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (16 * q >= cols) break;
                    drain_sync();  // the last ones have been read
#pragma unroll
                    for (int i = 0; i < 16; ++i) sts_f32(xch + ((half * 16 + i) * kXchPitch + row) * 4, acc[16 * q + i]);
                    drain_sync();
#pragma unroll 1
                    for (int i = dw; i < 32; i += kRoleWarps) {
                        const int in = 16 * q + (i & 15), tok = (i >> 4) * cols + in;
                        if (in >= cols || tok >= count) continue;
                        float hv[2];
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int at = lane * 2 + k, el = (at & 32) + tile_element(a.next_fmt, at & 31);
                            const uint32_t g = xch + (i * kXchPitch + el) * 4;
                            hv[k] = tile * 64 + el < a.out
                                        ? silu_mul(__uint_as_float(lds_u32(g)), __uint_as_float(lds_u32(g + 256)))
                                        : 0.0f;
                        }
                        const size_t pos = first + tok;
                        slice_64(hv[0], hv[1])
                            .store(a.h + (pos * a.next_groups + tile) * 256, a.hs + (size_t)tile * a.hs_pitch + pos, lane);
                    }
                }
            } else if constexpr (MODE == kDown) {
                const int o = tile * kUnitRows + row;
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                    if (i >= cols || tok0 + i >= count) break;
                    const int to = __shfl_sync(0xffffffffu, pair[i / 32], i % 32);
                    if (o < a.out) a.part[(size_t)to * a.out + o] = acc[i];
                }
            } else {
                // as above, then a loop of few instructions: 64 copies of it would come from memory each time
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (16 * q >= cols) break;
                    drain_sync();
#pragma unroll
                    for (int i = 0; i < 16; ++i) sts_f32(xch + ((half * 16 + i) * kXchPitch + row) * 4, acc[16 * q + i]);
                    drain_sync();
                    const int loc = threadIdx.x & 127, o = tile * kUnitRows + loc;
                    const float bias = a.bias && o < a.out ? a.bias[o] : 0.0f;
#pragma unroll 1
                    for (int i = dw >> 2; i < 32; i += 2) {
                        const int in = 16 * q + (i & 15), tok = (i >> 4) * cols + in;
                        if (in >= cols || tok >= count || o >= a.out) continue;
                        const int r = first + tok;
                        const size_t to = (size_t)r * a.out + o;
                        const float add = a.residual ? a.residual[to] : 0.0f;
                        float v = activate(__uint_as_float(lds_u32(xch + (i * kXchPitch + loc) * 4)) + bias, a.act);
                        if (a.row_scale) v *= a.row_scale[r];
                        a.y[to] = a.residual ? add + v : v;
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == 18) {
            // ---- products ----
            // the whole warp goes through the loop and one lane issues, with operands that are the same in all: so they
            // are in uniform registers (a lane on its own takes ~100 cycles per instruction)
            uint32_t n = 0;
            int k = 0;
            uint32_t k_phase = 0;
            while (alive && work.next(deal, id)) {
                int e, first, count;
                segment(work.u % nseg, e, first, count);
                const uint32_t idesc = idesc_f16kind(false, kUnitRows, 0) |
                                       (uint32_t)__shfl_sync(0xffffffffu, (count + 15) / 16 * 2, 0) << 17;
                int todo = 0;
                for (int c = work.r0; c < work.r1; ++c) todo += stages(c);
                todo = __shfl_sync(0xffffffffu, todo, 0);
                const uint32_t plane = (uint32_t)__shfl_sync(0xffffffffu, (count + 31) / 32, 0) * 4096;
                for (; todo > 0; --todo, ++n) {
                    const uint32_t s = n & (sums - 1), o = n % kOperands;
                    // mostly all three have come, and are looked at together
                    const bool x_here = mbar_try_wait(b_full + 8 * k, k_phase),
                               sum_free = mbar_try_wait(d_free + 8 * s, (n >> sum_shift & 1) ^ 1),
                               w_here = mbar_try_wait(a_full + 8 * o, n / kOperands & 1);
                    if (!__all_sync(0xffffffffu, (x_here || wait(b_full + 8 * k, k_phase, 47)) &&
                                                     (sum_free || wait(d_free + 8 * s, (n >> sum_shift & 1) ^ 1, 48)) &&
                                                     (w_here || wait(a_full + 8 * o, n / kOperands & 1, 49)))) {
                        alive = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t at = b_ring + k * b_bytes, hi = tmem + 256 + 64 * o, lo = hi + 32, d = tmem + sum_cols * s;
                    const uint64_t xhi = sw128_desc(at), xlo = sw128_desc(at + plane);
                    if (elect_one()) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            mma_f16kind_ta(d, hi + 8 * q, xlo + 2 * q, idesc, q > 0);
                            mma_f16kind_ta(d, lo + 8 * q, xhi + 2 * q, idesc, 1u);
                        }
#pragma unroll
                        for (int q = 0; q < 4; ++q) mma_f16kind_ta(d, hi + 8 * q, xhi + 2 * q, idesc, 1u);
                        mma_commit(done + 8 * (n % kDone));
                    }
                    __syncwarp();
                    if (++k == a.x_slots) k = 0, k_phase ^= 1;
                }
            }
        } else if (warp == 17) {
            // ---- x ----
            if (MODE != kPair) grid_dependency_wait();
            int n = 0, k = 0;
            while (alive && work.next(deal, id)) {
                int e, first, count;
                segment(work.u % nseg, e, first, count);
                first = __shfl_sync(0xffffffffu, first, 0);
                const int boxes = __shfl_sync(0xffffffffu, (count + 31) / 32, 0);
                int todo = 0;
                for (int c = work.r0; c < work.r1; ++c) todo += stages(c);
                todo = __shfl_sync(0xffffffffu, todo, 0);
                for (int g = 4 * work.r0; todo > 0; --todo, ++n, ++g) {
                    const int before = n - a.x_slots;  // had this place
                    if (before >= 0 && !__all_sync(0xffffffffu, wait(done + 8 * (before % kDone), before / kDone & 1, 50))) {
                        alive = false;
                        break;
                    }
                    const uint32_t at = b_ring + k * b_bytes, bar = b_full + 8 * k;
                    if (elect_one()) {
                        mbar_arrive_expect_tx(bar, boxes * (8192 + 128));
                        bulk_g2s(smem_u32(s_x[n % kXRing]), a.xs + (size_t)g * a.xs_pitch + first, boxes * 128, bar);
                        tma_load_3d(at, &maps.x[boxes - 1], 0, first, 2 * g, bar);
                    }
                    __syncwarp();
                    if (++k == a.x_slots) k = 0;
                }
            }
            if (lane == 0) s_b_issued = n;
        } else if (!ALN || warp == 16) {
            // ---- weights ----
            int slot = 0, n = 0;
            uint32_t slot_phase = 1;
            const int me = 32 * (warp == 19) + lane;
            while (alive && work.next(deal, id)) {
                int e, first, count;
                segment(work.u % nseg, e, first, count);
                const int row0 = __shfl_sync(0xffffffffu, e, 0) * a.out + work.u / nseg * tile_rows;
                for (int c = work.r0; c < work.r1; ++c, ++n) {
                    const uint32_t full = raw_full + 8 * slot, dst = raw_ring + slot * S::kBytes;
                    if (!__all_sync(0xffffffffu, wait(raw_empty + 8 * slot, slot_phase, 51))) {
                        alive = false;
                        break;
                    }
                    if constexpr (ALN) {
                        if (elect_one()) {
                            mbar_arrive_expect_tx(full, S::kBytes);
#pragma unroll
                            for (int b = 0; b < S::kBoxes; ++b) {
                                const int c0 = (c * S::kChunk + b * S::kPitch) / 2;
                                const uint32_t d = dst + b * kUnitRows * S::kPitch;
                                tma_load_2d(d, &maps.w[0], c0, row0, full);
                                if (MODE == kPair) tma_load_2d(d + 64 * S::kPitch, &maps.w[1], c0, row0, full);
                            }
                        }
                    } else {
                        // two rows a thread: the 16-byte windows that hold a row's blocks
                        bool stored = false;
#pragma unroll 1
                        for (int r = me; r < kUnitRows; r += 64) {
                            const uint8_t* base = MODE == kPair && r >= 64 ? a.w[1] : a.w[0];
                            const long long row = row0 + (MODE == kPair ? r & 63 : r);
                            if (row >= a.total_rows) continue;
                            long long left = a.row_bytes - (long long)c * S::kChunk;
                            if (left > S::kChunk) left = S::kChunk;
                            const uint8_t* src = base + row * a.row_bytes + (long long)c * S::kChunk;
                            const uint8_t* end = src + left;
                            const uint8_t* q =
                                reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(src) & ~(uintptr_t)15);
                            for (uint32_t to = dst + r * S::kPitch; q < end; q += 16, to += 16) {
                                if (q < base) {  // the stack starts inside this window: only its own bytes are read
                                    for (int b = (int)(base - q); b < 16 && q + b < end; ++b) sts_u8(to + b, q[b]);
                                    stored = true;
                                } else {
                                    const long long m = end - q;
                                    cp_async_16(to, q, m < 16 ? (uint32_t)m : 16u);
                                }
                            }
                        }
                        if (stored) {  // plain stores are ordered by a plain arrival
                            asm volatile("cp.async.wait_all;" ::: "memory");
                            mbar_arrive(full);
                        } else {
                            cp_async_arrive(full);
                        }
                    }
                    __syncwarp();
                    if (++slot == a.slots) slot = 0, slot_phase ^= 1;
                }
            }
            if (!ALN) asm volatile("cp.async.wait_all;" ::: "memory");
            if (lane == 0 && warp == 16) s_raw_issued = n;
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    // after a wait that ran out, copies and products may still be in flight: each is waited for once more, bounded
    if (*(volatile int*)&s_dead && warp == 18) {
        if (ALN)
            for (int i = max(0, s_raw_issued - a.slots); i < s_raw_issued; ++i)
                mbar_wait(raw_full + 8 * (i % a.slots), (i / a.slots) & 1);
        for (int i = max(0, s_b_issued - a.x_slots); i < s_b_issued; ++i)
            mbar_wait(b_full + 8 * (i % a.x_slots), (i / a.x_slots) & 1);
        if (elect_one()) mma_commit(done + 8 * kDone);  // a barrier of its own
        __syncwarp();
        mbar_wait(done + 8 * kDone, 0);
    }
    if (warp == 18) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// x as [plane: group and hi or lo][row][64], boxes of both planes of a group.
inline bool make_map_x(CUtensorMap* m, const ImmaArgs& a, int rows) {
    const EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[3] = {64, (cuuint64_t)a.x_rows, (cuuint64_t)a.groups * 2};
    const cuuint64_t strides[2] = {(cuuint64_t)a.groups * 256, 128};
    const cuuint32_t box[3] = {64, (cuuint32_t)rows, 2}, one[3] = {1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<uint8_t*>(a.x), dims, strides, box, one,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int F, int MODE, bool ALN>
cudaError_t launch_one(ImmaArgs a, int grid, int smem_per_sm, cudaStream_t stream) {
    using S = RawSlot<F, ALN>;
    auto k = imma_many_kernel<F, MODE, ALN>;
    const int xrows = (a.seg_cap + 31) / 32 * 32, stage = 256 * xrows;
    // the system's 1 KB per CTA, the static part (up to 1 KB besides the scales), alignment, barriers
    const int fixed = 1024 + (kScaleRing * kUnitRows + kXRing * 128) * 4 + 1024 + 1024 + 512 + (MODE == kDown ? 0 : kXchBytes);
    // x comes from L2, about 2 us ahead at 0.3 us a stage and 64 rows; the weights have the rest
    a.x_slots = xrows > 64 ? 3 : xrows > 32 ? 4 : kMaxBStages;
    a.slots = (smem_per_sm - fixed - a.x_slots * stage) / S::kBytes;
    if (a.slots > 8) a.slots = 8;
    if (a.slots < 2) return cudaErrorInvalidConfiguration;
    const size_t smem = (size_t)1024 + a.x_slots * stage + a.slots * S::kBytes + (MODE == kDown ? 0 : kXchBytes) + 512;
    ManyMaps maps{};
    for (int i = 0; ALN && i < (MODE == kPair ? 2 : 1); ++i)
        if (!make_map_2d(&maps.w[i], CU_TENSOR_MAP_DATA_TYPE_UINT16, const_cast<uint8_t*>(a.w[i]),
                         (uint64_t)a.row_bytes / 2, (uint64_t)a.total_rows, (uint64_t)a.row_bytes, S::kPitch / 2,
                         MODE == kPair ? kUnitRows / 2 : kUnitRows, CU_TENSOR_MAP_SWIZZLE_NONE))
            return cudaErrorInvalidValue;
    for (int i = 0; i < xrows / 32; ++i)
        if (!make_map_x(&maps.x[i], a, 32 * (i + 1))) return cudaErrorInvalidValue;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = ready_kernel(k, kManyLaunchRegs, done);
    if (e != cudaSuccess) return e;
    return launch_pdl(k, grid, kManyThreads, smem, stream, maps, a);
}

template <int MODE>
cudaError_t launch_many(int fmt, ImmaArgs a, int sm_count, int smem_per_sm, long long max_units, cudaStream_t stream) {
    const bool aln = aligned_rows(fmt, a.w[0], a.bpr) && (MODE != kPair || aligned_rows(fmt, a.w[1], a.bpr));
    a.row_bytes = (long long)a.bpr * block_bytes(fmt);
    const long long rounds = max_units * ((a.bpr + kChunkBlocks - 1) / kChunkBlocks);
    int grid = sm_count < kMaxTeams / 2 ? sm_count : kMaxTeams / 2;
    if (grid > rounds) grid = rounds < 1 ? 1 : (int)rounds;
    switch (fmt) {
        case kQ8_0:
            return aln ? launch_one<kQ8_0, MODE, true>(a, grid, smem_per_sm, stream)
                       : launch_one<kQ8_0, MODE, false>(a, grid, smem_per_sm, stream);
        case kQ4_0:
            return aln ? launch_one<kQ4_0, MODE, true>(a, grid, smem_per_sm, stream)
                       : launch_one<kQ4_0, MODE, false>(a, grid, smem_per_sm, stream);
        default:
            return aln ? launch_one<kQ4_1, MODE, true>(a, grid, smem_per_sm, stream)
                       : launch_one<kQ4_1, MODE, false>(a, grid, smem_per_sm, stream);
    }
}

}  // namespace
}  // namespace mlq
