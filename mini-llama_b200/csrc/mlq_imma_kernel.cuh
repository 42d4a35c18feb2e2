// mlq_imma_kernel.cuh -- the streaming kernel of the experts' products and of
// the linear with an epilogue (mathematics and operand layout:
// mlq_imma.cuh; the launches around it: mlq_imma.cu).
//
// One CTA per SM: a producer warp and 8 computing
// warps.  A unit is a tile of 32, 64 or 128 rows of one matrix against one
// segment; the computing warps split it in 32-row groups and the K axis in
// interleaved steps of 8 blocks.  A round is one step of every warp: 256
// (row, block) squares of 32 whatever the tile, so rounds cost the same and the
// launch's rounds are dealt out evenly, a contiguous range per CTA.  Each
// warp has a ring of weight slots of its own that the producer fills by TMA,
// running ahead across units, so the weight stream does not wait for a unit's
// end.  The K parts of a unit meet in shared memory in a fixed order; a unit
// whose rounds fall to several CTAs is added up (in order) by the last of
// them to finish.
#pragma once

#include "mlq_imma_args.cuh"
#include "mlq_tmap.h"

namespace mlq {
namespace {

// The accumulators of up to 2 NT rows of x by digits: an instruction's 8
// columns are the 4 digits of 2 rows, so lane t holds digits 3 and 2 (t even) or
// 1 and 0 (t odd) of row t / 2, and the two are added once, at the end.
template <int F, int NT>
struct FewRows {
    static constexpr int kSubs = 1;
    uint32_t bo[NT], so[NT];
    uint4 b[NT][2][2];  // [.][half of a K step][pair of blocks]
    float4 s[NT][2], m[F == kQ4_1 ? NT : 1][2];
    float acc[NT][2][2], accm[F == kQ4_1 ? NT : 1][2][2];

    template <class TokenOf>
    __device__ __forceinline__ void init(const ImmaArgs& a, int count, int lane, TokenOf token) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            // columns without a row of x repeat the first one's; nothing reads them
            const int r = 2 * i + (g >> 2), rs = 2 * i + (t >> 1);
            bo[i] = (uint32_t)token(r < count ? r : 0) * (uint32_t)a.bprp * kSlicedBytes + (g & 3) * 64 + t * 16;
            so[i] = (uint32_t)token(rs < count ? rs : 0) * (uint32_t)a.bprp;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                acc[i][j][0] = acc[i][j][1] = 0.0f;
                if (F == kQ4_1) accm[i][j][0] = accm[i][j][1] = 0.0f;
            }
        }
    }

    // Half h of the x registers: the four blocks from kb.
    __device__ __forceinline__ void load_x(const ImmaArgs& a, int kb, int h) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const uint4* x = reinterpret_cast<const uint4*>(a.few_x.data + bo[i] + (size_t)kb * kSlicedBytes);
            b[i][h][0] = x[0], b[i][h][1] = x[16];
            s[i][h] = *reinterpret_cast<const float4*>(a.few_x.scale + so[i] + kb);
            if (F == kQ4_1) m[i][h] = *reinterpret_cast<const float4*>(a.few_x.sum + so[i] + kb);
        }
    }

    __device__ __forceinline__ void prime(const ImmaArgs& a, int kb) { load_x(a, kb, 0); }

    // One K step of 8 blocks from kb: while four are multiplied, the next four (of this step, then of the next one
    // at kb_next) are fetched.
    template <bool ALN, class Wait, class Rows>
    __device__ __forceinline__ void step(const ImmaArgs& a, int kb, int kb_next, int valid, int lane, Wait wait, Rows rows) {
        const int t = lane & 3;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            load_x(a, h ? kb_next : kb + 4, h ^ 1);
            if (h == 0) wait();
#pragma unroll
            for (int p2 = 0; p2 < 2; ++p2) {
                const int p = 2 * h + p2;
                if (!ALN && 2 * p >= valid) continue;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    RawA A[2];
                    load_pair<F, ALN>(rows(j, 0), rows(j, 1), p, t, A[0], A[1]);
                    if (!ALN && 2 * p + 1 >= valid) A[1].d[0] = A[1].d[1] = A[1].m[0] = A[1].m[1] = 0.0f;
#pragma unroll
                    for (int o = 0; o < 2; ++o) {
                        uint32_t op[4];
                        int8_operand<F>(A[o], op);
#pragma unroll
                        for (int i = 0; i < NT; ++i) {
                            const uint4 x = b[i][h][p2];
                            const float4 s4 = s[i][h];
                            const float sx = p2 ? (o ? s4.w : s4.z) : (o ? s4.y : s4.x);
                            int c[4];
                            imma_s8(c, op, o ? make_uint2(x.z, x.w) : make_uint2(x.x, x.y));
                            acc[i][j][0] = fmaf(A[o].d[0] * sx, (float)(c[0] * 256 + c[1]), acc[i][j][0]);
                            acc[i][j][1] = fmaf(A[o].d[1] * sx, (float)(c[2] * 256 + c[3]), acc[i][j][1]);
                            if (F == kQ4_1) {
                                const float4 m4 = m[i][h];
                                const float mx = p2 ? (o ? m4.w : m4.z) : (o ? m4.y : m4.x);
                                accm[i][j][0] = fmaf(A[o].m[0], mx, accm[i][j][0]);
                                accm[i][j][1] = fmaf(A[o].m[1], mx, accm[i][j][1]);
                            }
                        }
                    }
                }
            }
        }
    }

    // put(row of x 0..7, 16-row strip j, row half q, value)
    template <class Put>
    __device__ __forceinline__ void store(int, int lane, Put put) {
        const int t = lane & 3;
        // digits 3 and 2 count 2^16 times digits 1 and 0; q4 codes count 16
        const float f = (t & 1 ? 1.0f : 65536.0f) * (F == kQ8_0 ? 1.0f : 0.0625f);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    float v = acc[i][j][q] * f;
                    v += __shfl_xor_sync(0xffffffffu, v, 1);
                    if (F == kQ4_1) v += accm[i][j][q];
                    if (!(t & 1)) put(2 * i + (t >> 1), j, q, v);
                }
    }
};

// Up to 8 S rows of x by halves: one column per row.
template <int F, int S>
struct ManyRows {
    static constexpr int kSubs = S;
    static constexpr int kG = S < 2 ? S : 2;  // groups of 8 rows per buffer
    uint32_t bo[S], so[S][2];
    uint4 hi[2][kG], lo[2][kG];
    float s[2][kG][2], m[2][kG][2];
    float acc[S][2][2][2];  // [.][strip][row half][row of x 2t, 2t + 1]

    template <class TokenOf>
    __device__ __forceinline__ void init(const ImmaArgs& a, int count, int lane, TokenOf token) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int r = 8 * i + g;
            bo[i] = (uint32_t)token(r < count ? r : 0) * (uint32_t)a.bprp * kSlicedBytes + t * 16;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int rs = 8 * i + 2 * t + x;
                so[i][x] = (uint32_t)token(rs < count ? rs : 0) * (uint32_t)a.bprp;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
                acc[i][j][0][0] = acc[i][j][0][1] = acc[i][j][1][0] = acc[i][j][1][1] = 0.0f;
        }
    }

    // Buffer q: x of rows 8 kG gr .. of block blk.
    __device__ __forceinline__ void load_x(const ImmaArgs& a, int blk, int gr, int q) {
#pragma unroll
        for (int k = 0; k < kG; ++k) {
            const int i = gr * kG + k;
            const uint4* x = reinterpret_cast<const uint4*>(a.many_x.data + bo[i] + (size_t)blk * kSlicedBytes);
            hi[q][k] = x[0], lo[q][k] = x[4];
#pragma unroll
            for (int x2 = 0; x2 < 2; ++x2) {
                s[q][k][x2] = a.many_x.scale[so[i][x2] + blk];
                if (F == kQ4_1) m[q][k][x2] = a.many_x.sum[so[i][x2] + blk];
            }
        }
    }

    __device__ __forceinline__ void prime(const ImmaArgs& a, int kb) { load_x(a, kb, 0, 0); }

    // One K step of 8 blocks from kb: while up to 16 rows of a block are multiplied, the next ones (then the next
    // block's, then the next step's) are fetched.
    template <bool ALN, class Wait, class Rows>
    __device__ __forceinline__ void step(const ImmaArgs& a, int kb, int kb_next, int valid, int lane, Wait wait, Rows rows) {
        const int t = lane & 3;
#pragma unroll
        for (int p = 0; p < kChunkBlocks / 2; ++p) {
            if (2 * p >= valid) break;
            if (p == 0) wait();
            RawA A[2][2];  // [strip][block]
#pragma unroll
            for (int j = 0; j < 2; ++j) load_pair<F, ALN>(rows(j, 0), rows(j, 1), p, t, A[j][0], A[j][1]);
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                const int n = 2 * p + o;
                if (n >= valid) break;
                uint32_t op[2][8];
                half_operand<F>(A[0][o], op[0]);
                half_operand<F>(A[1][o], op[1]);
#pragma unroll
                for (int gr = 0; gr < S / kG; ++gr) {
                    const int q = (n * (S / kG) + gr) & 1;
                    if (gr + 1 < S / kG)
                        load_x(a, kb + n, gr + 1, q ^ 1);
                    else
                        load_x(a, n + 1 < kChunkBlocks && n + 1 < valid ? kb + n + 1 : kb_next, 0, q ^ 1);
#pragma unroll
                    for (int k = 0; k < kG; ++k) {
                        const int i = gr * kG + k;
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            hmma_f16(c, op[j], lo[q][k].x, lo[q][k].y);
                            hmma_f16(c, op[j] + 4, lo[q][k].z, lo[q][k].w);
                            hmma_f16(c, op[j], hi[q][k].x, hi[q][k].y);
                            hmma_f16(c, op[j] + 4, hi[q][k].z, hi[q][k].w);
                            const RawA& A1 = A[j][o];
#pragma unroll
                            for (int r = 0; r < 2; ++r)
#pragma unroll
                                for (int x = 0; x < 2; ++x) {
                                    acc[i][j][r][x] = fmaf(A1.d[r] * s[q][k][x], c[2 * r + x], acc[i][j][r][x]);
                                    if (F == kQ4_1) acc[i][j][r][x] = fmaf(A1.m[r], m[q][k][x], acc[i][j][r][x]);
                                }
                        }
                    }
                }
            }
        }
    }

    template <class Put>
    __device__ __forceinline__ void store(int sub, int lane, Put put) {
        const int t = lane & 3;
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (i == sub) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        put(2 * t, j, q, acc[i][j][q][0]);
                        put(2 * t + 1, j, q, acc[i][j][q][1]);
                    }
            }
    }
};

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

// The barrier of the computing warps.
__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kImmaWarps) : "memory"); }

// 8 computing warps, and 1 producer warp (tensor maps) or 4 (16-byte copies)
template <bool ALN>
constexpr int kThreads = 32 * (kImmaWarps + (ALN ? 1 : 4));
constexpr int kRedFloats = kImmaWarps * 8 * 32;  // [warp][row of x][row of the group]

// How a launch's rounds are dealt out: CTA i takes [begin(i), begin(i + 1)).
// Whole units when that costs no CTA more than 2 rounds (a round takes about
// 0.8 us of a CTA's share of HBM, adding up a split unit about 2 us).
struct Deal {
    long long total;
    int units, per_unit, ctas;
    bool whole;
    __device__ Deal(int units_, int per_unit_, int ctas_) : units(units_), per_unit(per_unit_), ctas(ctas_) {
        total = (long long)units * per_unit;
        if (ctas > total) ctas = (int)total;
        const long long even = ctas ? (total + ctas - 1) / ctas : 0;
        const long long by_unit = ctas ? (long long)((units + ctas - 1) / ctas) * per_unit : 0;
        whole = by_unit <= even + 2;
        if (whole && ctas > units) ctas = units;
    }
    __device__ long long begin(int i) const {
        return whole ? (long long)units * i / ctas * per_unit : total * i / ctas;
    }
    // the CTA that has round t (not asked when units are whole)
    __device__ int owner(long long t) const { return (int)(((t + 1) * ctas - 1) / total); }
};

template <int F, int MODE, bool ALN>
__global__ void __launch_bounds__(kThreads<ALN>, 1) imma_kernel(const __grid_constant__ ImmaMaps maps, const ImmaArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    using S = Slot<F, ALN>;
    __shared__ int s_last, s_dead, s_issued[kImmaWarps];
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int kws = kImmaWarps / a.groups;
    const int steps = (a.bpr + kChunkBlocks - 1) / kChunkBlocks;
    const int per_unit = (steps + kws - 1) / kws;
    float* red = reinterpret_cast<float*>(smem + kImmaWarps * a.slots * S::kBytes);  // two buffers
    const uint32_t slots0 = smem_u32(smem), bars0 = smem_u32(red + 2 * kRedFloats);
    // barriers of warp w's slot i: full at bars0 + 16 (w slots + i), empty 8 bytes on
    if (threadIdx.x == 0) s_dead = 0;
    for (int i = threadIdx.x; i < kImmaWarps * a.slots; i += kThreads<ALN>) {
        mbar_init(bars0 + 16 * i, ALN ? 1 : 32);
        mbar_init(bars0 + 16 * i + 8, 1);
    }
    fence_mbar_init();

    // The segments come from prep.  kPair is prep's dependent, so it waits;
    // kDown started after every CTA of kPair had waited for prep, so prep has
    // completed: it reads the segments (past L1) and streams weights at once.
    if (MODE == kPair) grid_dependency_wait();
    if (MODE != kDown) launch_dependents();
    __syncthreads();
    const int nseg = MODE == kPlain ? (a.rows + kSegTokens - 1) / kSegTokens : __ldcg(a.nseg);
    const Deal deal(nseg * a.tiles, per_unit, gridDim.x);
    const bool has_work = (int)blockIdx.x < deal.ctas;
    const long long t0 = has_work ? deal.begin(blockIdx.x) : 0, t1 = has_work ? deal.begin(blockIdx.x + 1) : 0;
    // a tile's segments follow one another: segments with more rows take longer, so each CTA gets a mix, and the
    // CTAs that share a tile are few
    auto tile_of = [&](int u) { return u / nseg; };
    auto seg_of = [&](int u) { return u % nseg; };
    const int unit_rows = (MODE == kPair ? 16 : 32) * a.groups;

    if (warp >= kImmaWarps) {
        // ---- producers ----
        int u = t0 < t1 ? (int)(t0 / per_unit) : 0, r = t0 < t1 ? (int)(t0 % per_unit) : 0;
        long long row0 = 0;
        bool fresh = true;
        if constexpr (ALN) {
            // lane w fills the ring of warp w
            const int w = lane, grp = w % a.groups, kw = w / a.groups;
            int slot = 0, phase = 1, issued = 0;
            if (w < kImmaWarps) {
                for (long long t = t0; t < t1; ++t) {
                    if (fresh) {
                        const int e = MODE == kPlain ? 0 : __ldcg(&a.segs[seg_of(u)].expert);
                        row0 = (long long)e * a.out + (long long)tile_of(u) * unit_rows + grp * (MODE == kPair ? 16 : 32);
                        fresh = false;
                    }
                    const int c = r * kws + kw;
                    if (c < steps) {
                        const uint32_t bar = bars0 + 16 * (w * a.slots + slot);
                        const uint32_t dst = slots0 + (w * a.slots + slot) * S::kBytes;
                        if (!mbar_wait(bar + 8, phase)) {
                            report_error(a.err, 31);
                            *(volatile int*)&s_dead = 1;
                        }
                        if (*(volatile int*)&s_dead) break;
                        mbar_arrive_expect_tx(bar, S::kBytes);
#pragma unroll
                        for (int b = 0; b < S::kBoxes; ++b) {
                            const int c0 = (c * chunk_bytes(F) + b * S::kPitch) / 2;
                            const uint32_t d = dst + b * 32 * S::kPitch;
                            tma_load_2d(d, &maps.m[0], c0, (int)row0, bar);
                            if (MODE == kPair) tma_load_2d(d + 16 * S::kPitch, &maps.m[1], c0, (int)row0, bar);
                        }
                        ++issued;
                        if (++slot == a.slots) slot = 0, phase ^= 1;
                    }
                    if (++r == per_unit) r = 0, ++u, fresh = true;
                }
                s_issued[w] = issued;
            }
        } else {
            // Producer warp k fills the rings of computing warps 2k and 2k + 1: lane l takes every second 16-byte window of
            // rows l / 2 and l / 2 + 16 of a slot.
            const int half = warp - kImmaWarps;
            const int sub = lane & 1;
            int count[2] = {0, 0};
            bool alive = true;
            for (long long t = t0; t < t1 && alive; ++t) {
                if (fresh) {
                    const int e = MODE == kPlain ? 0 : __ldcg(&a.segs[seg_of(u)].expert);
                    row0 = (long long)e * a.out + (long long)tile_of(u) * unit_rows;
                    fresh = false;
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int w = 2 * half + k, c = r * kws + w / a.groups;
                    if (c >= steps || !alive) continue;
                    const int slot = count[k] % a.slots;
                    const uint32_t bar = bars0 + 16 * (w * a.slots + slot);
                    if (!__all_sync(0xffffffffu, mbar_wait(bar + 8, ((count[k] / a.slots) & 1) ^ 1))) {
                        if (lane == 0) report_error(a.err, 31), *(volatile int*)&s_dead = 1;
                        alive = false;
                        continue;
                    }
                    long long left = a.row_bytes - (long long)c * chunk_bytes(F);
                    if (left > chunk_bytes(F)) left = chunk_bytes(F);
                    bool stored = false;
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh) {
                        const uint8_t* base = MODE == kPair && hh ? a.w[1] : a.w[0];
                        const long long row =
                            row0 + (w % a.groups) * (MODE == kPair ? 16 : 32) + (lane >> 1) + (MODE == kPair ? 0 : 16 * hh);
                        if (row >= a.total_rows) continue;
                        const uint8_t* src = base + row * a.row_bytes + (long long)c * chunk_bytes(F);
                        const uint8_t* end = src + left;
                        const uint8_t* win = reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(src) & ~(uintptr_t)15);
                        const uint32_t dst = slots0 + (w * a.slots + slot) * S::kBytes + ((lane >> 1) + 16 * hh) * S::kPitch;
#pragma unroll
                        for (int i = 0; i < (chunk_bytes(F) + 31) / 32 + 1; ++i) {
                            const uint8_t* q = win + 32 * i + 16 * sub;
                            if (q >= end) break;
                            const uint32_t to = dst + 32 * i + 16 * sub;
                            if (q < base) {  // the stack starts inside this window: only its own bytes are read
                                for (int b = (int)(base - q); b < 16 && q + b < end; ++b) sts_u8(to + b, q[b]);
                                stored = true;
                            } else {
                                const long long n = end - q;
                                cp_async_16(to, q, n < 16 ? (uint32_t)n : 16u);
                            }
                        }
                    }
                    if (stored) {  // plain stores are ordered by a plain arrival
                        asm volatile("cp.async.wait_all;" ::: "memory");
                        mbar_arrive(bar);
                    } else {
                        cp_async_arrive(bar);
                    }
                    ++count[k];
                }
                if (*(volatile int*)&s_dead) alive = false;
                if (++r == per_unit) r = 0, ++u, fresh = true;
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (lane < 2) s_issued[2 * half + lane] = 0;  // nothing is in flight
        }
        __syncwarp();
        if (MODE != kPair) grid_dependency_wait();
        if (MODE == kDown) launch_dependents();
        __syncthreads();
        return;
    }

    // ---- computing warps ----
    if (MODE != kPair) grid_dependency_wait();
    if (MODE == kDown) launch_dependents();
    const int grp = warp % a.groups, kw = warp / a.groups, g = lane >> 2;
    const uint32_t bars = bars0 + 16 * warp * a.slots, slots = slots0 + warp * a.slots * S::kBytes;
    int slot = 0, phase = 0, taken = 0, buf = 0;
    bool alive = true;
    int finished_tile = -1, finished = 0;  // kDown: units of one tile whose parts this CTA has written

    // kDown: counts them, and the CTA that completes a tile sums it for every row of x
    auto settle = [&]() {
        if (MODE != kDown || !a.done || finished == 0) return;
        compute_sync();
        if (threadIdx.x == 0) {
            __threadfence();
            s_last = atomicAdd(a.done + finished_tile, (unsigned)finished) + finished == (unsigned)nseg;
            __threadfence();
        }
        compute_sync();
        if (s_last) {
            for (int i = threadIdx.x; i < unit_rows * a.rows; i += 32 * kImmaWarps) {
                const int o = finished_tile * unit_rows + i % unit_rows, x = i / unit_rows;
                if (o < a.out) a.y[(size_t)x * a.out + o] = combine(a, x, o);
            }
        }
        finished = 0;
    };

    auto run_unit = [&](auto& acc, const Sliced& in, int first, int count, int u, int e, int r0, int r1) {
        using Acc = typename std::remove_reference<decltype(acc)>::type;
        (void)in;
        const int tile = tile_of(u);
        acc.init(a, count, lane, [&](int r) -> int {
            if (MODE == kPair) return __ldcg(a.order + first + r) / a.top_k;
            return first + r;
        });
        if (r0 * kws + kw < steps) acc.prime(a, (r0 * kws + kw) * kChunkBlocks);
        for (int r = r0; r < r1; ++r) {
            const int c = r * kws + kw;
            if (c >= steps) break;
            const int cn = r + 1 < r1 && c + kws < steps ? c + kws : c;  // the step after this one
            const uint32_t at = slots + slot * S::kBytes;
            uint32_t shift[2] = {0, 0};
            if constexpr (!ALN) {
                // where each row starts in its window
                const long long off = ((long long)e * a.out + (long long)tile * unit_rows + grp * (MODE == kPair ? 16 : 32)) *
                                          a.row_bytes +
                                      (long long)c * chunk_bytes(F);
                shift[0] = (uint32_t)((reinterpret_cast<uintptr_t>(a.w[0]) + off) & 15);
                shift[1] = (uint32_t)((reinterpret_cast<uintptr_t>(a.w[MODE == kPair ? 1 : 0]) + off) & 15);
            }
            acc.template step<ALN>(
                a, c * kChunkBlocks, cn * kChunkBlocks, a.bpr - c * kChunkBlocks, lane,
                [&]() {
                    if (alive && !__all_sync(0xffffffffu, mbar_wait(bars + 16 * slot, phase))) {
                        alive = false;
                        if (lane == 0) report_error(a.err, 30), *(volatile int*)&s_dead = 1;
                    }
                },
                [&](int j, int q) -> uint32_t {
                    // slot row of strip j's row g + 8 q
                    const int row = MODE == kPair ? 16 * q + 8 * j + g : 16 * j + 8 * q + g;
                    if constexpr (ALN) return at + row * S::kPitch;
                    const int in_matrix = MODE == kPair ? 8 * j + g : row;
                    return at + row * S::kPitch +
                           ((shift[MODE == kPair ? q : 0] + (uint32_t)(in_matrix * (a.row_bytes & 15))) & 15);
                });
            __syncwarp();
            if (alive) ++taken;
            if (lane == 0) mbar_arrive(bars + 16 * slot + 8);
            if (++slot == a.slots) slot = 0, phase ^= 1;
        }

        // one row of x's sums of this unit: get(row of the tile as the slots have it)
        auto epilogue = [&](int sub, int n, auto get) {
            if (MODE == kPair) {
                // a warp takes a block of 32 hidden values of one row of x, in the lane order of the next product
                const int blocks = a.groups / 2;
                for (int i = warp; i < n * blocks; i += kImmaWarps) {
                    const int tok = i / blocks, b = tile * blocks + i % blocks;
                    if (32 * b >= a.out) continue;
                    const bool few = count <= a.few;
                    const int el = few ? imma_element(a.next_fmt, b & 1, lane) : half_element(a.next_fmt, b & 1, lane);
                    const int loc = 32 * (i % blocks) + el;
                    const int row = (loc >> 4) * 32 + (loc & 15);
                    const float h = 32 * b + el < a.out ? silu_mul(get(tok, row), get(tok, row + 16)) : 0.0f;
                    const size_t at = (size_t)(first + 8 * sub + tok) * a.next_bprp + b;
                    if (few)
                        slice_digits(h, a.h.data + (at - b) * kSlicedBytes + digit_block(b), a.h.scale + at, a.h.sum + at, lane);
                    else
                        slice_halves(h, a.h.data + at * kSlicedBytes, a.h.scale + at, a.h.sum + at, lane);
                }
            } else {
                for (int i = threadIdx.x; i < unit_rows * n; i += 32 * kImmaWarps) {
                    const int tok = i / unit_rows, row = i % unit_rows;
                    const int o = tile * unit_rows + row;
                    if (o >= a.out) continue;
                    float v = get(tok, row);
                    const int r = first + 8 * sub + tok;
                    if (MODE == kDown) {
                        a.part[(size_t)__ldcg(a.order + r) * a.out + o] = v;
                    } else {
                        if (a.bias) v += a.bias[o];
                        v = activate(v, a.act);
                        if (a.row_scale) v *= a.row_scale[r];
                        const size_t at = (size_t)r * a.out + o;
                        a.y[at] = a.residual ? a.residual[at] + v : v;
                    }
                }
            }
        };

        const bool whole = r0 == 0 && r1 == per_unit;
        const int slot_rows = 32 * a.groups;
        const size_t split_size = (size_t)a.split_tokens * slot_rows;
        int a0 = 0, a1 = 0;
        if (!whole) {
            a0 = deal.owner((long long)u * per_unit);
            a1 = deal.owner((long long)u * per_unit + per_unit - 1);
        }
        // a CTA's tail slot holds the unit that starts in its range, its head slot the one that started before
        float* mine = a.split + ((size_t)2 * blockIdx.x + ((int)blockIdx.x == a0 ? 1 : 0)) * split_size;
#pragma unroll 1
        for (int sub = 0; sub < Acc::kSubs; ++sub) {
            if (sub * 8 >= count) break;
            const int n = count - 8 * sub < 8 ? count - 8 * sub : 8;
            float* rb = red + buf * kRedFloats;
            buf ^= 1;
            acc.store(sub, lane, [&](int tok, int j, int q, float v) {
                const int row = MODE == kPair ? 16 * q + 8 * j + g : 16 * j + 8 * q + g;
                rb[(warp * 8 + tok) * 32 + row] = v;
            });
            compute_sync();
            auto sum_parts = [&](int tok, int row) {
                float v = 0.0f;
                for (int k = 0; k < kws; ++k) v += rb[((k * a.groups + (row >> 5)) * 8 + tok) * 32 + (row & 31)];
                return v;
            };
            if (whole) {
                epilogue(sub, n, sum_parts);
            } else {
                for (int i = threadIdx.x; i < slot_rows * n; i += 32 * kImmaWarps)
                    mine[(size_t)(8 * sub + i / slot_rows) * slot_rows + i % slot_rows] = sum_parts(i / slot_rows, i % slot_rows);
            }
        }
        bool complete = whole;
        if (!whole) {
            compute_sync();
            if (threadIdx.x == 0) {
                __threadfence();
                s_last = atomicAdd(a.split_done + a0, 1u) == (unsigned)(a1 - a0);
                __threadfence();
            }
            compute_sync();
            complete = s_last;
            compute_sync();  // s_last may be written again
            if (complete)
                for (int sub = 0; sub * 8 < count; ++sub)
                    epilogue(sub, count - 8 * sub < 8 ? count - 8 * sub : 8, [&](int tok, int row) {
                        const size_t at = (size_t)(8 * sub + tok) * slot_rows + row;
                        float v = __ldcg(a.split + ((size_t)2 * a0 + 1) * split_size + at);
                        for (int i = a0 + 1; i <= a1; ++i) v += __ldcg(a.split + (size_t)2 * i * split_size + at);
                        return v;
                    });
        }
        if (MODE == kDown && complete) {
            finished_tile = tile;
            ++finished;
        }
    };

    for (long long t = t0; t < t1;) {
        const int u = (int)(t / per_unit), r0 = (int)(t % per_unit);
        const int r1 = t1 - t < per_unit - r0 ? r0 + (int)(t1 - t) : per_unit;
        t += r1 - r0;
        const int seg = seg_of(u);
        int first, count, e = 0;
        if (MODE == kPlain) {
            first = seg * kSegTokens;
            count = a.rows - first < kSegTokens ? a.rows - first : kSegTokens;
        } else {
            e = __ldcg(&a.segs[seg].expert);
            first = __ldcg(&a.segs[seg].start);
            count = __ldcg(&a.segs[seg].count);
        }
        if (MODE == kDown && tile_of(u) != finished_tile) settle();
        if (count <= 2 && count <= a.few) {
            FewRows<F, 1> acc;
            run_unit(acc, a.few_x, first, count, u, e, r0, r1);
        } else if (count <= 4 && count <= a.few) {
            FewRows<F, 2> acc;
            run_unit(acc, a.few_x, first, count, u, e, r0, r1);
        } else if (count <= 8) {
            ManyRows<F, 1> acc;
            run_unit(acc, a.many_x, first, count, u, e, r0, r1);
        } else if (count <= 16) {
            ManyRows<F, 2> acc;
            run_unit(acc, a.many_x, first, count, u, e, r0, r1);
        } else {
            ManyRows<F, 4> acc;
            run_unit(acc, a.many_x, first, count, u, e, r0, r1);
        }
    }
    settle();
    if (MODE == kDown && nseg == 0 && a.done) {
        // no row names an expert
        const size_t n = (size_t)a.rows * a.out;
        for (size_t i = (size_t)blockIdx.x * 32 * kImmaWarps + threadIdx.x; i < n; i += (size_t)gridDim.x * 32 * kImmaWarps)
            a.y[i] = a.residual ? a.residual[i] : 0.0f;
    }
    __syncthreads();  // the producer has issued its last copy
    // after a wait that ran out, copies may still be in flight: each is waited for once more, bounded
    if (*(volatile int*)&s_dead)
        for (int i = taken; i < s_issued[warp]; ++i) mbar_wait(bars + 16 * (i % a.slots), (i / a.slots) & 1);
}

bool aligned_rows(int fmt, const void* w, int bpr) {
    return reinterpret_cast<uintptr_t>(w) % 16 == 0 && (long long)bpr * block_bytes(fmt) % 16 == 0 &&
           encode_fn() != nullptr;
}

// Ring depth: what the SM's shared memory leaves room for, 2..8.
template <int F, int MODE, bool ALN>
cudaError_t launch_one(ImmaArgs a, int grid, int smem_per_sm, cudaStream_t stream) {
    using S = Slot<F, ALN>;
    auto k = imma_kernel<F, MODE, ALN>;
    const int fixed = 2 * kRedFloats * 4 + 1024 + 256;  // the system's 1 KB per CTA, the static part
    a.slots = (smem_per_sm - fixed) / (kImmaWarps * (S::kBytes + 16));
    if (a.slots > 8) a.slots = 8;
    if (a.slots < 2) return cudaErrorInvalidConfiguration;
    const size_t smem = (size_t)kImmaWarps * a.slots * (S::kBytes + 16) + 2 * kRedFloats * 4;
    ImmaMaps maps{};
    if (ALN) {
        for (int i = 0; i < (MODE == kPair ? 2 : 1); ++i)
            if (!make_map_2d(&maps.m[i], CU_TENSOR_MAP_DATA_TYPE_UINT16, const_cast<uint8_t*>(a.w[i]),
                             (uint64_t)a.row_bytes / 2, (uint64_t)a.total_rows, (uint64_t)a.row_bytes, S::kPitch / 2,
                             MODE == kPair ? 16 : 32, CU_TENSOR_MAP_SWIZZLE_NONE))
                return cudaErrorInvalidValue;
    }
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(k, grid, kThreads<ALN>, smem, stream, maps, a);
}

template <int MODE>
cudaError_t launch_imma(int fmt, ImmaArgs a, int sm_count, int smem_per_sm, long long max_units, cudaStream_t stream) {
    const bool aln = aligned_rows(fmt, a.w[0], a.bpr) && (MODE != kPair || aligned_rows(fmt, a.w[1], a.bpr));
    a.row_bytes = (long long)a.bpr * block_bytes(fmt);
    const int steps = (a.bpr + kChunkBlocks - 1) / kChunkBlocks, kws = kImmaWarps / a.groups;
    const long long rounds = max_units * ((steps + kws - 1) / kws);
    int grid = sm_count < kMaxCtas ? sm_count : kMaxCtas;
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
