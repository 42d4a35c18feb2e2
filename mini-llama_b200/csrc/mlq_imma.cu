// mlq_imma.cu -- the experts' products and the linear with an epilogue
// (mathematics and operand layout: mlq_imma.cuh).
//
// A call is up to three launches, chained by programmatic dependent launch:
//   prep   sorts the (row, slot) pairs by expert into segments of at most 32
//          and slices x;
//   pair   h = silu(x Wg^T) * (x Wu^T) per segment, sliced in its epilogue;
//   down   h Wd^T per segment, weighed and summed per row by the CTA that
//          finishes a row tile last (fixed order), or by a fourth launch
//          when there are many rows;
// and two (prep, down in its plain form) for the linear with an epilogue.
//
// The streaming kernel.  One CTA per SM: a producer warp and 8 computing
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
#include "mlq_imma.cuh"
#include "mlq_tmap.h"

namespace mlq {
namespace {

enum Mode { kPlain = 0, kPair = 1, kDown = 2 };

struct ImmaMaps {
    CUtensorMap m[2];
};

// Sliced rows of x or h: [row][bprp][128 bytes], a scale and a sum per block.
struct Sliced {
    uint8_t* data;
    float* scale;
    float* sum;
};

struct ImmaArgs {
    const uint8_t* w[2];      // stacked matrices [n][out][bpr]; [1]: the up projections (kPair)
    long long row_bytes;      // bytes of a matrix row
    long long total_rows;     // rows of the whole stack
    int out;                  // rows of one matrix
    int bpr, bprp;            // blocks per row, and padded to whole steps
    int groups;               // 32-row groups of a unit (1, 2 or 4); kPair: 16 gate and 16 up rows each, 2 or 4
    int tiles;                // row tiles of one matrix
    int slots;                // ring depth of a warp
    int few;                  // segments of at most this many rows go by digits
    Sliced few_x, many_x;     // digits / halves (the same arrays for h: a segment has one form)
    // segments (kPair, kDown); kPlain: rows in order, one matrix
    const Segment* segs;
    const int* nseg;
    const int* order;         // expert-sorted position -> pair
    int top_k, rows;
    // kPair: sliced h by position
    int next_fmt, next_bprp;
    Sliced h;
    // kDown: one value per pair, then the weighed sum
    float* part;              // [pair][out]
    unsigned int* done;       // units finished per row tile, zero before the launch; null: a later launch sums
    const int32_t* ids;
    const float* weights;
    int n_experts;
    // units that several CTAs share
    float* split;             // [CTA][head, tail][row of x][row of the tile]
    unsigned int* split_done; // per CTA, zero before the launch
    int split_tokens;         // rows of x of a split slot
    // kPlain / kDown
    const float* bias;
    const float* row_scale;
    const float* residual;
    float* y;
    int act;
    int* err;
};

// The accumulators of up to 2 NT rows of x by digits: an instruction's 8
// columns are the 4 digits of 2 rows, so lane t holds digits 3 and 2 (t even) or
// 1 and 0 (t odd) of row t / 2, and the two are added once, at the end.
template <int F, int NT>
struct FewRows {
    static constexpr int kSubs = 1;
    uint32_t bo[NT], so[NT];
    float acc[NT][2][2], accm[F == kQ4_1 ? NT : 1][2][2];

    template <class TokenOf>
    __device__ __forceinline__ void init(const ImmaArgs& a, int count, int lane, TokenOf token) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            // columns without a row of x repeat the first one's; nothing reads them
            const int r = 2 * i + (g >> 2), rs = 2 * i + (t >> 1);
            bo[i] = (uint32_t)token(r < count ? r : 0) * (uint32_t)a.bprp * kSlicedBytes + (g & 3) * 32 + t * 8;
            so[i] = (uint32_t)token(rs < count ? rs : 0) * (uint32_t)a.bprp;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                acc[i][j][0] = acc[i][j][1] = 0.0f;
                if (F == kQ4_1) accm[i][j][0] = accm[i][j][1] = 0.0f;
            }
        }
    }

    template <bool ALN, class Rows, class Wait>
    __device__ __forceinline__ void step(const ImmaArgs& a, int kb, int valid, int lane, Wait wait, Rows rows) {
        const int t = lane & 3;
        uint2 b[NT][kChunkBlocks];
        float4 s[NT][2], m[F == kQ4_1 ? NT : 1][2];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const uint8_t* p = a.few_x.data + bo[i] + (size_t)kb * kSlicedBytes;
#pragma unroll
            for (int k = 0; k < kChunkBlocks; ++k) b[i][k] = *reinterpret_cast<const uint2*>(p + k * kSlicedBytes);
            const float4* sp = reinterpret_cast<const float4*>(a.few_x.scale + so[i] + kb);
            s[i][0] = sp[0], s[i][1] = sp[1];
            if (F == kQ4_1) {
                const float4* mp = reinterpret_cast<const float4*>(a.few_x.sum + so[i] + kb);
                m[i][0] = mp[0], m[i][1] = mp[1];
            }
        }
        wait();
#pragma unroll
        for (int p = 0; p < kChunkBlocks / 2; ++p) {
            if (!ALN && 2 * p >= valid) break;
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
                        int c[4];
                        imma_s8(c, op, b[i][2 * p + o]);
                        const float4 s4 = s[i][p >> 1];
                        const float sx = p & 1 ? (o ? s4.w : s4.z) : (o ? s4.y : s4.x);
                        acc[i][j][0] = fmaf(A[o].d[0] * sx, (float)(c[0] * 256 + c[1]), acc[i][j][0]);
                        acc[i][j][1] = fmaf(A[o].d[1] * sx, (float)(c[2] * 256 + c[3]), acc[i][j][1]);
                        if (F == kQ4_1) {
                            const float4 m4 = m[i][p >> 1];
                            const float mx = p & 1 ? (o ? m4.w : m4.z) : (o ? m4.y : m4.x);
                            accm[i][j][0] = fmaf(A[o].m[0], mx, accm[i][j][0]);
                            accm[i][j][1] = fmaf(A[o].m[1], mx, accm[i][j][1]);
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
    uint32_t bo[S], so[S][2];
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

    template <bool ALN, class Rows, class Wait>
    __device__ __forceinline__ void step(const ImmaArgs& a, int kb, int valid, int lane, Wait wait, Rows rows) {
        const int t = lane & 3;
        wait();
#pragma unroll
        for (int p = 0; p < kChunkBlocks / 2; ++p) {
            if (2 * p >= valid) break;
            RawA A[2][2];  // [strip][block]
#pragma unroll
            for (int j = 0; j < 2; ++j) load_pair<F, ALN>(rows(j, 0), rows(j, 1), p, t, A[j][0], A[j][1]);
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                if (2 * p + o >= valid) break;
                const int blk = kb + 2 * p + o;
                uint32_t op[2][8];
                half_operand<F>(A[0][o], op[0]);
                half_operand<F>(A[1][o], op[1]);
#pragma unroll
                for (int i = 0; i < S; ++i) {
                    const uint4* bp = reinterpret_cast<const uint4*>(a.many_x.data + bo[i] + (size_t)blk * kSlicedBytes);
                    const uint4 hi = bp[0], lo = bp[4];
                    const float s0 = a.many_x.scale[so[i][0] + blk], s1 = a.many_x.scale[so[i][1] + blk];
                    float m0 = 0.0f, m1 = 0.0f;
                    if (F == kQ4_1) m0 = a.many_x.sum[so[i][0] + blk], m1 = a.many_x.sum[so[i][1] + blk];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        hmma_f16(c, op[j], lo.x, lo.y);
                        hmma_f16(c, op[j] + 4, lo.z, lo.w);
                        hmma_f16(c, op[j], hi.x, hi.y);
                        hmma_f16(c, op[j] + 4, hi.z, hi.w);
                        const RawA& A1 = A[j][o];
                        acc[i][j][0][0] = fmaf(A1.d[0] * s0, c[0], acc[i][j][0][0]);
                        acc[i][j][0][1] = fmaf(A1.d[0] * s1, c[1], acc[i][j][0][1]);
                        acc[i][j][1][0] = fmaf(A1.d[1] * s0, c[2], acc[i][j][1][0]);
                        acc[i][j][1][1] = fmaf(A1.d[1] * s1, c[3], acc[i][j][1][1]);
                        if (F == kQ4_1) {
                            acc[i][j][0][0] = fmaf(A1.m[0], m0, acc[i][j][0][0]);
                            acc[i][j][0][1] = fmaf(A1.m[0], m1, acc[i][j][0][1]);
                            acc[i][j][1][0] = fmaf(A1.m[1], m0, acc[i][j][1][0]);
                            acc[i][j][1][1] = fmaf(A1.m[1], m1, acc[i][j][1][1]);
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

// y[r][o] = residual[r][o] + sum_j weights[r][j] part[r k + j][o], slots in
// order; a slot without an expert adds nothing.
__device__ __forceinline__ float combine(const ImmaArgs& a, int r, int o) {
    float v = 0.0f;
    for (int j = 0; j < a.top_k; ++j) {
        const int p = r * a.top_k + j;
        const int e = a.ids[p];
        if (e >= 0 && e < a.n_experts) v = fmaf(a.weights[p], __ldcg(a.part + (size_t)p * a.out + o), v);
    }
    const size_t at = (size_t)r * a.out + o;
    return a.residual ? a.residual[at] + v : v;
}

// The barrier of the computing warps.
__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kImmaWarps) : "memory"); }

constexpr int kThreads = 32 * (kImmaWarps + 1);
constexpr int kRedFloats = kImmaWarps * 8 * 32;  // [warp][row of x][row of the group]
constexpr int kMaxCtas = 192;                    // CTAs of a launch at most (split slots)

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
__global__ void __launch_bounds__(kThreads, 1) imma_kernel(const __grid_constant__ ImmaMaps maps, const ImmaArgs a) {
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
    for (int i = threadIdx.x; i < kImmaWarps * a.slots; i += kThreads) {
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
    // kPair: a segment's tiles follow one another (its rows of x stay near); kDown, kPlain: a tile's segments do
    auto tile_of = [&](int u) { return MODE == kPair ? u % a.tiles : u / nseg; };
    auto seg_of = [&](int u) { return MODE == kPair ? u / a.tiles : u % nseg; };
    const int unit_rows = (MODE == kPair ? 16 : 32) * a.groups;

    if (warp == kImmaWarps) {
        // ---- producer ----
        int issued = 0;  // of the ring of warp `lane` (aligned) or of every ring
        bool alive = true;
        int u = t0 < t1 ? (int)(t0 / per_unit) : 0, r = t0 < t1 ? (int)(t0 % per_unit) : 0;
        long long row0 = 0;
        bool fresh = true;
        if constexpr (ALN) {
            // lane w fills the ring of warp w
            const int w = lane, grp = w % a.groups, kw = w / a.groups;
            int slot = 0, phase = 1;
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
            // lane l copies row l of each warp's slot
            int count[kImmaWarps] = {};
            const uint8_t* base = MODE == kPair && lane >= 16 ? a.w[1] : a.w[0];
            const uint8_t* stack_end = base + a.total_rows * a.row_bytes;
            for (long long t = t0; t < t1 && alive; ++t) {
                if (fresh) {
                    const int e = MODE == kPlain ? 0 : __ldcg(&a.segs[seg_of(u)].expert);
                    row0 = (long long)e * a.out + (long long)tile_of(u) * unit_rows + (MODE == kPair ? lane & 15 : lane);
                    fresh = false;
                }
#pragma unroll
                for (int w = 0; w < kImmaWarps; ++w) {
                    const int c = r * kws + w / a.groups;
                    if (c >= steps || !alive) continue;
                    const int slot = count[w] % a.slots;
                    const uint32_t bar = bars0 + 16 * (w * a.slots + slot);
                    const bool ok = mbar_wait(bar + 8, ((count[w] / a.slots) & 1) ^ 1);
                    if (!__all_sync(0xffffffffu, ok)) {
                        if (lane == 0) report_error(a.err, 31), *(volatile int*)&s_dead = 1;
                        alive = false;
                        continue;
                    }
                    const long long row = row0 + (w % a.groups) * (MODE == kPair ? 16 : 32);
                    const uint32_t dst = slots0 + (w * a.slots + slot) * S::kBytes + lane * S::kPitch;
                    uint32_t bytes = 0;
                    const uint8_t* win = nullptr;
                    uint32_t into = dst;
                    if (row < a.total_rows) {
                        const uint8_t* src = base + row * a.row_bytes + (long long)c * chunk_bytes(F);
                        long long left = a.row_bytes - (long long)c * chunk_bytes(F);
                        if (left > chunk_bytes(F)) left = chunk_bytes(F);
                        const uintptr_t lo = reinterpret_cast<uintptr_t>(src) & ~(uintptr_t)15;
                        const uintptr_t hi = (reinterpret_cast<uintptr_t>(src) + left + 15) & ~(uintptr_t)15;
                        win = reinterpret_cast<const uint8_t*>(lo);
                        const uint8_t* wend = reinterpret_cast<const uint8_t*>(hi);
                        // windows that stick out of the stack: its own bytes there one by one, the rest not at all
                        if (win < base) {
                            const int skip = (int)(base - win);
                            for (int k = skip; k < 16 && base + (k - skip) < stack_end; ++k) sts_u8(dst + k, win[k]);
                            win += 16;
                            into += 16;
                        }
                        if (wend > stack_end && wend > win) {
                            wend -= 16;
                            for (int k = 0; wend + k < stack_end; ++k)
                                sts_u8(into + (uint32_t)(wend - win) + k, wend[k]);
                        }
                        bytes = wend > win ? (uint32_t)(wend - win) : 0;
                    }
                    if (bytes) {
                        mbar_arrive_expect_tx(bar, bytes);
                        bulk_g2s(into, win, bytes, bar);
                    } else {
                        mbar_arrive(bar);
                    }
                    ++count[w];
                }
                if (*(volatile int*)&s_dead) alive = false;
                if (++r == per_unit) r = 0, ++u, fresh = true;
            }
            if (lane == 0)
#pragma unroll
                for (int w = 0; w < kImmaWarps; ++w) s_issued[w] = count[w];
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
        for (int r = r0; r < r1; ++r) {
            const int c = r * kws + kw;
            if (c >= steps) break;
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
                a, c * kChunkBlocks, a.bpr - c * kChunkBlocks, lane,
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
                    return at + row * S::kPitch + ((shift[MODE == kPair ? q : 0] + (uint32_t)(in_matrix * (a.row_bytes & 15))) & 15);
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
                        slice_digits(h, a.h.data + at * kSlicedBytes, a.h.scale + at, a.h.sum + at, lane);
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

// y from the parts of every pair, for calls with many rows.
__global__ void combine_kernel(const ImmaArgs a) {
    launch_dependents();
    grid_dependency_wait();
    const size_t n = (size_t)a.rows * a.out;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x)
        a.y[i] = combine(a, (int)(i / a.out), (int)(i % a.out));
}

struct PrepArgs {
    const float* x;
    int rows, in, bpr, bprp, fmt;
    Sliced few, many;  // data null: that form is not needed
    unsigned int* split_done;
    // experts only (ids not null)
    const int32_t* ids;
    int pairs, n_experts;
    Segment* segs;
    int* nseg;
    int* order;
    unsigned int* done;
    int tiles;
    // padding blocks of the sliced h
    Sliced h;
    int h_bpr, h_bprp;
};

// Pairs by expert (CTA 0), x sliced (one warp per block).  Latency-bound:
// a decode call's x is a few KB.
__global__ void __launch_bounds__(256) prep_kernel(const PrepArgs a) {
    launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int first = blockIdx.x, ctas = gridDim.x;
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < 2 * kMaxCtas; i += 256) a.split_done[i] = 0;
    if (a.ids) {
        if (blockIdx.x == 0) {
            __shared__ int cnt[MLQ_MOE_MAX_EXPERTS];
            __shared__ int wsum[2][8];
            __shared__ unsigned char in_warp[8][MLQ_MOE_MAX_EXPERTS];
            for (int e = threadIdx.x; e < a.n_experts; e += 256) cnt[e] = 0;
            for (int i = threadIdx.x; i < a.tiles; i += 256) a.done[i] = 0;
            const int pad = a.h_bprp - a.h_bpr;
            for (int i = threadIdx.x; i < a.pairs * pad; i += 256) {
                const size_t at = (size_t)(i / pad) * a.h_bprp + a.h_bpr + i % pad;
                a.h.scale[at] = 0.0f;
                a.h.sum[at] = 0.0f;
            }
            __syncthreads();
            for (int p = threadIdx.x; p < a.pairs; p += 256) {
                const int e = a.ids[p];
                if (e >= 0 && e < a.n_experts) atomicAdd(&cnt[e], 1);
            }
            __syncthreads();
            // each thread: 4 consecutive experts; exclusive sums of pairs and of segments
            constexpr int kPer = MLQ_MOE_MAX_EXPERTS / 256;
            int n[kPer], np = 0, ns = 0;
            for (int i = 0; i < kPer; ++i) {
                const int e = threadIdx.x * kPer + i;
                n[i] = e < a.n_experts ? cnt[e] : 0;
                np += n[i];
                ns += (n[i] + kSegTokens - 1) / kSegTokens;
            }
            int ip = np, is = ns;
            for (int o = 1; o < 32; o <<= 1) {
                const int vp = __shfl_up_sync(0xffffffffu, ip, o), vs = __shfl_up_sync(0xffffffffu, is, o);
                if (lane >= o) ip += vp, is += vs;
            }
            if (lane == 31) wsum[0][warp] = ip, wsum[1][warp] = is;
            __syncthreads();
            int op = ip - np, os = is - ns;
            for (int w = 0; w < warp; ++w) op += wsum[0][w], os += wsum[1][w];
            for (int i = 0; i < kPer; ++i) {
                const int e = threadIdx.x * kPer + i;
                if (e < a.n_experts) cnt[e] = op;
                for (int k = 0; k < n[i]; k += kSegTokens)
                    a.segs[os++] = Segment{e, op + k, n[i] - k < kSegTokens ? n[i] - k : kSegTokens, 0};
                op += n[i];
            }
            if (threadIdx.x == 255) *a.nseg = os;
            __syncthreads();
            // pairs of an expert in their order (which segment a pair joins, and so how its sums round, must not
            // change from run to run): 256 at a time, ranked within the warp, then over the warps before it
            for (int e = threadIdx.x; e < 8 * a.n_experts; e += 256) in_warp[e / a.n_experts][e % a.n_experts] = 0;
            __syncthreads();
            for (int p0 = 0; p0 < a.pairs; p0 += 256) {
                const int p = p0 + threadIdx.x;
                int e = p < a.pairs ? a.ids[p] : -1;
                if (e >= a.n_experts) e = -1;
                const unsigned same = __match_any_sync(0xffffffffu, e);
                const int rank = __popc(same & ((1u << lane) - 1));
                if (e >= 0 && rank == 0) in_warp[warp][e] = (unsigned char)__popc(same);
                __syncthreads();
                if (e >= 0) {
                    int at = cnt[e] + rank;
                    for (int w = 0; w < warp; ++w) at += in_warp[w][e];
                    a.order[at] = p;
                }
                __syncthreads();
                if (e >= 0 && rank == 0) {
                    atomicAdd(&cnt[e], __popc(same));
                    in_warp[warp][e] = 0;
                }
                __syncthreads();
            }
            return;
        }
        first -= 1;
        ctas -= 1;
    }
    const long long n = (long long)a.rows * a.bprp;
    for (long long i = (long long)first * 8 + warp; i < n; i += (long long)ctas * 8) {
        const int r = (int)(i / a.bprp), b = (int)(i % a.bprp);
        const float* x = a.x + (long long)r * a.in;
        if (a.few.data) {
            const int at = b * kQK + imma_element(a.fmt, b & 1, lane);
            slice_digits(at < a.in ? x[at] : 0.0f, a.few.data + i * kSlicedBytes, a.few.scale + i, a.few.sum + i, lane);
        }
        if (a.many.data) {
            const int at = b * kQK + half_element(a.fmt, b & 1, lane);
            slice_halves(at < a.in ? x[at] : 0.0f, a.many.data + i * kSlicedBytes, a.many.scale + i, a.many.sum + i, lane);
        }
    }
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

bool aligned_rows(int fmt, const void* w, int bpr) {
    return reinterpret_cast<uintptr_t>(w) % 16 == 0 && (long long)bpr * block_bytes(fmt) % 16 == 0 &&
           encode_fn() != nullptr;
}

template <typename... Params, typename... Args>
cudaError_t launch_pdl(void (*kernel)(Params...), int grid, int block, size_t smem, cudaStream_t stream,
                       Args&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
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
    return launch_pdl(k, grid, kThreads, smem, stream, maps, a);
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

// 32-row groups of a unit: no more K parts than there are K steps, and the
// tallest tile whose units still give every SM one (a taller unit has fewer
// K parts to add up and reads its rows of x less often).
int choose_groups(int out, int bpr, long long nseg, int sm_count, int least) {
    const int steps = (bpr + kChunkBlocks - 1) / kChunkBlocks;
    int g = 4;
    while (g > least && kImmaWarps / (g / 2) <= steps && (out + 32 * g - 1) / (32 * g) * nseg < sm_count) g /= 2;
    return g;
}

struct Carve {
    uint8_t* p;
    template <class T>
    T* take(size_t n) {
        T* r = reinterpret_cast<T*>(p);
        p += align256(n * sizeof(T));
        return r;
    }
    Sliced take_sliced(size_t rows, int bprp) {
        Sliced s;
        s.data = take<uint8_t>(rows * bprp * kSlicedBytes);
        s.scale = take<float>(rows * bprp);
        s.sum = take<float>(rows * bprp);
        return s;
    }
};

size_t sliced_bytes(size_t rows, int bprp) {
    return align256(rows * bprp * kSlicedBytes) + 2 * align256(rows * bprp * sizeof(float));
}

constexpr int kMaxPairs = 8192;           // pairs of one pass at most
constexpr size_t kMaxSliced = 1u << 30;   // sliced bytes of one pass at most (offsets are 32 bits)
constexpr size_t kMaxParts = 1u << 30;    // bytes of the pairs' outputs of one pass at most
constexpr int kMaxPassRows = 16384;       // rows of one pass of a linear at most
constexpr int kCombineRows = 32;          // more rows: the sum over slots is a launch of its own

int split_tokens(int rows) { return rows < kSegTokens ? rows : kSegTokens; }

// Two slots per CTA of at most 128 rows, and the counters of two launches.
size_t split_bytes(int rows) {
    return align256((size_t)2 * kMaxCtas * split_tokens(rows) * 128 * sizeof(float)) +
           align256(2 * kMaxCtas * sizeof(unsigned int));
}

// Rows of x of one pass.
int experts_pass_rows(const MoeShape& s, int rows, int top_k) {
    long long n = kMaxPairs / top_k;
    const long long per = (long long)top_k * padded_blocks((s.hidden + kQK - 1) / kQK) * kSlicedBytes;
    const long long perx = (long long)padded_blocks((s.in + kQK - 1) / kQK) * kSlicedBytes;
    const long long cap = (long long)kMaxSliced / (per > perx ? per : perx);
    const long long capp = (long long)kMaxParts / ((long long)top_k * s.out * (long long)sizeof(float));
    if (n > cap) n = cap;
    if (n > capp) n = capp;
    if (n < 1) n = 1;
    return rows < n ? rows : (int)n;
}

int linear_pass_rows(int in, int rows) {
    long long n = (long long)kMaxSliced / ((long long)padded_blocks((in + kQK - 1) / kQK) * kSlicedBytes);
    if (n > kMaxPassRows) n = kMaxPassRows;
    return rows < n ? rows : (int)n;
}

int max_segments(int pairs, int n_experts) {
    const int full = pairs / kSegTokens + (pairs < n_experts ? pairs : n_experts);
    return full < pairs ? full : pairs;
}

int prep_ctas(long long blocks, int sm_count) {
    const long long n = (blocks + 7) / 8;
    return (int)(n < 8LL * sm_count ? n : 8LL * sm_count);
}

}  // namespace

size_t epilogue_workspace_bytes(int in, int rows) {
    const int n = linear_pass_rows(in, rows);
    return sliced_bytes(n, padded_blocks((in + kQK - 1) / kQK)) + split_bytes(n);
}

cudaError_t launch_linear_epilogue(int fmt, const uint8_t* w, int out, int in, const float* x, int rows,
                                   const mlq_epilogue& ep, float* y, void* ws, int sm_count, int smem_per_sm, int* err,
                                   cudaStream_t stream) {
    const int bpr = (in + kQK - 1) / kQK, bprp = padded_blocks(bpr);
    const int pass = linear_pass_rows(in, rows);
    for (int r0 = 0; r0 < rows;) {
        const int n = rows - r0 < pass ? rows - r0 : pass;
        Carve c{static_cast<uint8_t*>(ws)};
        PrepArgs p{};
        p.x = x + (long long)r0 * in;
        p.rows = n, p.in = in, p.bpr = bpr, p.bprp = bprp, p.fmt = fmt;
        (n <= kFewRows ? p.few : p.many) = c.take_sliced(n, bprp);
        float* split = c.take<float>((size_t)2 * kMaxCtas * split_tokens(n) * 128);
        p.split_done = c.take<unsigned int>(2 * kMaxCtas);
        cudaError_t e = launch_pdl(prep_kernel, prep_ctas((long long)n * bprp, sm_count), 256, 0, stream, p);
        if (e != cudaSuccess) return e;
        ImmaArgs a{};
        a.w[0] = w;
        a.total_rows = out, a.out = out, a.bpr = bpr, a.bprp = bprp;
        const int nseg = (n + kSegTokens - 1) / kSegTokens;
        a.groups = choose_groups(out, bpr, nseg, sm_count, 1);
        a.tiles = (out + 32 * a.groups - 1) / (32 * a.groups);
        a.few = n <= kFewRows ? kFewRows : 0;
        a.few_x = p.few, a.many_x = p.many;
        a.rows = n;
        a.split = split, a.split_done = p.split_done, a.split_tokens = split_tokens(n);
        a.bias = ep.bias;
        a.row_scale = ep.row_scale ? ep.row_scale + r0 : nullptr;
        a.residual = ep.residual ? ep.residual + (long long)r0 * out : nullptr;
        a.act = ep.activation;
        a.y = y + (long long)r0 * out;
        a.err = err;
        e = launch_imma<kPlain>(fmt, a, sm_count, smem_per_sm, (long long)nseg * a.tiles, stream);
        if (e != cudaSuccess) return e;
        r0 += n;
    }
    return cudaSuccess;
}

size_t experts_workspace_bytes(const MoeShape& s, int rows, int top_k) {
    const int n = experts_pass_rows(s, rows, top_k), pairs = n * top_k;
    const int bprp = padded_blocks((s.in + kQK - 1) / kQK), hp = padded_blocks((s.hidden + kQK - 1) / kQK);
    return 256 + align256((size_t)max_segments(pairs, s.n_experts) * sizeof(Segment)) +
           align256((size_t)pairs * sizeof(int)) + align256((size_t)((s.out + 31) / 32) * sizeof(unsigned int)) +
           (pairs > kFewRows ? 2 : 1) * sliced_bytes(n, bprp) + sliced_bytes(pairs, hp) +
           align256((size_t)pairs * s.out * sizeof(float)) + split_bytes(pairs);
}

cudaError_t launch_experts(const MoeShape& s, const uint8_t* gate, const uint8_t* up, const uint8_t* down,
                           const float* x, int rows, int top_k, const int32_t* ids, const float* weights,
                           const float* residual, float* y, void* ws, int sm_count, int smem_per_sm, int* err,
                           cudaStream_t stream) {
    const int pass = experts_pass_rows(s, rows, top_k);
    const int bpr = (s.in + kQK - 1) / kQK, bprp = padded_blocks(bpr);
    const int hb = (s.hidden + kQK - 1) / kQK, hp = padded_blocks(hb);
    for (int r0 = 0; r0 < rows; r0 += pass) {
        const int n = rows - r0 < pass ? rows - r0 : pass, pairs = n * top_k;
        const int nseg_max = max_segments(pairs, s.n_experts);
        const int nseg_likely = pairs < s.n_experts ? pairs : nseg_max;
        const int groups = choose_groups(s.out, hb, nseg_likely, sm_count, 1);
        const int tiles = (s.out + 32 * groups - 1) / (32 * groups);
        Carve c{static_cast<uint8_t*>(ws)};
        PrepArgs p{};
        p.nseg = c.take<int>(1);
        p.segs = c.take<Segment>(nseg_max);
        p.order = c.take<int>(pairs);
        p.done = c.take<unsigned int>((s.out + 31) / 32);
        p.tiles = tiles;
        p.x = x + (long long)r0 * s.in;
        p.rows = n, p.in = s.in, p.bpr = bpr, p.bprp = bprp, p.fmt = s.fmt;
        p.few = c.take_sliced(n, bprp);
        if (pairs > kFewRows) p.many = c.take_sliced(n, bprp);  // a row may name an expert more than once
        p.ids = ids + (long long)r0 * top_k;
        p.pairs = pairs, p.n_experts = s.n_experts;
        p.h = c.take_sliced(pairs, hp);
        p.h_bpr = hb, p.h_bprp = hp;
        float* part = c.take<float>((size_t)pairs * s.out);
        float* split = c.take<float>((size_t)2 * kMaxCtas * split_tokens(pairs) * 128);
        p.split_done = c.take<unsigned int>(2 * kMaxCtas);
        cudaError_t e = launch_pdl(prep_kernel, 1 + prep_ctas((long long)n * bprp, sm_count), 256, 0, stream, p);
        if (e != cudaSuccess) return e;

        ImmaArgs a{};
        a.w[0] = gate, a.w[1] = up;
        a.total_rows = (long long)s.n_experts * s.hidden;
        a.out = s.hidden, a.bpr = bpr, a.bprp = bprp;
        a.groups = choose_groups(2 * s.hidden, bpr, nseg_likely, sm_count, 2);
        a.tiles = (s.hidden + 16 * a.groups - 1) / (16 * a.groups);
        a.few = kFewRows;
        a.few_x = p.few, a.many_x = p.many;
        a.segs = p.segs, a.nseg = p.nseg, a.order = p.order;
        a.top_k = top_k, a.rows = n;
        a.next_fmt = s.fmt_down, a.next_bprp = hp;
        a.h = p.h;
        a.split = split, a.split_done = p.split_done, a.split_tokens = split_tokens(pairs);
        a.err = err;
        e = launch_imma<kPair>(s.fmt, a, sm_count, smem_per_sm, (long long)nseg_max * a.tiles, stream);
        if (e != cudaSuccess) return e;

        ImmaArgs d{};
        d.w[0] = down;
        d.total_rows = (long long)s.n_experts * s.out;
        d.out = s.out, d.bpr = hb, d.bprp = hp;
        d.groups = groups, d.tiles = tiles;
        d.few = kFewRows;
        d.few_x = p.h, d.many_x = p.h;
        d.segs = p.segs, d.nseg = p.nseg, d.order = p.order;
        d.top_k = top_k, d.rows = n;
        d.part = part;
        d.done = n <= kCombineRows ? p.done : nullptr;
        d.split = split, d.split_done = p.split_done + kMaxCtas, d.split_tokens = split_tokens(pairs);
        d.ids = p.ids;
        d.weights = weights + (long long)r0 * top_k;
        d.n_experts = s.n_experts;
        d.residual = residual ? residual + (long long)r0 * s.out : nullptr;
        d.y = y + (long long)r0 * s.out;
        d.err = err;
        e = launch_imma<kDown>(s.fmt_down, d, sm_count, smem_per_sm, (long long)nseg_max * tiles, stream);
        if (e != cudaSuccess) return e;
        if (!d.done) {
            const long long vals = (long long)n * s.out;
            e = launch_pdl(combine_kernel, (int)((vals + 255) / 256 < 16 * sm_count ? (vals + 255) / 256 : 16 * sm_count),
                           256, 0, stream, d);
            if (e != cudaSuccess) return e;
        }
    }
    return cudaSuccess;
}

}  // namespace mlq
