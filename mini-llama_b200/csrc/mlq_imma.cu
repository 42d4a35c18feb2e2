// mlq_imma.cu -- the experts' products and the linear with an epilogue
// (mathematics and operand layout: mlq_imma.cuh).
//
// A call is up to three launches, chained by programmatic dependent launch:
//   prep   sorts the (row, slot) pairs by expert into segments of at most 32
//          and slices x into digits;
//   pair   h = silu(x Wg^T) * (x Wu^T) per segment, sliced in its epilogue;
//   down   h Wd^T per segment, weighed and summed per row by the CTA that
//          finishes a row tile last (fixed order), or by a fourth launch
//          when there are many rows;
// and two (prep, down in its plain form) for the linear with an epilogue.
//
// The streaming kernel.  A unit is a row tile of one matrix against one
// segment.  Its 8 warps split the tile in 16-row strips and the K axis in
// interleaved steps of 8 blocks; every warp fetches its own 16 x 8 blocks by
// TMA into a ring of its own, so the weight stream never waits for another
// warp; units follow one another in a static order and the ring runs ahead
// across them.  The K parts of a unit meet in shared memory (fixed order), one
// barrier per unit.  Two CTAs per SM: one computes while the other drains.
#include "mlq_imma.cuh"
#include "mlq_tmap.h"

namespace mlq {
namespace {

enum Mode { kPlain = 0, kPair = 1, kDown = 2 };

struct ImmaMaps {
    CUtensorMap m[2];
};

struct ImmaArgs {
    const uint8_t* w[2];      // stacked matrices [n][out][bpr]; [1]: the up projections (kPair)
    long long row_bytes;      // bytes of a matrix row
    long long total_rows;     // rows of the whole stack
    int out;                  // rows of one matrix
    int bpr, bprp;            // blocks per row, and padded to whole steps
    int strips;               // 16-row strips of a unit (1, 2, 4 or 8); kPair: 4 (32 gate and 32 up rows)
    int tiles;                // row tiles of one matrix
    int slots;                // ring depth of a warp
    const uint8_t* dig;       // sliced rows of x / h: digits [row][bprp][96]
    const float* scale;       // [row][bprp]
    const float* sum;         // [row][bprp]
    // segments (kPair, kDown); kPlain: rows in order, one matrix
    const Segment* segs;
    const int* nseg;
    const int* order;         // expert-sorted position -> pair
    int top_k, rows;
    // kPair: sliced h by position
    int next_fmt, next_bprp;
    uint8_t* hdig;
    float* hscale;
    float* hsum;
    // kDown: one value per pair, then the weighed sum
    float* part;              // [pair][out]
    unsigned int* done;       // per row tile, zero before the launch; null: a later launch sums
    const int32_t* ids;
    const float* weights;
    int n_experts;
    // kPlain / kDown
    const float* bias;
    const float* row_scale;
    const float* residual;
    float* y;
    int act;
    int* err;
};

// The accumulators of up to 2 NT rows of x: a matrix instruction's 8 columns
// are the digits (hi, mid, lo, none) of 2 rows, so lane t holds (hi, mid)
// (t even) or lo (t odd) of row t / 2 and the two are added once, at the end.
template <int F, int NT>
struct FewRows {
    static constexpr int kSubs = 1;
    uint32_t bo[NT], so[NT];
    bool on[NT];
    float acc[NT][2], accm[NT][2];

    template <class TokenOf>
    __device__ __forceinline__ void init(const ImmaArgs& a, int count, int lane, TokenOf token) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int r = 2 * i + (g >> 2), s = g & 3;
            on[i] = s < 3 && r < count;
            bo[i] = (uint32_t)token(r < count ? r : 0) * (uint32_t)a.bprp * kDigitBytes + (s < 3 ? s : 0) * 32 + t * 8;
            const int rs = 2 * i + (t >> 1);
            so[i] = (uint32_t)token(rs < count ? rs : 0) * (uint32_t)a.bprp;
            acc[i][0] = acc[i][1] = accm[i][0] = accm[i][1] = 0.0f;
        }
    }

    template <bool ALN, class Wait>
    __device__ __forceinline__ void step(const ImmaArgs& a, int kb, uint32_t r0, uint32_t r1, int lane, Wait wait) {
        const int t = lane & 3;
        uint2 b[NT][kChunkBlocks];
        float s[NT][kChunkBlocks], m[NT][F == kQ4_1 ? kChunkBlocks : 1];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const uint8_t* p = a.dig + bo[i] + (size_t)kb * kDigitBytes;
#pragma unroll
            for (int k = 0; k < kChunkBlocks; ++k)
                b[i][k] = on[i] ? *reinterpret_cast<const uint2*>(p + k * kDigitBytes) : make_uint2(0, 0);
            const float4* sp = reinterpret_cast<const float4*>(a.scale + so[i] + kb);
            const float4 s0 = sp[0], s1 = sp[1];
            s[i][0] = s0.x, s[i][1] = s0.y, s[i][2] = s0.z, s[i][3] = s0.w;
            s[i][4] = s1.x, s[i][5] = s1.y, s[i][6] = s1.z, s[i][7] = s1.w;
            if (F == kQ4_1) {
                const float4* mp = reinterpret_cast<const float4*>(a.sum + so[i] + kb);
                const float4 m0 = mp[0], m1 = mp[1];
                m[i][0] = m0.x, m[i][1] = m0.y, m[i][2] = m0.z, m[i][3] = m0.w;
                m[i][4] = m1.x, m[i][5] = m1.y, m[i][6] = m1.z, m[i][7] = m1.w;
            }
        }
        wait();
#pragma unroll
        for (int p = 0; p < kChunkBlocks / 2; ++p) {
            BlockA A[2];
            load_pair<F, ALN>(r0, r1, p, t, A[0], A[1]);
#pragma unroll
            for (int o = 0; o < 2; ++o)
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    int c[4];
                    imma_s8(c, A[o].a, b[i][2 * p + o]);
                    const float sx = s[i][2 * p + o];
                    acc[i][0] = fmaf(A[o].d[0] * sx, (float)(c[0] * 256 + c[1]), acc[i][0]);
                    acc[i][1] = fmaf(A[o].d[1] * sx, (float)(c[2] * 256 + c[3]), acc[i][1]);
                    if (F == kQ4_1) {
                        accm[i][0] = fmaf(A[o].m[0], m[i][2 * p + o], accm[i][0]);
                        accm[i][1] = fmaf(A[o].m[1], m[i][2 * p + o], accm[i][1]);
                    }
                }
        }
    }

    // red: [row of x 0..7][weight row 0..15] of this warp
    __device__ __forceinline__ void store(float* red, int, int lane) {
        const int g = lane >> 2, t = lane & 3;
        // an accumulator holds 256 times its first digit plus the second: (hi, mid) is 256 too small, (lo, 0) 256
        // too large; q4 codes count 16
        const float f = (t & 1 ? 0.00390625f : 256.0f) * (F == kQ8_0 ? 1.0f : 0.0625f);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float v = acc[i][q] * f;
                v += __shfl_xor_sync(0xffffffffu, v, 1);
                if (F == kQ4_1) v += accm[i][q];
                if (!(t & 1)) red[(2 * i + (t >> 1)) * 16 + g + 8 * q] = v;
            }
    }
};

// Up to 8 S rows of x: three instructions (hi, mid, lo) whose 8 columns are 8
// rows of x, so a lane has all digits of rows 2t and 2t + 1.
template <int F, int S>
struct ManyRows {
    static constexpr int kSubs = S;
    uint32_t bo[S], so[S][2];
    float acc[S][2][2];  // [.][weight row g / g + 8][row of x]

    template <class TokenOf>
    __device__ __forceinline__ void init(const ImmaArgs& a, int count, int lane, TokenOf token) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int r = 8 * i + g;
            bo[i] = (uint32_t)token(r < count ? r : 0) * (uint32_t)a.bprp * kDigitBytes + t * 8;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int rs = 8 * i + 2 * t + q;
                so[i][q] = (uint32_t)token(rs < count ? rs : 0) * (uint32_t)a.bprp;
                acc[i][q][0] = acc[i][q][1] = 0.0f;
            }
        }
    }

    template <bool ALN, class Wait>
    __device__ __forceinline__ void step(const ImmaArgs& a, int kb, uint32_t r0, uint32_t r1, int lane, Wait wait) {
        const int t = lane & 3;
        wait();
#pragma unroll
        for (int p = 0; p < kChunkBlocks / 2; ++p) {
            BlockA A[2];
            load_pair<F, ALN>(r0, r1, p, t, A[0], A[1]);
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const uint8_t* bp = a.dig + bo[i] + (size_t)(kb + 2 * p) * kDigitBytes;
                const float2 s0 = *reinterpret_cast<const float2*>(a.scale + so[i][0] + kb + 2 * p);
                const float2 s1 = *reinterpret_cast<const float2*>(a.scale + so[i][1] + kb + 2 * p);
#pragma unroll
                for (int o = 0; o < 2; ++o) {
                    int hi[4], mid[4], lo[4];
                    imma_s8(hi, A[o].a, *reinterpret_cast<const uint2*>(bp + o * kDigitBytes));
                    imma_s8(mid, A[o].a, *reinterpret_cast<const uint2*>(bp + o * kDigitBytes + 32));
                    imma_s8(lo, A[o].a, *reinterpret_cast<const uint2*>(bp + o * kDigitBytes + 64));
                    const float sx[2] = {o ? s0.y : s0.x, o ? s1.y : s1.x};
#pragma unroll
                    for (int q = 0; q < 2; ++q)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const float v = fmaf((float)(hi[2 * q + x] * 256 + mid[2 * q + x]), 256.0f,
                                                 (float)lo[2 * q + x]);
                            acc[i][q][x] = fmaf(A[o].d[q] * sx[x], v, acc[i][q][x]);
                        }
                    if (F == kQ4_1) {
                        // the block's offset term, in the accumulator's unit (codes count 16)
                        const float2 m0 = *reinterpret_cast<const float2*>(a.sum + so[i][0] + kb + 2 * p);
                        const float2 m1 = *reinterpret_cast<const float2*>(a.sum + so[i][1] + kb + 2 * p);
                        const float mx[2] = {16.0f * (o ? m0.y : m0.x), 16.0f * (o ? m1.y : m1.x)};
#pragma unroll
                        for (int q = 0; q < 2; ++q)
#pragma unroll
                            for (int x = 0; x < 2; ++x) acc[i][q][x] = fmaf(A[o].m[q], mx[x], acc[i][q][x]);
                    }
                }
            }
        }
    }

    __device__ __forceinline__ void store(float* red, int sub, int lane) {
        const int g = lane >> 2, t = lane & 3;
        const float f = F == kQ8_0 ? 1.0f : 0.0625f;
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (i == sub) {
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int x = 0; x < 2; ++x) red[(2 * t + x) * 16 + g + 8 * q] = acc[i][q][x] * f;
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

constexpr int kRedFloats = kImmaWarps * 8 * 16;

template <int F, int MODE, bool ALN>
__global__ void __launch_bounds__(32 * kImmaWarps, 2)
    imma_kernel(const __grid_constant__ ImmaMaps maps, const ImmaArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    using S = Slot<F, ALN>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int strip = warp % a.strips, kw = warp / a.strips, kws = kImmaWarps / a.strips;
    const int steps = (a.bpr + kChunkBlocks - 1) / kChunkBlocks;
    const uint32_t slots = smem_u32(smem) + (uint32_t)warp * a.slots * S::kBytes;
    float* red = reinterpret_cast<float*>(smem + kImmaWarps * a.slots * S::kBytes);  // two buffers
    const uint32_t bars = smem_u32(red + 2 * kRedFloats) + warp * a.slots * 8;
    __shared__ int s_last;

    if (ALN && lane == 0) {
        for (int i = 0; i < a.slots; ++i) mbar_init(bars + 8 * i, 1);
        fence_mbar_init();
    }
    __syncwarp();

    // The segments come from prep.  kPair is prep's dependent, so it waits;
    // kDown started after every CTA of kPair had waited for prep, so prep has
    // completed: it reads the segments (past L1) and streams weights at once.
    if (MODE == kPair) {
        grid_dependency_wait();
        launch_dependents();
    }
    const int nseg = MODE == kPlain ? (a.rows + kSegTokens - 1) / kSegTokens : __ldcg(a.nseg);
    const int units = nseg * a.tiles;

    // what the ring fetches next: unit pu, K step pc
    int pu = blockIdx.x, pc = kw, p_slot = 0, in_flight = 0;
    long long p_row = 0;
    bool alive = true;  // false once a wait ran out: nothing more is fetched or waited for
    int lost = 0, lost_slot = 0, lost_phase = 0;
    auto unit_row = [&](int u) -> long long {
        const int seg = u % nseg, tile = u / nseg;
        const int e = MODE == kPlain ? 0 : __ldcg(&a.segs[seg].expert);
        return (long long)e * a.out + (long long)tile * (MODE == kPair ? 32 : 16 * a.strips) +
               strip * (MODE == kPair ? 8 : 16);
    };
    if (kw >= steps) pu = units;
    if (pu < units) p_row = unit_row(pu);
    auto fetch = [&]() {
        if (pu < units && alive) {
            const uint32_t dst = slots + p_slot * S::kBytes;
            if constexpr (ALN) {
                if (lane == 0) {
                    const uint32_t bar = bars + 8 * p_slot;
                    mbar_arrive_expect_tx(bar, S::kBytes);
#pragma unroll
                    for (int b = 0; b < S::kBoxes; ++b) {
                        const int c0 = (pc * chunk_bytes(F) + b * S::kBoxBytes) / 2;
                        const uint32_t d = dst + b * 16 * S::kBoxBytes;
                        tma_load_2d(d, &maps.m[0], c0, (int)p_row, bar);
                        if (MODE == kPair) tma_load_2d(d + 8 * S::kBoxBytes, &maps.m[1], c0, (int)p_row, bar);
                    }
                }
            } else {
                // two lanes per row, the 16-byte windows that hold its blocks
                const int r = lane >> 1;
                const uint8_t* base = MODE == kPair && r >= 8 ? a.w[1] : a.w[0];
                const long long row = p_row + (MODE == kPair ? (r & 7) : r);
                const long long off = row * a.row_bytes + (long long)pc * chunk_bytes(F);
                long long left = a.row_bytes - (long long)pc * chunk_bytes(F);
                if (left > chunk_bytes(F)) left = chunk_bytes(F);
                if (row >= a.total_rows) left = 0;
                const uint8_t* src = base + (left > 0 ? off : 0);
                const uint8_t* end = src + (left > 0 ? left : 0);
                const uint8_t* win = reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(src) & ~(uintptr_t)15);
                const uint32_t drow = dst + r * S::kPitch;
                for (int i = lane & 1; i < (chunk_bytes(F) + 15 + 15) / 16; i += 2) {
                    const uint8_t* q = win + 16 * i;
                    long long n = end - q;
                    n = n < 0 ? 0 : (n > 16 ? 16 : n);
                    if (q < base && n > 0) {
                        // the stack's first bytes, when it starts inside a window: nothing before it is read
                        for (int k = 0; k < 16; ++k)
                            sts_u8(drow + 16 * i + k, q + k >= base && k < n ? (uint32_t)q[k] : 0u);
                    } else {
                        cp_async_16(drow + 16 * i, n > 0 ? q : win + (win < base ? 16 : 0), (uint32_t)n);
                    }
                }
            }
            ++in_flight;
            if (++p_slot == a.slots) p_slot = 0;
            pc += kws;
            if (pc >= steps) {
                pc = kw;
                pu += gridDim.x;
                if (pu < units) p_row = unit_row(pu);
            }
        }
        if constexpr (!ALN) asm volatile("cp.async.commit_group;" ::: "memory");
    };

    if (MODE == kPlain) {
        launch_dependents();
    }
    for (int i = 0; i < a.slots; ++i) fetch();
    if (MODE != kPair) grid_dependency_wait();
    if (MODE == kDown) launch_dependents();

    int slot = 0, phase = 0, buf = 0;
    auto stream = [&](auto& acc, int seg_first, int count, int u) {
        // the rows of x of this segment, in the sliced arrays
        acc.init(a, count, lane, [&](int r) -> int {
            if (MODE == kPair) return __ldcg(a.order + seg_first + r) / a.top_k;
            return seg_first + r;
        });
        const int g = lane >> 2;
        const long long off0 = ALN ? 0 : unit_row(u) * a.row_bytes;  // for the byte shift of each row in its window
        for (int c = kw; c < steps; c += kws) {
            const uint32_t at = slots + slot * S::kBytes;
            uint32_t r0, r1;
            (void)off0;
            if constexpr (ALN) {
                r0 = at + g * S::kBoxBytes;
                r1 = r0 + 8 * S::kBoxBytes;
            } else {
                const long long o = off0 + (long long)c * chunk_bytes(F);
                const uintptr_t w0 = reinterpret_cast<uintptr_t>(a.w[0]) + o;
                const uintptr_t w1 = MODE == kPair ? reinterpret_cast<uintptr_t>(a.w[1]) + o : w0 + 8 * a.row_bytes;
                r0 = at + g * S::kPitch + (uint32_t)((w0 + g * a.row_bytes) & 15);
                r1 = at + (g + 8) * S::kPitch + (uint32_t)((w1 + g * a.row_bytes) & 15);
            }
            acc.template step<ALN>(a, c * kChunkBlocks, r0, r1, lane, [&]() {
                if constexpr (ALN) {
                    if (alive && !__all_sync(0xffffffffu, mbar_wait(bars + 8 * slot, phase))) {
                        alive = false;
                        lost = in_flight, lost_slot = slot, lost_phase = phase;
                        if (lane == 0) report_error(a.err, 30);
                    }
                } else {
                    // fetch() commits one group per step, so at most slots - 1 newer groups are in flight
                    switch (a.slots) {
                        case 2: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
                        case 3: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
                        default: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
                    }
                    __syncwarp();
                }
            });
            __syncwarp();
            --in_flight;
            if (++slot == a.slots) {
                slot = 0;
                phase ^= 1;
            }
            fetch();
        }

        using Acc = typename std::remove_reference<decltype(acc)>::type;
        const int tile = u / nseg;
#pragma unroll 1
        for (int sub = 0; sub < Acc::kSubs; ++sub) {
            if (sub * 8 >= count) break;
            float* rb = red + buf * kRedFloats;
            buf ^= 1;
            acc.store(rb + warp * 128, sub, lane);
            __syncthreads();
            const int n = count - 8 * sub < 8 ? count - 8 * sub : 8;
            if (MODE == kPair) {
                // warp w: row w of x, a block of 32 hidden values, lane l at the K position l of the next product
                if (warp < n) {
                    const int el = imma_element(a.next_fmt, tile & 1, lane);
                    const float* p = rb + (el >> 3) * 128 + warp * 16 + (el & 7);
                    float gate = 0.0f, up = 0.0f;
                    for (int k = 0; k < kws; ++k) {
                        gate += p[k * a.strips * 128];
                        up += p[k * a.strips * 128 + 8];
                    }
                    const float h = tile * 32 + el < a.out ? silu_mul(gate, up) : 0.0f;
                    const size_t at = (size_t)(seg_first + 8 * sub + warp) * a.next_bprp + tile;
                    slice_block(h, a.hdig + at * kDigitBytes, a.hscale + at, a.hsum + at, lane);
                }
            } else {
                const int rows = 16 * a.strips;
                for (int i = threadIdx.x; i < rows * n; i += blockDim.x) {
                    const int tok = i / rows, row = i % rows;
                    const int o = tile * rows + row;
                    if (o >= a.out) continue;
                    float v = 0.0f;
                    for (int k = 0; k < kws; ++k)
                        v += rb[(k * a.strips + (row >> 4)) * 128 + tok * 16 + (row & 15)];
                    const int r = seg_first + 8 * sub + tok;
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
        }
        if (MODE == kDown && a.done) {
            // the CTA that finishes a row tile last sums it for every row of x
            __syncthreads();
            if (threadIdx.x == 0) {
                __threadfence();
                s_last = atomicAdd(a.done + tile, 1u) + 1 == (unsigned)nseg;
                __threadfence();
            }
            __syncthreads();
            if (s_last) {
                const int rows = 16 * a.strips;
                for (int i = threadIdx.x; i < rows * a.rows; i += blockDim.x) {
                    const int o = tile * rows + i % rows, r = i / rows;
                    if (o < a.out) a.y[(size_t)r * a.out + o] = combine(a, r, o);
                }
            }
        }
    };

    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        const int seg = u % nseg;
        int first, count;
        if (MODE == kPlain) {
            first = seg * kSegTokens;
            count = a.rows - first < kSegTokens ? a.rows - first : kSegTokens;
        } else {
            first = __ldcg(&a.segs[seg].start);
            count = __ldcg(&a.segs[seg].count);
        }
        if (count <= 2) {
            FewRows<F, 1> acc;
            stream(acc, first, count, u);
        } else if (count <= 4) {
            FewRows<F, 2> acc;
            stream(acc, first, count, u);
        } else if (count <= 8) {
            ManyRows<F, 1> acc;
            stream(acc, first, count, u);
        } else if (count <= 16) {
            ManyRows<F, 2> acc;
            stream(acc, first, count, u);
        } else {
            ManyRows<F, 4> acc;
            stream(acc, first, count, u);
        }
    }
    if (MODE == kDown && nseg == 0 && a.done) {
        // no row names an expert
        const size_t n = (size_t)a.rows * a.out;
        for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x)
            a.y[i] = a.residual ? a.residual[i] : 0.0f;
    }
    // after a wait that ran out, copies may still be in flight: each is waited for once more, bounded
    if constexpr (ALN) {
        for (; lost > 0; --lost) {
            mbar_wait(bars + 8 * lost_slot, lost_phase);
            if (++lost_slot == a.slots) {
                lost_slot = 0;
                lost_phase ^= 1;
            }
        }
    } else {
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
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
    uint8_t* dig;
    float* scale;
    float* sum;
    // experts only (ids not null)
    const int32_t* ids;
    int pairs, n_experts;
    Segment* segs;
    int* nseg;
    int* order;
    unsigned int* done;
    int tiles;
    // padding blocks of the sliced h
    float* hscale;
    float* hsum;
    int h_bpr, h_bprp;
};

// Pairs by expert (CTA 0), x in digits (one warp per block).  Latency-bound:
// a decode call's x is a few KB.
__global__ void __launch_bounds__(256) prep_kernel(const PrepArgs a) {
    launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int first = blockIdx.x, ctas = gridDim.x;
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
                a.hscale[at] = 0.0f;
                a.hsum[at] = 0.0f;
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
        const int at = b * kQK + imma_element(a.fmt, b & 1, lane);
        const float v = at < a.in ? a.x[(long long)r * a.in + at] : 0.0f;
        slice_block(v, a.dig + i * kDigitBytes, a.scale + i, a.sum + i, lane);
    }
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

bool aligned_rows(int fmt, const void* w, int bpr) {
    return reinterpret_cast<uintptr_t>(w) % 16 == 0 && (long long)bpr * block_bytes(fmt) % 16 == 0 &&
           encode_fn() != nullptr;
}

int slot_bytes(int fmt, bool aln) {
    if (aln) return fmt == kQ8_0 ? Slot<kQ8_0, true>::kBytes : (fmt == kQ4_0 ? Slot<kQ4_0, true>::kBytes
                                                                             : Slot<kQ4_1, true>::kBytes);
    return fmt == kQ8_0 ? Slot<kQ8_0, false>::kBytes : (fmt == kQ4_0 ? Slot<kQ4_0, false>::kBytes
                                                                     : Slot<kQ4_1, false>::kBytes);
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

template <int F, int MODE, bool ALN>
cudaError_t launch_one(ImmaArgs a, const ImmaMaps& maps, int grid, size_t smem, cudaStream_t stream) {
    auto k = imma_kernel<F, MODE, ALN>;
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(k, grid, 32 * kImmaWarps, smem, stream, maps, a);
}

// Ring depth: what two CTAs per SM leave room for, 2..8 (2..4 without tensor maps).
template <int MODE>
cudaError_t launch_imma(int fmt, ImmaArgs a, int sm_count, int smem_per_sm, int max_units, cudaStream_t stream) {
    const bool aln = aligned_rows(fmt, a.w[0], a.bpr) && (MODE != kPair || aligned_rows(fmt, a.w[1], a.bpr));
    a.row_bytes = (long long)a.bpr * block_bytes(fmt);
    const int sb = slot_bytes(fmt, aln);
    const int fixed = 2 * kRedFloats * 4 + 1024 + 256;  // the system's 1 KB per CTA, the static part
    a.slots = (smem_per_sm / 2 - fixed) / (kImmaWarps * (sb + 8));
    if (a.slots > (aln ? 8 : 4)) a.slots = aln ? 8 : 4;
    if (a.slots < 2) return cudaErrorInvalidConfiguration;
    const size_t smem = (size_t)kImmaWarps * a.slots * (sb + 8) + 2 * kRedFloats * 4;
    ImmaMaps maps{};
    if (aln) {
        const int box = fmt == kQ8_0 ? 272 : (fmt == kQ4_0 ? 144 : 80);
        for (int i = 0; i < (MODE == kPair ? 2 : 1); ++i)
            if (!make_map_2d(&maps.m[i], CU_TENSOR_MAP_DATA_TYPE_UINT16, const_cast<uint8_t*>(a.w[i]),
                             (uint64_t)a.row_bytes / 2, (uint64_t)a.total_rows, (uint64_t)a.row_bytes, box / 2,
                             MODE == kPair ? 8 : 16, CU_TENSOR_MAP_SWIZZLE_NONE))
                return cudaErrorInvalidValue;
    }
    int grid = 2 * sm_count;
    if (grid > max_units) grid = max_units;
    if (grid < 1) grid = 1;
    switch (fmt) {
        case kQ8_0:
            return aln ? launch_one<kQ8_0, MODE, true>(a, maps, grid, smem, stream)
                       : launch_one<kQ8_0, MODE, false>(a, maps, grid, smem, stream);
        case kQ4_0:
            return aln ? launch_one<kQ4_0, MODE, true>(a, maps, grid, smem, stream)
                       : launch_one<kQ4_0, MODE, false>(a, maps, grid, smem, stream);
        default:
            return aln ? launch_one<kQ4_1, MODE, true>(a, maps, grid, smem, stream)
                       : launch_one<kQ4_1, MODE, false>(a, maps, grid, smem, stream);
    }
}

// 16-row strips of a unit: no more K parts than there are K steps, then
// taller units while there are enough of them to spread over the SMs (a
// taller unit has fewer K parts to add up).
int choose_strips(int out, int bpr, int nseg, int sm_count) {
    const int steps = (bpr + kChunkBlocks - 1) / kChunkBlocks;
    int kws = kImmaWarps;
    while (kws > steps) kws >>= 1;
    int strips = kImmaWarps / kws;
    while (strips < 4 && (long long)((out + 32 * strips - 1) / (32 * strips)) * nseg >= 6LL * sm_count) strips *= 2;
    return strips;
}

struct Carve {
    uint8_t* p;
    template <class T>
    T* take(size_t n) {
        T* r = reinterpret_cast<T*>(p);
        p += align256(n * sizeof(T));
        return r;
    }
};

size_t sliced_bytes(size_t rows, int bprp) {
    return align256(rows * bprp * kDigitBytes) + 2 * align256(rows * bprp * sizeof(float));
}

constexpr int kMaxPairs = 8192;           // pairs of one pass at most
constexpr size_t kMaxSliced = 1u << 30;   // digit bytes of one pass at most (offsets are 32 bits)
constexpr size_t kMaxParts = 1u << 30;    // bytes of the pairs' outputs of one pass at most
constexpr int kMaxPassRows = 16384;       // rows of one pass of a linear at most
constexpr int kCombineRows = 32;          // more rows: the sum over slots is a launch of its own

// Rows of x of one pass.
int experts_pass_rows(const MoeShape& s, int rows, int top_k) {
    long long n = kMaxPairs / top_k;
    const long long per = (long long)top_k * padded_blocks((s.hidden + kQK - 1) / kQK) * kDigitBytes;
    const long long perx = (long long)padded_blocks((s.in + kQK - 1) / kQK) * kDigitBytes;
    const long long cap = (long long)kMaxSliced / (per > perx ? per : perx);
    const long long capp = (long long)kMaxParts / ((long long)top_k * s.out * (long long)sizeof(float));
    if (n > cap) n = cap;
    if (n > capp) n = capp;
    if (n < 1) n = 1;
    return rows < n ? rows : (int)n;
}

int linear_pass_rows(int in, int rows) {
    long long n = (long long)kMaxSliced / ((long long)padded_blocks((in + kQK - 1) / kQK) * kDigitBytes);
    if (n > kMaxPassRows) n = kMaxPassRows;
    return rows < n ? rows : (int)n;
}

int max_segments(int pairs, int n_experts) {
    const int full = pairs / kSegTokens + (pairs < n_experts ? pairs : n_experts);
    return full < pairs ? full : pairs;
}

int down_strips(const MoeShape& s, int rows, int top_k, int sm_count) {
    const int pairs = rows * top_k;
    return choose_strips(s.out, (s.hidden + kQK - 1) / kQK, pairs < s.n_experts ? pairs : s.n_experts, sm_count);
}

}  // namespace

size_t epilogue_workspace_bytes(int in, int rows) {
    const int bprp = padded_blocks((in + kQK - 1) / kQK);
    return sliced_bytes(linear_pass_rows(in, rows), bprp);
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
        p.dig = c.take<uint8_t>((size_t)n * bprp * kDigitBytes);
        p.scale = c.take<float>((size_t)n * bprp);
        p.sum = c.take<float>((size_t)n * bprp);
        const long long blocks = (long long)n * bprp;
        cudaError_t e = launch_pdl(prep_kernel, (int)((blocks + 7) / 8 < 8 * sm_count ? (blocks + 7) / 8 : 8 * sm_count),
                                   256, 0, stream, p);
        if (e != cudaSuccess) return e;
        ImmaArgs a{};
        a.w[0] = w;
        a.total_rows = out, a.out = out, a.bpr = bpr, a.bprp = bprp;
        const int nseg = (n + kSegTokens - 1) / kSegTokens;
        a.strips = choose_strips(out, bpr, nseg, sm_count);
        a.tiles = (out + 16 * a.strips - 1) / (16 * a.strips);
        a.dig = p.dig, a.scale = p.scale, a.sum = p.sum;
        a.rows = n;
        a.bias = ep.bias;
        a.row_scale = ep.row_scale ? ep.row_scale + r0 : nullptr;
        a.residual = ep.residual ? ep.residual + (long long)r0 * out : nullptr;
        a.act = ep.activation;
        a.y = y + (long long)r0 * out;
        a.err = err;
        const long long units = (long long)nseg * a.tiles;
        e = launch_imma<kPlain>(fmt, a, sm_count, smem_per_sm, units > INT_MAX ? INT_MAX : (int)units, stream);
        if (e != cudaSuccess) return e;
        r0 += n;
    }
    return cudaSuccess;
}

size_t experts_workspace_bytes(const MoeShape& s, int rows, int top_k) {
    const int n = experts_pass_rows(s, rows, top_k), pairs = n * top_k;
    const int bprp = padded_blocks((s.in + kQK - 1) / kQK), hp = padded_blocks((s.hidden + kQK - 1) / kQK);
    return 256 + align256((size_t)max_segments(pairs, s.n_experts) * sizeof(Segment)) +
           align256((size_t)pairs * sizeof(int)) + align256((size_t)((s.out + 15) / 16) * sizeof(unsigned int)) +
           sliced_bytes(n, bprp) + sliced_bytes(pairs, hp) + align256((size_t)pairs * s.out * sizeof(float));
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
        const int strips = down_strips(s, n, top_k, sm_count);
        const int tiles = (s.out + 16 * strips - 1) / (16 * strips);
        Carve c{static_cast<uint8_t*>(ws)};
        PrepArgs p{};
        p.nseg = c.take<int>(1);
        p.segs = c.take<Segment>(nseg_max);
        p.order = c.take<int>(pairs);
        p.done = c.take<unsigned int>((s.out + 15) / 16);
        p.tiles = tiles;
        p.x = x + (long long)r0 * s.in;
        p.rows = n, p.in = s.in, p.bpr = bpr, p.bprp = bprp, p.fmt = s.fmt;
        p.dig = c.take<uint8_t>((size_t)n * bprp * kDigitBytes);
        p.scale = c.take<float>((size_t)n * bprp);
        p.sum = c.take<float>((size_t)n * bprp);
        p.ids = ids + (long long)r0 * top_k;
        p.pairs = pairs, p.n_experts = s.n_experts;
        uint8_t* hdig = c.take<uint8_t>((size_t)pairs * hp * kDigitBytes);
        p.hscale = c.take<float>((size_t)pairs * hp);
        p.hsum = c.take<float>((size_t)pairs * hp);
        p.h_bpr = hb, p.h_bprp = hp;
        float* part = c.take<float>((size_t)pairs * s.out);
        const long long blocks = (long long)n * bprp;
        cudaError_t e =
            launch_pdl(prep_kernel, 1 + (int)((blocks + 7) / 8 < 8 * sm_count ? (blocks + 7) / 8 : 8 * sm_count), 256, 0,
                       stream, p);
        if (e != cudaSuccess) return e;

        ImmaArgs a{};
        a.w[0] = gate, a.w[1] = up;
        a.total_rows = (long long)s.n_experts * s.hidden;
        a.out = s.hidden, a.bpr = bpr, a.bprp = bprp;
        a.strips = 4;
        a.tiles = (s.hidden + 31) / 32;
        a.dig = p.dig, a.scale = p.scale, a.sum = p.sum;
        a.segs = p.segs, a.nseg = p.nseg, a.order = p.order;
        a.top_k = top_k, a.rows = n;
        a.next_fmt = s.fmt_down, a.next_bprp = hp;
        a.hdig = hdig, a.hscale = p.hscale, a.hsum = p.hsum;
        a.err = err;
        long long units = (long long)nseg_max * a.tiles;
        e = launch_imma<kPair>(s.fmt, a, sm_count, smem_per_sm, units > INT_MAX ? INT_MAX : (int)units, stream);
        if (e != cudaSuccess) return e;

        ImmaArgs d{};
        d.w[0] = down;
        d.total_rows = (long long)s.n_experts * s.out;
        d.out = s.out, d.bpr = hb, d.bprp = hp;
        d.strips = strips, d.tiles = tiles;
        d.dig = hdig, d.scale = p.hscale, d.sum = p.hsum;
        d.segs = p.segs, d.nseg = p.nseg, d.order = p.order;
        d.top_k = top_k, d.rows = n;
        d.part = part;
        d.done = n <= kCombineRows ? p.done : nullptr;
        d.ids = p.ids;
        d.weights = weights + (long long)r0 * top_k;
        d.n_experts = s.n_experts;
        d.residual = residual ? residual + (long long)r0 * s.out : nullptr;
        d.y = y + (long long)r0 * s.out;
        d.err = err;
        units = (long long)nseg_max * tiles;
        e = launch_imma<kDown>(s.fmt_down, d, sm_count, smem_per_sm, units > INT_MAX ? INT_MAX : (int)units, stream);
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
