// mlq_imma_many.cuh -- the streaming kernel for many rows of x per matrix
// (halves, fp16 matrix instructions; mathematics and operand layout:
// mlq_imma.cuh; the launches around it: mlq_imma.cu).
//
// One CTA per SM: 16 computing and 4 producer warps.  A unit is a tile of 256
// rows of one matrix (kPair: 128 gate and 128 up rows) against one segment of
// up to 32 rows of x; a round is 8 blocks of K.  A stage holds a round's weights
// (16 strips of 16 rows) and records of x, both fetched asynchronously, so that
// x is read from L2 once per 256 weight rows.  A computing warp takes 2 strips
// x 16 rows of x (one strip where the segment has at most 16): per block ~20
// instructions turn codes to fp16 per strip and 4 matrix instructions per
// strip and 8 rows of x use them, so the matrix unit is what bounds a full
// segment (4 x 2.2 cycles per 16 x 8 x 32 products: 255 TFLOP/s on 148 SMs).
// Rounds are dealt out evenly as in mlq_imma_few.cuh.
#pragma once

#include "mlq_imma_common.cuh"

namespace mlq {
namespace {

constexpr int kStrips = 16;                       // 16-row strips of a unit
constexpr int kUnitRows = 16 * kStrips;
constexpr int kComputeWarps = 16, kProducers = 4;
constexpr int kManyThreads = 32 * (kComputeWarps + kProducers);
constexpr int kComputeThreads = 32 * kComputeWarps;
constexpr int kSumFloats = 32 * (128 + 4);        // sums of one pass: [row of x][128 or 256 rows + 4]
constexpr int kManyJoin = 2;                      // rounds; one takes ~2.4 us at a full segment
// registers: as in mlq_imma_few.cuh
constexpr int kManyLaunchRegs = 96, kManyProducerRegs = 32, kManyComputeRegs = 112;
static_assert((kProducers * kManyProducerRegs + kComputeWarps * kManyComputeRegs) * 32 <= kManyThreads * kManyLaunchRegs,
              "the shares must not exceed the launch's registers, or setmaxnreg would wait for ever");

// J strips against 8 S rows of x.
template <int F, int J, int S>
struct ManyRows {
    float acc[J][S][2][2];  // [.][.][row g / g + 8][row of x 2t, 2t + 1]

    __device__ __forceinline__ void init() {
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < S; ++i) acc[j][i][0][0] = acc[j][i][0][1] = acc[j][i][1][0] = acc[j][i][1][1] = 0.0f;
    }

    // One round; x: the lane's halves, s: the scales of its rows 2t (see run).
    template <bool ALN>
    __device__ __forceinline__ void step(uint32_t x, uint32_t s, int valid, const RowBase (&rows)[J]) {
        static_for<kChunkBlocks / 2>([&](auto pc) {
            constexpr int p = decltype(pc)::value;
            if (2 * p >= valid) return;
            RawA A[J][2];
#pragma unroll
            for (int j = 0; j < J; ++j) load_pair<F, ALN, p>(rows[j], A[j][0], A[j][1]);
            static_for<2>([&](auto oc) {
                constexpr int o = decltype(oc)::value, k = 2 * p + o;
                if (k >= valid) return;
                uint32_t op[J][8];
#pragma unroll
                for (int j = 0; j < J; ++j) half_operand<F>(A[j][o], op[j]);
#pragma unroll
                for (int i = 0; i < S; ++i) {
                    const uint32_t xi = x + i * 8 * kRecordBytes, si = s + i * 8 * kRecordBytes;
                    const uint4 hi = lds_u4_at<k * kSlicedBytes>(xi), lo = lds_u4_at<k * kSlicedBytes + 64>(xi);
                    const float sx[2] = {lds_f1_at<4 * k>(si), lds_f1_at<4 * k + kRecordBytes>(si)};
                    float mx[2] = {0.0f, 0.0f};
                    if (F == kQ4_1)
                        mx[0] = lds_f1_at<4 * k + 4 * kChunkBlocks>(si),
                        mx[1] = lds_f1_at<4 * k + 4 * kChunkBlocks + kRecordBytes>(si);
                    float c[J][4];
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.0f;
                        hmma_f16(c[j], op[j], lo.x, lo.y);
                    }
#pragma unroll
                    for (int j = 0; j < J; ++j) hmma_f16(c[j], op[j] + 4, lo.z, lo.w);
#pragma unroll
                    for (int j = 0; j < J; ++j) hmma_f16(c[j], op[j], hi.x, hi.y);
#pragma unroll
                    for (int j = 0; j < J; ++j) hmma_f16(c[j], op[j] + 4, hi.z, hi.w);
#pragma unroll
                    for (int j = 0; j < J; ++j)
#pragma unroll
                        for (int q = 0; q < 2; ++q)
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                acc[j][i][q][r] = fmaf(A[j][o].d[q] * sx[r], c[j][2 * q + r], acc[j][i][q][r]);
                                if (F == kQ4_1) acc[j][i][q][r] = fmaf(A[j][o].m[q], mx[r], acc[j][i][q][r]);
                            }
                }
            });
        });
    }

    // to: [row of x][pitch], this warp's first row of x and of the tile
    __device__ __forceinline__ void store(float* to, int pitch, int lane) const {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int r = 0; r < 2; ++r) to[(8 * i + 2 * t + r) * pitch + 16 * j + 8 * q + g] = acc[j][i][q][r];
    }
};

__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kComputeThreads) : "memory"); }

template <int F, int MODE, bool ALN>
__global__ void __launch_bounds__(kManyThreads, 1)
    imma_many_kernel(const __grid_constant__ ImmaMaps maps, const __grid_constant__ ImmaArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    using S = Slot<F, ALN>;
    __shared__ int s_last, s_dead, s_issued[kProducers];
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int steps = (a.bpr + kChunkBlocks - 1) / kChunkBlocks;
    // shared memory: stages (weights, records of x), sums, the stages' barriers (full, empty)
    const uint32_t stage_bytes = kStrips * S::kBytes + a.seg_cap * kRecordBytes;
    float* sums = reinterpret_cast<float*>(smem + a.slots * stage_bytes);
    const uint32_t ring = smem_u32(smem), bars = smem_u32(sums + kSumFloats);
    if (threadIdx.x == 0) {
        s_dead = 0;
        for (int i = 0; i < a.slots; ++i) {
            mbar_init(bars + 16 * i, ALN ? kProducers : 64 + 2);
            mbar_init(bars + 16 * i + 8, kComputeWarps);
        }
        fence_mbar_init();
    }
    // Segments: as in mlq_imma_few.cuh.
    if (MODE == kPair) grid_dependency_wait();
    if (MODE != kDown) launch_dependents();
    __syncthreads();
    const int nseg = MODE == kPlain ? (a.rows + a.seg_cap - 1) / a.seg_cap : __ldcg(a.nseg);
    const int id = blockIdx.x;
    const Deal deal(nseg * a.tiles, steps, gridDim.x, kManyJoin);
    Work work(deal, id);
    constexpr int tile_rows = MODE == kPair ? kUnitRows / 2 : kUnitRows;
    auto segment = [&](int seg, int& e, int& first, int& count) {
        e = MODE == kPlain ? 0 : __ldcg(&a.segs[seg].expert);
        first = MODE == kPlain ? seg * a.seg_cap : __ldcg(&a.segs[seg].start);
        count = MODE == kPlain ? min(a.rows - first, a.seg_cap) : __ldcg(&a.segs[seg].count);
    };

    if (warp >= kComputeWarps) {
        // ---- producers: 0 and 1 fetch the weights of 8 strips each, 2 and 3 the records of 16 rows of x each ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kManyProducerRegs));
        const int me = warp - kComputeWarps;
        if (MODE != kPair && me >= 2) grid_dependency_wait();
        int stage = 0, phase = 1, n = 0;
        bool alive = true;
        while (alive && work.next(deal, id)) {
            int e, first, count;
            segment(work.u % nseg, e, first, count);
            const int row0 = e * a.out + work.u / nseg * tile_rows;
            const int token = 16 * (me - 2) + (lane & 15);
            const int mine = me < 2 ? 8 : min(max(count - 16 * (me - 2), 0), 16);  // strips, rows of x
            const uint8_t* x = nullptr;
            if (me >= 2 && (lane & 15) < mine && lane < 16) {
                const int row = MODE == kPair ? __ldcg(a.order + first + token) / a.top_k : first + token;
                x = a.x + (size_t)row * (a.bprp / kChunkBlocks) * kRecordBytes;
            }
            for (int c = work.r0; c < work.r1; ++c, ++n) {
                const uint32_t full = bars + 16 * stage, dst = ring + stage * stage_bytes;
                if (!__all_sync(0xffffffffu, mbar_wait(full + 8, phase))) {
                    if (lane == 0) report_error(a.err, 33), *(volatile int*)&s_dead = 1;
                    alive = false;
                    break;
                }
                if (__any_sync(0xffffffffu, *(volatile int*)&s_dead)) {
                    alive = false;
                    break;
                }
                if (me >= 2) {
                    if (lane == 0) mbar_arrive_expect_tx(full, mine * kRecordBytes);
                    __syncwarp();
                    if (x) bulk_g2s(dst + kStrips * S::kBytes + token * kRecordBytes, x + (size_t)c * kRecordBytes, kRecordBytes, full);
                } else if constexpr (ALN) {
                    if (lane == 0) mbar_arrive_expect_tx(full, 8 * S::kBytes);
                    __syncwarp();
                    if (lane < 8) {
                        const int strip = 8 * me + lane, row = row0 + strip * (MODE == kPair ? 8 : 16);
#pragma unroll
                        for (int b = 0; b < S::kBoxes; ++b) {
                            const int c0 = (c * chunk_bytes(F) + b * S::kPitch) / 2;
                            const uint32_t d = dst + strip * S::kBytes + b * 16 * S::kPitch;
                            tma_load_2d(d, &maps.m[0], c0, row, full);
                            if (MODE == kPair) tma_load_2d(d + 8 * S::kPitch, &maps.m[1], c0, row, full);
                        }
                    }
                } else {
                    // lanes 2r, 2r + 1: the 16-byte windows that hold row r's blocks, strip by strip
                    const int r = lane >> 1, sub = lane & 1;
                    const uint8_t* base = MODE == kPair && r >= 8 ? a.w[1] : a.w[0];
                    bool stored = false;
#pragma unroll 1
                    for (int k = 0; k < 8; ++k) {
                        const int strip = 8 * me + k;
                        const long long row = row0 + strip * (MODE == kPair ? 8 : 16) + (MODE == kPair ? (r & 7) : r);
                        if (row >= a.total_rows) continue;
                        long long left = a.row_bytes - (long long)c * chunk_bytes(F);
                        if (left > chunk_bytes(F)) left = chunk_bytes(F);
                        const uint8_t* src = base + row * a.row_bytes + (long long)c * chunk_bytes(F);
                        const uint8_t* end = src + left;
                        const uint8_t* q =
                            reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(src) & ~(uintptr_t)15) + 16 * sub;
                        uint32_t to = dst + strip * S::kBytes + r * S::kPitch + 16 * sub;
#pragma unroll
                        for (int i = 0; i < (chunk_bytes(F) + 15 + 31) / 32; ++i, q += 32, to += 32) {
                            if (q >= end) break;
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
                if (++stage == a.slots) stage = 0, phase ^= 1;
            }
        }
        if (!ALN) asm volatile("cp.async.wait_all;" ::: "memory");
        if (lane == 0) s_issued[me] = n;
        if (MODE == kDown) launch_dependents();
        __syncthreads();
        return;
    }

    // ---- computing warps ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyComputeRegs));
    if (MODE != kPair) grid_dependency_wait();
    if (MODE == kDown) launch_dependents();
    const int tid = threadIdx.x, g = lane >> 2, t = lane & 3;
    int stage = 0, phase = 0, taken = 0;
    bool alive = true;

    while (work.next(deal, id)) {
        const int tile = work.u / nseg;
        int e, first, count;
        segment(work.u % nseg, e, first, count);
        const bool whole = work.r1 - work.r0 == deal.per;
        const int cap = a.seg_cap, pass_rows = cap > 16 ? 128 : 256, pitch = pass_rows + 4;

        // the unit's results: get(row of x, row of the tile as the stages have it), rows [from, from + pass_rows)
        auto epilogue = [&](int from, auto get) {
            if (MODE == kPair) {
                // a warp takes a block of 32 hidden values of one row of x, in the lane order of the next product
                const int blocks = pass_rows / 64;
                for (int i = warp; i < count * blocks; i += kComputeWarps) {
                    const int tok = i / blocks, loc0 = from / 2 + 32 * (i % blocks), b = (tile * tile_rows + loc0) / 32;
                    if (32 * b >= a.out) continue;
                    const int el = half_element(a.next_fmt, b & 1, lane), loc = loc0 + el;
                    const int row = (loc >> 3) * 16 + (loc & 7);
                    const float h = 32 * b + el < a.out ? silu_mul(get(tok, row), get(tok, row + 8)) : 0.0f;
                    slice_halves(h, a.h + (size_t)(first + tok) * (a.next_bprp / kChunkBlocks) * kRecordBytes, b, lane);
                }
            } else {
                for (int i = tid; i < pass_rows * count; i += kComputeThreads) {
                    const int tok = i / pass_rows, row = from + i % pass_rows;
                    const int o = tile * tile_rows + row;
                    if (o >= a.out) continue;
                    float v = get(tok, row);
                    const int r = first + tok;
                    if (MODE == kDown) {
                        a.part[(size_t)__ldcg(a.order + r) * a.out + o] = v;
                    } else {
                        if (a.bias) v += a.bias[o];
                        v = activate(v, a.act);
                        if (a.row_scale) v *= a.row_scale[r];
                        const size_t to = (size_t)r * a.out + o;
                        a.y[to] = a.residual ? a.residual[to] + v : v;
                    }
                }
            }
        };
        // a unit that several CTAs share: each leaves its sums in a slot (head: the unit started before its range, tail: in
        // it), and whoever comes last adds them up in order
        auto slot_of = [&](int c, bool tail) { return a.split + ((size_t)2 * c + (tail ? 1 : 0)) * a.split_size; };
        int j0 = 0, j1 = 0;
        if (!whole) {
            const long long r = (long long)(work.u - deal.each * deal.teams) * deal.per;
            j0 = deal.owner(r), j1 = deal.owner(r + deal.per - 1);
        }

        // the rounds of this piece for J strips from `strip` against 8 SUBS rows of x from `tok0`; SUBS 0: only keep step
        auto run = [&](auto& acc, auto jc, int strip, int tok0, bool idle) {
            constexpr int J = decltype(jc)::value;
            acc.init();
            [[maybe_unused]] uint32_t window[J][2] = {};
            if constexpr (!ALN) {
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    // where the lane's rows start in their windows
                    const long long off = ((long long)e * a.out + (long long)tile * tile_rows +
                                           (strip + j) * (MODE == kPair ? 8 : 16) + g) * a.row_bytes;
                    window[j][0] = (uint32_t)(reinterpret_cast<uintptr_t>(a.w[0]) + off) & 15;
                    window[j][1] = (uint32_t)(reinterpret_cast<uintptr_t>(a.w[MODE == kPair ? 1 : 0]) + off +
                                              (MODE == kPair ? 0 : 8 * a.row_bytes)) & 15;
                }
            }
            for (int c = work.r0; c < work.r1; ++c) {
                const uint32_t full = bars + 16 * stage, at = ring + stage * stage_bytes;
                if (!__all_sync(0xffffffffu, mbar_try_wait(full, phase)) && alive &&
                    !__all_sync(0xffffffffu, mbar_wait(full, phase))) {
                    alive = false;
                    if (lane == 0) report_error(a.err, 32), *(volatile int*)&s_dead = 1;
                }
                if (!idle) {
                    RowBase rows[J];
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        uint32_t r0 = at + (strip + j) * S::kBytes + g * S::kPitch, r1 = r0 + 8 * S::kPitch;
                        if constexpr (!ALN) {
                            const uint32_t k = (uint32_t)c * (chunk_bytes(F) & 15);
                            r0 += (window[j][0] + k) & 15;
                            r1 += (window[j][1] + k) & 15;
                        }
                        rows[j] = row_base(r0, r1, t);
                    }
                    const uint32_t x = at + kStrips * S::kBytes + tok0 * kRecordBytes;
                    acc.template step<ALN>(x + g * kRecordBytes + t * 16, x + 2 * t * kRecordBytes + kRecordScales,
                                           a.bpr - c * kChunkBlocks, rows);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(full + 8);
                if (++stage == a.slots) stage = 0, phase ^= 1;
            }
            if (alive) taken += work.r1 - work.r0;
            for (int from = 0; from < kUnitRows; from += pass_rows) {
                compute_sync();  // the last pass has been read
                if (!idle && 16 * strip >= from && 16 * strip < from + pass_rows)
                    acc.store(sums + tok0 * pitch + 16 * strip - from, pitch, lane);
                compute_sync();
                auto get = [&](int tok, int row) { return sums[tok * pitch + row - from]; };
                if (whole) {
                    epilogue(from, get);
                } else {
                    float* mine = slot_of(id, id == j0);
                    for (int i = tid; i < pass_rows * count; i += kComputeThreads)
                        mine[(size_t)(i / pass_rows) * kUnitRows + from + i % pass_rows] = get(i / pass_rows, from + i % pass_rows);
                }
            }
        };
        using One = std::integral_constant<int, 1>;
        using Two = std::integral_constant<int, 2>;
        const bool past = tile * tile_rows + (count > 16 ? warp / 2 * 2 : warp) * (MODE == kPair ? 8 : 16) >= a.out;
        if (count > 16) {
            const int tok0 = 16 * (warp & 1);
            if (count - tok0 > 8) {
                ManyRows<F, 2, 2> acc;
                run(acc, Two{}, warp / 2 * 2, tok0, past);
            } else {
                ManyRows<F, 2, 1> acc;
                run(acc, Two{}, warp / 2 * 2, tok0, past);
            }
        } else if (count > 8) {
            ManyRows<F, 1, 2> acc;
            run(acc, One{}, warp, 0, past);
        } else {
            ManyRows<F, 1, 1> acc;
            run(acc, One{}, warp, 0, past);
        }
        if (!whole) {
            compute_sync();
            if (tid == 0) {
                __threadfence();
                s_last = atomicAdd(a.split_done + j0, 1u) == (unsigned)(j1 - j0);
                __threadfence();
            }
            compute_sync();
            if (s_last)
                for (int from = 0; from < kUnitRows; from += pass_rows)
                    epilogue(from, [&](int tok, int row) {
                        const size_t in = (size_t)tok * kUnitRows + row;
                        float v = __ldcg(slot_of(j0, true) + in);
#pragma unroll 4
                        for (int c = j0 + 1; c <= j1; ++c) v += __ldcg(slot_of(c, false) + in);
                        return v;
                    });
        }
    }
    __syncthreads();  // the producers have issued their last copies
    // after a wait that ran out, copies may still be in flight: each is waited for once more, bounded
    if (*(volatile int*)&s_dead) {
        int n = 0;
        for (int p = 0; p < kProducers; ++p) n = max(n, s_issued[p]);
        for (int i = taken; i < n; ++i) mbar_wait(bars + 16 * (i % a.slots), (i / a.slots) & 1);
    }
}

template <int F, int MODE, bool ALN>
cudaError_t launch_one(ImmaArgs a, int grid, int smem_per_sm, cudaStream_t stream) {
    using S = Slot<F, ALN>;
    auto k = imma_many_kernel<F, MODE, ALN>;
    const int stage = kStrips * S::kBytes + a.seg_cap * kRecordBytes;
    const int fixed = kSumFloats * 4 + 1024 + 256;  // the system's 1 KB per CTA, the static part
    a.slots = (smem_per_sm - fixed) / (stage + 16);
    if (a.slots > 8) a.slots = 8;
    if (a.slots < 2) return cudaErrorInvalidConfiguration;
    const size_t smem = (size_t)a.slots * (stage + 16) + kSumFloats * 4;
    ImmaMaps maps{};
    if (ALN && !make_weight_maps(&maps, a, MODE == kPair, S::kPitch)) return cudaErrorInvalidValue;
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
