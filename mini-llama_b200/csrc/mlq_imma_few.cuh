// mlq_imma_few.cuh -- the streaming kernel for few rows of x per matrix
// (digits, int8 matrix instructions; mathematics and operand layout:
// mlq_imma.cuh; the launches around it: mlq_imma.cu).
//
// One CTA per SM: two teams of 8 computing warps, and two producer warps for
// each.  A unit is a tile of 16 to 128 rows of one matrix against one
// segment; a team's warps split it in 16-row strips and the K axis in
// interleaved steps of 8 blocks.  A round is one step of every warp: 128
// (row, block) squares of 16 x 8 whatever the tile, so rounds cost the same
// and the launch's rounds are dealt out evenly, a contiguous range per team.
// The producers fill a ring of stages (one round each) by TMA, running
// ahead across units, so the weight stream waits for no unit's end, and one
// team computes while the other is at one.  The K parts of a unit meet in
// shared memory in a fixed order; a unit whose rounds fall to several teams is
// added up (in order) by the last of them to finish.
//
// One row of 8192 values, with the slicing launch (us): 14336, 28672, 57344 and
// 114688 outputs take 26, 47, 82 and 153 in q8_0, 18, 32, 54 and 95 in q4_0, 20, 36, 59 and 105 in
// q4_1.  Past ~12 us for the slicing launch, the ramp and the last units, every
// format runs at 0.97 or more of a copy's 6.56 TB/s.  With 4 rows 28672 outputs take 51, 38 and 44:
// there the products and folds of the second pair of rows show.  Small matrices are
// bound by latency (4096 x 4096 q4_0, one row: 6.1 us, 1.4 us of HBM time).
#pragma once

#include "mlq_imma_common.cuh"

namespace mlq {
namespace {

// The accumulators of up to 2 NT rows of x by digits: an instruction's 8
// columns are the 4 digits of 2 rows, so lane t holds digits 3 and 2 (t even) or
// 1 and 0 (t odd) of row t / 2, and the two are added once, at the end.
template <int F, int NT>
struct FewRows {
    uint32_t xo[NT], so[NT];  // a lane's digits and scales in the step's records
    uint64_t acc[NT];         // of the lane's two weight rows

    __device__ __forceinline__ void init(int count, int lane) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            // columns without a row of x repeat the first one's; nothing reads them
            const int r = 2 * i + (g >> 2), rs = 2 * i + (t >> 1);
            xo[i] = (r < count ? r : 0) * record_bytes(F) + (g & 3) * 64 + t * 16;
            so[i] = (rs < count ? rs : 0) * record_bytes(F);
            acc[i] = 0;
        }
    }

    // One K step of 8 blocks; x: the records of the segment's rows.
    template <bool ALN>
    __device__ __forceinline__ void step(uint32_t x, int valid, uint32_t r0, uint32_t r1, int lane) {
        const RowBase rows = row_base(r0, r1, lane & 3);
        [[maybe_unused]] const uint32_t sums = x + block_sums(0, lane & 1);
        uint64_t part[NT] = {};  // of this step: a row of n blocks is a chain of n / 8 + 8 roundings, not of n
        static_for<kChunkBlocks / 2>([&](auto pc) {
            constexpr int p = decltype(pc)::value;
            if (!ALN && 2 * p >= valid) return;
            uint4 b[NT];
            float2 s[NT];
            [[maybe_unused]] float4 sum[NT];  // q4_1: the pair's sums of the lane's digits
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                b[i] = lds_u4_at<256 * p>(x + xo[i]);
                s[i] = lds_f2_at<8 * p + kRecordScales>(x + so[i]);
                if (F == kQ4_1) sum[i] = lds_f4_at<32 * p>(sums + so[i]);
            }
            RawA A[2];
            load_pair<F, ALN, p>(rows, A[0], A[1]);
            if (!ALN && 2 * p + 1 >= valid) A[1].d[0] = A[1].d[1] = A[1].m[0] = A[1].m[1] = 0.0f;
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                uint32_t op[4];
                int8_operand<F>(A[o], op);
                const uint64_t d = pack2(A[o].d[0], A[o].d[1]);
                [[maybe_unused]] const uint64_t m = F == kQ4_1 ? pack2(A[o].m[0], A[o].m[1]) : 0;
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const float sx = o ? s[i].y : s[i].x;
                    int c[4];
                    imma<F>(c, op, o ? make_uint2(b[i].z, b[i].w) : make_uint2(b[i].x, b[i].y));
                    const uint64_t v = pack2((float)(c[0] * 256 + c[1]), (float)(c[2] * 256 + c[3])), sx2 = pack2(sx, sx);
                    if constexpr (F == kQ4_1) {
                        // d v + m sum: m times the higher digits' sum is exact (11 and 12 bits), so the first step
                        // rounds what the parts leave of each other, and the second adds the lower digits' share
                        const float2 t = o ? make_float2(sum[i].z, sum[i].w) : make_float2(sum[i].x, sum[i].y);
                        const uint64_t left = fma2(d, v, mul2(m, pack2(t.x, t.x)));
                        part[i] = fma2(fma2(m, pack2(t.y, t.y), left), sx2, part[i]);
                    } else {
                        part[i] = fma2(d, mul2(v, sx2), part[i]);
                    }
                }
            }
        });
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i] = add2(acc[i], part[i]);
    }

    // red: [row of x][weight row 0..15] of this warp
    __device__ __forceinline__ void store(float* red, int lane) {
        const int t = lane & 3;
        // digits 3 and 2 count 2^16 times digits 1 and 0; q4 codes count 16
        const float f = (t & 1 ? 1.0f : 65536.0f) * (F == kQ8_0 ? 1.0f : 0.0625f);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const float2 both = unpack2(acc[i]);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float v = (q ? both.y : both.x) * f;
                v += __shfl_xor_sync(0xffffffffu, v, 1);
                if (!(t & 1)) red[(2 * i + (t >> 1)) * 16 + 8 * q + (lane >> 2)] = v;
            }
        }
    }
};

constexpr int kTeams = 2;
// Records of a round: (K parts) x (rows of x of a segment) <= 8, see choose_strips.
constexpr int x_stage(int fmt) { return 8 * record_bytes(fmt); }
constexpr int kThreads = 32 * kTeams * (kImmaWarps + 2);  // computing warps, then two producer warps per team
constexpr int kTeamThreads = 32 * kImmaWarps;
// Registers: the launch has 96 per thread (65536 / 640, in eights); the
// producers keep 32 and the computing warps take what that frees.
constexpr int kLaunchRegs = 96, kProducerRegs = 32, kComputeRegs = 112;
static_assert((2 * kTeams * kProducerRegs + kTeams * kImmaWarps * kComputeRegs) * 32 <= kThreads * kLaunchRegs,
              "the shares must not exceed the launch's registers, or setmaxnreg would wait for ever");
constexpr int kRedFloats = kImmaWarps * kFewRows * 16;  // [warp][row of x][row of the strip]
constexpr int kJoinRounds = 4;  // adding up a shared unit: ~2.5 us; a round takes ~0.8 us of a team's share of HBM

// The barrier of a team's computing warps.
__device__ __forceinline__ void team_sync(int team) {
    asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(kTeamThreads) : "memory");
}

// What a producer fetches next: round `round` of a tile against a segment, into `stage`.
struct Cursor {
    Work work;
    int r, tile, seg, round, row0, first, count, stage, phase, n;  // r: round of the piece; n: rounds so far
    bool on, fresh;
    __device__ __forceinline__ explicit Cursor(const Work& w)
        : work(w), r(0), tile(0), seg(0), round(0), row0(0), first(0), count(0), stage(0), phase(1), n(0), on(false),
          fresh(true) {}
};

// A computing warp's place in its team's ring.
struct WarpState {
    int stage, phase, taken;
    bool alive;  // false once a wait ran out: nothing is waited for any more
};

// What a computing warp needs for its part of a unit (by value: the function
// below has registers of its own).
struct UnitArgs {
    float* red;              // this warp's sums
    uint32_t full, slots;    // barrier of stage 0 (16 bytes each: full, empty), this warp's slot of stage 0
    uint32_t stage_bytes, to_x;  // from the slot to the records of this warp's K part
    int stages;
    int count;
    int c0, c_end, kws;      // K steps: c0, c0 + kws, .. below c_end
    int rounds, blocks;      // rounds of this part, blocks of a row
    uint32_t window0, window1, window_step;  // rows that are not aligned: where row g (g + 8) starts in its window
    int* err;
    volatile int* dead;
};

// The rounds of one unit: this warp's strip against the segment's rows of x,
// its sums to u.red.  A function of its own for each form of x.
template <class Acc, int F, bool ALN>
__device__ __forceinline__ WarpState unit_sums(const UnitArgs u, WarpState st) {
    using S = Slot<F, ALN>;
    const int lane = threadIdx.x & 31, g = lane >> 2;
    int c = u.c0;
    Acc acc;
    acc.init(u.count, lane);
    for (int r = 0; r < u.rounds; ++r, c += u.kws) {
        const uint32_t full = u.full + 16 * st.stage, at = u.slots + st.stage * u.stage_bytes;
        if (!__all_sync(0xffffffffu, mbar_try_wait(full, st.phase)) && st.alive &&
            !__all_sync(0xffffffffu, mbar_wait(full, st.phase))) {
            st.alive = false;
            if (lane == 0) report_error(u.err, 30), *u.dead = 1;
        }
        if (c < u.c_end) {
            uint32_t row0 = at + g * S::kPitch, row1 = row0 + 8 * S::kPitch;
            if constexpr (!ALN) {
                row0 += (u.window0 + (uint32_t)c * u.window_step) & 15;
                row1 += (u.window1 + (uint32_t)c * u.window_step) & 15;
            }
            const int valid = u.blocks - c * kChunkBlocks;
            acc.template step<ALN>(at + u.to_x, valid, row0, row1, lane);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(full + 8);
        if (++st.stage == u.stages) st.stage = 0, st.phase ^= 1;
    }
    if (st.alive) st.taken += u.rounds;
    acc.store(u.red, lane);
    return st;
}

template <int F, int MODE, bool ALN>
__global__ void __launch_bounds__(kThreads, 1)
    imma_few_kernel(const __grid_constant__ ImmaMaps maps, const __grid_constant__ ImmaArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    using S = Slot<F, ALN>;
    __shared__ int s_last[kTeams], s_dead, s_issued[kTeams][2];
    const int lane = threadIdx.x & 31, cta_warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const bool producer = cta_warp >= kTeams * kImmaWarps;
    const int team = producer ? (cta_warp - kTeams * kImmaWarps) >> 1 : cta_warp / kImmaWarps;
    const int kws = kImmaWarps / a.strips;
    const int steps = (a.bpr + kChunkBlocks - 1) / kChunkBlocks;
    const int per_seg = (steps + kws - 1) / kws;  // rounds of a tile against a segment
    // shared memory: stages [team][stage] of the warps' weights and the rounds' records of x, sums [team], (all_segs) y
    // [team], the stages' barriers [team][stage] (full, empty)
    constexpr uint32_t kRecord = record_bytes(F), kStage = kImmaWarps * S::kBytes + x_stage(F);
    const uint32_t red0 = kTeams * a.slots * kStage;
    const uint32_t y_floats = MODE == kDown && !a.part ? a.rows * 16 * a.strips : 0;
    const uint32_t bars0 = smem_u32(smem) + red0 + kTeams * (2 * kRedFloats + y_floats) * 4;
    const uint32_t bars = bars0 + 16 * team * a.slots;
    const uint32_t ring = smem_u32(smem) + team * a.slots * kStage;
    if (threadIdx.x == 0) {
        s_dead = 0;
        for (int i = 0; i < kTeams * a.slots; ++i) {
            mbar_init(bars0 + 16 * i, ALN ? 1 : 64);
            mbar_init(bars0 + 16 * i + 8, kImmaWarps);
        }
        fence_mbar_init();
    }

    // The segments come from prep.  kPair is prep's dependent, so it waits;
    // kDown started after every CTA of kPair had waited for prep, so prep has
    // completed: it reads the segments (past L1) and streams weights at once.
    if (MODE == kPair) grid_dependency_wait();
    if (MODE != kDown) launch_dependents();
    __syncthreads();
    const int nseg = MODE == kPlain ? (a.rows + a.seg_cap - 1) / a.seg_cap : __ldcg(a.nseg);
    // kDown with few rows (a.part null): a unit is a tile against every segment; otherwise against one, and the
    // segments of a tile are neighbours.
    const bool all_segs = MODE == kDown && !a.part;
    const int id = kTeams * blockIdx.x + team;
    const Deal deal(all_segs ? (nseg ? a.tiles : 0) : nseg * a.tiles, all_segs ? nseg * per_seg : per_seg,
                    kTeams * gridDim.x, kJoinRounds);
    Work work(deal, id);
    const int unit_rows = (MODE == kPair ? 8 : 16) * a.strips;

    if (producer) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegs));
        const int half = cta_warp & 1;
        // Tensor maps: the team's two producers take stages in turn (issuing a box takes ~70 cycles).  16-byte windows:
        // each takes the slots of four warps of every stage, the first one also x.
        Cursor cur(work);
        auto next_piece = [&](Cursor& c) {
            c.on = c.work.next(deal, id);
            if (!c.on) return;
            c.r = c.work.r0;
            c.tile = all_segs ? c.work.u : c.work.u / nseg;
            c.seg = all_segs ? c.work.r0 / per_seg : c.work.u % nseg;
            c.round = all_segs ? c.work.r0 % per_seg : c.work.r0;
            c.fresh = true;
        };
        auto advance = [&](Cursor& c) {
            ++c.n;
            if (++c.stage == a.slots) c.stage = 0, c.phase ^= 1;
            if (++c.round == per_seg) c.round = 0, ++c.seg, c.fresh = true;
            if (++c.r == c.work.r1) next_piece(c);
        };
        auto mine = [&](const Cursor& c) { return !ALN || (c.n & 1) == half; };
        // the segment's matrix and rows of x
        auto refresh = [&](Cursor& c) {
            if (!c.fresh) return;
            c.fresh = false;
            const int e = MODE == kPlain ? 0 : __ldcg(&a.segs[c.seg].expert);
            c.row0 = e * a.out + c.tile * unit_rows;
            c.first = MODE == kPlain ? c.seg * a.seg_cap : __ldcg(&a.segs[c.seg].start);
            c.count = MODE == kPlain ? (a.rows - c.first < a.seg_cap ? a.rows - c.first : a.seg_cap)
                                     : __ldcg(&a.segs[c.seg].count);
        };
        auto active = [&](const Cursor& c) { return min(steps - c.round * kws, kws); };  // K parts of the round
        auto fetch_weights = [&](Cursor& c) {
            const uint32_t full = bars + 16 * c.stage, dst = ring + c.stage * kStage;
            if constexpr (ALN) {
                if (lane == 0)
                    mbar_arrive_expect_tx(full, active(c) * (a.strips * S::kBytes + c.count * kRecord));
                __syncwarp();
                const int kw = lane / a.strips;
                if (kw < active(c)) {
                    const int row = c.row0 + (lane % a.strips) * (MODE == kPair ? 8 : 16);
#pragma unroll
                    for (int b = 0; b < S::kBoxes; ++b) {
                        const int c0 = ((c.round * kws + kw) * chunk_bytes(F) + b * S::kPitch) / 2;
                        const uint32_t d = dst + lane * S::kBytes + b * 16 * S::kPitch;
                        tma_load_2d(d, &maps.m[0], c0, row, full);
                        if (MODE == kPair) tma_load_2d(d + 8 * S::kPitch, &maps.m[1], c0, row, full);
                    }
                }
                __syncwarp();
            } else {
                if (half == 0 && lane == 0) mbar_expect_tx(full, active(c) * c.count * kRecord);
                // lanes 2r, 2r + 1: the windows that hold row r's blocks
                const int r = lane >> 1, sub = lane & 1;
                const uint8_t* base = MODE == kPair && r >= 8 ? a.w[1] : a.w[0];
                bool stored = false;
#pragma unroll 1
                for (int k = 0; k < kImmaWarps / 2; ++k) {
                    const int w = kImmaWarps / 2 * half + k, step = c.round * kws + w / a.strips;
                    const long long row =
                        c.row0 + (w % a.strips) * (MODE == kPair ? 8 : 16) + (MODE == kPair ? (r & 7) : r);
                    if (step >= steps || row >= a.total_rows) continue;
                    long long left = a.row_bytes - (long long)step * chunk_bytes(F);
                    if (left > chunk_bytes(F)) left = chunk_bytes(F);
                    const uint8_t* src = base + row * a.row_bytes + (long long)step * chunk_bytes(F);
                    const uint8_t* end = src + left;
                    const uint8_t* q =
                        reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(src) & ~(uintptr_t)15) + 16 * sub;
                    uint32_t to = dst + w * S::kBytes + r * S::kPitch + 16 * sub;
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
                __syncwarp();  // the bytes of x are expected before anyone arrives for good
                if (stored) {  // plain stores are ordered by a plain arrival
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    mbar_arrive(full);
                } else {
                    cp_async_arrive(full);
                }
            }
        };
        // lane (K part, row of x): its record
        auto fetch_x = [&](Cursor& c) {
            if (!ALN && half) return;
            const int kw = lane / a.seg_cap, r = lane % a.seg_cap;
            if (kw < active(c) && r < c.count) {
                const int row = MODE == kPair ? __ldcg(a.order + c.first + r) / a.top_k : c.first + r;
                bulk_g2s(ring + c.stage * kStage + kImmaWarps * S::kBytes + lane * kRecord,
                         a.x + ((size_t)row * (a.bprp / kChunkBlocks) + c.round * kws + kw) * kRecord, kRecord,
                         bars + 16 * c.stage);
            }
            __syncwarp();
        };
        next_piece(cur);
        if (MODE != kPair) {
            // the ring's first weights are on their way while the launch before this one writes x
            Cursor xs = cur;
            for (int i = 0; i < a.slots && cur.on; ++i, advance(cur))
                if (mine(cur)) refresh(cur), fetch_weights(cur);
            grid_dependency_wait();
            for (; xs.on && xs.n < cur.n; advance(xs))
                if (mine(xs)) refresh(xs), fetch_x(xs);
        }
        for (; cur.on; advance(cur)) {
            if (!mine(cur)) continue;
            refresh(cur);
            if (!__all_sync(0xffffffffu, mbar_wait(bars + 16 * cur.stage + 8, cur.phase))) {
                if (lane == 0) report_error(a.err, 31), *(volatile int*)&s_dead = 1;
                break;
            }
            if (__any_sync(0xffffffffu, *(volatile int*)&s_dead)) break;
            fetch_weights(cur);
            fetch_x(cur);
        }
        if (!ALN) asm volatile("cp.async.wait_all;" ::: "memory");
        if (lane == 0) s_issued[team][half] = ALN ? cur.n : 0;
        if (MODE == kDown) launch_dependents();
        __syncthreads();
        return;
    }

    // ---- computing warps ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kComputeRegs));
    if (MODE != kPair) grid_dependency_wait();
    if (MODE == kDown) launch_dependents();
    const int warp = cta_warp % kImmaWarps, tid = threadIdx.x % kTeamThreads;
    const int strip = warp % a.strips, kw = warp / a.strips;
    float* red = reinterpret_cast<float*>(smem + red0) + team * 2 * kRedFloats;
    WarpState st{0, 0, 0, true};
    int half = 0;
    float* ysum = reinterpret_cast<float*>(smem + red0) + kTeams * 2 * kRedFloats + team * y_floats;  // all_segs: [row][row of the tile]

    // Units that several teams share.  A team's tail slot holds the piece of the unit that starts in its range, its head
    // slot that of the unit that started before.
    auto slot_of = [&](int t, bool tail) { return a.split + ((size_t)2 * t + (tail ? 1 : 0)) * a.split_size; };
    int j0 = 0, j1 = 0;  // the teams that share the piece's unit
    auto join = [&](int n, auto value) -> int {
        const long long t = (long long)(work.u - deal.each * deal.teams) * deal.per;
        j0 = deal.owner(t), j1 = deal.owner(t + deal.per - 1);
        float* mine = slot_of(id, id == j0);
        for (int i = tid; i < n; i += kTeamThreads) mine[i] = value(i);
        team_sync(team);
        if (tid == 0) {
            __threadfence();
            s_last[team] = atomicAdd(a.split_done + j0, 1u) == (unsigned)(j1 - j0);
            __threadfence();
        }
        team_sync(team);
        return s_last[team];
    };
    auto joined = [&](int i) {
        float v = __ldcg(slot_of(j0, true) + i);
#pragma unroll 4
        for (int t = j0 + 1; t <= j1; ++t) v += __ldcg(slot_of(t, false) + i);
        return v;
    };

    while (work.next(deal, id)) {
        const bool whole = work.r1 - work.r0 == deal.per;
        const int tile = all_segs ? work.u : work.u / nseg;
        if (all_segs)
            for (int i = tid; i < (int)y_floats; i += kTeamThreads) ysum[i] = 0.0f;
        int seg = all_segs ? work.r0 / per_seg : work.u % nseg;
        for (int done = work.r0; done < work.r1; ++seg) {
            const int base = all_segs ? seg * per_seg : 0;
            const int r0 = done - base, r1 = work.r1 - base < per_seg ? work.r1 - base : per_seg;
            done = base + r1;
            int first, count, e = 0;
            if (MODE == kPlain) {
                first = seg * a.seg_cap;
                count = a.rows - first < a.seg_cap ? a.rows - first : a.seg_cap;
            } else {
                e = __ldcg(&a.segs[seg].expert);
                first = __ldcg(&a.segs[seg].start);
                count = __ldcg(&a.segs[seg].count);
            }
            float* rb = red + half * kRedFloats;  // the buffers alternate
            half ^= 1;
            UnitArgs u{};
            u.red = rb + warp * kFewRows * 16;
            u.full = bars, u.slots = ring + warp * S::kBytes, u.stages = a.slots, u.stage_bytes = kStage;
            u.to_x = (kImmaWarps - warp) * S::kBytes + kw * a.seg_cap * kRecord;
            u.count = count;
            u.c0 = r0 * kws + kw, u.kws = kws, u.rounds = r1 - r0, u.blocks = a.bpr;
            u.c_end = r1 * kws < steps ? r1 * kws : steps;
            u.err = a.err, u.dead = &s_dead;
            if constexpr (!ALN) {
                const long long off =
                    ((long long)e * a.out + (long long)tile * unit_rows + strip * (MODE == kPair ? 8 : 16) + (lane >> 2)) * a.row_bytes;
                u.window0 = (uint32_t)(reinterpret_cast<uintptr_t>(a.w[0]) + off) & 15;
                u.window1 = (uint32_t)(reinterpret_cast<uintptr_t>(a.w[MODE == kPair ? 1 : 0]) + off +
                                       (MODE == kPair ? 0 : 8 * a.row_bytes)) & 15;
                u.window_step = chunk_bytes(F) & 15;
            }
            if (count <= 2)
                st = unit_sums<FewRows<F, 1>, F, ALN>(u, st);
            else
                st = unit_sums<FewRows<F, 2>, F, ALN>(u, st);
            team_sync(team);
            auto sum_parts = [&](int tok, int row) {
                float v = 0.0f;
                for (int k = 0; k < kws; ++k) v += rb[((k * a.strips + (row >> 4)) * kFewRows + tok) * 16 + (row & 15)];
                return v;
            };

            if (all_segs) {
                // a thread takes a row of the tile and every second row of x, so that no other adds to its sums
                for (int i = tid; i < 2 * unit_rows; i += kTeamThreads) {
                    const int row = i % unit_rows, odd = i / unit_rows;
                    for (int tok = 0; tok < count; ++tok) {
                        const int pair = __ldcg(a.order + first + tok), x = pair / a.top_k;
                        if ((x & 1) != odd) continue;
                        float* to = ysum + x * unit_rows + row;
                        *to = fmaf(a.weights[pair], sum_parts(tok, row), *to);
                    }
                }
                continue;
            }

            // the unit's results: get(row of x of the segment, row of the tile as the slots have it)
            auto epilogue = [&](auto get) {
                if (MODE == kPair) {
                    // a warp takes a block of 32 hidden values of one row of x, in the lane order of the next product
                    const int blocks = a.strips / 4;
                    for (int i = warp; i < count * blocks; i += kImmaWarps) {
                        const int tok = i / blocks, b = tile * blocks + i % blocks;
                        if (32 * b >= a.out) continue;
                        const int el = imma_element(a.next_fmt, b & 1, lane);
                        const int loc = 32 * (i % blocks) + el;
                        const int row = (loc >> 3) * 16 + (loc & 7);
                        const float h = 32 * b + el < a.out ? silu_mul(get(tok, row), get(tok, row + 8)) : 0.0f;
                        slice_digits(h, a.next_fmt,
                                     a.h + (size_t)(first + tok) * (a.next_bprp / kChunkBlocks) * record_bytes(a.next_fmt), b,
                                     lane);
                    }
                } else {
                    for (int i = tid; i < unit_rows * count; i += kTeamThreads) {
                        const int tok = i / unit_rows, row = i % unit_rows;
                        const int o = tile * unit_rows + row;
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
            if (whole) {
                epilogue(sum_parts);
            } else {
                // leave the sums of this piece; whoever comes last adds the pieces up in order, in its buffer
                const int slot_rows = 16 * a.strips, n = slot_rows * count;
                const int last = join(n, [&](int i) { return sum_parts(i / slot_rows, i % slot_rows); });
                if (last) {
                    for (int i = tid; i < n; i += kTeamThreads) rb[i] = joined(i);
                    team_sync(team);
                    epilogue([&](int tok, int row) { return rb[tok * slot_rows + row]; });
                }
                team_sync(team);  // s_last and, where this was the last piece, rb may be written again
            }
        }
        if (all_segs) {
            team_sync(team);
            const int n = a.rows * unit_rows;
            bool last = true;
            if (!whole) last = join(n, [&](int i) { return ysum[i]; });
            if (last)
                for (int i = tid; i < n; i += kTeamThreads) {
                    const int o = tile * unit_rows + i % unit_rows;
                    if (o >= a.out) continue;
                    const float v = whole ? ysum[i] : joined(i);
                    const size_t to = (size_t)(i / unit_rows) * a.out + o;
                    a.y[to] = a.residual ? a.residual[to] + v : v;
                }
            team_sync(team);  // ysum and s_last may be written again
        }
    }
    if (all_segs && nseg == 0) {
        // no row names an expert
        const size_t n = (size_t)a.rows * a.out;
        for (size_t i = (size_t)id * kTeamThreads + tid; i < n; i += (size_t)kTeams * gridDim.x * kTeamThreads)
            a.y[i] = a.residual ? a.residual[i] : 0.0f;
    }
    __syncthreads();  // the producers have issued their last copies
    // after a wait that ran out, copies may still be in flight: each is waited for once more, bounded
    if (*(volatile int*)&s_dead)
        for (int i = st.taken; i < s_issued[team][i & 1]; ++i) mbar_wait(bars + 16 * (i % a.slots), (i / a.slots) & 1);
}

// Ring depth: what the SM's shared memory leaves room for, 2..8 stages.
template <int F, int MODE, bool ALN>
cudaError_t launch_one(ImmaArgs a, int grid, int smem_per_sm, cudaStream_t stream) {
    using S = Slot<F, ALN>;
    auto k = imma_few_kernel<F, MODE, ALN>;
    const int sums = kTeams * (2 * kRedFloats + (MODE == kDown && !a.part ? a.rows * 16 * a.strips : 0)) * 4;
    const int fixed = sums + 1024 + 256;  // the system's 1 KB per CTA, the static part
    constexpr int stage = kImmaWarps * S::kBytes + x_stage(F);
    a.slots = (smem_per_sm - fixed) / (kTeams * (stage + 16));
    if (a.slots > 8) a.slots = 8;
    if (a.slots < 2) return cudaErrorInvalidConfiguration;
    const size_t smem = (size_t)kTeams * a.slots * (stage + 16) + sums;
    ImmaMaps maps{};
    if (ALN && !make_weight_maps(&maps, a, MODE == kPair, S::kPitch)) return cudaErrorInvalidValue;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = ready_kernel(k, kLaunchRegs, done);
    if (e != cudaSuccess) return e;
    return launch_pdl(k, grid, kThreads, smem, stream, maps, a);
}

template <int MODE>
cudaError_t launch_few(int fmt, ImmaArgs a, int sm_count, int smem_per_sm, long long max_units, cudaStream_t stream) {
    const bool aln = aligned_rows(fmt, a.w[0], a.bpr) && (MODE != kPair || aligned_rows(fmt, a.w[1], a.bpr));
    a.row_bytes = (long long)a.bpr * block_bytes(fmt);
    const int steps = (a.bpr + kChunkBlocks - 1) / kChunkBlocks, kws = kImmaWarps / a.strips;
    const long long rounds = max_units * ((steps + kws - 1) / kws);
    int grid = sm_count < kMaxTeams / kTeams ? sm_count : kMaxTeams / kTeams;
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
