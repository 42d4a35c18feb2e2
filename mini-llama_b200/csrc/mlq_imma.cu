// mlq_imma.cu -- the experts' products and the linear with an epilogue
// (mathematics and operand layout: mlq_imma.cuh).
//
// A call is three to five launches, chained by programmatic dependent launch:
//   prep   sorts the (row, slot) pairs by expert into segments and slices x (many
//          rows: slices in a launch of its own, by sorted position);
//   pair   h = silu(x Wg^T) * (x Wu^T) per segment, sliced in its epilogue;
//   down   h Wd^T, weighed and summed per row over the segments of a tile in
//          order, or, with many rows, by a fourth launch over the slots;
// and two (prep, down in its plain form) for the linear with an epilogue.
#include "mlq_imma_args.cuh"

namespace mlq {
namespace {

// y from the parts of every pair, for calls with many rows; V consecutive
// values per thread.
template <int V>
__global__ void __launch_bounds__(256) combine_kernel(const ImmaArgs a) {
    launch_dependents();
    grid_dependency_wait();
    const int per = a.out / V;
    const size_t n = (size_t)a.rows * per;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const int r = (int)(i / per), o = (int)(i % per) * V;
        if constexpr (V == 1) {
            a.y[i] = combine(a, r, o);
        } else {
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
            for (int j = 0; j < a.top_k; ++j) {  // as combine() does it
                const int p = r * a.top_k + j, e = a.ids[p];
                if (e < 0 || e >= a.n_experts) continue;
                const float w = a.weights[p];
                const float4 q = __ldcg(reinterpret_cast<const float4*>(a.part + (size_t)p * a.out + o));
                v.x = fmaf(w, q.x, v.x), v.y = fmaf(w, q.y, v.y), v.z = fmaf(w, q.z, v.z), v.w = fmaf(w, q.w, v.w);
            }
            const size_t at = (size_t)r * a.out + o;
            if (a.residual) {
                const float4 q = *reinterpret_cast<const float4*>(a.residual + at);
                v.x = q.x + v.x, v.y = q.y + v.y, v.z = q.z + v.z, v.w = q.w + v.w;
            }
            *reinterpret_cast<float4*>(a.y + at) = v;
        }
    }
}

constexpr int kMaxPairs = 8192;  // pairs of one pass at most

struct PrepArgs {
    const float* x;
    int rows, in, bpr, bprp, fmt;
    uint8_t* sliced;  // records
    int seg_cap;      // rows of a segment at most
    unsigned int* split_done;
    // experts only (ids not null)
    const int32_t* ids;
    int pairs, n_experts;
    int positions;    // many rows: of order, an expert's first one a multiple of 8; else 0
    Segment* segs;
    int* nseg;
    int* order;       // position -> pair
    int* place;       // many rows: pair -> position, -1: no expert
    // padding blocks of the sliced h
    uint8_t* h;
    int h_bpr, h_bprp, h_fmt;
};

// Pairs by expert (CTA 0), x sliced (one warp per block).  Latency-bound:
// a decode call's x is a few KB.
__global__ void __launch_bounds__(256) prep_kernel(const PrepArgs a) {
    launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int first = blockIdx.x, ctas = gridDim.x;
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < 2 * kMaxTeams; i += 256) a.split_done[i] = 0;
    if (a.ids) {
        if (blockIdx.x == 0) {
            __shared__ int cnt[MLQ_MOE_MAX_EXPERTS];
            __shared__ int wsum[2][8];
            __shared__ unsigned char in_warp[8][MLQ_MOE_MAX_EXPERTS];
            __shared__ short s_ids[kMaxPairs];  // -1: none of the experts
            for (int e = threadIdx.x; e < a.n_experts; e += 256) cnt[e] = 0;
            const int pad = a.h ? a.h_bprp - a.h_bpr : 0;
            const int align = a.positions ? 8 : 1;
            for (int i = threadIdx.x; i < a.pairs * pad; i += 256) {
                const int b = a.h_bpr + i % pad;
                uint8_t* record = a.h + ((size_t)(i / pad) * (a.h_bprp / kChunkBlocks) + b / kChunkBlocks) * record_bytes(a.h_fmt);
                reinterpret_cast<float*>(record + kRecordScales)[b % kChunkBlocks] = 0.0f;
                if (a.h_fmt == kQ4_1)
                    for (int odd = 0; odd < 2; ++odd)
                        *reinterpret_cast<float2*>(record + block_sums(b % kChunkBlocks, odd)) = make_float2(0.0f, 0.0f);
            }
            __syncthreads();
#pragma unroll 8
            for (int p = threadIdx.x; p < a.pairs; p += 256) {
                const int e = a.ids[p];
                const bool is = e >= 0 && e < a.n_experts;
                s_ids[p] = (short)(is ? e : -1);
                if (is) atomicAdd(&cnt[e], 1);
            }
            __syncthreads();
            // each thread: 4 consecutive experts; exclusive sums of pairs and of segments
            constexpr int kPer = MLQ_MOE_MAX_EXPERTS / 256;
            int n[kPer], np = 0, ns = 0;
            for (int i = 0; i < kPer; ++i) {
                const int e = threadIdx.x * kPer + i;
                n[i] = e < a.n_experts ? cnt[e] : 0;
                np += (n[i] + align - 1) / align * align;
                ns += (n[i] + a.seg_cap - 1) / a.seg_cap;
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
                // many rows: segments of one length, not a full one and a rest
                const int parts = (n[i] + a.seg_cap - 1) / a.seg_cap;
                const int each = a.positions && parts ? ((n[i] + parts - 1) / parts + 15) / 16 * 16 : a.seg_cap;
                for (int k = 0; k < parts; ++k)
                    a.segs[os++] = Segment{e, op + k * each, min(n[i] - k * each, each), 0};
                op += (n[i] + align - 1) / align * align;
            }
            if (threadIdx.x == 255) *a.nseg = os;
            __syncthreads();
            // pairs of an expert in their order (which segment a pair joins, and so how its sums round, must not
            // change from run to run): 256 at a time, ranked within the warp, then over the warps before it
            for (int e = threadIdx.x; e < 8 * a.n_experts; e += 256) in_warp[e / a.n_experts][e % a.n_experts] = 0;
            __syncthreads();
            for (int p0 = 0; p0 < a.pairs; p0 += 256) {
                const int p = p0 + threadIdx.x;
                const int e = p < a.pairs ? s_ids[p] : -1;
                const unsigned same = __match_any_sync(0xffffffffu, e);
                const int rank = __popc(same & ((1u << lane) - 1));
                if (e >= 0 && rank == 0) in_warp[warp][e] = (unsigned char)__popc(same);
                __syncthreads();
                if (e >= 0) {
                    int at = cnt[e] + rank;
                    for (int w = 0; w < warp; ++w) at += in_warp[w][e];
                    a.order[at] = p;
                    if (a.place) a.place[p] = at;
                } else if (a.place && p < a.pairs) {
                    a.place[p] = -1;
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
        uint8_t* row = a.sliced + (size_t)r * (a.bprp / kChunkBlocks) * record_bytes(a.fmt);
        const int at = b * kQK + imma_element(a.fmt, b & 1, lane);
        slice_digits(at < a.in ? x[at] : 0.0f, a.fmt, row, b, lane);
    }
}

struct HalvesArgs {
    const float* x;
    const int* place;  // [rows][top_k] positions of a row's pairs, -1: none; null: rows are positions
    int rows, positions, top_k, in, groups, fmt;
    uint8_t* halves;   // [position][groups][hi, lo][64]
    float* scales;     // [groups][pitch]
    int pitch;
    unsigned int* split_done;
};

// x by position for many rows: a warp per 64 values, sliced once for all of
// the row's experts.
__global__ void __launch_bounds__(256) halves_kernel(const HalvesArgs a) {
    launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < 2 * kMaxTeams; i += 256) a.split_done[i] = 0;
    const long long n = (long long)a.rows * a.groups, step = (long long)gridDim.x * 8;
    for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += step) {
        const int r = (int)(i / a.groups), g = (int)(i % a.groups);
        const float* x = a.x + (long long)r * a.in;
        float v[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int p = 2 * lane + k, at = 64 * g + (p & 32) + tile_element(a.fmt, p & 31);
            v[k] = at < a.in ? x[at] : 0.0f;
        }
        const Sliced64 s = slice_64(v[0], v[1]);
        if (!a.place) {
            s.store(a.halves + (size_t)i * 256, a.scales + (size_t)g * a.pitch + r, lane);
            continue;
        }
        for (int j = 0; j < a.top_k; ++j) {
            const int pos = a.place[r * a.top_k + j];
            if (pos >= 0) s.store(a.halves + ((size_t)pos * a.groups + g) * 256, a.scales + (size_t)g * a.pitch + pos, lane);
        }
    }
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// About how many rounds the busiest team has (see Deal): `units` of `per`
// rounds, each with an end that takes `end` rounds' time.
double deal_cost(long long units, long long per, double end, int teams) {
    const long long each = units / teams, rest = units % teams;
    double c = each * (per + end);
    if (rest) {
        const double split = (double)((rest * per + teams - 1) / teams) + 4;
        c += end + (split < per ? split : per);
    }
    return c;
}

// 16-row strips of a unit (at least `least`): the K axis is then split in 8 /
// strips parts.  all_segs: a unit meets every segment.
int choose_strips(int out, int bpr, int nseg, bool all_segs, int sm_count, int least, double* cost = nullptr) {
    const int steps = (bpr + kChunkBlocks - 1) / kChunkBlocks;
    int best = kImmaWarps;
    double best_cost = 1e300;
    for (int n = kImmaWarps; n >= least; n /= 2) {
        const int kws = kImmaWarps / n;
        const long long per = (steps + kws - 1) / kws, tiles = (out + 16 * n - 1) / (16 * n);
        const double c = all_segs ? deal_cost(tiles, per * nseg, 0.5 * nseg + 0.5, 2 * sm_count)
                                  : deal_cost(tiles * nseg, per, 0.7, 2 * sm_count);
        if (c < best_cost) best_cost = c, best = n;
    }
    if (cost) *cost = best_cost;
    return best;
}

// Rows of x of a segment of a linear that goes by digits: 2 while that ends sooner by the count of rounds, mostly for
// small matrices (4 rows of q4_0, 2048 x 2048: 8.1 us with one segment and 5.6 with two; 4096 x 4096: 14.0 and 8.4).
int linear_cap(int rows, int out, int bpr, int sm_count) {
    if (rows < 3) return rows;
    double two, four;
    choose_strips(out, bpr, (rows + 1) / 2, false, sm_count, 2, &two);
    choose_strips(out, bpr, (rows + kFewRows - 1) / kFewRows, false, sm_count, kFewRows, &four);
    return two < four ? 2 : kFewRows;
}

struct Carve {
    uint8_t* p;
    template <class T>
    T* take(size_t n) {
        T* r = reinterpret_cast<T*>(p);
        p += align256(n * sizeof(T));
        return r;
    }
    uint8_t* take_sliced(size_t rows, int bprp, int fmt) {
        return take<uint8_t>(rows * (bprp / kChunkBlocks) * record_bytes(fmt));
    }
    // Whether what was taken lies within `bytes` bytes from `ws` on.
    bool within(const void* ws, size_t bytes) const { return (size_t)(p - static_cast<const uint8_t*>(ws)) <= bytes; }
};

size_t sliced_bytes(size_t rows, int bprp, int fmt) { return align256(rows * (bprp / kChunkBlocks) * record_bytes(fmt)); }

constexpr size_t kMaxSliced = 1u << 30;   // sliced bytes of one pass at most (offsets are 32 bits)
constexpr size_t kMaxParts = 1u << 30;    // bytes of the pairs' outputs of one pass at most
constexpr int kMaxPassRows = 16384;       // rows of one pass of a linear at most
// Rows of a linear that go by digits, in segments of 4 whose weights come from L2 after the first.  3584 x 18944, us by
// digits and by halves: q4_0 5 rows 26 and 38, 12 rows 35 and 40, 16 rows 42 and 41; q8_0 31 and 40, 40 and 43, 50 and 45.
constexpr int kLinearFewRows = 12;
constexpr int kCombineRows = 32;          // more rows: the sum over slots is a launch of its own

// Rows of x of a segment at most in the form of few rows.  A stage holds 8
// records of x, so a unit of fewer rows may have its K axis split further: with about a
// row per expert, 2 (an expert with more has several segments).
int few_cap(int rows, int pairs, int n_experts) { return rows < 3 ? rows : pairs <= n_experts ? 2 : kFewRows; }

// And in that of many: half as many again as an expert has on average, so
// that most experts are one segment.
constexpr int kManyCapStep = 32;
int many_cap(int pairs, int n_experts) {
    const int n = (pairs / n_experts * 3 / 2 + 8 + kManyCapStep - 1) / kManyCapStep * kManyCapStep;
    return n < kSegTokens ? n : kSegTokens;
}

// Positions of `pairs` pairs when every expert starts at a multiple of 8.
int many_positions(int pairs, int n_experts) { return (pairs + 7 * (pairs < n_experts ? pairs : n_experts) + 7) / 8 * 8; }

int groups_of(int in) { return (in + 63) / 64; }

// A copy of up to 128 scales may start at the last position.
int scale_pitch(int positions) { return (positions + 7) / 8 * 8 + kSegTokens; }

size_t halves_bytes(int positions, int groups) {
    return align256((size_t)positions * groups * 256) + align256((size_t)groups * scale_pitch(positions) * sizeof(float));
}

// Floats of a slot for a shared unit's sums: rows of x x rows of the tile.  n:
// rows of the call (a unit of few rows that meets every segment has them all).
size_t split_floats(bool few, int n, int strips) {
    if (!few) return (size_t)kSegTokens * 128;
    return (size_t)(n <= kCombineRows && n > kFewRows ? n : kFewRows) * 16 * strips;
}

// Two slots per team at most, and the counters of two launches.
size_t split_count(bool few) { return few ? 2 * kMaxTeams : kMaxTeams; }
size_t split_bytes(bool few, int n) {
    return align256(split_floats(few, n, kImmaWarps) * split_count(few) * sizeof(float)) +
           align256(2 * kMaxTeams * sizeof(unsigned int));
}

// Rows of x of one pass.
int experts_pass_rows(const MoeShape& s, int rows, int top_k) {
    long long n = kMaxPairs / top_k;
    // many rows: x too is by pair
    const long long per = (long long)top_k * padded_blocks((s.hidden + kQK - 1) / kQK) * (kSlicedBytes + 8);
    const long long perx = (long long)top_k * padded_blocks((s.in + kQK - 1) / kQK) * (kSlicedBytes + 8);
    const long long cap = (long long)kMaxSliced / (per > perx ? per : perx);
    const long long capp = (long long)kMaxParts / ((long long)top_k * s.out * (long long)sizeof(float));
    if (n > cap) n = cap;
    if (n > capp) n = capp;
    if (n < 1) n = 1;
    return rows < n ? rows : (int)n;
}

int linear_pass_rows(int in, int rows) {
    long long n = (long long)kMaxSliced / ((long long)padded_blocks((in + kQK - 1) / kQK) * (kSlicedBytes + 8));
    if (n > kMaxPassRows) n = kMaxPassRows;
    return rows < n ? rows : (int)n;
}

int max_segments(int pairs, int n_experts, int cap) {
    const int full = pairs / cap + (pairs < n_experts ? pairs : n_experts);
    return full < pairs ? full : pairs;
}

// Places in the segment list: as many as the form's smallest cap gives.  The
// cap in use grows with the rows, and a list of just its segments would get shorter
// where it does: a pass of fewer rows would then need more than a full one.
int segment_places(bool few, int pairs, int n_experts) {
    return max_segments(pairs, n_experts, few ? 1 : kManyCapStep);
}

// Whether a call's rows of x go by digits, in segments of at most 4: an
// expert with more rows has several segments, whose weights come from L2 after the
// first, so the time grows with the rows, while that of the other form hardly does below
// 16 rows per expert.  60 experts of 3584 x 2560, us by digits and by halves: q4_0 6 rows
// per expert 386 and 701, 10 rows 588 and 704, 11 rows 639 and 705, 12 rows 689 and 706; q8_0 447 and
// 708, 664 and 713, 727 and 715, 774 and 721; q4_1 453 and 987, 691 and 991, 750 and 991, 811 and 991, and 14
// rows 920 and 993.  One border for all: q8_0's own is 10 rows, q4_0's 12, q4_1's 14 (whose calls of
// 12 to 14 rows take up to a fifth longer than they need).  The ids are on the device, so the average decides: where
// most rows go to few experts, those are unpacked again for each 4 rows although their number would call for the other form.
constexpr int kFewPerExpert = 11;
bool few_rows(int pairs, int n_experts) { return pairs <= kFewPerExpert * n_experts; }

int prep_ctas(long long blocks, int sm_count) {
    const long long n = (blocks + 7) / 8;
    return (int)(n < 8LL * sm_count ? n : 8LL * sm_count);
}

// `rows` rows of x (null: made by a product) as halves in `positions` places.
HalvesArgs halves_args(Carve& c, const float* x, int rows, int positions, int in, int fmt) {
    HalvesArgs h{};
    h.x = x, h.rows = rows, h.positions = positions, h.in = in, h.fmt = fmt;
    h.groups = groups_of(in), h.pitch = scale_pitch(positions);
    h.halves = c.take<uint8_t>((size_t)positions * h.groups * 256);
    h.scales = c.take<float>((size_t)h.groups * h.pitch);
    return h;
}

void set_halves(ImmaArgs& a, const HalvesArgs& h) {
    a.x = h.halves, a.xs = h.scales, a.xs_pitch = h.pitch, a.x_rows = h.positions, a.groups = h.groups;
}

}  // namespace

size_t epilogue_workspace_bytes(int fmt, int in, int rows) {
    const int n = linear_pass_rows(in, rows);
    // more rows never need less
    const int few_rows = n < kLinearFewRows ? n : kLinearFewRows;
    const size_t few = sliced_bytes(few_rows, padded_blocks((in + kQK - 1) / kQK), fmt) + split_bytes(true, few_rows);
    const size_t many = n <= kLinearFewRows ? 0 : halves_bytes(n, groups_of(in)) + split_bytes(false, n);
    return few > many ? few : many;
}

cudaError_t launch_linear_epilogue(int fmt, const uint8_t* w, int out, int in, const float* x, int rows,
                                   const mlq_epilogue& ep, float* y, void* ws, size_t ws_bytes, int sm_count,
                                   int smem_per_sm, int* err, cudaStream_t stream) {
    const int bpr = (in + kQK - 1) / kQK, bprp = padded_blocks(bpr);
    const int pass = linear_pass_rows(in, rows);
    for (int r0 = 0; r0 < rows;) {
        const int n = rows - r0 < pass ? rows - r0 : pass;
        Carve c{static_cast<uint8_t*>(ws)};
        PrepArgs p{};
        p.x = x + (long long)r0 * in;
        p.rows = n, p.in = in, p.bpr = bpr, p.bprp = bprp, p.fmt = fmt;
        const bool few = n <= kLinearFewRows;
        HalvesArgs hv{};
        if (few)
            p.sliced = c.take_sliced(n, bprp, fmt);
        else
            hv = halves_args(c, p.x, n, n, in, fmt);
        float* split = c.take<float>(split_floats(few, n, kImmaWarps) * split_count(few));
        p.split_done = hv.split_done = c.take<unsigned int>(2 * kMaxTeams);
        if (!c.within(ws, ws_bytes)) return cudaErrorInvalidValue;
        cudaError_t e = few ? launch_pdl(prep_kernel, prep_ctas((long long)n * bprp, sm_count), 256, 0, stream, p)
                            : launch_pdl(halves_kernel, prep_ctas((long long)n * hv.groups, sm_count), 256, 0, stream, hv);
        if (e != cudaSuccess) return e;
        ImmaArgs a{};
        a.w[0] = w;
        a.total_rows = out, a.out = out, a.bpr = bpr, a.bprp = bprp;
        const int parts = (n + kSegTokens - 1) / kSegTokens;
        a.seg_cap = few ? linear_cap(n, out, bpr, sm_count) : ((n + parts - 1) / parts + 15) / 16 * 16;
        const int nseg = (n + a.seg_cap - 1) / a.seg_cap;
        a.strips = few ? choose_strips(out, bpr, nseg, false, sm_count, a.seg_cap) : 8;
        a.tiles = (out + 16 * a.strips - 1) / (16 * a.strips);
        if (few)
            a.x = p.sliced;
        else
            set_halves(a, hv);
        a.rows = n;
        a.split = split, a.split_done = p.split_done, a.split_size = split_floats(few, n, a.strips);
        a.bias = ep.bias;
        a.row_scale = ep.row_scale ? ep.row_scale + r0 : nullptr;
        a.residual = ep.residual ? ep.residual + (long long)r0 * out : nullptr;
        a.act = ep.activation;
        a.y = y + (long long)r0 * out;
        a.err = err;
        e = (few ? launch_few_plain : launch_many_plain)(fmt, a, sm_count, smem_per_sm, (long long)nseg * a.tiles, stream);
        if (e != cudaSuccess) return e;
        r0 += n;
    }
    return cudaSuccess;
}

size_t experts_workspace_bytes(const MoeShape& s, int rows, int top_k) {
    const int pass = experts_pass_rows(s, rows, top_k);
    const int bprp = padded_blocks((s.in + kQK - 1) / kQK), hp = padded_blocks((s.hidden + kQK - 1) / kQK);
    auto bytes = [&](int n) {
        const int pairs = n * top_k;
        const bool few = few_rows(pairs, s.n_experts);
        const size_t lists = 256 + align256((size_t)segment_places(few, pairs, s.n_experts) * sizeof(Segment));
        if (few)
            return lists + align256((size_t)pairs * sizeof(int)) + sliced_bytes(n, bprp, s.fmt) +
                   sliced_bytes(pairs, hp, s.fmt_down) +
                   (n <= kCombineRows ? 0 : align256((size_t)pairs * s.out * sizeof(float))) + split_bytes(few, n);
        const int positions = many_positions(pairs, s.n_experts);
        return lists + align256((size_t)positions * sizeof(int)) + align256((size_t)pairs * sizeof(int)) +
               halves_bytes(positions, groups_of(s.in)) + halves_bytes(positions, groups_of(s.hidden)) +
               align256((size_t)pairs * s.out * sizeof(float)) +
               split_bytes(few, n);
    };
    // never less than for fewer rows (the last pass is one of those): within a form, and on either side of kCombineRows,
    // every array grows with the rows, so the most is at one of these
    size_t most = 0;
    for (const long long n : {(long long)pass, (long long)kCombineRows, (long long)kFewPerExpert * s.n_experts / top_k})
        if (n >= 1 && n <= pass) {
            const size_t b = bytes((int)n);
            if (b > most) most = b;
        }
    return most;
}

cudaError_t launch_experts(const MoeShape& s, const uint8_t* gate, const uint8_t* up, const uint8_t* down,
                           const float* x, int rows, int top_k, const int32_t* ids, const float* weights,
                           const float* residual, float* y, void* ws, size_t ws_bytes, int sm_count, int smem_per_sm,
                           int* err, cudaStream_t stream) {
    const int pass = experts_pass_rows(s, rows, top_k);
    const int bpr = (s.in + kQK - 1) / kQK, bprp = padded_blocks(bpr);
    const int hb = (s.hidden + kQK - 1) / kQK, hp = padded_blocks(hb);
    for (int r0 = 0; r0 < rows; r0 += pass) {
        const int n = rows - r0 < pass ? rows - r0 : pass, pairs = n * top_k;
        const bool few = few_rows(pairs, s.n_experts);
        const int cap = few ? few_cap(n, pairs, s.n_experts) : many_cap(pairs, s.n_experts);
        const bool at_once = few && n <= kCombineRows;  // the down product meets all segments of a tile in one unit
        const int nseg_max = max_segments(pairs, s.n_experts, cap);
        const int nseg_likely = pairs < s.n_experts ? pairs : nseg_max;
        const int strips = few ? choose_strips(s.out, hb, nseg_likely, at_once, sm_count, cap) : 8;
        const int tiles = (s.out + 16 * strips - 1) / (16 * strips);
        Carve c{static_cast<uint8_t*>(ws)};
        PrepArgs p{};
        HalvesArgs hx{}, hh{};
        p.nseg = c.take<int>(1);
        p.segs = c.take<Segment>(segment_places(few, pairs, s.n_experts));
        p.positions = few ? 0 : many_positions(pairs, s.n_experts);
        p.order = c.take<int>(few ? pairs : p.positions);
        p.x = x + (long long)r0 * s.in;
        p.in = s.in, p.bpr = bpr, p.bprp = bprp, p.fmt = s.fmt;
        p.seg_cap = cap;
        p.ids = ids + (long long)r0 * top_k;
        p.pairs = pairs, p.n_experts = s.n_experts;
        if (few) {
            p.rows = n;
            p.sliced = c.take_sliced(n, bprp, s.fmt);
            p.h = c.take_sliced(pairs, hp, s.fmt_down);
            p.h_bpr = hb, p.h_bprp = hp, p.h_fmt = s.fmt_down;
        } else {
            p.place = c.take<int>(pairs);
            hx = halves_args(c, p.x, n, p.positions, s.in, s.fmt);
            hh = halves_args(c, nullptr, n, p.positions, s.hidden, s.fmt_down);
            hx.place = p.place, hx.top_k = top_k;
        }
        float* part = c.take<float>(at_once ? 0 : (size_t)pairs * s.out);
        float* split = c.take<float>(split_floats(few, n, kImmaWarps) * split_count(few));
        p.split_done = hx.split_done = c.take<unsigned int>(2 * kMaxTeams);
        if (!c.within(ws, ws_bytes)) return cudaErrorInvalidValue;
        cudaError_t e = launch_pdl(prep_kernel, few ? 1 + prep_ctas((long long)n * bprp, sm_count) : 1, 256, 0, stream, p);
        if (e == cudaSuccess && !few)
            e = launch_pdl(halves_kernel, prep_ctas((long long)n * hx.groups, sm_count), 256, 0, stream, hx);
        if (e != cudaSuccess) return e;

        ImmaArgs a{};
        a.w[0] = gate, a.w[1] = up;
        a.total_rows = (long long)s.n_experts * s.hidden;
        a.out = s.hidden, a.bpr = bpr, a.bprp = bprp;
        a.strips = few ? choose_strips(2 * s.hidden, bpr, nseg_likely, false, sm_count, 4) : 8;
        a.tiles = (s.hidden + 8 * a.strips - 1) / (8 * a.strips);
        a.seg_cap = cap;
        a.x = p.sliced;
        if (!few) set_halves(a, hx);
        a.segs = p.segs, a.nseg = p.nseg, a.order = p.order;
        a.top_k = top_k, a.rows = n;
        a.next_fmt = s.fmt_down, a.next_bprp = hp;
        a.h = few ? p.h : hh.halves;
        a.hs = hh.scales, a.hs_pitch = hh.pitch, a.next_groups = hh.groups;
        a.split = split, a.split_done = p.split_done, a.split_size = split_floats(few, n, a.strips);
        a.err = err;
        e = (few ? launch_few_pair : launch_many_pair)(s.fmt, a, sm_count, smem_per_sm, (long long)nseg_max * a.tiles, stream);
        if (e != cudaSuccess) return e;

        ImmaArgs d{};
        d.w[0] = down;
        d.total_rows = (long long)s.n_experts * s.out;
        d.out = s.out, d.bpr = hb, d.bprp = hp;
        d.strips = strips, d.tiles = tiles;
        d.seg_cap = cap;
        d.x = p.h;
        if (!few) set_halves(d, hh);
        d.segs = p.segs, d.nseg = p.nseg, d.order = p.order;
        d.top_k = top_k, d.rows = n;
        d.part = at_once ? nullptr : part;
        d.split = split, d.split_done = p.split_done + kMaxTeams;
        d.split_size = split_floats(few, n, strips);
        d.ids = p.ids;
        d.weights = weights + (long long)r0 * top_k;
        d.n_experts = s.n_experts;
        d.residual = residual ? residual + (long long)r0 * s.out : nullptr;
        d.y = y + (long long)r0 * s.out;
        d.err = err;
        e = (few ? launch_few_down : launch_many_down)(s.fmt_down, d, sm_count, smem_per_sm, (long long)nseg_max * tiles, stream);
        if (e != cudaSuccess) return e;
        if (d.part) {
            const bool four = s.out % 4 == 0 && reinterpret_cast<uintptr_t>(d.y) % 16 == 0 &&
                              reinterpret_cast<uintptr_t>(d.residual) % 16 == 0;
            const long long ctas = ((long long)n * s.out / (four ? 4 : 1) + 255) / 256;
            e = launch_pdl(four ? combine_kernel<4> : combine_kernel<1>, (int)(ctas < 16 * sm_count ? ctas : 16 * sm_count),
                           256, 0, stream, d);
            if (e != cudaSuccess) return e;
        }
    }
    return cudaSuccess;
}

}  // namespace mlq
