// mlq_imma_args.cuh -- what the launches of mlq_imma.cu share.
#pragma once

#include "mlq_imma.cuh"

namespace mlq {

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
    int strips;               // 16-row strips of a unit (1, 2, 4 or 8); kPair: 8 gate and 8 up rows each, 4 or 8
    int tiles;                // row tiles of one matrix
    int slots;                // ring depth of a warp (many rows: of the CTA)
    int x_slots;              // many rows: ring depth of x
    int seg_cap;              // rows of x of a segment at most
    const uint8_t* x;         // records of the rows of x or h; many rows: [x_rows][groups][hi, lo][64] fp16, by position
    // many rows
    const float* xs;          // [groups][xs_pitch] scales of x
    int xs_pitch, x_rows, groups;
    float* hs;                // kPair: [next_groups][hs_pitch] scales of h
    int hs_pitch, next_groups;
    // segments (kPair, kDown); kPlain: rows in order, one matrix
    const Segment* segs;
    const int* nseg;
    const int* order;         // expert-sorted position -> pair
    int top_k, rows;
    // kPair: sliced h by position
    int next_fmt, next_bprp;
    uint8_t* h;
    // kDown: one value per pair for a later launch to sum; null: a unit meets every segment and is summed at once
    float* part;              // [pair][out]
    const int32_t* ids;
    const float* weights;
    int n_experts;
    // units that several teams share
    float* split;             // [team][head, tail][split_size]: row of x, row of the tile
    unsigned int* split_done; // per team, zero before the launch
    size_t split_size;
    // kPlain / kDown
    const float* bias;
    const float* row_scale;
    const float* residual;
    float* y;
    int act;
    int* err;
};

constexpr int kMaxTeams = 320;  // teams of a launch at most (split slots)

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

template <typename... Params, typename... Args>
inline cudaError_t launch_pdl(void (*kernel)(Params...), int grid, int block, size_t smem, cudaStream_t stream,
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

// One streaming launch (mlq_imma_{few,many}_{plain,pair,down}.cu).
// max_units: an upper bound of its units.
#define MLQ_IMMA_LAUNCH(name)                                                                                    \
    cudaError_t name(int fmt, const ImmaArgs& a, int sm_count, int smem_per_sm, long long max_units, cudaStream_t stream)
MLQ_IMMA_LAUNCH(launch_few_plain);
MLQ_IMMA_LAUNCH(launch_few_pair);
MLQ_IMMA_LAUNCH(launch_few_down);
MLQ_IMMA_LAUNCH(launch_many_plain);
MLQ_IMMA_LAUNCH(launch_many_pair);
MLQ_IMMA_LAUNCH(launch_many_down);

}  // namespace mlq
