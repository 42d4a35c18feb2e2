// mlq_imma_plain.cu -- the streaming kernel's linear with an epilogue (a file of its
// own so that the three forms compile side by side).
#include "mlq_imma_kernel.cuh"

namespace mlq {

cudaError_t launch_imma_plain(int fmt, const ImmaArgs& a, int sm_count, int smem_per_sm, long long max_units,
                           cudaStream_t stream) {
    return launch_imma<kPlain>(fmt, a, sm_count, smem_per_sm, max_units, stream);
}

}  // namespace mlq
