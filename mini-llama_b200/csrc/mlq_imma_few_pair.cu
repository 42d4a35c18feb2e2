// mlq_imma_few_pair.cu -- the few-rows kernel's gate and up products (a file
// of its own so that the forms compile side by side).
#include "mlq_imma_few.cuh"

namespace mlq {

MLQ_IMMA_LAUNCH(launch_few_pair) { return launch_few<kPair>(fmt, a, sm_count, smem_per_sm, max_units, stream); }

}  // namespace mlq
