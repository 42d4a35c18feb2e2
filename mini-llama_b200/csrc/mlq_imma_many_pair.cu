// mlq_imma_many_pair.cu -- the many-rows kernel's gate and up products (a file
// of its own so that the forms compile side by side).
#include "mlq_imma_many.cuh"

namespace mlq {

MLQ_IMMA_LAUNCH(launch_many_pair) { return launch_many<kPair>(fmt, a, sm_count, smem_per_sm, max_units, stream); }

}  // namespace mlq
