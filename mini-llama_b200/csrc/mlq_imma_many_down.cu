// mlq_imma_many_down.cu -- the many-rows kernel's down products (a file
// of its own so that the forms compile side by side).
#include "mlq_imma_many.cuh"

namespace mlq {

MLQ_IMMA_LAUNCH(launch_many_down) { return launch_many<kDown>(fmt, a, sm_count, smem_per_sm, max_units, stream); }

}  // namespace mlq
