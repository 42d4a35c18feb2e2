// mlq_imma_few_down.cu -- the few-rows kernel's down products (a file
// of its own so that the forms compile side by side).
#include "mlq_imma_few.cuh"

namespace mlq {

MLQ_IMMA_LAUNCH(launch_few_down) { return launch_few<kDown>(fmt, a, sm_count, smem_per_sm, max_units, stream); }

}  // namespace mlq
