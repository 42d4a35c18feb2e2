// mlq_imma_few_plain.cu -- the few-rows kernel's linear with an epilogue (a file
// of its own so that the forms compile side by side).
#include "mlq_imma_few.cuh"

namespace mlq {

MLQ_IMMA_LAUNCH(launch_few_plain) { return launch_few<kPlain>(fmt, a, sm_count, smem_per_sm, max_units, stream); }

}  // namespace mlq
