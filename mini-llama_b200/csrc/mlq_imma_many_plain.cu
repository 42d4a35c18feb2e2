// mlq_imma_many_plain.cu -- the many-rows kernel's linear with an epilogue (a file
// of its own so that the forms compile side by side).
#include "mlq_imma_many.cuh"

namespace mlq {

MLQ_IMMA_LAUNCH(launch_many_plain) { return launch_many<kPlain>(fmt, a, sm_count, smem_per_sm, max_units, stream); }

}  // namespace mlq
