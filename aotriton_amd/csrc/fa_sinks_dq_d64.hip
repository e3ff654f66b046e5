// dQ kernels of attention with a window and sinks, head dim 64 (fp16 and bf16).
#include "fa_sinks.h"

// Compiled twice, as the other per-head-dim files: FA_PADDED = the columns to compute for smaller head dims.
#ifndef FA_PADDED
#define FA_PADDED 0
#endif
#if FA_PADDED
#define FA_RUN run_sinks_dq_d64_padded
#else
#define FA_RUN run_sinks_dq_d64
#endif

namespace fa {
hipError_t FA_RUN(int dtype, const SinkBwdArgs& a, hipStream_t s) {
  if (dtype == kDtypeBF16) return launch_dq_variant<bf16_t, 64, FA_PADDED, true, false, false, true>(a, s);
  return launch_dq_variant<f16_t, 64, FA_PADDED, true, false, false, true>(a, s);
}
}  // namespace fa
