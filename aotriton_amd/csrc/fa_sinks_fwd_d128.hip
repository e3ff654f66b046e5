// Forward kernels of attention with a window and sinks, head dim 128 (fp16 and bf16).
#include "fa_sinks.h"

// Compiled three times, as the other per-head-dim files: FA_PADDED = the columns to compute for smaller head dims.
#ifndef FA_PADDED
#define FA_PADDED 0
#endif
#if FA_PADDED == 96
#define FA_RUN run_sinks_fwd_d128_cols96
#elif FA_PADDED
#define FA_RUN run_sinks_fwd_d128_padded
#else
#define FA_RUN run_sinks_fwd_d128
#endif

namespace fa {
hipError_t FA_RUN(int dtype, const SinkFwdArgs& a, hipStream_t s) {
  if (dtype == kDtypeBF16) return launch_fwd_sinks<bf16_t, 128, FA_PADDED>(a, s);
  return launch_fwd_sinks<f16_t, 128, FA_PADDED>(a, s);
}
}  // namespace fa
