// Kernels with 64 rows per wave (fa_fwd_wide.h, fa_bwd_wide.h) of attention with a window and sinks, head dims above 64 and up to 128.
#include "fa_bwd_wide.h"
#include "fa_fwd_wide.h"

// Compiled three times, as the other per-head-dim files: FA_PADDED = the columns to compute for smaller head dims.
#ifndef FA_PADDED
#define FA_PADDED 0
#endif
#if FA_PADDED == 96
#define FA_NAME(name) name##_cols96
#elif FA_PADDED
#define FA_NAME(name) name##_padded
#else
#define FA_NAME(name) name
#endif

namespace fa {
hipError_t FA_NAME(run_sinks_fwd_wide_d128)(int dtype, const SinkFwdArgs& a, hipStream_t s) {
  return dtype == kDtypeBF16 ? launch_fwd_wide_sinks<bf16_t, FA_PADDED>(a, s) : launch_fwd_wide_sinks<f16_t, FA_PADDED>(a, s);
}
hipError_t FA_NAME(run_sinks_dkdv_wide_d128)(int dtype, const SinkBwdArgs& a, hipStream_t s) {
  if (dtype == kDtypeBF16) return launch_dkdv_wide<bf16_t, true, FA_PADDED, true>(a, s);
  return launch_dkdv_wide<f16_t, true, FA_PADDED, true>(a, s);
}
hipError_t FA_NAME(run_sinks_dq_wide_d128)(int dtype, const SinkBwdArgs& a, hipStream_t s) {
  if (dtype == kDtypeBF16) return launch_dq_wide<bf16_t, true, FA_PADDED, true>(a, s);
  return launch_dq_wide<f16_t, true, FA_PADDED, true>(a, s);
}
}  // namespace fa
