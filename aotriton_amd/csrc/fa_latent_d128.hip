// Attention over keys that are part per head, part shared: K and V of 65 to 128 columns (fp16 and bf16).
#include "fa_kernels.h"
#include "fa_latent.h"

namespace fa {
hipError_t run_latent_fwd_d128(int dtype, const LatentArgs& a, hipStream_t s) {
  return dtype == kDtypeBF16 ? launch_latent_fwd<bf16_t, 128>(a, s) : launch_latent_fwd<f16_t, 128>(a, s);
}
hipError_t run_latent_bwd_d128(int dtype, const LatentBwdArgs& a, hipStream_t s) {
  const hipError_t e = a.alone ? run_latent_dq_alone_d128(dtype, a, s) : dtype == kDtypeBF16 ? launch_latent_dq<bf16_t, 128>(a, s) : launch_latent_dq<f16_t, 128>(a, s);
  return e != hipSuccess ? e : run_latent_keys_d128(dtype, a, s);
}
}  // namespace fa
