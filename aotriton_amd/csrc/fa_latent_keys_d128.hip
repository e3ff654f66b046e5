// Gradients of keys that are part per head, part shared: K and V of 65 to 128 columns (fp16 and bf16).
#include "fa_kernels.h"
#include "fa_latent_keys.h"

namespace fa {
hipError_t run_latent_keys_d128(int dtype, const LatentBwdArgs& a, hipStream_t s) {
  return dtype == kDtypeBF16 ? launch_latent_keys<bf16_t, 128>(a, s) : launch_latent_keys<f16_t, 128>(a, s);
}
hipError_t run_latent_dq_alone_d128(int dtype, const LatentBwdArgs& a, hipStream_t s) {
  return dtype == kDtypeBF16 ? launch_latent_dq_alone<bf16_t, 128>(a, s) : launch_latent_dq_alone<f16_t, 128>(a, s);
}
}  // namespace fa
