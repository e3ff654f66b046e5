// Attention over a cache of latent rows, values of up to 512 columns, rows of up to 576 (fp16 and bf16): blocks of 32 rows.
#include "fa_kernels.h"
#include "fa_latent_cache.h"

namespace fa {
hipError_t run_latent_cache_d512(int dtype, const LatentCacheArgs& a, hipStream_t s) {
  if (a.block_rows == 128) return run_latent_cache_d512_full(dtype, a, s);
  return dtype == kDtypeBF16 ? launch_latent_cache_rows<bf16_t, 512, 1>(a, s) : launch_latent_cache_rows<f16_t, 512, 1>(a, s);
}
}  // namespace fa
