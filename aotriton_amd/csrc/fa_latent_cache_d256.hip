// Attention over a cache of latent rows, values of up to 256 columns, rows of up to 320 (fp16 and bf16).
#include "fa_kernels.h"
#include "fa_latent_cache.h"

namespace fa {
namespace {
template <typename T> hipError_t launch(const LatentCacheArgs& a, hipStream_t s) {
  switch (a.block_rows) {
    case 32: return launch_latent_cache_rows<T, 256, 1>(a, s);
    case 64: return launch_latent_cache_rows<T, 256, 2>(a, s);
    default: return launch_latent_cache_rows<T, 256, 4>(a, s);
  }
}
}  // namespace
hipError_t run_latent_cache_d256(int dtype, const LatentCacheArgs& a, hipStream_t s) {
  return dtype == kDtypeBF16 ? launch<bf16_t>(a, s) : launch<f16_t>(a, s);
}
}  // namespace fa
