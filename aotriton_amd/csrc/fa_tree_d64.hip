// Attention of drafted tokens over a cache of pages, head dim 64 (fp16 and bf16).
#include "fa_cache.h"
#include "fa_kernels.h"

// Compiled twice, as the other per-head-dim files: FA_PADDED=64 for smaller head dims (a multiple of 8).
#ifndef FA_PADDED
#define FA_PADDED 0
#endif
#if FA_PADDED
#define FA_RUN run_tree_d64_padded
#else
#define FA_RUN run_tree_d64
#endif

namespace fa {
hipError_t FA_RUN(int dtype, const TreeArgs& a, hipStream_t s) {
  if (dtype == kDtypeBF16) return launch_tree<bf16_t, 64, FA_PADDED != 0>(a, s);
  return launch_tree<f16_t, 64, FA_PADDED != 0>(a, s);
}
}  // namespace fa
