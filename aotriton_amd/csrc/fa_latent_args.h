// Argument blocks of the kernels for keys and values that come from one latent vector a token, and their launchers: attention over keys
// that are part per head, part shared (fa_latent.h), attention over a cache of the latent rows (fa_latent_cache.h).
#pragma once
#include <hip/hip_runtime.h>

#include "fa_args.h"
#include "fa_cache_args.h"

namespace fa {

struct LatentArgs {
  const void* q; const void* k; const void* v; const void* c;      // c: the keys' shared part, (batch, rows, r)
  void* out; float* lse;                                           // lse: may be null
  Strides3 sq, sk, sv, so;
  int64_t c_z, c_s;
  int32_t batch, heads;
  int32_t e, r, ev;              // columns of K, of the shared part, of V
  float sm_scale;
  int32_t causal;                // query i sees keys up to i + Sk - Sq
  SeqArgs seq;
  int32_t rows_q, rows_k;        // of the tensors: packed offsets are held inside them
  int32_t group;                 // fa_latent.h: latent_item
  // The keys of a tile cut into `parts` (> 1), for calls with few queries: the parts' sums, side by side for every slab of 32 rows.  A batch's
  // head has `slabs` of them (fa_latent.h: latent_slab).
  int32_t parts, slabs;
  float* part_o; float* part_ml;
};

struct LatentBwdArgs : LatentArgs {
  const void* dout;
  void* dq; void* dk; void* dv; void* dc;
  Strides3 sdo, sdq, sdk, sdv;
  int64_t dc_z, dc_s;
  // Written by the dQ kernel for the dK/dV kernel, one value for every row as in lse: L / ln 2, and delta = rowsum(dO O).
  float* stat_lse; float* stat_delta;
  // Every head's sum for the shared part, fp32 (sequence or batch and head, key, 64 columns): summed over the heads by a launch of its own.
  float* part_c;
  int64_t part_rows;             // keys of a (batch, head) slab of part_c
  bool alone;                    // dQ in its form for few workgroups (fa_latent_keys.h)
};

// A block of rows that lies in several pieces: the first of them (two times its worker, plus its place there), how many (0: the block is one
// piece), first row of the sequence, number in it, rows of it.
struct LatentHead { int32_t piece, pieces, start, block, rows; };

// Attention over a cache of latent rows (CacheArgs: K is the cache, of one head; head_dim_v of its columns are the values).
struct LatentCacheArgs {
  const void* q; void* out; float* lse;
  int64_t q_row, q_head, o_row, o_head;
  CacheArgs cache;
  const int32_t* starts;
  int32_t rows, hq;              // packed tokens of all sequences
  float sm_scale;
  // Work, in tiles of 32 slots for block_rows packed (token, head) rows of a sequence.  The list of all sequences' tiles is cut into
  // `workers` equal pieces of at least `least`, one for a workgroup; the sums of a block that lies in several pieces go to
  // part_o, two places for every worker.
  int32_t block_rows, workers, least;
  int32_t margin;                // tiles that a block's beginning and its end take each (fa_latent_list.h: LatentSeq::units); negative: blocks stay whole
  int32_t block_shift;           // block_rows as a power of two; so, rounded, blocks that 32 tokens make (one at least), and tiles that a group's tokens make
  int32_t group_shift, step_shift;
  float* part_o; float* part_ml;
  LatentHead* heads;             // of the blocks, `blocks` of them (fa_latent_cache.h: latent_block)
  int32_t blocks;
};

// compiled columns of K and V (64 or 128; of the shared part 64)
hipError_t run_latent_fwd_d64(int dtype, const LatentArgs& a, hipStream_t s);
hipError_t run_latent_fwd_d128(int dtype, const LatentArgs& a, hipStream_t s);
hipError_t run_latent_bwd_d64(int dtype, const LatentBwdArgs& a, hipStream_t s);
hipError_t run_latent_bwd_d128(int dtype, const LatentBwdArgs& a, hipStream_t s);
hipError_t run_latent_dq_alone_d64(int dtype, const LatentBwdArgs& a, hipStream_t s);
hipError_t run_latent_dq_alone_d128(int dtype, const LatentBwdArgs& a, hipStream_t s);
hipError_t run_latent_keys_d64(int dtype, const LatentBwdArgs& a, hipStream_t s);      // dK, dV and dC, behind dQ
hipError_t run_latent_keys_d128(int dtype, const LatentBwdArgs& a, hipStream_t s);
// compiled columns in front of the last 64 (256 or 512)
hipError_t run_latent_cache_d256(int dtype, const LatentCacheArgs& a, hipStream_t s);
hipError_t run_latent_cache_d512(int dtype, const LatentCacheArgs& a, hipStream_t s);
hipError_t run_latent_cache_d512_full(int dtype, const LatentCacheArgs& a, hipStream_t s);      // blocks of 128 rows

}  // namespace fa
