/*
 * C ABI of attention whose keys and values come from one latent vector a token: over keys that are part per head and part shared by all
 * heads (training, prompts), and over a cache of pages of the latent rows themselves (serving).  Conventions (views, hipError_t
 * values, asynchronous launches on the caller's stream) as in flash.h, of the cache as in cache.h; no counterpart in the reference.
 *
 * Tensors are fp16 or bf16, any strides with a unit last one, made of aligned 16-byte pieces (columns and strides multiples of 8, 16-byte
 * aligned bases).  Scratch memory comes from `alloc`, nothing else is kept; all of it can be captured into a graph.
 *
 * Errors: FA_ERROR_INVALID_VALUE for null or inconsistent views, FA_ERROR_NOT_SUPPORTED for strides, alignments and sizes that are
 * not built, both before any HIP call; FA_ERROR_NO_BINARY_FOR_GPU off gfx950; FA_ERROR_OUT_OF_MEMORY where a call that needs scratch memory gets none.
 */
#ifndef AOTRITON_AMD_LATENT_H
#define AOTRITON_AMD_LATENT_H

#include "aotriton_amd/cache.h"
#include "aotriton_amd/flash.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The expanded form.  Head h scores query i against key j with
 *   Sm_scale (Q[h, i, :E] . K[h, j] + Q[h, i, E:] . S[j]);
 * with `causal` query i sees keys up to i + Sk - Sq, without it all.  E and Ev up to 128, R up to 64.  A query that sees no key gives 0 and
 * a logsumexp of +inf, and has no gradient.  Packed sequences: batch 1, ascending offsets in cu_seqlens_q and cu_seqlens_k (int32, sequences + 1
 * values on the device), held inside the tensors, and greatest lengths in max_seqlen_q and max_seqlen_k, which a longer sequence is cut to.  Rows that no
 * sequence has (in front of the first offset, past the greatest length, behind the last offset) are neither read nor written (fa_zero_gaps). */
typedef struct fa_latent_fwd_params {
  fa_tensor4 Q;              /* (batch, heads, Sq, E + R) */
  fa_tensor4 K;              /* (batch, heads, Sk, E) */
  fa_tensor4 V;              /* (batch, heads, Sk, Ev) */
  fa_tensor4 S;              /* (batch, 1, Sk, R): the keys' part that all heads share */
  fa_tensor4 Out;            /* (batch, heads, Sq, Ev) */
  fa_tensor2 L;              /* fp32 (batch * heads, Sq); null in the forward: not wanted */
  fa_tensor1 cu_seqlens_q;   /* null: batches of equal lengths */
  fa_tensor1 cu_seqlens_k;
  int32_t max_seqlen_q;      /* packed sequences only */
  int32_t max_seqlen_k;
  float Sm_scale;
  int32_t causal;
} fa_latent_fwd_params;
/* Calls with few queries cut the keys into parts, if they get scratch memory (alloc may be null). */
FA_API int fa_latent_fwd(const fa_latent_fwd_params* params, void* hip_stream, fa_allocator* alloc);

typedef struct fa_latent_bwd_params {
  fa_latent_fwd_params fwd;  /* of the forward, with its results Out and L */
  fa_tensor4 DO;             /* as Out */
  fa_tensor4 DQ, DK, DV, DS; /* as Q, K, V, S */
} fa_latent_bwd_params;
/* Scratch memory: two words for every row and head, and 64 for every key and head, whose sum over the heads is DS.  No atomics: results
 * do not change from call to call. */
FA_API int fa_latent_bwd(const fa_latent_bwd_params* params, void* hip_stream, fa_allocator* alloc);

/* The absorbed form, over a cache of pages of latent rows: a row is the key of all heads, and its first Ev columns are their value.  The
 * new tokens of all sequences are packed: rows [starts[z], starts[z + 1]) of Q are those of sequence z, whose own latent rows lie in the cache
 * already, in the slots behind lengths[z] (fa_cache_append_packed).  Token t of a sequence sees slots up to lengths[z] + t.  Head
 * h scores it with Sm_scale Q[row, h] . slot.  E up to 576, Ev up to 512 and no more than E.  What is not there (a page outside the cache, a
 * slot outside the table) is not seen; rows that see nothing, and rows of no sequence, give 0 and a logsumexp of +inf.  Slots that no token of
 * the call sees may hold anything; what lies in those of its own tokens has to be finite.  max_length bounds the lengths: it
 * decides how finely the slots are cut, and nothing else. */
typedef struct fa_latent_cache_params {
  fa_tensor4 Q;       /* (1, rows, Hq, E) */
  fa_tensor4 Out;     /* (1, rows, Hq, Ev) */
  fa_tensor2 L;       /* fp32 (rows, Hq) or null */
  fa_tensor4 latent;  /* (pages, 1, slots, E) */
  fa_tensor2 table;   /* int32 (sequences, columns) */
  fa_tensor1 lengths; /* int32 (sequences): filled slots, without the new tokens */
  fa_tensor1 starts;  /* int32 (sequences + 1), ascending */
  float Sm_scale;
  int32_t max_length;
} fa_latent_cache_params;
FA_API int fa_latent_cache_attn(const fa_latent_cache_params* params, void* hip_stream, fa_allocator* alloc);

#ifdef __cplusplus
}
#endif
#endif /* AOTRITON_AMD_LATENT_H */
