/*
 * C ABI of the cache of pages: its rows, pages and sequences, and the attention of drafted tokens over it.  Conventions (views,
 * hipError_t values, asynchronous launches on the caller's stream, no device memory of its own) as in flash.h; no counterpart in
 * the reference.
 *
 * A cache is two tensors (pages, heads, slots of a page, head dim) of fp16 or bf16: any strides with a unit last one, made of aligned
 * 16-byte pieces (head dims, up to 256, and strides multiples of 8, 16-byte aligned bases, pages less than 2^31 elements apart), so that (pages, slots, heads, head dim) storage
 * is as good; the slots of a page are a power of two from 16 up.  A sequence is a row of the page table, int32 with -1 where
 * there is no page, and a length: slot n of the sequence is slot n % slots of the page in column n / slots.  All indices are read on the
 * device, and none is trusted: pages outside the cache, sequences outside the table, slots outside a row of the table are not
 * read and not written (what would have stood there is not there); a negative length is a sequence that is not there.
 *
 * Errors: FA_ERROR_INVALID_VALUE for null or inconsistent views, FA_ERROR_NOT_SUPPORTED for strides, alignments and sizes that are
 * not built, both before any HIP call; FA_ERROR_NO_BINARY_FOR_GPU off gfx950.
 */
#ifndef AOTRITON_AMD_CACHE_H
#define AOTRITON_AMD_CACHE_H

#include "aotriton_amd/flash.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct fa_cache {
  fa_tensor4 K;       /* (pages, Hk, slots, D) */
  fa_tensor4 V;       /* (pages, Hk, slots, Dv) */
  fa_tensor2 table;   /* int32 (sequences, columns) */
  fa_tensor1 lengths; /* int32 (sequences): filled slots, without the drafted tokens */
} fa_cache;

/* Attention of up to 64 drafted tokens per sequence over its cache; one token is plain decoding.  The drafted tokens' own K and V
 * lie in the cache already, token t in slot length + t (fa_cache_append).  parents[t] is the token that t follows, an earlier one, or -1
 * for one that follows the cache; anything else says that t is not there, nor what hangs on it.  Without parents every token
 * follows the one before it.  Token t sees the filled slots, its ancestors and itself.  With a window (> 0) of these only
 * the last `window` by position, itself included, and positions below `sinks`; a drafted token stands at length + its number of
 * ancestors.  A token that is not there, or sees nothing, gives 0 and a logsumexp of +inf.  Slots that no token sees may hold anything.
 * max_length bounds the lengths; it decides into how many parts the keys are split (and nothing else: longer sequences are only slower).
 * The parts' sums take scratch memory from `alloc` (fa_attn_fwd_alloc); without it the keys are not split. */
typedef struct fa_tree_params {
  fa_tensor4 Q;       /* (sequences, Hq, tokens, D) */
  fa_tensor4 Out;     /* (sequences, Hq, tokens, Dv) */
  fa_tensor2 L;       /* fp32 (sequences * Hq, tokens) or null */
  fa_cache cache;
  fa_tensor2 parents; /* int32 (sequences, tokens) or null */
  float Sm_scale;
  int32_t max_length;
  int32_t window;     /* 0: none */
  int32_t sinks;      /* with a window only */
} fa_tree_params;
FA_API int fa_tree_attn(const fa_tree_params* params, void* hip_stream, fa_allocator* alloc);

/* Rows t < counts[z] (null: all) of k (sequences, Hk, tokens, D) and v into slots lengths[z] + t.  Lengths stay as they are.  Two
 * sequences that share the page written to race. */
FA_API int fa_cache_append(const fa_tensor4* k, const fa_tensor4* v, const fa_cache* cache, const fa_tensor1* counts, void* hip_stream);

/* Page target[i] becomes a copy of page source[i].  No target may be named twice or be a source of the same call. */
FA_API int fa_cache_copy_pages(const fa_tensor4* k_cache, const fa_tensor4* v_cache, const fa_tensor1* source, const fa_tensor1* target, void* hip_stream);

/* Sequence target[i] becomes sequence source[i]: it shares its full pages, whose uses[] go up by one, and gets the rows of the last, partial
 * one in page spare[i] (not looked at where the length is a multiple of the slots or that page is not there), whose count goes up
 * as well; the rest of its table is -1.  A source that is not there (a negative length) has no fork.  The target's table is overwritten, not
 * freed (fa_cache_free).  No target may be named twice or be a source of the same call. */
FA_API int fa_cache_fork(const fa_cache* cache, const fa_tensor1* uses, const fa_tensor1* source, const fa_tensor1* target,
                         const fa_tensor1* spare, void* hip_stream);

/* The accepted drafted tokens move together: the row in slot lengths[z] + path[z][i] goes to slot lengths[z] + i for i < counts[z], and
 * new_lengths[z] = lengths[z] + counts[z].  A path ascends.  path is int32 (sequences, steps); a count above steps is steps. */
FA_API int fa_cache_keep_path(const fa_cache* cache, const fa_tensor2* path, const fa_tensor1* counts, const fa_tensor1* new_lengths, void* hip_stream);

/* Columns [first[i], last[i]) of the table's row sequences[i] become -1, and the uses[] of the pages that stood there go down by one.  A page
 * without a use is free; the caller hands it out again. */
FA_API int fa_cache_free(const fa_tensor2* table, const fa_tensor1* uses, const fa_tensor1* sequences, const fa_tensor1* first,
                         const fa_tensor1* last, void* hip_stream);

#ifdef __cplusplus
}
#endif
#endif /* AOTRITON_AMD_CACHE_H */
