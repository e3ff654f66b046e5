// Argument blocks of the kernels over a cache of pages, and their launchers.
//
// The cache is two tensors (pages, heads, slots of a page, columns) of any strides with unit columns; slot n of a sequence is slot
// n % page of the page that the sequence's row of the page table names in column n / page.  Entries outside [0, pages), columns
// outside the table and slots outside a sequence are never read or written through: what they stand for is not there.
#pragma once
#include <hip/hip_runtime.h>

#include "fa_args.h"

namespace fa {

constexpr int kTreeTokens = 64;      // a drafted token's ancestors are a 64-bit word

struct CacheArgs {
  void* k; void* v;
  Strides3 sk, sv;               // page, head, slot
  const int32_t* table;          // (sequences, columns)
  int64_t table_row;
  const int32_t* lengths;        // slots of a sequence that are filled, without the drafted tokens
  int32_t sequences, columns, pages, heads, page_shift;
  int32_t head_dim, head_dim_v;
};

struct TreeArgs {
  const void* q; void* out; float* lse;
  Strides3 sq, so;
  CacheArgs cache;
  const int32_t* parents;        // (sequences, tokens); null: a chain
  int64_t parents_row;
  int32_t hq, tokens;
  float sm_scale;
  int32_t window, sinks;         // window 0: none
  // Work, in blocks of 1 << block_shift slots for row_rows packed rows of a head.  workers > 0: the blocks of all sequences, one after the
  // other, are cut into that many equal pieces of at least `least` blocks, one for a workgroup.  Otherwise every sequence is cut into
  // pieces of part_blocks blocks, at most `parts`, the last of which has what is left.  The rows' sums over a sequence that lies in several
  // pieces go to part_o (null: none does) as (head, block of rows, tree_sums' place, row of the block, compiled columns) and, maximum and
  // row sum, to part_ml.
  int32_t workers, least, parts, part_blocks, block_shift;
  int32_t row_blocks, row_rows, part_rows;      // part_rows: stored per block of rows
  float* part_o; float* part_ml;
};

struct AppendArgs {
  CacheArgs cache;
  const void* new_k; const void* new_v;      // (sequences, heads, tokens, columns)
  Strides3 snk, snv;
  const int32_t* counts;                     // rows of each sequence; null: all
  int32_t tokens, chunks;                    // chunks: workgroups of a sequence (the launcher's)
};

struct CopyArgs {
  CacheArgs cache;                           // (without a table)
  const int32_t* source; const int32_t* target;
  int32_t flat_k, flat_v;                    // a page is one run of memory
  int32_t chunks;                            // workgroups per page (launcher)
};

struct ForkArgs {
  CacheArgs cache;
  int32_t* table_out; int32_t* lengths_out; int32_t* uses;      // the cache's own table and lengths
  const int32_t* source; const int32_t* target; const int32_t* spare;
  int32_t chunks, table_chunks;              // workgroups per fork (launcher)
};

struct KeepArgs {
  CacheArgs cache;
  const int32_t* path; int64_t path_row;     // (sequences, steps)
  const int32_t* counts;
  int32_t* lengths_out;
  int32_t steps;
  int32_t chunks;                            // workgroups per sequence (launcher)
};

struct FreeArgs {
  int32_t* table; int64_t table_row;
  int32_t sequences, columns, pages;
  int32_t* uses;
  const int32_t* which; const int32_t* first; const int32_t* last;
  int32_t chunks;                            // workgroups per sequence (launcher)
};

// dtype: kDtypeF16 or kDtypeBF16; the others move 16-bit columns whatever they stand for.  Scratch of TreeArgs is the caller's.
hipError_t run_tree(int dtype, const TreeArgs& a, hipStream_t s);
hipError_t run_cache_append(const AppendArgs& a, hipStream_t s);
hipError_t run_cache_copy(const CopyArgs& a, int count, hipStream_t s);
hipError_t run_cache_fork(const ForkArgs& a, int count, hipStream_t s);
hipError_t run_cache_keep(const KeepArgs& a, hipStream_t s);
hipError_t run_cache_free(const FreeArgs& a, int count, hipStream_t s);

}  // namespace fa
