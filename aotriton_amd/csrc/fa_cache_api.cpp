// C entry points of the cache of pages and of the attention of drafted tokens over it: argument checks, and how many parts the
// keys are split into.  No state of their own; the device is looked up through fa_check_gpu and fa_get_multiprocessor_count.
#include <algorithm>

#include "aotriton_amd/cache.h"
#include "fa_cache_args.h"
#include "fa_kernels.h"

namespace fa {

#define FA_DECL(d)                                                   \
  hipError_t run_tree_d##d(int, const TreeArgs&, hipStream_t);       \
  hipError_t run_tree_d##d##_padded(int, const TreeArgs&, hipStream_t);
FA_DECL(64)
FA_DECL(128)
FA_DECL(256)
#undef FA_DECL

static int compiled_columns(const CacheArgs& c) {
  const int d = std::max(c.head_dim, c.head_dim_v);
  return d <= 64 ? 64 : d <= 128 ? 128 : 256;
}

hipError_t run_tree(int dtype, const TreeArgs& a, hipStream_t s) {
  const int d = compiled_columns(a.cache);
  const bool padded = a.cache.head_dim != d || a.cache.head_dim_v != d;
  switch (d) {
    case 64: return (padded ? run_tree_d64_padded : run_tree_d64)(dtype, a, s);
    case 128: return (padded ? run_tree_d128_padded : run_tree_d128)(dtype, a, s);
    default: return (padded ? run_tree_d256_padded : run_tree_d256)(dtype, a, s);
  }
}

}  // namespace fa

namespace {

constexpr int64_t kMaxRowStride = 1 << 21;      // elements, as in the other entry points
constexpr uint64_t kMaxCount = 0x7fffffff;

bool empty(const fa_tensor4& t) { return t.sizes[0] == 0 || t.sizes[1] == 0 || t.sizes[2] == 0; }

// rows of aligned 16-byte pieces, no negative stride
int check_rows(const fa_tensor4& t, int dtype) {
  if (t.dtype != dtype || (t.ptr == nullptr && !empty(t))) return FA_ERROR_INVALID_VALUE;
  for (int i = 0; i < 4; ++i)
    if (t.sizes[i] > kMaxCount) return FA_ERROR_INVALID_VALUE;
  if (t.sizes[3] == 0 || t.sizes[3] > 256 || t.sizes[3] % 8 != 0 || (t.strides[3] != 1 && t.sizes[3] > 1)) return FA_ERROR_NOT_SUPPORTED;
  if ((reinterpret_cast<uintptr_t>(t.ptr) & 15u) != 0) return FA_ERROR_NOT_SUPPORTED;
  for (int i = 0; i < 3; ++i)
    if (t.sizes[i] > 1 && ((int64_t)t.strides[i] < 0 || t.strides[i] % 8 != 0)) return FA_ERROR_NOT_SUPPORTED;
  if (t.sizes[2] > 1 && (int64_t)t.strides[2] > kMaxRowStride) return FA_ERROR_NOT_SUPPORTED;
  return FA_SUCCESS;
}

// int32 values next to each other, `n` of them
int check_ints(const fa_tensor1& t, uint64_t n) {
  if (t.dtype != FA_DTYPE_INT32 || t.sizes[0] != n || (t.ptr == nullptr && n > 0)) return FA_ERROR_INVALID_VALUE;
  if (n > 1 && t.strides[0] != 1) return FA_ERROR_NOT_SUPPORTED;
  return FA_SUCCESS;
}

// int32 rows with adjacent columns
int check_int_rows(const fa_tensor2& t, uint64_t rows) {
  if (t.dtype != FA_DTYPE_INT32 || t.sizes[0] != rows || t.sizes[1] > kMaxCount) return FA_ERROR_INVALID_VALUE;
  if (t.ptr == nullptr && t.sizes[0] * t.sizes[1] > 0) return FA_ERROR_INVALID_VALUE;
  if ((t.sizes[1] > 1 && t.strides[1] != 1) || (t.sizes[0] > 1 && (int64_t)t.strides[0] < 0)) return FA_ERROR_NOT_SUPPORTED;
  return FA_SUCCESS;
}

// Rows of a tensor that is written have to lie apart.
bool rows_apart(const fa_tensor2& t) { return t.sizes[0] <= 1 || t.strides[0] >= t.sizes[1]; }
// (an expanded cache has one row for many)
bool written_apart(const fa_tensor4& t) {
  for (int i = 0; i < 3; ++i)
    if (t.sizes[i] > 1 && t.strides[i] < t.sizes[3]) return false;
  return true;
}
bool written_apart(const fa_cache& c) { return written_apart(c.K) && written_apart(c.V); }

fa::Strides3 strides3(const fa_tensor4& t) {
  return fa::Strides3{(int64_t)t.strides[0], (int64_t)t.strides[1], (int64_t)t.strides[2]};
}

// K and V of a cache
int check_pages(const fa_tensor4& k, const fa_tensor4& v, fa::CacheArgs* out) {
  int e = FA_SUCCESS;
  if (k.dtype != FA_DTYPE_FLOAT16 && k.dtype != FA_DTYPE_BFLOAT16) return FA_ERROR_INVALID_VALUE;
  if ((e = check_rows(k, k.dtype)) != FA_SUCCESS || (e = check_rows(v, k.dtype)) != FA_SUCCESS) return e;
  for (int i = 0; i < 3; ++i)
    if (k.sizes[i] != v.sizes[i] || k.sizes[i] == 0) return FA_ERROR_INVALID_VALUE;
  // (kernels multiply with the strides of pages and rows in 32 bits)
  for (const fa_tensor4* t : {&k, &v})
    if (t->sizes[0] > 1 && (int64_t)t->strides[0] > 0x7fffffff) return FA_ERROR_NOT_SUPPORTED;
  const uint64_t page = k.sizes[2];
  if (page < 16 || page > (1 << 20) || (page & (page - 1)) != 0) return FA_ERROR_NOT_SUPPORTED;
  fa::CacheArgs& c = *out;
  c = fa::CacheArgs{};
  c.k = k.ptr; c.v = v.ptr;
  c.sk = strides3(k); c.sv = strides3(v);
  c.pages = (int32_t)k.sizes[0];
  c.heads = (int32_t)k.sizes[1];
  c.page_shift = __builtin_ctzll(page);
  c.head_dim = (int32_t)k.sizes[3];
  c.head_dim_v = (int32_t)v.sizes[3];
  return FA_SUCCESS;
}

int check_cache(const fa_cache* p, fa::CacheArgs* out) {
  if (p == nullptr) return FA_ERROR_INVALID_VALUE;
  int e = check_pages(p->K, p->V, out);
  if (e != FA_SUCCESS) return e;
  fa::CacheArgs& c = *out;
  if (p->lengths.sizes[0] > kMaxCount) return FA_ERROR_INVALID_VALUE;
  if ((e = check_ints(p->lengths, p->lengths.sizes[0])) != FA_SUCCESS) return e;
  if ((e = check_int_rows(p->table, p->lengths.sizes[0])) != FA_SUCCESS) return e;
  // slots, and the blocks of 64 sequences, are counted in 32 bits
  if ((p->table.sizes[1] << c.page_shift) > 1ull << 29) return FA_ERROR_NOT_SUPPORTED;
  c.table = static_cast<const int32_t*>(p->table.ptr);
  c.table_row = (int64_t)p->table.strides[0];
  c.lengths = static_cast<const int32_t*>(p->lengths.ptr);
  c.sequences = (int32_t)p->lengths.sizes[0];
  c.columns = (int32_t)p->table.sizes[1];
  return FA_SUCCESS;
}

// a launch's workgroups have to fit 31 bits
bool fits(double workgroups) { return workgroups < 2147483648.0; }

// Rows per workgroup, how the keys are cut, and the scratch for the sums of sequences that lie in several pieces.
struct TreePlan { int64_t o_bytes, bytes; };
TreePlan tree_plan(fa::TreeArgs* a, int64_t max_length, int num_cu) {
  TreePlan p{};
  const int d = fa::compiled_columns(a->cache);
  const int64_t rows = (int64_t)a->tokens * (a->hq / a->cache.heads), sequences = a->cache.sequences;
  // (the blocks that a sequence of that length has, at the most)
  auto blocks_of = [&](int64_t length, int64_t size) {
    int64_t slots = length + a->tokens;
    if (a->window > 0) slots = std::min<int64_t>(slots, (int64_t)a->window + a->tokens + std::min<int64_t>(a->sinks, length) + 3 * size);
    return std::max<int64_t>(1, (slots + size - 1) / size);
  };
  // 32 rows per workgroup where it has few blocks of 32 slots to do, tiles where it has many.  (us, 32 rows / 128 / 256, D128 Hq 32 Hk 8 unless
  // said: one token, B1 4096 slots 11.5 / 12.7, B8 up to 2048 14.5 / 16.8, B64 up to 8192 129 / 129, D64 75 / 72; 4 tokens, B16 up to 8192
  // 37 / 35, 16 tokens 46 / 40 / 42, B4 800 slots 15.3 / 16.8 / 17; 32 tokens, B1 4096 slots 21 / 26 / 22, B8 up to 6000 40 / 31 / 31; 48 tokens, B8 700
  // slots 34 / 29 / 27, 4900 80 / 62 / 54; 64 tokens, B1 4000 slots 25 / 29 / 32.)
  const int64_t work = blocks_of(max_length, 32) * sequences * a->cache.heads * ((rows + 31) / 32) / (2 * num_cu);
  a->row_rows = d > 128 || work <= (rows <= 64 ? 32 : 16) ? 32 : rows <= 128 ? 128 : 256;
  a->row_blocks = (int)((rows + a->row_rows - 1) / a->row_rows);
  a->part_rows = (int)std::min<int64_t>(rows, a->row_rows);
  a->block_shift = a->row_rows == 32 ? 5 : 6;
  a->least = a->row_rows == 32 ? 8 : 2;
  const int64_t size = 1 << a->block_shift;
  // One round of workgroups: two on a CU, one with tiles of 256 rows or more than 128 columns.  What else the table has room for plays no
  // part.  (us, cut for a table of 131072 slots / for max_length, D128 Hq 32 Hk 8: B64 512 slots, one token, 391 / 24, B8 4096 slots, 64 tokens,
  // 122 / 57.)
  const int64_t heads = (int64_t)a->cache.heads * a->row_blocks, chip = (int64_t)(d > 128 || a->row_rows == 256 ? 1 : 2) * num_cu;
  const int64_t blocks = blocks_of(max_length, size);
  const int64_t per = std::max<int64_t>(a->least, (blocks * sequences * heads + chip - 1) / chip);
  int64_t stored = 0;      // (at most two places for a workgroup of the round, whatever the table and the sequences are)
  // Short pieces: a workgroup has one, of one sequence, so that nothing waits for the lengths of the others or for an item before.
  // Long ones: equal pieces of all keys, whatever the lengths: a piece may hold the ends of two sequences, 12 us more with tiles.  (us,
  // the one / the other, D128 unless said, Hq 32 Hk 8: B1 4096 slots 11.7 / 13.3, B8 up to 2048 14.9 / 18.2, B32 Hq 16 Hk 2 D64 7 tokens window 1024
  // 15.4 / 22.3, B8 48 tokens 4900 54 / 66; B64 up to 8192 145 / 132, D64 87 / 79, B8 48 tokens up to 16384 117 / 63.)
  const int64_t short_piece = a->row_rows == 32 ? 32 : 24;
  if (per <= short_piece) {
    a->part_blocks = (int)per;
    a->parts = (int)((blocks + per - 1) / per);
    if (a->parts > 1) stored = heads * sequences * a->parts * a->part_rows;
  } else if (chip / heads > 1) {
    a->workers = (int)(chip / heads);
    stored = heads * a->workers * 2 * a->part_rows;
  }
  p.o_bytes = stored * d * 4;
  p.bytes = stored * (d * 4 + 8);
  return p;
}

}  // namespace

extern "C" {

int fa_tree_attn(const fa_tree_params* p, void* hip_stream, fa_allocator* alloc) {
  if (p == nullptr) return FA_ERROR_INVALID_VALUE;
  fa::TreeArgs a{};
  int e = check_cache(&p->cache, &a.cache);
  if (e != FA_SUCCESS) return e;
  const fa::CacheArgs& c = a.cache;
  const int dtype = p->cache.K.dtype;
  if ((e = check_rows(p->Q, dtype)) != FA_SUCCESS || (e = check_rows(p->Out, dtype)) != FA_SUCCESS) return e;
  const uint64_t tokens = p->Q.sizes[2], hq = p->Q.sizes[1];
  if (p->Q.sizes[0] != (uint64_t)c.sequences || p->Q.sizes[3] != (uint64_t)c.head_dim || hq == 0 || hq % (uint64_t)c.heads != 0) return FA_ERROR_INVALID_VALUE;
  for (int i = 0; i < 3; ++i)
    if (p->Out.sizes[i] != p->Q.sizes[i]) return FA_ERROR_INVALID_VALUE;
  if (p->Out.sizes[3] != (uint64_t)c.head_dim_v) return FA_ERROR_INVALID_VALUE;
  if (tokens > fa::kTreeTokens || hq > 65536) return FA_ERROR_NOT_SUPPORTED;
  if (p->max_length < 0 || p->window < 0 || p->sinks < 0 || (p->window == 0 && p->sinks != 0)) return FA_ERROR_INVALID_VALUE;
  if (p->parents.ptr != nullptr) {
    if ((e = check_int_rows(p->parents, (uint64_t)c.sequences)) != FA_SUCCESS) return e;
    if (p->parents.sizes[1] != tokens) return FA_ERROR_INVALID_VALUE;
  }
  if (p->L.ptr != nullptr) {
    const fa_tensor2& l = p->L;
    if (l.dtype != FA_DTYPE_FLOAT32 || l.sizes[0] != (uint64_t)c.sequences * hq || l.sizes[1] != tokens) return FA_ERROR_INVALID_VALUE;
    if ((l.sizes[1] > 1 && l.strides[1] != 1) || (l.sizes[0] > 1 && l.strides[0] != l.sizes[1])) return FA_ERROR_NOT_SUPPORTED;
  }
  if ((e = fa_check_gpu(hip_stream)) != FA_SUCCESS) return e;
  if (c.sequences == 0 || tokens == 0) return FA_SUCCESS;
  a.q = p->Q.ptr; a.out = p->Out.ptr; a.lse = static_cast<float*>(p->L.ptr);
  a.sq = strides3(p->Q); a.so = strides3(p->Out);
  a.parents = static_cast<const int32_t*>(p->parents.ptr);
  a.parents_row = (int64_t)p->parents.strides[0];
  a.hq = (int32_t)hq; a.tokens = (int32_t)tokens;
  a.sm_scale = p->Sm_scale;
  // (the kernels add the window to positions)
  a.window = std::min(p->window, 1 << 30);
  a.sinks = std::min(p->sinks, 1 << 30);
  const int64_t room = (int64_t)c.columns << c.page_shift;
  const TreePlan plan = tree_plan(&a, std::min<int64_t>(p->max_length, room), fa_get_multiprocessor_count(hip_stream));
  if (plan.bytes > 0) {
    void* scratch = alloc != nullptr ? alloc->alloc(alloc, (uint64_t)plan.bytes) : nullptr;
    if (scratch != nullptr) {
      a.part_o = static_cast<float*>(scratch);
      a.part_ml = reinterpret_cast<float*>(static_cast<char*>(scratch) + plan.o_bytes);
    }
  }
  if (a.part_o == nullptr) {      // every sequence is one piece
    a.workers = 0;
    a.parts = 1;
  }
  if (!fits(((double)c.heads * (a.workers > 0 ? a.workers : (double)c.sequences * a.parts) + 8) * a.row_blocks) || !fits((double)c.sequences * c.heads * a.row_blocks * 256)) return FA_ERROR_NOT_SUPPORTED;
  return (int)fa::run_tree(dtype, a, static_cast<hipStream_t>(hip_stream));
}

int fa_cache_append(const fa_tensor4* k, const fa_tensor4* v, const fa_cache* cache, const fa_tensor1* counts, void* hip_stream) {
  if (k == nullptr || v == nullptr) return FA_ERROR_INVALID_VALUE;
  fa::AppendArgs a{};
  int e = check_cache(cache, &a.cache);
  if (e != FA_SUCCESS) return e;
  if (!written_apart(*cache)) return FA_ERROR_NOT_SUPPORTED;
  const fa::CacheArgs& c = a.cache;
  if ((e = check_rows(*k, cache->K.dtype)) != FA_SUCCESS || (e = check_rows(*v, cache->K.dtype)) != FA_SUCCESS) return e;
  for (const fa_tensor4* t : {k, v})
    if (t->sizes[0] != (uint64_t)c.sequences || t->sizes[1] != (uint64_t)c.heads || t->sizes[2] != k->sizes[2]) return FA_ERROR_INVALID_VALUE;
  if (k->sizes[3] != (uint64_t)c.head_dim || v->sizes[3] != (uint64_t)c.head_dim_v) return FA_ERROR_INVALID_VALUE;
  if (counts != nullptr && counts->ptr != nullptr) {
    if ((e = check_ints(*counts, (uint64_t)c.sequences)) != FA_SUCCESS) return e;
    a.counts = static_cast<const int32_t*>(counts->ptr);
  }
  a.new_k = k->ptr; a.new_v = v->ptr;
  a.snk = strides3(*k); a.snv = strides3(*v);
  a.tokens = (int32_t)k->sizes[2];
  const double pieces = (double)a.tokens * c.heads * ((c.head_dim + c.head_dim_v) / 8);
  if (!fits(pieces) || !fits(c.sequences * (pieces / 256 + 1))) return FA_ERROR_NOT_SUPPORTED;
  if ((e = fa_check_gpu(hip_stream)) != FA_SUCCESS) return e;
  return (int)fa::run_cache_append(a, static_cast<hipStream_t>(hip_stream));
}

int fa_cache_copy_pages(const fa_tensor4* k_cache, const fa_tensor4* v_cache, const fa_tensor1* source, const fa_tensor1* target, void* hip_stream) {
  if (k_cache == nullptr || v_cache == nullptr || source == nullptr || target == nullptr) return FA_ERROR_INVALID_VALUE;
  fa::CopyArgs a{};
  int e = check_pages(*k_cache, *v_cache, &a.cache);
  if (e != FA_SUCCESS) return e;
  if (!written_apart(*k_cache) || !written_apart(*v_cache)) return FA_ERROR_NOT_SUPPORTED;
  const uint64_t n = source->sizes[0];
  if (n > kMaxCount) return FA_ERROR_INVALID_VALUE;
  if ((e = check_ints(*source, n)) != FA_SUCCESS || (e = check_ints(*target, n)) != FA_SUCCESS) return e;
  // heads and slots in either order without a gap
  auto flat = [&](const fa_tensor4& t) {
    const uint64_t heads = t.sizes[1], slots = t.sizes[2], d = t.sizes[3];
    return ((heads == 1 || t.strides[1] == slots * d) && t.strides[2] == d) || (t.strides[2] == heads * d && (heads == 1 || t.strides[1] == d));
  };
  a.flat_k = flat(*k_cache);
  a.flat_v = flat(*v_cache);
  a.source = static_cast<const int32_t*>(source->ptr);
  a.target = static_cast<const int32_t*>(target->ptr);
  const fa::CacheArgs& c = a.cache;
  const double pieces = (double)std::max(c.head_dim, c.head_dim_v) / 8 * c.heads * (1 << c.page_shift);
  if (pieces > 1e9 || !fits((double)n * 2 * (pieces / 1024 + 1))) return FA_ERROR_NOT_SUPPORTED;
  if ((e = fa_check_gpu(hip_stream)) != FA_SUCCESS) return e;
  return (int)fa::run_cache_copy(a, (int)n, static_cast<hipStream_t>(hip_stream));
}

int fa_cache_fork(const fa_cache* cache, const fa_tensor1* uses, const fa_tensor1* source, const fa_tensor1* target, const fa_tensor1* spare, void* hip_stream) {
  if (uses == nullptr || source == nullptr || target == nullptr || spare == nullptr) return FA_ERROR_INVALID_VALUE;
  fa::ForkArgs a{};
  int e = check_cache(cache, &a.cache);
  if (e != FA_SUCCESS) return e;
  const fa::CacheArgs& c = a.cache;
  const uint64_t n = source->sizes[0];
  if (n > kMaxCount) return FA_ERROR_INVALID_VALUE;
  if ((e = check_ints(*uses, (uint64_t)c.pages)) != FA_SUCCESS) return e;
  for (const fa_tensor1* t : {source, target, spare})
    if ((e = check_ints(*t, n)) != FA_SUCCESS) return e;
  if (!rows_apart(cache->table) || !written_apart(*cache)) return FA_ERROR_NOT_SUPPORTED;
  a.table_out = static_cast<int32_t*>(cache->table.ptr);
  a.lengths_out = static_cast<int32_t*>(cache->lengths.ptr);
  a.uses = static_cast<int32_t*>(uses->ptr);
  a.source = static_cast<const int32_t*>(source->ptr);
  a.target = static_cast<const int32_t*>(target->ptr);
  a.spare = static_cast<const int32_t*>(spare->ptr);
  const double pieces = (double)(c.head_dim + c.head_dim_v) / 8 * c.heads * (1 << c.page_shift);
  if (pieces > 1e9 || !fits((double)n * (pieces / 1024 + c.columns / 256 + 2))) return FA_ERROR_NOT_SUPPORTED;
  if ((e = fa_check_gpu(hip_stream)) != FA_SUCCESS) return e;
  return (int)fa::run_cache_fork(a, (int)n, static_cast<hipStream_t>(hip_stream));
}

int fa_cache_keep_path(const fa_cache* cache, const fa_tensor2* path, const fa_tensor1* counts, const fa_tensor1* new_lengths, void* hip_stream) {
  if (path == nullptr || counts == nullptr || new_lengths == nullptr) return FA_ERROR_INVALID_VALUE;
  fa::KeepArgs a{};
  int e = check_cache(cache, &a.cache);
  if (e != FA_SUCCESS) return e;
  const fa::CacheArgs& c = a.cache;
  if (!written_apart(*cache)) return FA_ERROR_NOT_SUPPORTED;
  if ((e = check_int_rows(*path, (uint64_t)c.sequences)) != FA_SUCCESS) return e;
  if ((e = check_ints(*counts, (uint64_t)c.sequences)) != FA_SUCCESS || (e = check_ints(*new_lengths, (uint64_t)c.sequences)) != FA_SUCCESS) return e;
  // (workgroups of one sequence read its length while another one writes the new one)
  if (c.sequences > 0 && new_lengths->ptr == cache->lengths.ptr) return FA_ERROR_INVALID_VALUE;
  a.path = static_cast<const int32_t*>(path->ptr);
  a.path_row = (int64_t)path->strides[0];
  a.steps = (int32_t)path->sizes[1];
  a.counts = static_cast<const int32_t*>(counts->ptr);
  a.lengths_out = static_cast<int32_t*>(new_lengths->ptr);
  if (!fits((double)c.sequences * ((double)(c.head_dim + c.head_dim_v) / 8 * c.heads / 64 + 1))) return FA_ERROR_NOT_SUPPORTED;
  if ((e = fa_check_gpu(hip_stream)) != FA_SUCCESS) return e;
  return (int)fa::run_cache_keep(a, static_cast<hipStream_t>(hip_stream));
}

int fa_cache_free(const fa_tensor2* table, const fa_tensor1* uses, const fa_tensor1* sequences, const fa_tensor1* first, const fa_tensor1* last, void* hip_stream) {
  if (table == nullptr || uses == nullptr || sequences == nullptr || first == nullptr || last == nullptr) return FA_ERROR_INVALID_VALUE;
  fa::FreeArgs a{};
  int e = check_int_rows(*table, table->sizes[0]);
  if (e != FA_SUCCESS) return e;
  if (!rows_apart(*table)) return FA_ERROR_NOT_SUPPORTED;
  const uint64_t n = sequences->sizes[0];
  if (n > kMaxCount || table->sizes[0] > kMaxCount || uses->sizes[0] > kMaxCount) return FA_ERROR_INVALID_VALUE;
  if ((e = check_ints(*uses, uses->sizes[0])) != FA_SUCCESS) return e;
  for (const fa_tensor1* t : {sequences, first, last})
    if ((e = check_ints(*t, n)) != FA_SUCCESS) return e;
  a.table = static_cast<int32_t*>(table->ptr);
  a.table_row = (int64_t)table->strides[0];
  a.sequences = (int32_t)table->sizes[0];
  a.columns = (int32_t)table->sizes[1];
  a.pages = (int32_t)uses->sizes[0];
  a.uses = static_cast<int32_t*>(uses->ptr);
  a.which = static_cast<const int32_t*>(sequences->ptr);
  a.first = static_cast<const int32_t*>(first->ptr);
  a.last = static_cast<const int32_t*>(last->ptr);
  if (!fits((double)n * (a.columns / 256 + 1))) return FA_ERROR_NOT_SUPPORTED;
  if ((e = fa_check_gpu(hip_stream)) != FA_SUCCESS) return e;
  return (int)fa::run_cache_free(a, (int)n, static_cast<hipStream_t>(hip_stream));
}

}  // extern "C"
