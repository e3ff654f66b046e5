// C entry points of attention over keys and values from one latent vector a token: argument checks, and how the keys are cut.  No state of
// their own; the device is looked up through fa_check_gpu and fa_get_multiprocessor_count.
#include <algorithm>

#include "aotriton_amd/latent.h"
#include "fa_checks.h"
#include "fa_latent_args.h"

namespace {

using namespace fa::checks;

constexpr uint64_t kColumns = 128, kShared = 64;                       // of the expanded form
constexpr uint64_t kLatent = 576, kLatentValue = 512;                  // of the absorbed form

// (rows of what has none may lie anywhere)
bool apart(const fa_tensor4& t) { return empty(t) || written_apart(t); }

bool same_sizes(const fa_tensor4& a, const fa_tensor4& b) { return std::equal(a.sizes, a.sizes + 4, b.sizes); }

// int32 offsets of the sequences of packed tensors; 0 where the tensors are not packed, -1: not such
int64_t offsets_of(const fa_tensor1& t) {
  if (t.ptr == nullptr) return 0;
  return t.dtype == FA_DTYPE_INT32 && t.sizes[0] >= 2 && t.sizes[0] <= kMaxCount && t.strides[0] == 1 ? (int64_t)t.sizes[0] - 1 : -1;
}

int64_t sequences(const fa::LatentArgs& a) { return a.seq.num_seqlens != 0 ? a.seq.num_seqlens : a.batch; }

int check_fwd(const fa_latent_fwd_params* p, bool lse_needed, fa::LatentArgs* out) {
  const int dtype = p->Q.dtype;
  if (dtype != FA_DTYPE_FLOAT16 && dtype != FA_DTYPE_BFLOAT16) return FA_ERROR_INVALID_VALUE;
  int e = check_rows(p->Q, dtype, kColumns + kShared);
  if (e == FA_SUCCESS) e = check_rows(p->K, dtype, kColumns);
  if (e == FA_SUCCESS) e = check_rows(p->V, dtype, kColumns);
  if (e == FA_SUCCESS) e = check_rows(p->S, dtype, kShared);
  if (e == FA_SUCCESS) e = check_rows(p->Out, dtype, kColumns);
  if (e != FA_SUCCESS) return e;
  const uint64_t batch = p->Q.sizes[0], heads = p->Q.sizes[1], sq = p->Q.sizes[2], sk = p->K.sizes[2];
  for (const fa_tensor4* t : {&p->K, &p->V})
    if (t->sizes[0] != batch || t->sizes[1] != heads || t->sizes[2] != sk) return FA_ERROR_INVALID_VALUE;
  if (p->S.sizes[0] != batch || p->S.sizes[1] != 1 || p->S.sizes[2] != sk) return FA_ERROR_INVALID_VALUE;
  if (p->Q.sizes[3] != p->K.sizes[3] + p->S.sizes[3]) return FA_ERROR_INVALID_VALUE;
  for (int i = 0; i < 3; ++i)
    if (p->Out.sizes[i] != p->Q.sizes[i]) return FA_ERROR_INVALID_VALUE;
  if (p->Out.sizes[3] != p->V.sizes[3]) return FA_ERROR_INVALID_VALUE;
  if (!apart(p->Out)) return FA_ERROR_NOT_SUPPORTED;
  if (p->L.ptr != nullptr || (lse_needed && batch * heads * sq > 0)) {
    const fa_tensor2& l = p->L;
    if (l.ptr == nullptr || l.dtype != FA_DTYPE_FLOAT32 || l.sizes[0] != batch * heads || l.sizes[1] != sq) return FA_ERROR_INVALID_VALUE;
    if ((l.sizes[1] > 1 && l.strides[1] != 1) || (l.sizes[0] > 1 && l.strides[0] != l.sizes[1])) return FA_ERROR_NOT_SUPPORTED;
  }
  const int64_t nq = offsets_of(p->cu_seqlens_q), nk = offsets_of(p->cu_seqlens_k);
  if (nq < 0 || nk != nq) return FA_ERROR_INVALID_VALUE;
  if (nq > 0 && (batch != 1 || p->max_seqlen_q < 0 || p->max_seqlen_k < 0)) return FA_ERROR_INVALID_VALUE;
  if (heads > 65536 || batch > 65536 || sq > (1u << 30) || sk > (1u << 30)) return FA_ERROR_NOT_SUPPORTED;

  fa::LatentArgs& a = *out;
  a.q = p->Q.ptr; a.k = p->K.ptr; a.v = p->V.ptr; a.c = p->S.ptr; a.out = p->Out.ptr;
  a.lse = static_cast<float*>(p->L.ptr);
  a.sq = strides3(p->Q); a.sk = strides3(p->K); a.sv = strides3(p->V); a.so = strides3(p->Out);
  a.c_z = (int64_t)p->S.strides[0]; a.c_s = (int64_t)p->S.strides[2];
  a.batch = (int32_t)batch; a.heads = (int32_t)heads;
  a.e = (int32_t)p->K.sizes[3]; a.r = (int32_t)p->S.sizes[3]; a.ev = (int32_t)p->V.sizes[3];
  a.sm_scale = p->Sm_scale;
  a.causal = p->causal != 0;
  a.rows_q = (int32_t)sq; a.rows_k = (int32_t)sk;
  a.parts = 1;
  if (nq > 0) {
    a.seq.cu_q = static_cast<const int32_t*>(p->cu_seqlens_q.ptr);
    a.seq.cu_k = static_cast<const int32_t*>(p->cu_seqlens_k.ptr);
    a.seq.num_seqlens = (int32_t)nq;
    a.seq.max_seqlen_q = (int32_t)std::min<uint64_t>(p->max_seqlen_q, sq);
    a.seq.max_seqlen_k = (int32_t)std::min<uint64_t>(p->max_seqlen_k, sk);
  } else {
    a.seq.max_seqlen_q = a.rows_q;
    a.seq.max_seqlen_k = a.rows_k;
  }
  const double pairs = (double)sequences(a) * a.heads;
  if (!fits(pairs * (a.seq.max_seqlen_q / 128 + 1.0) * 16) || !fits(pairs * (a.seq.max_seqlen_k / 128 + 1.0))) return FA_ERROR_NOT_SUPPORTED;
  return FA_SUCCESS;
}

int compiled(const fa::LatentArgs& a) { return a.e <= 64 && a.ev <= 64 ? 64 : 128; }

// Tiles of 128 queries of all heads; of packed sequences about as many.
int64_t query_tiles(const fa::LatentArgs& a) {
  const int64_t nseq = sequences(a);
  return a.heads * (a.seq.num_seqlens > 0 ? a.rows_q / 128 + (nseq + 1) / 2 : nseq * ((a.rows_q + 127) / 128));
}

// Parts that the keys are cut into: where the tiles of 128 queries do not fill the chip, as many as do, of eight tiles of keys at least.
// (4 heads, 128 queries, 8192 keys: uncut 181 us, in 4 parts 54, in 16, the rule's, 30; 16 heads, 128 queries, 4096 keys: 95, 33, in 8 25, in 16 28;
// 16 heads, 1024 queries, 4096 keys: 102, in 4, the rule's, 53, in 8 65.)
int latent_parts(const fa::LatentArgs& a, int num_cu) {
  const int64_t tiles = query_tiles(a);
  const int64_t chip = 2 * (int64_t)num_cu, keys = (a.seq.max_seqlen_k + 63) / 64;
  if (tiles == 0) return 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>({chip / tiles, keys / 8, 16}));
}

}  // namespace

extern "C" {

int fa_latent_fwd(const fa_latent_fwd_params* p, void* hip_stream, fa_allocator* alloc) {
  if (p == nullptr) return FA_ERROR_INVALID_VALUE;
  fa::LatentArgs a{};
  int e = check_fwd(p, false, &a);
  if (e != FA_SUCCESS) return e;
  if ((e = fa_check_gpu(hip_stream)) != FA_SUCCESS) return e;
  const int d = compiled(a), parts = alloc != nullptr ? latent_parts(a, fa_get_multiprocessor_count(hip_stream)) : 1;
  if (parts > 1) {
    a.slabs = a.rows_q / 32 + (int32_t)(a.seq.num_seqlens != 0 ? a.seq.num_seqlens : 1);
    const int64_t slabs = (int64_t)a.batch * a.heads * a.slabs * parts;
    const int64_t o_bytes = slabs * 32 * d * 4;
    void* scratch = alloc->alloc(alloc, (uint64_t)(o_bytes + slabs * 64 * 4));
    if (scratch != nullptr) {
      a.parts = parts;
      a.part_o = static_cast<float*>(scratch);
      a.part_ml = reinterpret_cast<float*>(static_cast<char*>(scratch) + o_bytes);
    }
  }
  return (int)(d == 64 ? fa::run_latent_fwd_d64 : fa::run_latent_fwd_d128)(p->Q.dtype, a, static_cast<hipStream_t>(hip_stream));
}

int fa_latent_bwd(const fa_latent_bwd_params* p, void* hip_stream, fa_allocator* alloc) {
  if (p == nullptr) return FA_ERROR_INVALID_VALUE;
  fa::LatentBwdArgs a{};
  int e = check_fwd(&p->fwd, true, &a);
  if (e != FA_SUCCESS) return e;
  const fa_latent_fwd_params& f = p->fwd;
  const struct { const fa_tensor4 *t, *like; bool written; } all[] = {{&p->DO, &f.Out, false}, {&p->DQ, &f.Q, true}, {&p->DK, &f.K, true}, {&p->DV, &f.V, true}, {&p->DS, &f.S, true}};
  for (const auto& x : all) {
    if ((e = check_rows(*x.t, f.Q.dtype, x.like->sizes[3])) != FA_SUCCESS) return e;
    if (!same_sizes(*x.t, *x.like)) return FA_ERROR_INVALID_VALUE;
    if (x.written && !apart(*x.t)) return FA_ERROR_NOT_SUPPORTED;
  }
  a.dout = p->DO.ptr;
  a.dq = p->DQ.ptr; a.dk = p->DK.ptr; a.dv = p->DV.ptr; a.dc = p->DS.ptr;
  a.sdo = strides3(p->DO); a.sdq = strides3(p->DQ); a.sdk = strides3(p->DK); a.sdv = strides3(p->DV);
  a.dc_z = (int64_t)p->DS.strides[0]; a.dc_s = (int64_t)p->DS.strides[2];
  a.part_rows = a.rows_k;
  if (!fits((double)a.batch * a.rows_k / 16 + 1)) return FA_ERROR_NOT_SUPPORTED;
  if ((e = fa_check_gpu(hip_stream)) != FA_SUCCESS) return e;
  const int64_t stats = (int64_t)a.batch * a.heads * a.rows_q, shared = (int64_t)a.batch * a.heads * a.rows_k * kShared;
  if (stats + (int64_t)a.batch * a.rows_k == 0) return FA_SUCCESS;
  const int64_t stat_bytes = (stats * 2 * 4 + 255) / 256 * 256;
  void* scratch = nullptr;      // (without heads DS is 0)
  if (a.heads > 0) {
    scratch = alloc != nullptr ? alloc->alloc(alloc, (uint64_t)(stat_bytes + shared * 4)) : nullptr;
    if (scratch == nullptr) return FA_ERROR_OUT_OF_MEMORY;
  }
  a.stat_lse = static_cast<float*>(scratch);
  a.stat_delta = a.stat_lse + stats;
  a.part_c = reinterpret_cast<float*>(static_cast<char*>(scratch) + stat_bytes);
  // (steps of 1 to 16 heads, E = Ev = 128, R = 64: 128 tiles 361 us with two waves on a SIMD, 311 alone, 256 tiles 399 and 350, 512 480 and 443, 752 878 and
  // 881, 2800 1655 and 1705)
  a.alone = query_tiles(a) <= 2 * (int64_t)fa_get_multiprocessor_count(hip_stream);
  return (int)(compiled(a) == 64 ? fa::run_latent_bwd_d64 : fa::run_latent_bwd_d128)(f.Q.dtype, a, static_cast<hipStream_t>(hip_stream));
}

int fa_latent_cache_attn(const fa_latent_cache_params* p, void* hip_stream, fa_allocator* alloc) {
  if (p == nullptr) return FA_ERROR_INVALID_VALUE;
  const fa_tensor4& x = p->latent;
  if (x.dtype != FA_DTYPE_FLOAT16 && x.dtype != FA_DTYPE_BFLOAT16) return FA_ERROR_INVALID_VALUE;
  int e = check_rows(x, x.dtype, kLatent);
  if (e == FA_SUCCESS) e = check_rows(p->Q, x.dtype, kLatent);
  if (e == FA_SUCCESS) e = check_rows(p->Out, x.dtype, kLatentValue);
  if (e != FA_SUCCESS) return e;
  if (x.sizes[0] == 0 || x.sizes[1] != 1 || x.sizes[2] == 0) return FA_ERROR_INVALID_VALUE;
  const uint64_t slots = x.sizes[2], rows = p->Q.sizes[1], hq = p->Q.sizes[2], n = p->lengths.sizes[0];
  if (slots < 16 || slots > (1 << 20) || (slots & (slots - 1)) != 0) return FA_ERROR_NOT_SUPPORTED;
  if (p->Q.sizes[0] != 1 || p->Q.sizes[3] != x.sizes[3] || hq == 0) return FA_ERROR_INVALID_VALUE;
  for (int i = 0; i < 3; ++i)
    if (p->Out.sizes[i] != p->Q.sizes[i]) return FA_ERROR_INVALID_VALUE;
  if (p->Out.sizes[3] > x.sizes[3]) return FA_ERROR_INVALID_VALUE;
  if (!apart(p->Out)) return FA_ERROR_NOT_SUPPORTED;
  if (n >= kMaxCount || p->max_length < 0) return FA_ERROR_INVALID_VALUE;
  if ((e = check_ints(p->lengths, n)) != FA_SUCCESS || (e = check_ints(p->starts, n + 1)) != FA_SUCCESS || (e = check_int_rows(p->table, n)) != FA_SUCCESS) return e;
  if (p->L.ptr != nullptr) {
    const fa_tensor2& l = p->L;
    if (l.dtype != FA_DTYPE_FLOAT32 || l.sizes[0] != rows || l.sizes[1] != hq) return FA_ERROR_INVALID_VALUE;
    if ((l.sizes[1] > 1 && l.strides[1] != 1) || (l.sizes[0] > 1 && l.strides[0] != l.sizes[1])) return FA_ERROR_NOT_SUPPORTED;
  }
  fa::LatentCacheArgs a{};
  fa::CacheArgs& c = a.cache;
  c.k = x.ptr;
  c.sk = strides3(x);
  c.page_shift = __builtin_ctzll(slots);
  c.pages = (int32_t)x.sizes[0]; c.heads = 1;
  c.head_dim = (int32_t)x.sizes[3]; c.head_dim_v = (int32_t)p->Out.sizes[3];
  c.table = static_cast<const int32_t*>(p->table.ptr);
  c.table_row = (int64_t)p->table.strides[0];
  c.columns = (int32_t)p->table.sizes[1];
  c.sequences = (int32_t)n;
  c.lengths = static_cast<const int32_t*>(p->lengths.ptr);
  a.starts = static_cast<const int32_t*>(p->starts.ptr);
  a.q = p->Q.ptr; a.out = p->Out.ptr; a.lse = static_cast<float*>(p->L.ptr);
  a.q_row = rows > 1 ? (int64_t)p->Q.strides[1] : 0; a.q_head = hq > 1 ? (int64_t)p->Q.strides[2] : 0;
  a.o_row = (int64_t)p->Out.strides[1]; a.o_head = (int64_t)p->Out.strides[2];
  a.rows = (int32_t)rows; a.hq = (int32_t)hq;
  a.sm_scale = p->Sm_scale;
  // slots are counted in 32 bits, and a block's 128 rows of Q and Out are reached with 32-bit offsets; (rows, heads) pairs of a sequence are 31 bits
  if ((p->table.sizes[1] << c.page_shift) > 1ull << 29 || hq > 65536 || (double)rows * (double)hq >= (double)(1 << 30)) return FA_ERROR_NOT_SUPPORTED;
  auto near = [&](int64_t row, int64_t head) { return (double)row * (double)(128 / hq + 1) + (double)head * (double)hq + kLatent < (double)(1 << 29); };
  if (!near(a.q_row, a.q_head) || !near(rows > 1 ? a.o_row : 0, hq > 1 ? a.o_head : 0)) return FA_ERROR_NOT_SUPPORTED;
  if ((e = fa_check_gpu(hip_stream)) != FA_SUCCESS) return e;
  if (rows == 0) return FA_SUCCESS;

  const int num_cu = fa_get_multiprocessor_count(hip_stream), d = c.head_dim <= 320 && c.head_dim_v <= 256 ? 256 : 512;
  // Rows of a workgroup.  32 where a sequence has no more on average, or where blocks of 128, which take longer to begin and to end, would leave a CU
  // a few tiles of 32 slots.  64 sequences of 4096 slots, 576 columns: 32 heads 90 us with blocks of 32 and of 128, 40 heads 124 and 94, 128 heads 211
  // and 114; 16 sequences (8 tiles a CU) with 64 heads 45 and 43; 8 sequences (4 tiles) 32 and 35, with 128 heads 44 and 46; 2 sequences 25 and 29.
  // 64 rows only up to 256 columns of values (64 sequences, 64 heads, 320 columns: 75, 58, 59 us for 32, 64, 128 rows); above, 40 heads took 111 with them.
  // (Sequences without a new token count, too: 64 with 128 heads take 111 us in a table of 64 rows, 204 to 215 in one of 256.)
  const int64_t mean = n > 0 ? (int64_t)(rows * hq / n) : 0;
  const int64_t room = (int64_t)c.columns << c.page_shift;
  const int64_t most = std::max<int64_t>(1, (int64_t)rows - (int64_t)n + 1);      // new tokens of a sequence, if all have some
  const int64_t tiles = (std::min<int64_t>((int64_t)p->max_length + most, room) + 31) / 32;
  const bool much = (int64_t)n * ((mean + 127) / 128) * tiles >= 6 * (int64_t)num_cu;
  a.block_rows = mean <= 32 || !much ? 32 : mean <= 64 && d == 256 ? 64 : 128;
  // One workgroup on a CU, one round of them.
  const int64_t blocks = (int64_t)rows * (int64_t)hq / a.block_rows + (int64_t)n;
  if (!fits((double)blocks * 4 * 16)) return FA_ERROR_NOT_SUPPORTED;
  a.blocks = (int32_t)blocks;
  a.least = 4;       // (one sequence of 4096 slots with 16 heads: 24.9 us with 6, 23.5 with 2 to 4, 25.9 with 1)
  a.margin = 5;      // (a batch of prompts' chunks and single tokens 84 us with 2, 67 with 4, 65 with 5 and 6; 64 sequences with 128 heads 92, 84, 84 and 83)
  a.block_shift = a.block_rows == 32 ? 5 : a.block_rows == 64 ? 6 : 7;
  a.group_shift = a.step_shift = 0;
  while ((2ull << a.group_shift) * a.block_rows <= 32 * hq) ++a.group_shift;
  while ((32ull * hq << a.step_shift) < (uint64_t)a.block_rows) ++a.step_shift;
  // Blocks of short sequences stay whole: no pieces, and no second launch.  8 sequences with 16 heads: 100 slots 19.5 us in pieces, 14.4 whole, 250 slots
  // 18.7 and 19.3, 400 slots 19.1 and 25.3; 64 sequences of 250 slots 24.9 and 20.5, with 128 heads and 100 slots 20.3 and 16.9.
  const bool whole = tiles <= 9;
  if (whole) {
    a.least = 1;
    a.margin = -1;
  }
  a.workers = (int32_t)std::max<int64_t>(1, std::min<int64_t>(num_cu, whole ? blocks : blocks * ((tiles + a.least - 1) / a.least)));
  const int64_t places = 2 * (int64_t)a.workers * (a.block_rows / 32), o_bytes = places * 32 * d * 4;
  void* scratch = alloc != nullptr && a.workers > 1 && !whole ? alloc->alloc(alloc, (uint64_t)(o_bytes + places * 64 * 4 + blocks * (int64_t)sizeof(fa::LatentHead))) : nullptr;
  if (scratch != nullptr) {
    a.part_o = static_cast<float*>(scratch);
    a.part_ml = reinterpret_cast<float*>(static_cast<char*>(scratch) + o_bytes);
    a.heads = reinterpret_cast<fa::LatentHead*>(a.part_ml + places * 64);
  } else if (a.workers > 1 && !whole) {
    return FA_ERROR_OUT_OF_MEMORY;
  }
  return (int)(d == 256 ? fa::run_latent_cache_d256 : fa::run_latent_cache_d512)(x.dtype, a, static_cast<hipStream_t>(hip_stream));
}

}  // extern "C"
