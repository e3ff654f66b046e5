// The pages of a cache: appending rows, copying pages, forking and freeing sequences, compacting the accepted path of a tree.
//
// All of it moves bytes: 16 bytes per lane, consecutive lanes along a row.  What bounds the bulk copy is HBM (2048 pages of 64 slots,
// 8 heads, D128, bf16: 1.07 GB in 218 us, 4.9 TB/s); the others move a few MB and are bound by their launch and two dependent round trips
// to memory, the page table, then the rows (32 sequences, 24 rows each: append 3.6 us, a path of 6 of them 6.0-6.4; 16 forks 4.0, 16 frees of
// 63 pages 2.7 us; a caller in Python takes longer to ask for them).
#include "fa_cache.h"
#include "fa_kernels.h"

namespace fa {
namespace {

using piece_t = u32x4_t;      // eight columns

__device__ __forceinline__ bool page_at(const CacheArgs& c, int z, int64_t slot, int& page) {
  if (slot < 0) return false;
  const int64_t col = slot >> c.page_shift;
  if (col >= c.columns) return false;
  page = c.table[z * c.table_row + col];
  return page >= 0 && page < c.pages;
}
__device__ __forceinline__ int slot_in_page(const CacheArgs& c, int64_t slot) { return (int)(slot & ((1 << c.page_shift) - 1)); }
__device__ __forceinline__ uint16_t* row_of(void* base, const Strides3& s, int page, int head, int slot) {
  return reinterpret_cast<uint16_t*>(base) + (int64_t)page * s.z + (int64_t)head * s.h + (int64_t)slot * s.s;
}

// ---- append: row t of sequence z to slot lengths[z] + t ----------------------------------------------------------
// A thread per piece, a.chunks workgroups per sequence (one list of all pieces divides 64-bit numbers).
__global__ __launch_bounds__(256) void append_kernel(const AppendArgs a) {
  const CacheArgs& c = a.cache;
  const uint32_t per_k = c.head_dim / 8, per = per_k + c.head_dim_v / 8;
  const int z = blockIdx.x / a.chunks;
  const int n = c.lengths[z], count = a.counts != nullptr ? a.counts[z] : a.tokens;
  const uint32_t e = blockIdx.x % a.chunks * 256 + threadIdx.x, th = e / per;
  const int t = th / (uint32_t)c.heads, h = th % (uint32_t)c.heads;
  const uint32_t ch = e % per;
  if (t >= a.tokens || t >= count) return;
  int page;
  if (n < 0 || !page_at(c, z, (int64_t)n + t, page)) return;
  const int slot = slot_in_page(c, (int64_t)n + t);
  const bool v = ch >= per_k;
  const Strides3& from = v ? a.snv : a.snk;
  const uint16_t* src = reinterpret_cast<const uint16_t*>(v ? a.new_v : a.new_k) + (int64_t)z * from.z + (int64_t)h * from.h + (int64_t)t * from.s;
  uint16_t* dst = row_of(v ? c.v : c.k, v ? c.sv : c.sk, page, h, slot);
  const int col = (v ? ch - per_k : ch) * 8;
  *reinterpret_cast<piece_t*>(dst + col) = *reinterpret_cast<const piece_t*>(src + col);
}

// ---- copies of whole pages --------------------------------------------------------------------------------------------
// A workgroup takes kCopyPieces * 256 pieces of one page of K or V.  `flat`: the page is one run of memory, whatever the order of
// its heads and slots.
constexpr int kCopyPieces = 4;
__global__ __launch_bounds__(256) void copy_pages_kernel(const CopyArgs a) {
  const CacheArgs& c = a.cache;
  const int chunk = blockIdx.x % a.chunks, which = blockIdx.x / a.chunks % 2, i = blockIdx.x / a.chunks / 2;
  const int from = a.source[i], to = a.target[i];
  if (from < 0 || from >= c.pages || to < 0 || to >= c.pages || from == to) return;
  void* base = which ? c.v : c.k;
  const Strides3& st = which ? c.sv : c.sk;
  const int per = (which ? c.head_dim_v : c.head_dim) / 8, slots = 1 << c.page_shift;
  const int total = per * slots * c.heads;
  const uint16_t* src = reinterpret_cast<const uint16_t*>(base) + (int64_t)from * st.z;
  uint16_t* dst = reinterpret_cast<uint16_t*>(base) + (int64_t)to * st.z;
  const bool flat = which ? a.flat_v : a.flat_k;
  piece_t x[kCopyPieces];
  int64_t at[kCopyPieces];
  const int e0 = chunk * (kCopyPieces * 256) + threadIdx.x;
#pragma unroll
  for (int k = 0; k < kCopyPieces; ++k) {
    const int e = e0 + k * 256;
    at[k] = (int64_t)e * 8;
    if (!flat) {
      const int col = e % per * 8, row = e / per;
      at[k] = (int64_t)(row / slots) * st.h + (int64_t)(row % slots) * st.s + col;
    }
    if (e < total) x[k] = *reinterpret_cast<const piece_t*>(src + at[k]);
  }
#pragma unroll
  for (int k = 0; k < kCopyPieces; ++k)
    if (e0 + k * 256 < total) *reinterpret_cast<piece_t*>(dst + at[k]) = x[k];
}

// ---- fork: sequence target[i] becomes source[i] -----------------------------------------------------------------------
// It shares the full pages (their use counts go up) and gets a copy of the filled rows of the last, partial one in page spare[i].
// The first a.chunks workgroups of a fork copy, the rest write the target's row of the table.
__global__ __launch_bounds__(256) void fork_kernel(const ForkArgs a) {
  const CacheArgs& c = a.cache;
  const int per_fork = a.chunks + a.table_chunks, i = blockIdx.x / per_fork, b = blockIdx.x % per_fork;
  const int from = a.source[i], to = a.target[i];
  if (from < 0 || from >= c.sequences || to < 0 || to >= c.sequences || from == to) return;
  const int length = c.lengths[from];
  if (length < 0) return;      // (a sequence that is not there has no forks)
  const int full = length >> c.page_shift, tail = slot_in_page(c, length), spare = a.spare[i];
  const bool spare_ok = spare >= 0 && spare < c.pages;
  if (b == 0 && threadIdx.x == 0) a.lengths_out[to] = length;
  if (b >= a.chunks) {
    const int col = (b - a.chunks) * 256 + threadIdx.x;
    if (col >= c.columns) return;
    // (a partial page that is not there has no copy, and leaves the spare one alone)
    int page = -1;
    if (col < full || (col == full && tail > 0)) {
      page = c.table[(int64_t)from * c.table_row + col];
      if (page < 0 || page >= c.pages) page = -1;
      else if (col == full) page = spare_ok ? spare : -1;
    }
    if (page >= 0) atomicAdd(a.uses + page, 1);      // (whole numbers: the order does not matter)
    a.table_out[(int64_t)to * c.table_row + col] = page;
    return;
  }
  int page;
  if (tail == 0 || !spare_ok || !page_at(c, from, length - 1, page) || page == spare) return;
  const int per_k = c.head_dim / 8, per = per_k + c.head_dim_v / 8;
  const int total = per * c.heads * tail;
  for (int e = b * 256 + threadIdx.x; e < total; e += a.chunks * 256) {
    const int ch = e % per, h = e / per % c.heads, slot = e / per / c.heads;
    const bool v = ch >= per_k;
    const int col = (v ? ch - per_k : ch) * 8;
    void* base = v ? c.v : c.k;
    const Strides3& st = v ? c.sv : c.sk;
    *reinterpret_cast<piece_t*>(row_of(base, st, spare, h, slot) + col) = *reinterpret_cast<const piece_t*>(row_of(base, st, page, h, slot) + col);
  }
}

// ---- keep: the rows of a tree's accepted path move together ------------------------------------------------------------
// Slot lengths[z] + path[i] goes to lengths[z] + i.  The path ascends, so path[i] >= i and a row is overwritten only after it has been
// read if one thread takes all rows of its piece in order; up to kKeepRows of them are in flight, read before any is written.
constexpr int kKeepRows = 8;
__global__ __launch_bounds__(64) void keep_path_kernel(const KeepArgs a) {
  const CacheArgs& c = a.cache;
  const int per_k = c.head_dim / 8, per = per_k + c.head_dim_v / 8;
  const int z = blockIdx.x / a.chunks, e = blockIdx.x % a.chunks * 64 + threadIdx.x;
  const int length = c.lengths[z];
  int count = a.counts[z] < a.steps ? a.counts[z] : a.steps;
  if (count < 0 || length < 0) count = 0;
  if (blockIdx.x % a.chunks == 0 && threadIdx.x == 0) a.lengths_out[z] = length + count;
  if (e >= per * c.heads) return;
  const int ch = e % per, h = e / per;
  const bool v = ch >= per_k;
  const int col = (v ? ch - per_k : ch) * 8;
  void* base = v ? c.v : c.k;
  const Strides3& st = v ? c.sv : c.sk;
  const int32_t* path = a.path + (int64_t)z * a.path_row;
  if (c.columns == 0) return;
  const int32_t* row = c.table + (int64_t)z * c.table_row;
  // (a look-up without a branch: all of a step's are on their way together, and in front of its stores, which the compiler must not
  // pass with loads)
  auto look = [&](int64_t slot, int& page) {
    const int64_t at = slot >> c.page_shift;
    const bool ok = at >= 0 && at < c.columns;
    page = row[ok ? at : 0];
    return ok && page >= 0 && page < c.pages;
  };
  for (int i0 = 0; i0 < count; i0 += kKeepRows) {
    piece_t x[kKeepRows];
    int from[kKeepRows], page[kKeepRows], to[kKeepRows];
    bool live[kKeepRows];
#pragma unroll
    for (int k = 0; k < kKeepRows; ++k) from[k] = path[i0 + k < count ? i0 + k : i0];
#pragma unroll
    for (int k = 0; k < kKeepRows; ++k) {
      const bool there = look((int64_t)length + from[k], page[k]), room = look((int64_t)length + i0 + k, to[k]);
      live[k] = i0 + k < count && from[k] > i0 + k && there && room;      // (from == i: it is there already)
    }
#pragma unroll
    for (int k = 0; k < kKeepRows; ++k)
      if (live[k]) x[k] = *reinterpret_cast<const piece_t*>(row_of(base, st, page[k], h, slot_in_page(c, (int64_t)length + from[k])) + col);
#pragma unroll
    for (int k = 0; k < kKeepRows; ++k)
      if (live[k]) *reinterpret_cast<piece_t*>(row_of(base, st, to[k], h, slot_in_page(c, (int64_t)length + i0 + k)) + col) = x[k];
  }
}

// ---- free: columns [first, last) of a sequence's row of the table ------------------------------------------------------
// An entry is taken with an exchange, so that one that is named twice counts once.
__global__ __launch_bounds__(256) void free_pages_kernel(const FreeArgs a) {
  const int i = blockIdx.x / a.chunks, col = blockIdx.x % a.chunks * 256 + threadIdx.x;
  const int z = a.which[i];
  if (z < 0 || z >= a.sequences || col >= a.columns || col < a.first[i] || col >= a.last[i]) return;
  const int page = atomicExch(a.table + (int64_t)z * a.table_row + col, -1);
  if (page >= 0 && page < a.pages) atomicSub(a.uses + page, 1);
}

// ---- append_packed: row t to the slot that is named for it -----------------------------------------------------------------
// A thread per piece; a token's pieces lie next to each other.  Bound by memory: 30011 rows of K and V with 8 heads of 128 columns, 234 MiB moved,
// 44 us (5.4 TB/s); 200 latent rows 2.9 us, which the host's 5 hide.
__global__ __launch_bounds__(256) void append_packed_kernel(const PackedAppendArgs a) {
  const CacheArgs& c = a.cache;
  const uint32_t per_k = c.head_dim / 8 * c.heads, per = per_k + c.head_dim_v / 8 * c.heads;
  const uint32_t e = blockIdx.x * 256 + threadIdx.x;
  const int t = (int)(e / per);
  if (t >= a.tokens) return;
  const int64_t slot = a.slots[t], page = slot >> c.page_shift;
  if (slot < 0 || page >= c.pages) return;
  uint32_t x = e % per;
  const bool v = x >= per_k;
  if (v) x -= per_k;
  const uint32_t pieces = (v ? c.head_dim_v : c.head_dim) / 8, h = x / pieces;
  const int col = (int)(x % pieces) * 8;
  const Strides3& from = v ? a.snv : a.snk;
  const uint16_t* src = reinterpret_cast<const uint16_t*>(v ? a.new_v : a.new_k) + (int64_t)t * from.z + (int64_t)h * from.h;
  uint16_t* dst = row_of(v ? c.v : c.k, v ? c.sv : c.sk, (int)page, h, slot_in_page(c, slot));
  *reinterpret_cast<piece_t*>(dst + col) = *reinterpret_cast<const piece_t*>(src + col);
}

// ---- reserve: pages for the rows that a batch adds, and where each goes ----------------------------------------------------
// The k-th column that needs a page, in the order of sequences and columns, gets the k-th free page.  Two launches: the first notes which
// pages are free and counts what each sequence asks for; the second gives each sequence its pages from there, so that nothing it reads is
// what another workgroup writes.  Bound by dependent round trips to memory: 200 sequences and 16384 pages 3.8 + 6 us, 500 with prompts of up to
// 6000 tokens and 400000 pages 4.8 + 10.4 (one workgroup with all of it in LDS: 15.6 for the former).
struct Reserve {
  int32_t start, count;          // first row of the sequence in the batch, rows
  int32_t first, last;           // columns that they touch, as far as the table goes
};
// Sum of the values in front of place z of n, and of all.  All threads of the workgroup call it; `sums` has room for a word per wave.
template <typename Value>
__device__ __forceinline__ void sum_before(int n, int z, Value value, int64_t* sums, int64_t& before, int64_t& all) {
  int64_t b = 0, s = 0;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int64_t x = value(i);
    s += x;
    b += i < z ? x : 0;
  }
#pragma unroll
  for (int i = 1; i < 64; i *= 2) { b += __shfl_xor(b, i); s += __shfl_xor(s, i); }
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) { sums[wave] = b; sums[4 + wave] = s; }
  __syncthreads();
  before = sums[0] + sums[1] + sums[2] + sums[3];
  all = sums[4] + sums[5] + sums[6] + sums[7];
  __syncthreads();
}
__device__ __forceinline__ int rows_asked(const ReserveArgs& a, int z) { return a.lengths[z] < 0 || a.counts[z] < 0 ? 0 : a.counts[z]; }
__device__ __forceinline__ Reserve reserve_of(const ReserveArgs& a, int z, int64_t start) {
  Reserve r;
  const int length = a.lengths[z], asked = rows_asked(a, z);
  r.start = (int)(start < a.tokens ? start : a.tokens);
  r.count = asked < a.tokens - r.start ? asked : a.tokens - r.start;
  const int64_t first = (int64_t)length >> a.page_shift, last = ((int64_t)length + r.count + (1 << a.page_shift) - 1) >> a.page_shift;
  r.first = (int)(r.count > 0 && first < a.columns ? first : 0);
  r.last = (int)(r.count > 0 && first < a.columns ? (last < a.columns ? last : a.columns) : 0);
  return r;
}
__device__ __forceinline__ bool no_page(const ReserveArgs& a, int entry) { return entry < 0 || entry >= a.pages; }

// workgroups below a.runs: a run of pages each; the others: a sequence each
__global__ __launch_bounds__(256) void reserve_count_kernel(const ReserveArgs a) {
  __shared__ int64_t sums[8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if ((int)blockIdx.x < a.runs) {
    int n = 0;
    const int w0 = (int)blockIdx.x << a.run_shift, w1 = w0 + (1 << a.run_shift) < a.words ? w0 + (1 << a.run_shift) : a.words;
    for (int w = w0 + wave; w < w1; w += 4) {
      const int64_t page = (int64_t)w * 64 + lane;
      const uint64_t bits = __builtin_amdgcn_ballot_w64(page < a.pages && a.uses[page < a.pages ? page : 0] == 0);
      if (lane == 0) a.free_bits[w] = bits;
      n += __builtin_popcountll(bits);
    }
    if (lane == 0) sums[wave] = n;
    __syncthreads();
    if (tid == 0) a.run_free[blockIdx.x] = (int)(sums[0] + sums[1] + sums[2] + sums[3]);
    return;
  }
  const int z = blockIdx.x - a.runs;
  int64_t before, all;
  sum_before(a.sequences, z, [&](int i) { return (int64_t)rows_asked(a, i); }, sums, before, all);
  if (z >= a.sequences) {      // (of no sequence: the end)
    if (tid == 0) a.starts[a.sequences] = (int)(all < a.tokens ? all : a.tokens);
    return;
  }
  const Reserve r = reserve_of(a, z, before);
  int n = 0;
  for (int c = r.first + tid; c < r.last; c += 256) n += no_page(a, a.table[(int64_t)z * a.table_row + c]) ? 1 : 0;
#pragma unroll
  for (int i = 1; i < 64; i *= 2) n += __shfl_xor(n, i);
  if (lane == 0) sums[wave] = n;
  __syncthreads();
  if (tid == 0) {
    a.starts[z] = r.start;
    a.wanted[z] = (int)(sums[0] + sums[1] + sums[2] + sums[3]);
  }
}

// Free page number k: the run by its sums in LDS, the word in the run, the bit in the word.
__device__ __forceinline__ int free_page(const ReserveArgs& a, const int32_t* run_sum, int k) {
  int lo = 0, n = a.runs;        // the last run with no more than k free pages in front of it
  while (n > 1) {
    const int half = n / 2;
    if (run_sum[lo + half] <= k) lo += half;
    n -= half;
  }
  k -= run_sum[lo];
  // (16 words at a time, a run's where the pool is of ordinary size: one after the other they took a round trip to memory each)
  constexpr int N = 16;
  int w = -1;
  uint64_t bits = 0;
  for (int w0 = lo << a.run_shift; w < 0 && w0 < a.words; w0 += N) {
    uint64_t b[N];
#pragma unroll
    for (int i = 0; i < N; ++i) b[i] = a.free_bits[w0 + i < a.words ? w0 + i : a.words - 1];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = __builtin_popcountll(b[i]);
      if (w < 0 && k < c) {
        bits = b[i];
        w = w0 + i;
      } else if (w < 0) {
        k -= c;
      }
    }
  }
  int at = 0;
#pragma unroll
  for (int half = 32; half >= 1; half /= 2) {
    const uint64_t low = bits & ((1ull << half) - 1);
    const int c = __builtin_popcountll(low);
    if (k >= c) { k -= c; at += half; bits >>= half; }
    else bits = low;
  }
  return w * 64 + at;
}

__global__ __launch_bounds__(256) void reserve_kernel(const ReserveArgs a) {
  __shared__ int64_t sums[8];
  __shared__ int32_t run_sum[kReserveRuns + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, z = blockIdx.x;
  // (what is read from memory whatever comes of it, in front of the first wait)
  const bool is = z < a.sequences;
  const int end = a.starts[a.sequences], length = is ? a.lengths[z] : 0, wanted = is ? a.wanted[z] : 0;
  const Reserve r = is ? reserve_of(a, z, a.starts[z]) : Reserve{0, 0, 0, 0};
  int32_t* row = a.table + (int64_t)z * a.table_row;
  int own = r.first + tid < r.last ? row[r.first + tid] : 0, in_run[kReserveRuns / 256];
#pragma unroll
  for (int i = 0; i < kReserveRuns / 256; ++i) in_run[i] = i * 256 + tid < a.runs ? a.run_free[i * 256 + tid] : 0;
  // free pages in front of each run
  int base = 0;
#pragma unroll
  for (int i = 0; i < kReserveRuns / 256; ++i) {
    if (i * 256 >= a.runs) break;
    const int n = in_run[i];
    int s = n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) { const int y = __shfl_up(s, d); s += lane >= d ? y : 0; }
    if (lane == 63) sums[wave] = s;
    __syncthreads();
    for (int w = 0; w < 4; ++w) {
      if (w < wave) s += (int)sums[w];
    }
    if (i * 256 + tid < a.runs) run_sum[i * 256 + tid] = base + s - n;
    base += (int)(sums[0] + sums[1] + sums[2] + sums[3]);
    __syncthreads();
  }
  const int free = base;
  int64_t rank, all;
  sum_before(a.sequences, z, [&](int i) { return (int64_t)a.wanted[i]; }, sums, rank, all);
  if (z == 0 && tid == 0) *a.missing = (int)(all > free ? all - free : 0);
  // rows of no sequence
  for (int64_t i = (int64_t)end + blockIdx.x * 256 + tid; i < a.tokens; i += (int64_t)gridDim.x * 256) a.slots[i] = -1;
  if (!is) return;
  if (wanted > 0)
    for (int c0 = r.first; c0 < r.last; c0 += 256) {
      const int c = c0 + tid, entry = own;
      own = c + 256 < r.last ? row[c + 256] : 0;
      const bool want = c < r.last && no_page(a, entry);
      const uint64_t ask = __builtin_amdgcn_ballot_w64(want);
      if (lane == 0) sums[wave] = __builtin_popcountll(ask);
      __syncthreads();
      int64_t k = rank + __builtin_popcountll(ask & ((1ull << lane) - 1));
      for (int w = 0; w < 4; ++w) {
        if (w < wave) k += sums[w];
        rank += sums[w];
      }
      if (want && k < free) {
        const int page = free_page(a, run_sum, (int)k);
        row[c] = page;
        a.uses[page] = 1;
      }
      __syncthreads();
    }
  // (eight look-ups on their way: one after the other 6000 rows took 6 us)
  constexpr int N = 8;
  for (int i0 = tid; i0 < r.count; i0 += 256 * N) {
    int page[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int64_t c = ((int64_t)length + i0 + 256 * k) >> a.page_shift;
      page[k] = -1;
      if (i0 + 256 * k < r.count && c < a.columns) page[k] = row[c];
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = i0 + 256 * k;
      const int64_t slot = (int64_t)length + i;
      if (i < r.count) a.slots[(int64_t)r.start + i] = !no_page(a, page[k]) ? ((int64_t)page[k] << a.page_shift) + (slot & ((1 << a.page_shift) - 1)) : -1;
    }
  }
}

unsigned blocks_of(int64_t n, int per) { return (unsigned)((n + per - 1) / per); }

}  // namespace

hipError_t run_cache_append(const AppendArgs& a0, hipStream_t s) {
  AppendArgs a = a0;
  a.chunks = (int)blocks_of((int64_t)a.tokens * a.cache.heads * ((a.cache.head_dim + a.cache.head_dim_v) / 8), 256);
  if (a.cache.sequences == 0 || a.chunks == 0) return hipSuccess;
  hipLaunchKernelGGL(append_kernel, dim3((unsigned)(a.cache.sequences * a.chunks)), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t run_cache_copy(const CopyArgs& a0, int count, hipStream_t s) {
  CopyArgs a = a0;
  const int widest = a.cache.head_dim > a.cache.head_dim_v ? a.cache.head_dim : a.cache.head_dim_v;
  a.chunks = (int)blocks_of(((int64_t)widest / 8 * a.cache.heads) << a.cache.page_shift, 256 * kCopyPieces);
  if (count == 0) return hipSuccess;
  hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)(count * 2 * a.chunks)), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t run_cache_fork(const ForkArgs& a0, int count, hipStream_t s) {
  ForkArgs a = a0;
  const int64_t pieces = ((int64_t)(a.cache.head_dim + a.cache.head_dim_v) / 8 * a.cache.heads) << a.cache.page_shift;
  a.chunks = (int)blocks_of(pieces, 256 * 4);
  a.table_chunks = (int)blocks_of(a.cache.columns, 256);
  if (count == 0) return hipSuccess;
  hipLaunchKernelGGL(fork_kernel, dim3((unsigned)(count * (a.chunks + a.table_chunks))), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t run_cache_keep(const KeepArgs& a0, hipStream_t s) {
  KeepArgs a = a0;
  a.chunks = (int)blocks_of((int64_t)(a.cache.head_dim + a.cache.head_dim_v) / 8 * a.cache.heads, 64);
  if (a.cache.sequences == 0) return hipSuccess;
  hipLaunchKernelGGL(keep_path_kernel, dim3((unsigned)(a.cache.sequences * a.chunks)), dim3(64), 0, s, a);
  return hipGetLastError();
}

hipError_t run_cache_free(const FreeArgs& a0, int count, hipStream_t s) {
  FreeArgs a = a0;
  a.chunks = (int)blocks_of(a.columns, 256);
  if (count == 0 || a.columns == 0) return hipSuccess;
  hipLaunchKernelGGL(free_pages_kernel, dim3((unsigned)(count * a.chunks)), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t run_cache_append_packed(const PackedAppendArgs& a, hipStream_t s) {
  const int64_t pieces = (int64_t)a.tokens * a.cache.heads * ((a.cache.head_dim + a.cache.head_dim_v) / 8);
  if (pieces == 0) return hipSuccess;
  hipLaunchKernelGGL(append_packed_kernel, dim3(blocks_of(pieces, 256)), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t run_cache_reserve(const ReserveArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(reserve_count_kernel, dim3((unsigned)(a.runs + a.sequences + 1)), dim3(256), 0, s, a);
  hipLaunchKernelGGL(reserve_kernel, dim3((unsigned)(a.sequences > 0 ? a.sequences : 1)), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace fa
