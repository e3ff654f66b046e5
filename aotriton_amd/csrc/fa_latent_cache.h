// Attention over a cache of pages of latent rows (the absorbed form): gfx950, MFMA 32x32x16.
//
//   S = scale Q X^T,  O = softmax(S) X[:, :Ev]     X: the rows of a sequence, the keys of all heads and, in front, their values
//
// A row of the score matrix is a (token, head) pair of a sequence.  A tile of 32 slots comes into swizzled LDS once and serves both
// products: row reads for S^T = X Q^T, transposing reads for O^T += X^T P^T.  Its first EA columns (256 or 512) and the 64 behind them lie
// in two areas, as rows of 2 EA and 128 bytes.
// RW waves side by side take 32 rows each; the 4 / RW groups of them share the columns of O, and each forms all of S, so that nothing
// is exchanged between waves.  With 128 rows (RW = 4) nothing is formed twice, and O takes all 256 accumulation registers at
// EA = 512; with few rows the cache's bytes bound the kernel and not what it computes.
//
// Work is a list of blocks of rows times tiles of slots, cut into one piece for a CU wherever the cut falls; the sums of a block that lies in
// several pieces are put together by a launch of its own (with one workgroup for a sequence, 64 sequences with 128 heads would take four times
// as long).  576 columns, values of 512: a tile of 128 rows takes 3600 cycles, 2180 of them MFMAs (the products alone 2700, with the
// exponentials 3100); 64 sequences with 128 heads 78 to 84 us, of which 63 to 68 here and 16 for the pieces (86 MiB of fp32 sums, written and read); 16 heads
// over up to 16384 slots 79 us, 4.2 TB/s.
#pragma once
#include "fa_cache.h"
#include "fa_latent_args.h"
#include "fa_latent_list.h"
#include "fa_latent_parts.h"

namespace fa {

constexpr int kLatentTail = 64;

template <int EA> struct LatentCacheSmem {
  static constexpr int A = 32 * EA * 2, STAGE = A + 32 * kLatentTail * 2, STAGES = 4;
  static constexpr int LIST = STAGES * STAGE;           // words of latent_find
  static constexpr int BYTES = EA == 256 ? 2 * LIST : LIST + 128 + 8192;      // (with 128 rows of Q)
  // Q of RW x 32 rows: in how many parts of its columns it comes, with how many tiles of the cache in front of it.  (Where it lies on the list, that
  // has been read.)
  template <int RW> struct Q {
    static constexpr int HALVES = EA == 512 && RW == 4 ? 2 : 1, COLUMNS = EA / HALVES, FIRST = EA == 256 || RW == 1 ? 3 : 2;
    __host__ __device__ static constexpr int at(int half, int group) {
      const int size = 32 * COLUMNS * 2 + (half == HALVES - 1 ? 32 * kLatentTail * 2 : 0);
      return (EA == 256 ? LIST : FIRST * STAGE) + group * size;
    }
    static_assert(EA == 256 || 2 * STAGE + 4 * 32 * (COLUMNS + kLatentTail) * 2 <= BYTES || RW < 4, "Q fits");
  };
};

__device__ __forceinline__ LatentSeq latent_cache_seq(const LatentCacheArgs& a, int z) {
  auto hold = [](int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; };
  const int start = hold(a.starts[z], 0, a.rows);
  return latent_seq_of(a, start, hold(hold(a.starts[z + 1], 0, a.rows) - start, 0, a.rows), a.cache.lengths[z], (int64_t)a.cache.columns << a.cache.page_shift);
}

// Number of a sequence's first block, with a gap or two: that of its first row, divided by the rows of a block, and one more for every sequence in
// front.  LatentCacheArgs::blocks bounds them.
__device__ __forceinline__ int latent_block(const LatentCacheArgs& a, int z, int start) { return (start * a.hq >> a.block_shift) + z; }

// The cut of the list: its length, that of a piece, and of the sequence looked for its number and where it starts in the list.  `mine(z, first
// unit, sequence)` says which one that is.  All 256 threads call this.
struct LatentCut { int64_t per, total, first; int z; LatentSeq seq; };
template <typename Mine>
__device__ __forceinline__ LatentCut latent_find(const LatentCacheArgs& a, char* words, Mine mine) {
  int64_t* sums = reinterpret_cast<int64_t*>(words);      // of the four waves; then the answer
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.cache.sequences;
  LatentCut cut{0, 0, 0, -1, {}};
  int64_t base = 0;
  LatentSeq s;
  int64_t before = 0;
  auto chunk = [&](int z0) {      // this thread's sequence and the units in front of it
    const int z = z0 + tid;
    int64_t u = 0;
    if (z < n) {
      s = latent_cache_seq(a, z);
      u = s.units(a);
    }
    int64_t sum = u;
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
      const int64_t y = __shfl_up(sum, i);
      if (lane >= i) sum += y;
    }
    if (lane == 63) sums[wave] = sum;
    __syncthreads();
    before = base + sum - u;
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before += sums[w];
      base += sums[w];
    }
    __syncthreads();
  };
  for (int z0 = 0; z0 < n; z0 += 256) chunk(z0);
  cut.total = base;
  const int64_t even = latent_div(base + a.workers - 1, a.workers);
  cut.per = even > a.least ? even : a.least;
  if (tid == 0) sums[5] = -1;
  __syncthreads();
  if (n > 256) base = 0;
  for (int z0 = 0; z0 < n; z0 += 256) {
    if (n > 256) chunk(z0);
    const int z = z0 + tid;
    if (z < n && s.blocks > 0 && mine(cut, z, before, s)) {
      sums[4] = before;
      sums[5] = z;
      *reinterpret_cast<LatentSeq*>(sums + 6) = s;
    }
    if (n > 256) __syncthreads();
  }
  __syncthreads();
  cut.first = sums[4];
  cut.z = (int)sums[5];
  cut.seq = *reinterpret_cast<const LatentSeq*>(sums + 6);
  __syncthreads();      // (Q may come to lie on the words)
  return cut;
}

// kCut: rows have fewer than EA columns; those past them are zero.
template <typename T, int EA, int RW, bool kCut>
__global__ __launch_bounds__(256, 1) void latent_cache_kernel(const LatentCacheArgs a) {
  using Tr = Traits<T>;
  using op_t = typename Tr::op_t;
  using SM = LatentCacheSmem<EA>;
  constexpr int KE = EA / 16, KR = kLatentTail / 16, CG = 4 / RW, DB = EA / 32 / CG;
  // O takes all accumulation registers: its MFMAs are written as asm (fa_wide.h), and scores have to be in vector registers; the compiler, left
  // to place the two, spills a thousand bytes.
  constexpr bool kFull = DB == 16;
  extern __shared__ __attribute__((aligned(kSwzAlign))) char smem[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rw = wave % RW, cg = wave / RW;
  const CacheArgs& ca = a.cache;
  const int e = ca.head_dim, ev = ca.head_dim_v;

  const int n_seq = ca.sequences, starts_first = n_seq > 0 ? a.starts[0] : a.rows, starts_last = n_seq > 0 ? a.starts[n_seq] : 0;
  // (workgroups go round the XCDs: those of neighbouring pieces, which read the same Q, stand on one)
  const int xcd = blockIdx.x % 8, each = a.workers / 8, more = a.workers % 8;
  const int64_t worker = xcd * each + (xcd < more ? xcd : more) + (int)blockIdx.x / 8;
  const LatentCut cut = latent_find(a, smem + SM::LIST, [&](const LatentCut& t, int, int64_t first, const LatentSeq& s) {
    return first <= worker * t.per && worker * t.per < first + s.units(a);
  });
  // rows of no sequence
  {
    const int gap = starts_first < 0 ? 0 : starts_first > a.rows ? a.rows : starts_first, end = starts_last < gap ? gap : starts_last;
    for (int i = blockIdx.x; i < gap + (a.rows - end); i += gridDim.x) {
      const int row = i < gap ? i : end + i - gap;
      for (int x = threadIdx.x; x < a.hq * (ev / 8); x += 256) {
        const int h = x / (ev / 8), col = x % (ev / 8) * 8;
        *reinterpret_cast<u32x4_t*>(reinterpret_cast<T*>(a.out) + (int64_t)row * a.o_row + (int64_t)h * a.o_head + col) = u32x4_t{0, 0, 0, 0};
        if (a.lse != nullptr && col == 0) a.lse[(int64_t)row * a.hq + h] = __builtin_inff();
      }
    }
  }
  const int64_t u = worker * cut.per;
  const int64_t u_end = u + cut.per < cut.total ? u + cut.per : cut.total;
  // (for the kernel that puts the pieces together: a block's head is written by the worker that begins it, and where blocks are numbered with a
  // gap by the one that begins the block in front, or the first)
  auto put_heads = [&](int from, int to) {
    for (int i = (from < 0 ? 0 : from) + (int)threadIdx.x; i < to && i < a.blocks; i += 256) a.heads[i] = LatentHead{0, 0, 0, 0, 0};
  };
  if (a.heads != nullptr && cut.total == 0 && worker == 0) put_heads(0, a.blocks);
  if (u >= u_end) return;
  int z = __builtin_amdgcn_readfirstlane(cut.z);

  const int smem0 = lds_offset(smem);
  // What depends on the lane alone is formed where it is needed: held through the loop over tiles, which Q and O leave little room, it would be
  // spilled, and a reload waits for the tiles that are on their way.
  auto own_lane = [&]() __attribute__((always_inline)) { int l = threadIdx.x; if constexpr (kFull) asm volatile("" : "+v"(l)); return l & 63; };
  const int x_row = (int)ca.sk.s * 2;
  constexpr int LPR = EA / 8, RPL = 64 / LPR;      // lanes of a row, rows of an access
  LatentSeq s = cut.seq;
  int block = 0;
  int64_t at_unit = u;      // where the block begins
  for (bool again = false; at_unit < u_end; again = true) {
    if (again) s = latent_cache_seq(a, z);
    s.start = __builtin_amdgcn_readfirstlane(s.start); s.tokens = __builtin_amdgcn_readfirstlane(s.tokens);
    s.length = __builtin_amdgcn_readfirstlane(s.length); s.end = __builtin_amdgcn_readfirstlane(s.end);
    s.tiles = __builtin_amdgcn_readfirstlane(s.tiles); s.blocks = __builtin_amdgcn_readfirstlane(s.blocks);
    s.filled = __builtin_amdgcn_readfirstlane(s.filled);
    if (!again) {
      int unit;
      block = __builtin_amdgcn_readfirstlane(s.block_of(a, u - cut.first, unit));
      at_unit = u - __builtin_amdgcn_readfirstlane(unit);
    }
    if (block >= s.blocks) {      // (the next one that has rows)
      block = 0;
      ++z;
      continue;
    }
    const int lane = own_lane(), c = lane & 31, hi = lane >> 5;
    const int block_tiles = __builtin_amdgcn_readfirstlane(s.tiles_of(a, block));
    // (a cut beside the tiles leaves the block to one side of it)
    const int span = a.margin < 0 ? 1 : block_tiles + 2 * a.margin;
    auto tile_of = [&](int64_t x) {
      const int64_t n = a.margin < 0 ? (x > at_unit ? block_tiles : 0) : x - at_unit - a.margin;
      return __builtin_amdgcn_readfirstlane(n < 0 ? 0 : n < block_tiles ? (int)n : block_tiles);
    };
    const int j0 = tile_of(u), n_tiles = tile_of(u_end) - j0;
    if (n_tiles <= 0) {
      at_unit += span;
      ++block;
      continue;
    }
    auto slot_of = [&](int entry) { const int n = (j0 + entry / 2) * 32 + entry % 2 * 16; return entry < 2 * n_tiles && n < s.end ? n : -1; };
    PageRun<decltype(slot_of)> pages(ca, z, lane, slot_of);
    const int rows = s.tokens * a.hq, w0 = block * a.block_rows + rw * 32, w_last = w0 + 31 < rows ? w0 + 31 : rows - 1;
    const bool row_ok = w0 + c < rows;
    const int row = row_ok ? w0 + c : rows - 1, token = row / a.hq, head = row - token * a.hq;
    // the last slot that the row sees, that the wave's first and last rows see
    const int see = s.last_slot(token);
    const int see_least = __builtin_amdgcn_readfirstlane(s.last_slot(w0 / a.hq));
    const int see_most = __builtin_amdgcn_readfirstlane(s.last_slot(w_last / a.hq));
    const int j1 = j0 + n_tiles, wave_end = w0 < rows ? see_most / 32 + 1 : 0;

    const char* xbase = reinterpret_cast<const char*>(ca.k);
    auto stage_of = [&](int j) { return smem0 + ((j - j0) & (SM::STAGES - 1)) * SM::STAGE; };
    constexpr int kLoads = 8 / RPL + 1, kPieces = 4 / RPL + 1;      // of a tile, and the pairs they come in
    u32x4_t f_rs;
    int f_lds;
    // What a tile's fetch needs, in steps that stand behind different MFMAs; fetch_holes says which of its halves have no page.
    int f_page, f_left, f_entry;
    const char* f_from;
    auto fetch_page = [&](int j) __attribute__((always_inline)) {
      f_entry = (j - j0) * 2;
      f_page = pages.at(f_entry + wave / 2);
      f_lds = __builtin_amdgcn_readfirstlane(stage_of(j));
    };
    auto fetch_rows = [&](int j) __attribute__((always_inline)) {
      const int n = j * 32 + wave * 8;
      f_left = s.end - n < 8 ? s.end - n : 8;
      f_from = xbase + (int64_t)(n & ((1 << ca.page_shift) - 1)) * ca.sk.s * 2;
    };
    auto fetch_rsrc = [&]() __attribute__((always_inline)) {      // (a page that is not there: zeros, no traffic)
      f_rs = wave_rsrc_words(f_from + (int64_t)(f_page < 0 ? 0 : f_page) * ca.sk.z * 2, f_page < 0 ? 0 : rows_extent(f_left, x_row, e * 2));
    };
    auto fetch_holes = [&]() __attribute__((always_inline)) { return pages.holes(f_entry) & 3; };
    auto fetch_piece = [&](int i) __attribute__((always_inline)) {
      const int l = own_lane();
      if (i < kPieces - 1) {
        // a lane's piece of its row: the lane's number, swizzled by the row's
        const int lrow = l / LPR, base = (l % LPR) ^ Swz<EA>::f(lrow + 8 * (wave & 1)), lds = f_lds + wave * 8 * EA * 2;
        static_assert(RPL == 1 || RPL == 2, "f of a row is that of its access and that of its place in it");
        int voff[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) voff[t] = lrow * x_row + ((base ^ Swz<EA>::f((2 * i + t) * RPL)) << 4);
        if (kCut) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if ((base ^ Swz<EA>::f((2 * i + t) * RPL)) * 8 >= e) voff[t] = kVoffOutOfRange;
        }
        load_to_lds(f_rs, voff[0], 2 * i * RPL * x_row, lds + 2 * i * 1024, voff[1], (2 * i + 1) * RPL * x_row, lds + (2 * i + 1) * 1024);
      } else {
        const int ch = (l % 8) ^ Swz<kLatentTail>::f(8 * (wave & 1) + l / 8);      // (a wave's eight rows are the first or second of 16)
        load_to_lds1(f_rs, EA + ch * 8 < e ? l / 8 * x_row + (EA + ch * 8) * 2 : kVoffOutOfRange, f_lds + SM::A + wave * 1024);
      }
    };
    auto fetch = [&](int j) __attribute__((always_inline)) {
      pages.to((j - j0) * 2);
      fetch_page(j);
      fetch_rows(j);
      fetch_rsrc();
#pragma unroll
      for (int i = 0; i < kPieces; ++i) fetch_piece(i);
      return fetch_holes();
    };
    // Q passes through LDS as tiles of 32 rows, as the latent rows do: whole rows of memory, each once (as a lane's row in pieces straight into
    // registers it took 11 us for 128 rows).  It lies behind the first kFirst stages, whose tiles are on their way with it; where it does not fit
    // there, it comes in two halves of its columns.
    // (lane l has the place of row l % 8 of the wave's eight of the l / 8-th 32)
    const int r0 = block * a.block_rows, tb = r0 / a.hq, r_lane = r0 + lane / 8 * 32 + wave * 8 + lane % 8, t_lane = r_lane / a.hq;
    const int q_off = r_lane < rows && lane < 8 * RW ? (t_lane - tb) * ((int)a.q_row * 2) + (r_lane - t_lane * a.hq) * ((int)a.q_head * 2) : -1;
    const int t_end = (r0 + a.block_rows - 1 < rows ? r0 + a.block_rows - 1 : rows - 1) / a.hq;
    const u32x4_t q_rs = wave_rsrc_words(reinterpret_cast<const T*>(a.q) + (int64_t)(s.start + tb) * a.q_row,
                                         (int)(((t_end - tb) * a.q_row + (a.hq - 1) * a.q_head + e) * 2));
    auto fetch_q = [&](auto half) __attribute__((always_inline)) {
      constexpr int H = decltype(half)::value, at_col = H * SM::template Q<RW>::COLUMNS, QC = SM::template Q<RW>::COLUMNS, QL = QC / 8, QR = 64 / QL;
      constexpr bool ends = H == SM::template Q<RW>::HALVES - 1;
      static_assert(QR == 1 || QR == 2, "f of a row is that of its access and that of its place in it");
      const int l = own_lane(), lrow = l / QL, base = (l % QL) ^ Swz<QC>::f(lrow + 8 * (wave & 1)), tail_ch = (l % 8) ^ Swz<kLatentTail>::f(8 * (wave & 1) + l / 8);
#pragma unroll
      for (int g = 0; g < RW; ++g) {
        const int lds = smem0 + SM::template Q<RW>::at(H, g), lds_a = lds + wave * 8 * QC * 2;
        auto off = [&](int i) { return __builtin_amdgcn_readlane(q_off, 8 * g + i); };
#pragma unroll
        for (int i = 0; i < 8 / QR; i += 2) {
          int voff[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int at = QR == 1 ? off(i + k) : lrow ? off((i + k) * QR + QR - 1) : off((i + k) * QR), ch = base ^ Swz<QC>::f((i + k) * QR);
            voff[k] = at >= 0 && (!kCut || at_col + ch * 8 < e) ? at + at_col * 2 + (ch << 4) : kVoffOutOfRange;
          }
          load_to_lds(q_rs, voff[0], 0, lds_a + i * 1024, voff[1], 0, lds_a + (i + 1) * 1024);
        }
        if (ends) {
          const int at = __shfl(q_off, 8 * g + l / 8);
          load_to_lds1(q_rs, at >= 0 && EA + tail_ch * 8 < e ? at + (EA + tail_ch * 8) * 2 : kVoffOutOfRange, lds + 32 * QC * 2 + wave * 1024);
        }
      }
    };
    op_t q[KE + KR];
    auto take_q = [&](auto half) __attribute__((always_inline)) {
      constexpr int H = decltype(half)::value, QC = SM::template Q<RW>::COLUMNS, N = QC / 16;
      const int X = smem0 + SM::template Q<RW>::at(H, rw), q_e = Swz<QC>::row_base(own_lane()), q_r = Swz<kLatentTail>::row_base(own_lane());
#pragma unroll
      for (int k = 0; k < N; ++k) q[H * N + k] = lds_read<op_t>((q_e ^ ((k & 7) << 5)) + X + (k >> 3) * 256);
      if (H == SM::template Q<RW>::HALVES - 1) {
#pragma unroll
        for (int k = 0; k < KR; ++k) q[KE + k] = lds_read<op_t>((q_r ^ (k << 5)) + X + 32 * QC * 2);
      }
    };
    using zero = std::integral_constant<int, 0>;
    using one = std::integral_constant<int, 1>;
    // (pages are looked up 32 tiles at a time, and where the compiler waits for them it waits for Q too)
    constexpr int kFirst = SM::template Q<RW>::FIRST;
    int holes = 0, holes1 = 0, holes2 = 0;      // of this tile, the next, the one behind it
    fetch_q(zero{});
    holes = fetch(j0);
    holes1 = fetch(j0 + 1);
    if (kFirst > 2) holes2 = fetch(j0 + 2);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(kFirst * kLoads) : "memory");
    take_q(zero{});
    if constexpr (SM::template Q<RW>::HALVES == 2) {
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      fetch_q(one{});
      asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
      take_q(one{});
    }
    arrived(q);
    if (kFirst < SM::STAGES - 1) {
      asm volatile("s_barrier" ::: "memory");      // (all waves have their rows)
      holes2 = fetch(j0 + 2);
    }
    f32x16 o[DB];
#pragma unroll
    for (int b = 0; b < DB; ++b) {
      if constexpr (kFull) acc_zero<T>(o[b]);
      else o[b] = f32x16{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    }
    RowSoftmax sm(a.sm_scale);

    constexpr int kRing = 8, kS = KE + KR, kV = 2 * DB;      // operands on their way: left to itself the compiler keeps dozens
    f32x16 x[1];
    op_t p[2], p_next[2], ring[kRing];
    // Addresses of the operands in the tiles of S and of the values, which move from stage to stage (formed for every read they cost an
    // instruction each, where the compiler does not see that an offset would do; of the number of the group's first block of columns the lower
    // two bits are swizzled).
    int at_e[8], at_r[KR], at_v[8];
    {
      const int first_block = cg * DB, block_xor = (first_block & 3) << 6, block_off = (first_block >> 2) * 256;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        at_e[i] = smem0 + (Swz<EA>::row_base(lane) ^ (i << 5));
        at_v[i] = smem0 + (Swz<EA>::tr_base(lane, i >> 2) ^ block_xor ^ ((i & 3) << 6)) + block_off;
      }
#pragma unroll
      for (int i = 0; i < KR; ++i) at_r[i] = smem0 + SM::A + (Swz<kLatentTail>::row_base(lane) ^ (i << 5));
      arrived(at_e);
      arrived(at_r);
      arrived(at_v);
    }
    auto onward = [&](auto& at, int j) __attribute__((always_inline)) {      // from the stage of tile j to that of j + 1
      const int by = ((j - j0) & (SM::STAGES - 1)) == SM::STAGES - 1 ? -(SM::STAGES - 1) * SM::STAGE : SM::STAGE;
#pragma unroll
      for (auto& x : at) x += by;
      arrived(at);
    };
    auto read_s = [&](int k) __attribute__((always_inline)) { return k < KE ? lds_read<op_t>(at_e[k & 7] + (k >> 3) * 256) : lds_read<op_t>(at_r[k - KE]); };
    auto read_v = [&](int i) __attribute__((always_inline)) {
      const int b = i % DB, off = i / DB * 16 * Swz<EA>::ROWB + (b >> 2) * 256;
      const auto lo = __builtin_bit_cast(typename Tr::q4_t, lds_read_tr_at(at_v[b & 3] + off));
      const auto up = __builtin_bit_cast(typename Tr::q4_t, lds_read_tr_at(at_v[4 + (b & 3)] + off));
      return __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    // x = S of a tile.  Behind its MFMAs: tile `next` is fetched, and the first operands of the values that come next are read.
    auto scores = [&](int next, int& holes_next, auto goes_on) __attribute__((always_inline)) {
      constexpr bool on = decltype(goes_on)::value;
#pragma unroll
      for (int k = 0; k < kRing - 1; ++k) ring[k] = read_s(k);
#pragma unroll
      for (int k = 0; k < kS; ++k) {
        constexpr int kAhead = kRing - 1;
        if (k + kAhead < kS) ring[(k + kAhead) % kRing] = read_s(k + kAhead);
        else if (on && k + kAhead - kS < kV) ring[(k + kAhead) % kRing] = read_v(k + kAhead - kS);
        x[0] = Tr::mfma(ring[k % kRing], q[k], k == 0 ? f32x16{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f} : x[0]);
        if (on) {
          if (k == 0) fetch_page(next);
          if (k == 1) fetch_rows(next);
          if (k == 2) fetch_rsrc();
          if (k == 3) holes_next = fetch_holes();
          if (k % 3 == 1 && k > 3 && k / 3 - 1 < kPieces) fetch_piece(k / 3 - 1);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // scores that a lane's row does not see of tile j (x[i] is key 8 (i / 4) + 4 hi + i % 4), where there may be some
    auto hide = [&](int j, int hol, float to) __attribute__((always_inline)) {
      if (hol == 0 && j * 32 + 31 <= see_least) return;
      const int n = see - j * 32 - 4 * hi, limit[2] = {hol & 1 ? -1 : n, hol & 2 ? -1 : n};
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (8 * (i / 4) + i % 4 > limit[i / 8]) x[0][i] = to;
    };
    // P of tile j from x, with the rows' maxima as they are after it
    auto full_step = [&](int j, int hol, auto rescale) __attribute__((always_inline)) {
      hide(j, hol, sm.hidden());
      sm.step(x, rescale);
#pragma unroll
      for (int t = 0; t < 2; ++t) p_next[t] = pack8<T>(x[0], t);
    };
    // O += X(j)^T P(j)^T, and P of tile j + 1 from x behind its MFMAs, against the maxima that the rows have (an element's three parts behind
    // different ones, as in fa_fwd_wide.h); returns whether they will do.  The first operands are there or on their way.
    auto values = [&](int j, int hol) __attribute__((always_inline)) {
      constexpr int kLag = 2, kFrom = kV > 8 ? 2 : 0;      // (S comes out of its last MFMA meanwhile)
      hide(j + 1, hol, -__builtin_inff());
      const float msc = sm.m * sm.sc;
      float sum = 0.f;
      uint32_t words[8];
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        if (i + kRing - 1 < kV) ring[(kS + i + kRing - 1) % kRing] = read_v(i + kRing - 1);
        if constexpr (kFull) mfma_acc<T>(o[i % DB], ring[(kS + i) % kRing], p[i / DB]);
        else o[i % DB] = Tr::mfma(ring[(kS + i) % kRing], p[i / DB], o[i % DB]);
#pragma unroll
        for (int E = i < kFrom ? 0 : first_of(i - kFrom, 16 + kLag, kV - kFrom); E < (i < kFrom ? 0 : first_of(i + 1 - kFrom, 16 + kLag, kV - kFrom)); ++E) {
          if (E < 16) x[0][E] = __builtin_fmaf(x[0][E], sm.sc, -msc);
          if (E >= kLag / 2 && E < 16 + kLag / 2) x[0][E - kLag / 2] = fast_exp2(x[0][E - kLag / 2]);
          if (E >= kLag) {
            const int e2 = E - kLag;
            sum += x[0][e2];
            if (e2 & 1) words[e2 / 2] = __builtin_bit_cast(uint32_t, Tr::cvt2(x[0][e2 - 1], x[0][e2]));
            // (here and not behind the last MFMA, where the compiler would have them)
            asm volatile("" : "+v"(sum));
            if (e2 & 1) asm volatile("" : "+v"(words[e2 / 2]));
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      // (also catches inf and NaN)
      if ((sm.prescale && hol != 3) || __builtin_amdgcn_ballot_w64(!(sum < 4096.f)) != 0) return false;
      sm.l += sum;
#pragma unroll
      for (int t = 0; t < 2; ++t) p_next[t] = __builtin_bit_cast(op_t, u32x4_t{words[4 * t], words[4 * t + 1], words[4 * t + 2], words[4 * t + 3]});
      return true;
    };
    using yes = std::true_type;
    using no = std::false_type;
    const int jw = j1 < wave_end ? j1 : wave_end;      // the wave's tiles end here
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(2 * kLoads) : "memory");
    if (j0 < jw) {
      scores(0, holes, no{});
      full_step(j0, holes, [](float) {});
    }
    // In a round: S of the next tile, then the values of this one with the exponentials of the next behind them.  Tiles are fetched three
    // ahead, into the stage of the one before this; those behind the last are empty.
    for (int j = j0; j < j1; ++j) {
#pragma unroll
      for (int t = 0; t < 2; ++t) p[t] = p_next[t];
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(kLoads) : "memory");
      pages.to((j + 3 - j0) * 2);
      int holes3 = 0;
      if (j + 1 < jw) {
        onward(at_e, j);
        onward(at_r, j);
        scores(j + 3, holes3, yes{});
      } else {
        holes3 = fetch(j + 3);
#pragma unroll
        for (int i = 0; i < kRing - 1 && i < kV; ++i) ring[(kS + i) % kRing] = read_v(i);
      }
      const bool done = j >= jw || values(j, j + 1 < jw ? holes1 : 3);
      onward(at_v, j);
      if (!done) {
        scores(0, holes3, no{});
        full_step(j + 1, holes1, [&](float f) __attribute__((always_inline)) {
#pragma unroll
          for (int b = 0; b < DB; ++b) {
            if constexpr (kFull) asm volatile("s_nop 15\n\ts_nop 7" : "+a"(o[b]));
            f32x16 t = o[b];
            t *= f;
            if constexpr (kFull) asm volatile("" : "+v"(t));
            o[b] = t;
            if constexpr (kFull) asm volatile("s_nop 3" : "+a"(o[b]));
          }
        });
      }
      holes1 = holes2;
      holes2 = holes3;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");      // (all waves have left the stages)
    if constexpr (kFull) settle(o);
    // (the row once more, as above)
    const int tail_lane = own_lane(), up = tail_lane >> 5, out_row = w0 + (tail_lane & 31);
    const float sum = cross_sum(sm.l);
    if (a.heads != nullptr && j0 == 0) {
      const int at = latent_block(a, z, s.start) + block;
      if (at < a.blocks && threadIdx.x == 0) {
        a.heads[at] = n_tiles < block_tiles ? LatentHead{(int)worker * 2 + 1, (int)latent_div(at_unit + a.margin + block_tiles - 1 - u, cut.per) + 1, s.start, block, rows}
                                        : LatentHead{0, 0, 0, 0, 0};
      }
      if (at_unit == 0) put_heads(0, at);
      if (block == s.blocks - 1) {
        int next = a.blocks;
        for (int y = z + 1; y < ca.sequences; ++y) {
          const LatentSeq t = latent_cache_seq(a, y);
          if (t.blocks > 0) {
            next = latent_block(a, y, t.start);
            break;
          }
        }
        put_heads(at + 1, next);
      }
    }
    if (n_tiles < block_tiles) {      // a piece, the first of the worker or its last
      if (w0 < rows) {
        const int place = j0 > 0 ? 0 : 1;
        const int64_t at = (worker * 2 + place) * RW + rw;
        float* to = a.part_o + at * (EA / 32 * 1024) + cg * DB * 1024 + tail_lane * 4;
  #pragma unroll
        for (int b = 0; b < DB; ++b) {
  #pragma unroll
          for (int g = 0; g < 4; ++g) *reinterpret_cast<f32x4*>(to + (4 * b + g) * 256) = f32x4{o[b][4 * g], o[b][4 * g + 1], o[b][4 * g + 2], o[b][4 * g + 3]};
          __builtin_amdgcn_sched_barrier(0);
        }
        if (cg == 0) a.part_ml[at * 64 + tail_lane] = tail_lane < 32 ? sm.m : sum;
      }
    } else {
      // O passes through the wave's stage, so that rows go out whole (as a lane's row in pieces of 8 bytes: 19 us for 128 rows)
      constexpr int W = DB * 32, ROW = W * 2 + 16, LPO = W / 8, RPO = 64 / LPO;
      static_assert(32 * ROW <= SM::STAGE, "the rows fit");
      const int r = out_row < rows ? out_row : rows - 1, t = r / a.hq, h = r - t * a.hq, t0 = __builtin_amdgcn_readfirstlane(t);
      const float f = sum == 0.f ? 0.f : 1.0f / sum;
      const int place = smem0 + wave * SM::STAGE;
#pragma unroll
      for (int b = 0; b < DB; ++b) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          typename Tr::q4_t y;
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = Tr::cvt(o[b][4 * g + i] * f);
          lds_write(place + (tail_lane & 31) * ROW + (32 * b + 8 * g + 4 * up) * 2, y);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (a.lse != nullptr && up == 0 && cg == 0 && out_row < rows) a.lse[(int64_t)(s.start + t) * a.hq + h] = sm.lse(sum);
      const int off = (int)((t - t0) * a.o_row + h * a.o_head), lpo = tail_lane % LPO, col = cg * W + lpo * 8;
      T* to = reinterpret_cast<T*>(a.out) + (int64_t)(s.start + t0) * a.o_row + col;
#pragma unroll
      for (int i = 0; i < 32 / RPO; ++i) {
        const int r1 = i * RPO + tail_lane / LPO, at = RPO == 1 ? __builtin_amdgcn_readlane(off, i) : __shfl(off, r1);
        const u32x4_t y = lds_read<u32x4_t>(place + r1 * ROW + lpo * 16);
        if (w0 + r1 < rows && col < ev) *reinterpret_cast<u32x4_t*>(to + at) = y;
      }
    }
    at_unit += span;
    ++block;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");      // (what comes next takes the rows' place)
  }
}

// The pieces of a block put together: a workgroup per 32 rows and `wide` blocks of 32 columns.  A block that one worker had is written already.
// Bound by round trips to memory for few rows (hence 16 loads at a time: 33 pieces one after the other took 22 us), by the pieces' bytes for many.
template <typename T, int EA, int RW>
__global__ __launch_bounds__(256) void latent_cache_sum_kernel(const LatentCacheArgs a, int wide) {
  constexpr int DB = EA / 32;
  const int per = DB / wide, db0 = blockIdx.x % per * wide, rw = blockIdx.x / per % RW;
  const LatentHead head_of = a.heads[blockIdx.x / per / RW];
  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5, c = lane & 31, row = head_of.block * a.block_rows + rw * 32 + c;
  const int w0 = head_of.piece / 2, w1 = w0 + head_of.pieces - 1;
  // (offsets of sequences that do not ascend leave heads that nobody wrote)
  if (head_of.pieces <= 0 || w0 < 0 || w1 < w0 || w1 >= a.workers || head_of.block < 0 || row < 0 || row >= head_of.rows) return;
  if (head_of.start < 0 || (int64_t)head_of.start * a.hq + row >= (int64_t)a.rows * a.hq) return;
  auto at = [&](int w) { return (int64_t)(w == w0 ? head_of.piece : w * 2) * RW + rw; };
  const float sc = score_scale(a.sm_scale, false);
  const int token = row / a.hq, head = row - token * a.hq;
  T* out = reinterpret_cast<T*>(a.out) + (int64_t)(head_of.start + token) * a.o_row + (int64_t)head * a.o_head;
  // N pieces of W blocks of columns at a time
  auto columns = [&](auto n, auto w, int db) __attribute__((always_inline)) {
    constexpr int N = decltype(n)::value, W = decltype(w)::value;
    float m = kNegBig, l = 0.f;
    f32x4 x[W];
#pragma unroll
    for (int k = 0; k < W; ++k) x[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int w = w0; w <= w1; w += N) {
      float pm[N], pl[N];
      f32x4 px[N][W];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t p = at(w + i < w1 ? w + i : w1);
        pm[i] = a.part_ml[p * 64 + c];
        pl[i] = a.part_ml[p * 64 + 32 + c];
#pragma unroll
        for (int k = 0; k < W; ++k) px[i][k] = *reinterpret_cast<const f32x4*>(a.part_o + p * (DB * 1024) + (db + k) * 1024 + tid * 4);
      }
      float top = m;
#pragma unroll
      for (int i = 0; i < N; ++i) top = fmaxf(top, pm[i]);
      const float f = fast_exp2((m - top) * sc);
      m = top;
      l *= f;
#pragma unroll
      for (int k = 0; k < W; ++k) x[k] *= f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (w + i > w1) continue;
        const float g = fast_exp2((pm[i] - top) * sc);
        l += g * pl[i];
#pragma unroll
        for (int k = 0; k < W; ++k) x[k] += g * px[i][k];
      }
    }
    const float f = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const int col = 32 * (db + k) + 8 * (tid >> 6) + 4 * hi;
      typename Traits<T>::q4_t y;
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] = Traits<T>::cvt(x[k][r] * f);
      if (col < a.cache.head_dim_v) *reinterpret_cast<typename Traits<T>::q4_t*>(out + col) = y;
    }
    if (a.lse != nullptr && db == 0 && tid < 32)
      a.lse[(int64_t)(head_of.start + token) * a.hq + head] = l == 0.f ? __builtin_inff() : __builtin_fmaf(m, sc, fast_log2(l)) * kLn2;
  };
  using std::integral_constant;
  int db = db0;
  if (head_of.pieces <= 4)
    for (; db + 4 <= db0 + wide; db += 4) columns(integral_constant<int, 4>{}, integral_constant<int, 4>{}, db);
  if (head_of.pieces <= 8)
    for (; db + 2 <= db0 + wide; db += 2) columns(integral_constant<int, 8>{}, integral_constant<int, 2>{}, db);
  for (; db < db0 + wide; ++db) columns(integral_constant<int, 16>{}, integral_constant<int, 1>{}, db);
}

template <typename T, int EA, int RW, bool kCut> hipError_t launch_latent_cache_main(const LatentCacheArgs& a, hipStream_t s) {
  static std::atomic<uint64_t> done{0};
  const hipError_t e = allow_large_lds(reinterpret_cast<const void*>(&latent_cache_kernel<T, EA, RW, kCut>), LatentCacheSmem<EA>::BYTES, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((latent_cache_kernel<T, EA, RW, kCut>), dim3((unsigned)a.workers), dim3(256), LatentCacheSmem<EA>::BYTES, s, a);
  return hipGetLastError();
}
template <typename T, int EA, int RW> hipError_t launch_latent_cache_rows(const LatentCacheArgs& a, hipStream_t s) {
  const hipError_t e = (a.cache.head_dim < EA ? launch_latent_cache_main<T, EA, RW, true> : launch_latent_cache_main<T, EA, RW, false>)(a, s);
  if (e != hipSuccess) return e;
  if (a.part_o != nullptr && a.cache.sequences > 0) {
    int wide = 1;      // (two rounds of workgroups, or nearly)
    while (wide < EA / 32 && (int64_t)a.blocks * RW * (EA / 32) / wide > 4096) wide *= 2;
    hipLaunchKernelGGL((latent_cache_sum_kernel<T, EA, RW>), dim3((unsigned)(a.blocks * RW * (EA / 32 / wide))), dim3(256), 0, s, a, wide);
  }
  return hipGetLastError();
}


}  // namespace fa
