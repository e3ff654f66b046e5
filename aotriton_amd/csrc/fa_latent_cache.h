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
#pragma once
#include "fa_cache.h"
#include "fa_latent_args.h"
#include "fa_latent_parts.h"

namespace fa {

constexpr int kLatentTail = 64;

template <int EA> struct LatentCacheSmem {
  static constexpr int A = 32 * EA * 2, STAGE = A + 32 * kLatentTail * 2, STAGES = 4;
  static constexpr int LIST = STAGES * STAGE;           // words of latent_find
  static constexpr int BYTES = LIST + 64;
};

// A sequence as the list of work has it: `blocks` blocks of rows, `tiles` tiles each (one at least, for rows that see nothing).
struct LatentSeq {
  int32_t start, tokens, length, end;      // first row of Q, tokens, filled slots, slots with the new ones as far as the table goes
  int32_t blocks, tiles;
  __device__ __forceinline__ int64_t units() const { return (int64_t)blocks * tiles; }
};
__device__ __forceinline__ LatentSeq latent_cache_seq(const LatentCacheArgs& a, int z) {
  auto hold = [](int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; };
  LatentSeq s;
  s.start = hold(a.starts[z], 0, a.rows);
  s.tokens = hold(hold(a.starts[z + 1], 0, a.rows) - s.start, 0, a.rows);
  s.length = a.cache.lengths[z];
  const int64_t room = (int64_t)a.cache.columns << a.cache.page_shift, end = (int64_t)s.length + s.tokens;
  s.end = s.length < 0 ? 0 : (int)(end < room ? end : room);
  s.blocks = (int)(((int64_t)s.tokens * a.hq + a.block_rows - 1) / a.block_rows);
  s.tiles = s.end > 32 ? (s.end + 31) / 32 : 1;
  return s;
}

// The cut of the list: its length, that of a piece, and of the sequence looked for its number and where it starts in the list.  `mine(z, first
// unit, sequence)` says which one that is.  All 256 threads call this.
struct LatentCut { int64_t per, total, first; int z; };
template <typename Mine>
__device__ __forceinline__ LatentCut latent_find(const LatentCacheArgs& a, char* words, Mine mine) {
  int64_t* sums = reinterpret_cast<int64_t*>(words);      // of the four waves; then the answer
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.cache.sequences;
  LatentCut cut{0, 0, 0, -1};
  int64_t base = 0;
  LatentSeq s;
  int64_t before = 0;
  auto chunk = [&](int z0) {      // this thread's sequence and the units in front of it
    const int z = z0 + tid;
    int64_t u = 0;
    if (z < n) {
      s = latent_cache_seq(a, z);
      u = s.units();
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
  const int64_t even = (base + a.workers - 1) / a.workers;
  cut.per = even > a.least ? even : a.least;
  if (tid == 0) sums[5] = -1;
  __syncthreads();
  if (n > 256) base = 0;
  for (int z0 = 0; z0 < n; z0 += 256) {
    if (n > 256) chunk(z0);
    const int z = z0 + tid;
    if (z < n && s.units() > 0 && mine(cut, z, before, s)) {
      sums[4] = before;
      sums[5] = z;
    }
    if (n > 256) __syncthreads();
  }
  __syncthreads();
  cut.first = sums[4];
  cut.z = (int)sums[5];
  return cut;
}

// Behind the last MFMA onto the accumulators, which the compiler does not see (fa_wide.h): 16 passes and what the register file takes.
template <int DB> __device__ __forceinline__ void settle(f32x16 (&o)[DB]) {
#pragma unroll
  for (int b = 0; b < DB; ++b) asm volatile("" : "+a"(o[b]));
  asm volatile("s_nop 15\n\ts_nop 15");
#pragma unroll
  for (int b = 0; b < DB; ++b) asm volatile("" : "+a"(o[b]));
}

template <typename T, int EA, int RW>
__global__ __launch_bounds__(256, 1) void latent_cache_kernel(const LatentCacheArgs a) {
  using Tr = Traits<T>;
  using op_t = typename Tr::op_t;
  using SM = LatentCacheSmem<EA>;
  constexpr int KE = EA / 16, KR = kLatentTail / 16, CG = 4 / RW, DB = EA / 32 / CG;
  // O takes all accumulation registers: its MFMAs are written as asm (fa_wide.h), and scores have to be in vector registers; the compiler, left
  // to place the two, spills a thousand bytes.
  constexpr bool kFull = DB == 16;
  extern __shared__ __attribute__((aligned(kSwzAlign))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), rw = wave % RW, cg = wave / RW;
  const CacheArgs& ca = a.cache;
  const int e = ca.head_dim, ev = ca.head_dim_v;

  // rows of no sequence
  {
    const int n = ca.sequences;
    const int first = n > 0 ? a.starts[0] : a.rows, last = n > 0 ? a.starts[n] : 0;
    const int gap = first < 0 ? 0 : first > a.rows ? a.rows : first, end = last < gap ? gap : last;
    for (int i = blockIdx.x; i < gap + (a.rows - end); i += gridDim.x) {
      const int row = i < gap ? i : end + i - gap;
      for (int x = tid; x < a.hq * (ev / 8); x += 256) {
        const int h = x / (ev / 8), col = x % (ev / 8) * 8;
        *reinterpret_cast<u32x4_t*>(reinterpret_cast<T*>(a.out) + (int64_t)row * a.o_row + (int64_t)h * a.o_head + col) = u32x4_t{0, 0, 0, 0};
        if (a.lse != nullptr && col == 0) a.lse[(int64_t)row * a.hq + h] = __builtin_inff();
      }
    }
    if (n == 0) return;
  }
  const int64_t worker = blockIdx.x;
  const LatentCut cut = latent_find(a, smem + SM::LIST, [&](const LatentCut& t, int, int64_t first, const LatentSeq& s) {
    return first <= worker * t.per && worker * t.per < first + s.units();
  });
  int64_t u = worker * cut.per;
  const int64_t u_end = u + cut.per < cut.total ? u + cut.per : cut.total;
  if (u >= u_end) return;
  int z = __builtin_amdgcn_readfirstlane(cut.z);
  int64_t first = cut.first;

  const int smem0 = lds_offset(smem);
  // What depends on the lane alone is formed where it is needed: held through the loop over tiles, which Q and O leave little room, it would be
  // spilled, and a reload waits for the tiles that are on their way.
  auto own_lane = [&]() __attribute__((always_inline)) { int l = threadIdx.x; asm volatile("" : "+v"(l)); return l & 63; };
  const int x_row = (int)ca.sk.s * 2;
  constexpr int LPR = EA / 8, RPL = 64 / LPR;      // lanes of a row, rows of an access
  while (u < u_end) {
    LatentSeq s = latent_cache_seq(a, z);
    s.start = __builtin_amdgcn_readfirstlane(s.start); s.tokens = __builtin_amdgcn_readfirstlane(s.tokens);
    s.length = __builtin_amdgcn_readfirstlane(s.length); s.end = __builtin_amdgcn_readfirstlane(s.end);
    s.tiles = __builtin_amdgcn_readfirstlane(s.tiles); s.blocks = __builtin_amdgcn_readfirstlane(s.blocks);
    if (u - first >= s.units()) {      // (the next one that has rows)
      first += s.units();
      ++z;
      continue;
    }
    const int block = (int)((u - first) / s.tiles), j0 = (int)((u - first) % s.tiles);
    const int n_tiles = (int)(u_end - u < s.tiles - j0 ? u_end - u : s.tiles - j0);
    const int rows = s.tokens * a.hq, w0 = block * a.block_rows + rw * 32, w_last = w0 + 31 < rows ? w0 + 31 : rows - 1;
    const bool row_ok = w0 + c < rows;
    const int row = row_ok ? w0 + c : rows - 1, token = row / a.hq, head = row - token * a.hq;
    // the last slot that the row sees, that the wave's first and last rows see
    auto sees = [&](int t) { const int n = s.length + t; return n < s.end ? n : s.end - 1; };
    const int see = sees(token);
    const int see_least = __builtin_amdgcn_readfirstlane(sees(w0 / a.hq)), see_most = __builtin_amdgcn_readfirstlane(sees(w_last / a.hq));
    const int j1 = j0 + n_tiles, wave_end = w0 < rows ? see_most / 32 + 1 : 0;

    auto slot_of = [&](int entry) { const int n = (j0 + entry / 2) * 32 + entry % 2 * 16; return entry < 2 * n_tiles && n < s.end ? n : -1; };
    PageRun<decltype(slot_of)> pages(ca, z, lane, slot_of);
    const char* xbase = reinterpret_cast<const char*>(ca.k);
    auto fetch = [&](int j) __attribute__((always_inline)) {      // returns which of the tile's halves have no page
      pages.to((j - j0) * 2);
      const int n = j * 32 + wave * 8, left = s.end - n < 8 ? s.end - n : 8;
      const int p = pages.at((j - j0) * 2 + wave / 2);
      const char* from = xbase + ((int64_t)(p < 0 ? 0 : p) * ca.sk.z + (int64_t)(n & ((1 << ca.page_shift) - 1)) * ca.sk.s) * 2;
      const u32x4_t rs = wave_rsrc_words(from, p < 0 ? 0 : rows_extent(left, x_row, e * 2));
      const int lds = smem0 + ((j - j0) & (SM::STAGES - 1)) * SM::STAGE, lds_a = lds + wave * 8 * EA * 2;
      const int l = own_lane(), lrow = l / LPR, lch = l % LPR;
#pragma unroll
      for (int i = 0; i < 8 / RPL; i += 2) {
        int voff[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int ch = lch ^ Swz<EA>::f((i + t) * RPL + lrow + 8 * (wave & 1));
          voff[t] = ch * 8 < e ? lrow * x_row + ch * 16 : kVoffOutOfRange;
        }
        load_to_lds(rs, voff[0], i * RPL * x_row, lds_a + i * 1024, voff[1], (i + 1) * RPL * x_row, lds_a + (i + 1) * 1024);
      }
      const int ch = (l % 8) ^ Swz<kLatentTail>::f(8 * (wave & 1) + l / 8);      // (a wave's eight rows are the first or second of 16)
      load_to_lds1(rs, EA + ch * 8 < e ? l / 8 * x_row + (EA + ch * 8) * 2 : kVoffOutOfRange, lds + SM::A + wave * 1024);
      return pages.holes((j - j0) * 2) & 3;
    };
    // (tiles are fetched two ahead; their pages are looked up 32 tiles at a time)
    int holes = fetch(j0), holes1 = 0, holes2 = 0;

    op_t q[KE + KR];
    {
      const int t0 = w0 < rows ? w0 / a.hq : 0, t1 = w_last / a.hq;
      const T* qp = reinterpret_cast<const T*>(a.q) + (int64_t)(s.start + t0) * a.q_row;
      const auto rs = wave_rsrc(qp, w0 < rows ? (int)(((t1 - t0) * a.q_row + (a.hq - 1) * a.q_head + e) * 2) : 0);
      const int at = row_ok ? (int)(((token - t0) * a.q_row + head * a.q_head) * 2) : kVoffOutOfRange;
#pragma unroll
      for (int k = 0; k < KE + KR; ++k) {
        const int col = 16 * k + 8 * hi;
        q[k] = __builtin_bit_cast(op_t, __builtin_amdgcn_raw_buffer_load_b128(rs, col < e ? at + col * 2 : kVoffOutOfRange, 0, 0));
      }
    }
    // (Q has to be there before the loop: left to the first use in it the compiler waits there, in every round, for all that is on its way)
    arrived(q);
    if (n_tiles > 1) holes1 = fetch(j0 + 1);
    f32x16 o[DB];
#pragma unroll
    for (int b = 0; b < DB; ++b) {
      if constexpr (kFull) acc_zero<T>(o[b]);
      else o[b] = f32x16{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    }
    RowSoftmax sm(a.sm_scale);

    for (int j = j0; j < j1; ++j, holes = holes1, holes1 = holes2) {
      constexpr int kLoads = 8 / RPL + 1;      // of a tile
      if (j + 1 < j1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(kLoads) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (j + 2 < j1) holes2 = fetch(j + 2);
      if (j >= wave_end) continue;
      // (a few operands at a time are on their way: left to itself the compiler keeps dozens)
      const int X = smem0 + ((j - j0) & (SM::STAGES - 1)) * SM::STAGE;
      const int at_e = Swz<EA>::row_base(own_lane()), at_r = Swz<kLatentTail>::row_base(own_lane());
      auto k_read = [&](int k) __attribute__((always_inline)) {
        return k < KE ? lds_read<op_t>((at_e ^ ((k & 7) << 5)) + X + (k >> 3) * 256) : lds_read<op_t>((at_r ^ ((k - KE) << 5)) + X + SM::A);
      };
      constexpr int kRing = 5;
      f32x16 x[1];
      op_t xa[kRing];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[0][i] = 0.f;
#pragma unroll
      for (int k = 0; k < kRing - 1; ++k) xa[k] = k_read(k);
#pragma unroll
      for (int k = 0; k < KE + KR; ++k) {
        if (k + kRing - 1 < KE + KR) xa[(k + kRing - 1) % kRing] = k_read(k + kRing - 1);
        x[0] = Tr::mfma(xa[k % kRing], q[k], x[0]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (holes != 0) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (holes >> (i / 8) & 1) x[0][i] = -__builtin_inff();
      }
      sm.step(x, j * 32 + 31 > see_least, see - j * 32 - 4 * hi, [&](float f) __attribute__((always_inline)) {
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
      op_t p[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) p[t] = pack8<T>(x[0], t);
      if constexpr (kFull) asm volatile("s_nop 1" : "+v"(p[0]), "+v"(p[1]));
      // (the group's first block of columns: of its number the lower two bits are swizzled)
      const int first_block = cg * DB, block_xor = (first_block & 3) << 6, block_off = (first_block >> 2) * 256;
      const int at_0 = (Swz<EA>::tr_base(own_lane(), 0) ^ block_xor) + block_off, at_1 = (Swz<EA>::tr_base(own_lane(), 1) ^ block_xor) + block_off;
      auto v_read = [&](int i) __attribute__((always_inline)) {
        const int b = i % DB, off = X + i / DB * 16 * Swz<EA>::ROWB + (b >> 2) * 256;
        const auto lo = __builtin_bit_cast(typename Tr::q4_t, lds_read_tr_at((at_0 ^ ((b & 3) << 6)) + off));
        const auto up = __builtin_bit_cast(typename Tr::q4_t, lds_read_tr_at((at_1 ^ ((b & 3) << 6)) + off));
        return __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
      };
#pragma unroll
      for (int i = 0; i < kRing - 1; ++i) xa[i] = v_read(i);
#pragma unroll
      for (int i = 0; i < 2 * DB; ++i) {
        if (i + kRing - 1 < 2 * DB) xa[(i + kRing - 1) % kRing] = v_read(i + kRing - 1);
        if constexpr (kFull) mfma_acc<T>(o[i % DB], xa[i % kRing], p[i / DB]);
        else o[i % DB] = Tr::mfma(xa[i % kRing], p[i / DB], o[i % DB]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (kFull) settle(o);
    // (the row once more, as above)
    const int tail_lane = own_lane(), up = tail_lane >> 5, out_row = w0 + (tail_lane & 31);
    const float sum = cross_sum(sm.l);
    if (n_tiles < s.tiles) {      // a piece: the first of the worker, or its last
      const int place = u == worker * cut.per ? 0 : 1;
      const int64_t at = (worker * 2 + place) * RW + rw;
      float* to = a.part_o + at * (EA / 32 * 1024) + cg * DB * 1024 + tail_lane * 4;
#pragma unroll
      for (int b = 0; b < DB; ++b) {
#pragma unroll
        for (int g = 0; g < 4; ++g) *reinterpret_cast<f32x4*>(to + (4 * b + g) * 256) = f32x4{o[b][4 * g], o[b][4 * g + 1], o[b][4 * g + 2], o[b][4 * g + 3]};
        __builtin_amdgcn_sched_barrier(0);
      }
      if (cg == 0) a.part_ml[at * 64 + tail_lane] = tail_lane < 32 ? sm.m : sum;
    } else if (out_row < rows) {
      const float f = sum == 0.f ? 0.f : 1.0f / sum;
      const int t = out_row / a.hq, h = out_row - t * a.hq;
      T* to = reinterpret_cast<T*>(a.out) + (int64_t)(s.start + t) * a.o_row + (int64_t)h * a.o_head;
#pragma unroll
      for (int b = 0; b < DB; ++b) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int col = 32 * (cg * DB + b) + 8 * g + 4 * up;
          typename Tr::q4_t y;
#pragma unroll
          for (int r = 0; r < 4; ++r) y[r] = Tr::cvt(o[b][4 * g + r] * f);
          if (col < ev) *reinterpret_cast<typename Tr::q4_t*>(to + col) = y;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (a.lse != nullptr && up == 0 && cg == 0) a.lse[(int64_t)(s.start + t) * a.hq + h] = sm.lse(sum);
    }
    u += n_tiles;
    __syncthreads();      // (the next segment's first tile takes the place of one that may still be read)
  }
}

// The pieces of a block put together: a workgroup per 32 rows and `wide` blocks of 32 columns.  A block that one worker had is written already.
// Bound by round trips to memory for few rows (hence eight pieces at a time: 33 of them one after the other took 22 us), by the pieces' bytes for many.
template <typename T, int EA, int RW>
__global__ __launch_bounds__(256) void latent_cache_sum_kernel(const LatentCacheArgs a, int wide) {
  __shared__ __attribute__((aligned(8))) char words[64];
  constexpr int DB = EA / 32;
  const int per = DB / wide, db0 = blockIdx.x % per * wide, rw = blockIdx.x / per % RW, vb = blockIdx.x / per / RW;
  // (blocks numbered with a gap or two: those of sequence z start at its first row's number divided by the rows of a block, plus z)
  auto base_of = [&](int z, const LatentSeq& s) { return (int)((int64_t)s.start * a.hq / a.block_rows) + z; };
  const LatentCut cut = latent_find(a, words, [&](const LatentCut&, int z, int64_t, const LatentSeq& s) {
    const int base = base_of(z, s);
    return base <= vb && vb < base + s.blocks;
  });
  if (cut.z < 0) return;
  const LatentSeq s = latent_cache_seq(a, cut.z);
  const int block = vb - base_of(cut.z, s);
  const int64_t u0 = cut.first + (int64_t)block * s.tiles, u1 = u0 + s.tiles;
  const int w0 = (int)(u0 / cut.per), w1 = (int)((u1 - 1) / cut.per);
  if (w0 == w1) return;
  const int tid = threadIdx.x, lane = tid & 63, hi = lane >> 5, c = lane & 31, row = block * a.block_rows + rw * 32 + c;
  if (row >= s.tokens * a.hq) return;
  const int first_place = u0 != w0 * cut.per ? 1 : 0;
  auto at = [&](int w) { return ((int64_t)w * 2 + (w == w0 ? first_place : 0)) * RW + rw; };
  const float sc = score_scale(a.sm_scale, false);
  const int token = row / a.hq, head = row - token * a.hq;
  T* out = reinterpret_cast<T*>(a.out) + (int64_t)(s.start + token) * a.o_row + (int64_t)head * a.o_head;
  for (int db = db0; db < db0 + wide; ++db) {
    float m = kNegBig, l = 0.f;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    constexpr int N = 8;
    for (int w = w0; w <= w1; w += N) {
      float pm[N], pl[N];
      f32x4 px[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t p = at(w + i < w1 ? w + i : w1);
        pm[i] = a.part_ml[p * 64 + c];
        pl[i] = a.part_ml[p * 64 + 32 + c];
        px[i] = *reinterpret_cast<const f32x4*>(a.part_o + p * (DB * 1024) + db * 1024 + tid * 4);
      }
      float top = m;
#pragma unroll
      for (int i = 0; i < N; ++i) top = fmaxf(top, pm[i]);
      const float f = fast_exp2((m - top) * sc);
      m = top;
      l *= f;
      x *= f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float g = w + i <= w1 ? fast_exp2((pm[i] - top) * sc) : 0.f;
        l += g * pl[i];
        if (w + i <= w1) x += g * px[i];
      }
    }
    const float f = l == 0.f ? 0.f : 1.0f / l;
    const int col = 32 * db + 8 * (tid >> 6) + 4 * hi;
    typename Traits<T>::q4_t y;
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = Traits<T>::cvt(x[r] * f);
    if (col < a.cache.head_dim_v) *reinterpret_cast<typename Traits<T>::q4_t*>(out + col) = y;
    if (a.lse != nullptr && db == 0 && tid < 32)
      a.lse[(int64_t)(s.start + token) * a.hq + head] = l == 0.f ? __builtin_inff() : __builtin_fmaf(m, sc, fast_log2(l)) * kLn2;
  }
}

template <typename T, int EA, int RW> hipError_t launch_latent_cache_rows(const LatentCacheArgs& a, hipStream_t s) {
  static std::atomic<uint64_t> done{0};
  const hipError_t e = allow_large_lds(reinterpret_cast<const void*>(&latent_cache_kernel<T, EA, RW>), LatentCacheSmem<EA>::BYTES, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((latent_cache_kernel<T, EA, RW>), dim3((unsigned)a.workers), dim3(256), LatentCacheSmem<EA>::BYTES, s, a);
  if (a.part_o != nullptr && a.cache.sequences > 0) {
    const int64_t blocks = (int64_t)a.rows * a.hq / a.block_rows + a.cache.sequences;
    int wide = 1;      // (two rounds of workgroups, or nearly)
    while (wide < EA / 32 && blocks * RW * (EA / 32) / wide > 4096) wide *= 2;
    hipLaunchKernelGGL((latent_cache_sum_kernel<T, EA, RW>), dim3((unsigned)(blocks * RW * (EA / 32 / wide))), dim3(256), 0, s, a, wide);
  }
  return hipGetLastError();
}


}  // namespace fa
