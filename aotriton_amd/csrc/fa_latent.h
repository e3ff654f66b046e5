// Attention whose keys are part per head, part shared by all heads, forward and dQ (dK, dV and dC, and dQ of few workgroups: fa_latent_keys.h): gfx950, MFMA 32x32x16.
//
//   S = scale (Qe K^T + Qr C^T),  P = softmax(S),  O = P V
//   dV = P^T dO,  dS = P (dO V^T - rowsum(dO O)),  dQ = scale [dS K | dS C],  dK = scale dS^T Qe,  dC = scale sum over heads of dS^T Qr
//
// The shared part is never copied per head: its tile stands next to that of K in LDS, and a key is the two of them.  K and V (64 or 128
// compiled columns) and C (64) may have fewer columns each; what is past them reads as zero.
//
// Layouts and products as in fa_fwd_impl.h: a wave owns 32 rows (dK/dV: keys), a lane one of them; tiles come straight into swizzled LDS
// (fa_device.h: Swz), the next one while this one is worked on, and serve row reads and transposing reads alike.
//
// Bound by the matrix pipe, and by what the card's power leaves of its rate: two waves on a SIMD keep it busy 60 % of the time.  16 heads of 8192
// causal tokens, E = Ev = 128, R = 64, bf16: forward 346-360 us (970 TFLOP/s; a product of 8192^3 reaches 1160-1190), dQ 570-580 (950), dK, dV and dC
// 690.  dQ and dK/dV each form S and dP, 25 % of the backward's products, rather than dQ in pieces from the other's blocks: no atomics, results that
// do not change.
#pragma once
#include <algorithm>
#include "fa_device.h"
#include "fa_latent_args.h"
#include "fa_latent_parts.h"
#include "fa_wide.h"

namespace fa {

constexpr int kLatentShared = 64;      // compiled columns of the shared part
constexpr int kLatentFewTiles = 4;     // tiles of 64 keys up to which dQ sums delta itself

// A tile's 64 rows as they come into LDS: 16 rows a wave, 1 KB an access.  A lane's byte offsets of its accesses; the columns start at
// `col0` of the row, and there are `cols` of them.
template <int D> struct TileRows {
  static constexpr int LPR = D / 8, RPL = 64 / LPR, N = 16 / RPL;      // lanes of a row, rows of an access, accesses
  int voff[N];
  __device__ __forceinline__ TileRows(int lane, int row_bytes, int col0, int cols) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = i * RPL + lane / LPR, ch = (lane % LPR) ^ Swz<D>::f(row);
      voff[i] = ch * 8 < cols ? row * row_bytes + (col0 + ch * 8) * 2 : kVoffOutOfRange;
    }
  }
  __device__ __forceinline__ void fetch(u32x4_t rsrc, int lds) const {
#pragma unroll
    for (int i = 0; i < N; ++i) load_to_lds1(rsrc, voff[i], lds + i * 1024);
  }
};

// A wave's 32 rows on their way into `lds`, as TileRows has them: columns [col0, col0 + cols) of the first `rows` rows, zeros elsewhere.  From there they
// go into registers, and results back the same way: whole rows of memory, which a lane's row in pieces of 8 or 16 bytes leaves to the caches
// (a block of dK/dV spent 35 us on that, as much as on twelve of its tiles).
template <int D>
__device__ __forceinline__ void fetch_rows(const void* base, int row_bytes, int rows, int lane, int col0, int cols, int lds) {
  const TileRows<D> t(lane, row_bytes, col0, cols);
#pragma unroll
  for (int i = 0; i < 2; ++i)
    t.fetch(wave_rsrc_words(reinterpret_cast<const char*>(base) + (int64_t)(16 * i) * row_bytes, rows_extent(rows - 16 * i < 16 ? rows - 16 * i : 16, row_bytes, (col0 + cols) * 2)),
            lds + i * 16 * 2 * D);
}
// as MFMA operands, row lane % 32
template <typename T, int D>
__device__ __forceinline__ void take_rows(typename Traits<T>::op_t* x, int lane, int lds) {
  const int at = Swz<D>::row_base(lane);
#pragma unroll
  for (int k = 0; k < D / 16; ++k) x[k] = lds_read<typename Traits<T>::op_t>((at ^ (k << 5)) + lds);
}

// A transposed accumulator (columns x 32 rows) times `f` to the first `rows` rows of a tensor, columns [0, cols), through the wave's piece of LDS (RowsOut bytes).
template <typename T, int NB> constexpr int kRowsOut = 32 * (NB * 32 * (int)sizeof(T) + 16);
template <typename T, int NB>
__device__ __forceinline__ void store_rows(const f32x16* x, float f, T* to, int64_t stride, int rows, int cols, int lane, int lds) {
  constexpr int ROW = NB * 32 * (int)sizeof(T) + 16, LPR = NB * 32 * (int)sizeof(T) / 16, RPL = 64 / LPR, PER = 16 / (int)sizeof(T);
  const int c = lane & 31, hi = lane >> 5;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      vec<T, 4> y;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (sizeof(T) == 4) y[r] = x[b][4 * g + r] * f;
        else y[r] = Traits<T>::cvt(x[b][4 * g + r] * f);
      }
      lds_write(lds + c * ROW + (32 * b + 8 * g + 4 * hi) * (int)sizeof(T), y);
    }
  const int ch = lane % LPR;
#pragma unroll
  for (int i = 0; i < 32 / RPL; ++i) {
    const int r = i * RPL + lane / LPR;
    const u32x4_t y = lds_read<u32x4_t>(lds + r * ROW + ch * 16);
    if (r < rows && ch * PER < cols) *reinterpret_cast<u32x4_t*>(to + r * stride + ch * PER) = y;
  }
}

__device__ __forceinline__ void latent_meet() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int EC> struct LatentSmem {
  static constexpr int TILE = 64 * EC * 2, SHARED = 64 * kLatentShared * 2;
  static constexpr int C_OFF = TILE, V_OFF = TILE + SHARED;
  static constexpr int STAGE = 2 * TILE + SHARED;      // K, C, V (dK/dV: Q, its shared part, dO)
  static constexpr int STATS = 2 * 64 * 4;
  static constexpr int BYTES = 2 * STAGE, BWD_STAGE = STAGE + STATS, BWD_BYTES = 3 * BWD_STAGE, DQ_BYTES = 3 * STAGE;
  // a wave's own rows before and after the loop over tiles: two tensors of EC columns, then one of the shared part
  static constexpr int WAVE = STAGE / 2, WAVE_V = 32 * EC * 2, WAVE_C = 2 * WAVE_V;
};

// (The offsets of packed sequences are held inside the tensors, and lengths inside the greatest: what lies past them is not there, and no kernel reads or
// writes it.)
__device__ __forceinline__ SeqInfo latent_seq(const LatentArgs& a, int z) {
  SeqInfo r{a.seq.max_seqlen_q, a.seq.max_seqlen_k, 0, 0, z, a.rows_q};
  if (a.seq.num_seqlens != 0) {
    auto hold = [](int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; };
    r.q_start = hold(a.seq.cu_q[z], 0, a.rows_q);
    r.k_start = hold(a.seq.cu_k[z], 0, a.rows_k);
    r.seqlen_q = hold(hold(a.seq.cu_q[z + 1], 0, a.rows_q) - r.q_start, 0, a.seq.max_seqlen_q);
    r.seqlen_k = hold(hold(a.seq.cu_k[z + 1], 0, a.rows_k) - r.k_start, 0, a.seq.max_seqlen_k);
    r.batch_index = 0;
  }
  return uniform(r);
}

// (sequence, head, tile) of a workgroup.  LatentArgs::group heads (of all sequences side by side, the last ones the rest) stand side by side, their
// tiles of a kind one behind the other.  Causal tiles have the more keys the later they stand: those first.
__device__ __forceinline__ void latent_item(const LatentArgs& a, int id, int nseq, int tiles, bool backwards, int& z, int& h, int& t) {
  const int pairs = nseq * a.heads, front = id / (a.group * tiles) * a.group, have = pairs - front < a.group ? pairs - front : a.group;
  const int rest = id - front * tiles, zh = front + rest % have;
  t = rest / have;
  if (backwards) t = tiles - 1 - t;
  h = zh % a.heads;
  z = zh / a.heads;
}

template <typename T> __device__ __forceinline__ T* row_at(const void* base, const Strides3& s, const SeqInfo& si, int h, int64_t row) {
  return const_cast<T*>(reinterpret_cast<const T*>(base)) + (int64_t)si.batch_index * s.z + (int64_t)h * s.h + row * s.s;
}

// Number of the slab of a sequence's rows from 32 `block` on.  Packed sequences have theirs one behind the other, each from q_start / 32 + z on: that
// is past those of the sequence in front, ceil(n / 32) of them, and a head has no more than rows / 32 + sequences.  (As many for every sequence as the
// longest has would be 850 MB where one of 2048 tokens stands beside 199 of 4 with one head; so they are 19.)
__device__ __forceinline__ int64_t latent_slab(const LatentArgs& a, const SeqInfo& si, int z, int h, int block) {
  return ((int64_t)si.batch_index * a.heads + h) * a.slabs + si.q_start / 32 + (a.seq.num_seqlens != 0 ? z : 0) + block;
}

// ---- forward -------------------------------------------------------------------------------------------------------
template <typename T, int EC>
__global__ __launch_bounds__(256, 2) void latent_fwd_kernel(const LatentArgs a, int nseq, int tiles) {
  using Tr = Traits<T>;
  using op_t = typename Tr::op_t;
  using SM = LatentSmem<EC>;
  constexpr int KE = EC / 16, KR = kLatentShared / 16, DB = EC / 32;
  extern __shared__ __attribute__((aligned(kSwzAlign))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int z, h, mt;
  const int part = blockIdx.x / (nseq * a.heads) % a.parts;
  latent_item(a, blockIdx.x % (nseq * a.heads) + blockIdx.x / (nseq * a.heads * a.parts) * (nseq * a.heads), nseq, tiles, a.causal != 0, z, h, mt);
  const SeqInfo si = latent_seq(a, z);
  const int q0 = mt * 128;
  if (q0 >= si.seqlen_q) return;
  const int shift = si.seqlen_k - si.seqlen_q;
  const int w0 = q0 + wave * 32, row = w0 + c, rows = si.seqlen_q - w0;
  // key tiles of the workgroup, of the part, of the wave
  auto last_key = [&](int r) { return a.causal ? (r < si.seqlen_q ? r : si.seqlen_q - 1) + shift : si.seqlen_k - 1; };
  auto tiles_of = [&](int r) { const int n = last_key(r) + 1; return n > 0 ? (n + 63) / 64 : 0; };
  const int all = tiles_of(q0 + 127), per = (all + a.parts - 1) / a.parts;
  const int j0 = part * per, j1 = j0 + per < all ? j0 + per : all, wave_end = tiles_of(w0 + 31);
  const int see = last_key(row);

  const int smem0 = lds_offset(smem);
  const int k_row = (int)a.sk.s * 2, v_row = (int)a.sv.s * 2, c_row = (int)a.c_s * 2;
  const TileRows<EC> kt(lane, k_row, 0, a.e), vt(lane, v_row, 0, a.ev);
  const TileRows<kLatentShared> ct(lane, c_row, 0, a.r);
  auto fetch = [&](int stage, int j) __attribute__((always_inline)) {
    const int n = j * 64 + wave * 16, left = si.seqlen_k - n < 16 ? si.seqlen_k - n : 16;
    const int64_t at = si.k_start + n;
    const int lds = smem0 + stage * SM::STAGE + wave * 16 * 2 * EC;
    kt.fetch(wave_rsrc_words(row_at<T>(a.k, a.sk, si, h, at), rows_extent(left, k_row, a.e * 2)), lds);
    vt.fetch(wave_rsrc_words(row_at<T>(a.v, a.sv, si, h, at), rows_extent(left, v_row, a.ev * 2)), lds + SM::V_OFF);
    ct.fetch(wave_rsrc_words(row_at<T>(a.c, Strides3{a.c_z, 0, a.c_s}, si, 0, at), rows_extent(left, c_row, a.r * 2)),
             smem0 + stage * SM::STAGE + SM::C_OFF + wave * 16 * 2 * kLatentShared);
  };
  op_t q[KE + KR];
  {
    const T* qp = row_at<T>(a.q, a.sq, si, h, (int64_t)si.q_start + w0);
    const int own = smem0 + wave * SM::WAVE;
    fetch_rows<EC>(qp, (int)a.sq.s * 2, rows, lane, 0, a.e, own);
    fetch_rows<kLatentShared>(qp, (int)a.sq.s * 2, rows, lane, a.e, a.r, own + SM::WAVE_C);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    take_rows<T, EC>(q, lane, own);
    take_rows<T, kLatentShared>(q + KE, lane, own + SM::WAVE_C);
  }
  // (Q has to be there before the loop: left to the first use in it the compiler waits there, in every round, for all that is on its way)
  arrived(q);
  latent_meet();
  if (j0 < j1) fetch(0, j0);
  f32x16 o[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[b][i] = 0.f;
  RowSoftmax sm(a.sm_scale);
  const int row_e = Swz<EC>::row_base(lane), row_r = Swz<kLatentShared>::row_base(lane);
  const int tr0 = Swz<EC>::tr_base(lane, 0), tr1 = Swz<EC>::tr_base(lane, 1);

  for (int j = j0; j < j1; ++j) {
    latent_meet();
    const int stage = (j - j0) & 1;
    if (j + 1 < j1) fetch(stage ^ 1, j + 1);
    if (j >= wave_end) continue;
    const char* K = smem + stage * SM::STAGE;
    f32x16 s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
#pragma unroll
      for (int k = 0; k < KE; ++k) s[b] = Tr::mfma(swz_read_row<T, EC>(K, row_e, k, b), q[k], s[b]);
#pragma unroll
      for (int k = 0; k < KR; ++k) s[b] = Tr::mfma(swz_read_row<T, kLatentShared>(K + SM::C_OFF, row_r, k, b), q[KE + k], s[b]);
    }
    const int n0 = j * 64;
    const bool masked = n0 + 64 > si.seqlen_k || (a.causal && n0 + 63 > w0 + shift);
    if (masked) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * b + 8 * (i / 4) + i % 4 > see - n0 - 4 * hi) s[b][i] = sm.hidden();
    }
    sm.step(s, [&](float f) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[b][i] *= f;
    });
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const op_t p = pack8<T>(s[t / 2], t % 2);
#pragma unroll
      for (int b = 0; b < DB; ++b) o[b] = Tr::mfma(swz_read_tr<T, EC>(K + SM::V_OFF, tr0, tr1, t, b), p, o[b]);
    }
  }
  if (a.parts > 1) {
    if (rows > 0) store_part<DB>(a.part_o, a.part_ml, latent_slab(a, si, z, h, mt * 4 + wave) * a.parts + part, o, sm, lane);
    return;
  }
  const float l = cross_sum(sm.l);
  if (a.lse != nullptr && hi == 0 && row < si.seqlen_q) a.lse[lse_offset(si, h, a.heads) + row] = sm.lse(l);
  latent_meet();
  store_rows<T, DB>(o, l == 0.f ? 0.f : 1.0f / l, row_at<T>(a.out, a.so, si, h, (int64_t)si.q_start + w0), a.so.s, rows, a.ev, lane, smem0 + wave * SM::WAVE);
}

// the parts' sums of 32 rows and 32 columns put together
template <typename T, int EC>
__global__ __launch_bounds__(256) void latent_fwd_sum_kernel(const LatentArgs a, int nseq, int tiles) {
  constexpr int DB = EC / 32;
  const int db = blockIdx.x % DB, item = blockIdx.x / DB, wave = item % 4, mt = item / 4 % tiles, zh = item / 4 / tiles;
  const int h = zh % a.heads, z = zh / a.heads;
  const SeqInfo si = latent_seq(a, z);
  const int lane = threadIdx.x & 63, hi = lane >> 5, row = mt * 128 + wave * 32 + (lane & 31);
  if (row >= si.seqlen_q) return;
  float lse;
  const vec<float, 4> x = sum_parts<DB>(a.part_o, a.part_ml, latent_slab(a, si, z, h, mt * 4 + wave) * a.parts, a.parts, a.sm_scale, db, threadIdx.x, lse);
  const int col = 32 * db + 8 * (threadIdx.x >> 6) + 4 * hi;
  typename Traits<T>::q4_t y;
#pragma unroll
  for (int r = 0; r < 4; ++r) y[r] = Traits<T>::cvt(x[r]);
  if (col < a.ev) *reinterpret_cast<typename Traits<T>::q4_t*>(row_at<T>(a.out, a.so, si, h, (int64_t)si.q_start + row) + col) = y;
  if (a.lse != nullptr && db == 0 && threadIdx.x < 32) a.lse[lse_offset(si, h, a.heads) + row] = lse;
}

// ---- dQ ------------------------------------------------------------------------------------------------------------
// Rows as in the forward; also delta.
template <typename T, int EC>
__global__ __launch_bounds__(256, 2) void latent_dq_kernel(const LatentBwdArgs a, int nseq, int tiles) {
  using Tr = Traits<T>;
  using op_t = typename Tr::op_t;
  using SM = LatentSmem<EC>;
  constexpr int KE = EC / 16, KR = kLatentShared / 16, DB = EC / 32, RB = kLatentShared / 32;
  extern __shared__ __attribute__((aligned(kSwzAlign))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int z, h, mt;
  latent_item(a, blockIdx.x, nseq, tiles, a.causal != 0, z, h, mt);
  const SeqInfo si = latent_seq(a, z);
  const int q0 = mt * 128;
  if (q0 >= si.seqlen_q) return;
  const int shift = si.seqlen_k - si.seqlen_q;
  const int w0 = q0 + wave * 32, row = w0 + c, rows = si.seqlen_q - w0;
  auto last_key = [&](int r) { return a.causal ? (r < si.seqlen_q ? r : si.seqlen_q - 1) + shift : si.seqlen_k - 1; };
  auto tiles_of = [&](int r) { const int n = last_key(r) + 1; return n > 0 ? (n + 63) / 64 : 0; };
  const int j1 = tiles_of(q0 + 127), wave_end = tiles_of(w0 + 31), see = last_key(row);

  const int smem0 = lds_offset(smem);
  const int k_row = (int)a.sk.s * 2, v_row = (int)a.sv.s * 2, c_row = (int)a.c_s * 2;
  // (what depends on the lane alone is formed anew for every tile: held, it would be spilled, and a reload waits for the tile on its way)
  auto own_lane = [&]() __attribute__((always_inline)) { int l = threadIdx.x; asm volatile("" : "+v"(l)); return l & 63; };
  auto fetch = [&](int stage, int j) __attribute__((always_inline)) {
    const int l = own_lane();
    const TileRows<EC> kt(l, k_row, 0, a.e), vt(l, v_row, 0, a.ev);
    const TileRows<kLatentShared> ct(l, c_row, 0, a.r);
    const int n = j * 64 + wave * 16, left = si.seqlen_k - n < 16 ? si.seqlen_k - n : 16;
    const int64_t at = si.k_start + n;
    const int lds = smem0 + stage * SM::STAGE + wave * 16 * 2 * EC;
    kt.fetch(wave_rsrc_words(row_at<T>(a.k, a.sk, si, h, at), rows_extent(left, k_row, a.e * 2)), lds);
    vt.fetch(wave_rsrc_words(row_at<T>(a.v, a.sv, si, h, at), rows_extent(left, v_row, a.ev * 2)), lds + SM::V_OFF);
    ct.fetch(wave_rsrc_words(row_at<T>(a.c, Strides3{a.c_z, 0, a.c_s}, si, 0, at), rows_extent(left, c_row, a.r * 2)),
             smem0 + stage * SM::STAGE + SM::C_OFF + wave * 16 * 2 * kLatentShared);
  };
  op_t q[KE + KR], dout[KE];
  const int own = smem0 + wave * SM::WAVE;
  {
    const T* qp = row_at<T>(a.q, a.sq, si, h, (int64_t)si.q_start + w0);
    fetch_rows<EC>(qp, (int)a.sq.s * 2, rows, lane, 0, a.e, own);
    fetch_rows<EC>(row_at<T>(a.dout, a.sdo, si, h, (int64_t)si.q_start + w0), (int)a.sdo.s * 2, rows, lane, 0, a.ev, own + SM::WAVE_V);
    fetch_rows<kLatentShared>(qp, (int)a.sq.s * 2, rows, lane, a.e, a.r, own + SM::WAVE_C);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    take_rows<T, EC>(q, lane, own);
    take_rows<T, EC>(dout, lane, own + SM::WAVE_V);
    take_rows<T, kLatentShared>(q + KE, lane, own + SM::WAVE_C);
  }
  arrived(q);
  arrived(dout);
  latent_meet();
  if (j1 > 0) fetch(0, 0);
  // delta of few keys is summed from P and dP in a pass of its own, else from O: of O's rounding as much is left as the keys that weigh in
  // have not averaged out, and with few of them it is the largest error of the gradients (two thirds of dQ's products once more, for rows
  // whose tiles are few).
  const bool few = j1 <= kLatentFewTiles;
  float delta = 0.f, lse = __builtin_inff();
  if (row < si.seqlen_q) lse = a.lse[lse_offset(si, h, a.heads) + row] * kLog2e;
  if (!few) {
    op_t out[KE];
    const int place = smem0 + SM::STAGE + wave * SM::WAVE_V;      // (in the other stage)
    fetch_rows<EC>(row_at<T>(a.out, a.so, si, h, (int64_t)si.q_start + w0), (int)a.so.s * 2, rows, lane, 0, a.ev, place);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    take_rows<T, EC>(out, lane, place);
#pragma unroll
    for (int k = 0; k < KE; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) delta += (float)out[k][i] * (float)dout[k][i];
  }
  const float qs = a.sm_scale * kLog2e, qs_or_1 = qs == 0.f ? 1.f : qs;
  // P and dP of 32 keys of tile j
  auto products = [&](const char* K, int j, int b, f32x16& p, f32x16& dp) __attribute__((always_inline)) {
    const int l = own_lane(), n0 = j * 64;
    const bool masked = n0 + 64 > si.seqlen_k || (a.causal && n0 + 63 > w0 + shift);
    const int row_e = Swz<EC>::row_base(l), row_r = Swz<kLatentShared>::row_base(l);
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = dp[i] = 0.f;
#pragma unroll
    for (int k = 0; k < KE; ++k) p = Tr::mfma(swz_read_row<T, EC>(K, row_e, k, b), q[k], p);
#pragma unroll
    for (int k = 0; k < KR; ++k) p = Tr::mfma(swz_read_row<T, kLatentShared>(K + SM::C_OFF, row_r, k, b), q[KE + k], p);
#pragma unroll
    for (int k = 0; k < KE; ++k) dp = Tr::mfma(swz_read_row<T, EC>(K + SM::V_OFF, row_e, k, b), dout[k], dp);
    if (masked || qs == 0.f) {      // (of what a row does not see S is what P of 0 comes from)
      const int limit = see - n0 - 32 * b - 4 * hi;
      const float never = qs < 0.f ? __builtin_inff() : -__builtin_inff();
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = 8 * (i / 4) + i % 4 > limit ? never : qs == 0.f ? 0.f : p[i];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = fast_exp2(__builtin_fmaf(p[i], qs_or_1, -lse));
  };
  int stage = 0;      // of the tile that comes next
  if (few) {
    for (int j = 0; j < j1; ++j, stage ^= 1) {
      latent_meet();
      fetch(stage ^ 1, j + 1 < j1 ? j + 1 : 0);
      if (j >= wave_end) continue;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        f32x16 p, dp;
        products(smem + stage * SM::STAGE, j, b, p, dp);
#pragma unroll
        for (int i = 0; i < 16; ++i) delta = __builtin_fmaf(p[i], dp[i], delta);
      }
    }
  }
  delta = cross_sum(delta);
  if (row < si.seqlen_q && hi == 0) {
    const int64_t at = lse_offset(si, h, a.heads) + row;
    a.stat_lse[at] = lse;
    a.stat_delta[at] = delta;
  }
  f32x16 dq[DB + RB];
#pragma unroll
  for (int b = 0; b < DB + RB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) dq[b][i] = 0.f;
  for (int j = 0; j < j1; ++j, stage ^= 1) {
    latent_meet();
    if (j + 1 < j1) fetch(stage ^ 1, j + 1);
    if (j >= wave_end) continue;
    const char* K = smem + stage * SM::STAGE;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      f32x16 s, dp;
      products(K, j, b, s, dp);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] *= dp[i] - delta;
      const int m = own_lane();
      const int tr0 = Swz<EC>::tr_base(m, 0), tr1 = Swz<EC>::tr_base(m, 1), rr0 = Swz<kLatentShared>::tr_base(m, 0), rr1 = Swz<kLatentShared>::tr_base(m, 1);
      op_t ds[2];
      auto add = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int x = 0; x < DB; ++x) dq[x] = Tr::mfma(swz_read_tr<T, EC>(K, tr0, tr1, 2 * b + t, x), ds[t], dq[x]);
#pragma unroll
          for (int x = 0; x < RB; ++x) dq[DB + x] = Tr::mfma(swz_read_tr<T, kLatentShared>(K + SM::C_OFF, rr0, rr1, 2 * b + t, x), ds[t], dq[DB + x]);
        }
      };
#pragma unroll
      for (int t = 0; t < 2; ++t) ds[t] = pack8<T>(s, t);
      add();
      if (j1 == 1) {      // (what dS lost in 16 bits, where few keys do not average it out: fa_latent_keys.h)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] -= (float)ds[i / 8][i % 8];
#pragma unroll
        for (int t = 0; t < 2; ++t) ds[t] = pack8<T>(s, t);
        add();
      }
    }
  }
  latent_meet();
  T* to = row_at<T>(a.dq, a.sdq, si, h, (int64_t)si.q_start + w0);
  const int out_lane = own_lane();
  store_rows<T, DB>(dq, a.sm_scale, to, a.sdq.s, rows, a.e, out_lane, own);
  store_rows<T, RB>(dq + DB, a.sm_scale, to + a.e, a.sdq.s, rows, a.r, out_lane, own + kRowsOut<T, DB>);
}

// Heads whose tiles are worked on side by side: as many as have two workgroups for a CU, a multiple of 8 (an XCD keeps its heads).  Those that run at a
// time then share what passes by in L2: the step of 12 packed sequences of 200 to 4000 tokens with 16 heads takes 1830 us, with all heads side by
// side 2010, with one an XCD 1900; three long sequences, the last of which ends by itself, 1490 for 1410; equal lengths the same.
inline int latent_group(int pairs, int tiles) {
  const int n = (512 / std::max(tiles, 1) + 7) / 8 * 8;
  return std::min(std::max(n, 8), pairs);
}

// ---- launches ------------------------------------------------------------------------------------------------------
template <typename T, int EC> hipError_t launch_latent_fwd(const LatentArgs& args, hipStream_t s) {
  static std::atomic<uint64_t> done{0};
  const int nseq = nseq_of(args.seq, args.batch), tiles = (args.seq.max_seqlen_q + 127) / 128;
  if (nseq * args.heads == 0 || tiles == 0) return hipSuccess;
  LatentArgs a = args;
  a.group = a.parts > 1 ? nseq * a.heads : latent_group(nseq * a.heads, tiles);
  hipError_t e = allow_large_lds(reinterpret_cast<const void*>(&latent_fwd_kernel<T, EC>), LatentSmem<EC>::BYTES, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((latent_fwd_kernel<T, EC>), dim3((unsigned)(nseq * a.heads * tiles * a.parts)), dim3(256), LatentSmem<EC>::BYTES, s, a, nseq, tiles);
  if (a.parts > 1)
    hipLaunchKernelGGL((latent_fwd_sum_kernel<T, EC>), dim3((unsigned)(nseq * a.heads * tiles * 4 * (EC / 32))), dim3(256), 0, s, a, nseq, tiles);
  return hipGetLastError();
}

template <typename T, int EC> hipError_t launch_latent_dq(const LatentBwdArgs& args, hipStream_t s) {
  static std::atomic<uint64_t> done{0};
  const int nseq = nseq_of(args.seq, args.batch), tiles = (args.seq.max_seqlen_q + 127) / 128;
  if (nseq * args.heads == 0 || tiles == 0) return hipSuccess;
  LatentBwdArgs a = args;
  a.group = latent_group(nseq * a.heads, tiles);
  hipError_t e = allow_large_lds(reinterpret_cast<const void*>(&latent_dq_kernel<T, EC>), LatentSmem<EC>::BYTES, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((latent_dq_kernel<T, EC>), dim3((unsigned)(nseq * a.heads * tiles)), dim3(256), LatentSmem<EC>::BYTES, s, a, nseq, tiles);
  return hipGetLastError();
}

}  // namespace fa
