// dK, dV and dC of attention whose keys are part per head, part shared by all heads (fa_latent.h), and dQ of few workgroups: gfx950, MFMA 32x32x16.
#pragma once
#include "fa_latent.h"

namespace fa {

// ---- dK, dV and every head's part of dC -----------------------------------------------------------------------------
// A wave owns 32 keys, a lane one of them, with K, C and V as operands in registers; tiles of 64 queries pass, 32 of them at a time: in a round the
// MFMAs of S and dP of the next 32 stand over the exponentials of these, then those of dV, dK and dC follow.  The wave is the only one on its
// SIMD (dK, dV and dC take 160 accumulators), so that what is not behind an MFMA costs its time.  16 heads of 8192 causal tokens, E = Ev = 128,
// R = 64: 690 us (one after the other, as the compiler orders them, 843), 53 % of it MFMAs, 1000 TFLOP/s; 12 packed sequences of 200 to 4000
// tokens 780 (1120).
template <typename T, int EC>
__global__ __launch_bounds__(256, 1) void latent_dkdv_kernel(const LatentBwdArgs a, int nseq, int tiles) {
  using Tr = Traits<T>;
  using op_t = typename Tr::op_t;
  using SM = LatentSmem<EC>;
  constexpr int KE = EC / 16, KR = kLatentShared / 16, DB = EC / 32, RB = kLatentShared / 32;
  extern __shared__ __attribute__((aligned(kSwzAlign))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int z, h, nt;
  latent_item(a, blockIdx.x, nseq, tiles, false, z, h, nt);
  const SeqInfo si = latent_seq(a, z);
  if (nt * 128 >= si.seqlen_k) return;
  const int shift = si.seqlen_k - si.seqlen_q;
  const int w0 = nt * 128 + wave * 32, key = w0 + c, keys = si.seqlen_k - w0;
  // the first query that sees a key
  auto first_query = [&](int n) { return a.causal && n - shift > 0 ? n - shift : 0; };
  const int j0 = first_query(nt * 128) / 64, j1 = (si.seqlen_q + 63) / 64;

  const int smem0 = lds_offset(smem);
  const int q_row = (int)a.sq.s * 2, do_row = (int)a.sdo.s * 2;
  const TileRows<EC> qt(lane, q_row, 0, a.e), dt(lane, do_row, 0, a.ev);
  const TileRows<kLatentShared> rt(lane, q_row, a.e, a.r);
  const float* stats = (wave & 1 ? a.stat_delta : a.stat_lse) + lse_offset(si, h, a.heads);
  auto fetch = [&](int stage, int j) __attribute__((always_inline)) {
    const int m = j * 64 + wave * 16, left = si.seqlen_q - m < 16 ? si.seqlen_q - m : 16;
    const int64_t at = si.q_start + m;
    const int base = smem0 + stage * SM::BWD_STAGE, lds = base + wave * 16 * 2 * EC;
    const auto q_rs = wave_rsrc_words(row_at<T>(a.q, a.sq, si, h, at), rows_extent(left, q_row, (a.e + a.r) * 2));
    qt.fetch(q_rs, lds);
    rt.fetch(q_rs, base + SM::C_OFF + wave * 16 * 2 * kLatentShared);
    dt.fetch(wave_rsrc_words(row_at<T>(a.dout, a.sdo, si, h, at), rows_extent(left, do_row, a.ev * 2)), lds + SM::V_OFF);
    // (of a row past the sequence both statistics are 0)
    if (wave < 2) {
      const int n = si.seqlen_q - j * 64 < 64 ? si.seqlen_q - j * 64 : 64;
      load_word_to_lds(wave_rsrc_words(stats + j * 64, n > 0 ? n * 4 : 0), lane * 4, base + SM::STAGE + wave * 256);
    }
  };
  op_t k[KE + KR], v[KE];
  const int own = smem0 + wave * SM::WAVE;
  fetch_rows<EC>(row_at<T>(a.k, a.sk, si, h, (int64_t)si.k_start + w0), (int)a.sk.s * 2, keys, lane, 0, a.e, own);
  fetch_rows<EC>(row_at<T>(a.v, a.sv, si, h, (int64_t)si.k_start + w0), (int)a.sv.s * 2, keys, lane, 0, a.ev, own + SM::WAVE_V);
  fetch_rows<kLatentShared>(row_at<T>(a.c, Strides3{a.c_z, 0, a.c_s}, si, 0, (int64_t)si.k_start + w0), (int)a.c_s * 2, keys, lane, 0, a.r, own + SM::WAVE_C);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  take_rows<T, EC>(k, lane, own);
  take_rows<T, EC>(v, lane, own + SM::WAVE_V);
  take_rows<T, kLatentShared>(k + KE, lane, own + SM::WAVE_C);
  arrived(k);
  arrived(v);
  latent_meet();
  if (j0 < j1) fetch(0, j0);
  // (accumulators are written as asm, fa_wide.h, so that S and dP lie in vector registers, where the exponentials are)
  f32x16 dk[DB + RB], dv[DB];
#pragma unroll
  for (int b = 0; b < DB + RB; ++b) acc_zero<T>(dk[b]);
#pragma unroll
  for (int b = 0; b < DB; ++b) acc_zero<T>(dv[b]);
  const float qs = a.sm_scale * kLog2e, qs_or_1 = qs == 0.f ? 1.f : qs;
  constexpr int kS = KE + KR, kA = kS + KE, kB = 2 * (2 * DB + RB), kRing = 6;      // MFMAs of S, of both; of the products with P and dS; operands on their way
  // addresses of the operands in the stages of S and of the products (fa_latent_cache.h)
  int at_e[8], at_r[KR], at_t[8], at_c[4], at_stats = smem0 + SM::STAGE + 16 * hi;
  static_assert(KE <= 8 && DB <= 4, "a tile's row is one period of the swizzle");
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    at_e[i] = smem0 + (Swz<EC>::row_base(lane) ^ (i % KE << 5));
    at_t[i] = smem0 + (Swz<EC>::tr_base(lane, i >> 2) ^ ((i & 3) % DB << 6));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    at_r[i] = smem0 + SM::C_OFF + (Swz<kLatentShared>::row_base(lane) ^ (i << 5));
    at_c[i] = smem0 + SM::C_OFF + (Swz<kLatentShared>::tr_base(lane, i >> 1) ^ ((i & 1) << 6));
  }
  auto onward = [&](auto& at, int by) __attribute__((always_inline)) {
#pragma unroll
    for (auto& x : at) x += by;
    arrived(at);
  };
  op_t ring[kRing];
  f32x16 s[2], dp[2];
  // operand n of the products of S and dP of half b of a tile: Q, the shared part of Q, dO
  auto read_a = [&](int b, int n) __attribute__((always_inline)) {
    if (n < KE) return lds_read<op_t>(at_e[n] + b * 32 * Swz<EC>::ROWB);
    if (n < kS) return lds_read<op_t>(at_r[n - KE] + b * 32 * Swz<kLatentShared>::ROWB);
    return lds_read<op_t>(at_e[n - kS] + SM::V_OFF + b * 32 * Swz<EC>::ROWB);
  };
  // of dV, dK and dC, 16 queries after the other
  auto read_b = [&](int b, int n) __attribute__((always_inline)) {
    const int t = 2 * b + n / (kB / 2), x = n % (kB / 2);
    int lo, hi2;
    if (x < 2 * DB) {
      const int off = t * 16 * Swz<EC>::ROWB + (x < DB ? SM::V_OFF : 0);
      lo = at_t[x % DB] + off;
      hi2 = at_t[4 + x % DB] + off;
    } else {
      lo = at_c[x - 2 * DB] + t * 16 * Swz<kLatentShared>::ROWB;
      hi2 = at_c[2 + x - 2 * DB] + t * 16 * Swz<kLatentShared>::ROWB;
    }
    return __builtin_shufflevector(__builtin_bit_cast(typename Tr::q4_t, lds_read_tr_at(lo)), __builtin_bit_cast(typename Tr::q4_t, lds_read_tr_at(hi2)), 0, 1, 2, 3, 4, 5, 6, 7);
  };
  op_t p_op[2], ds_op[2];
  f32x4 st_lse, st_delta;
  // P and dS of the 32 queries in s[b] and dp[b], element e of the lane's 16
  auto element = [&](int b, int e) __attribute__((always_inline)) {
    if (e % 4 == 0) {
      const int st = at_stats + 128 * b + 32 * (e / 4);
      st_lse = lds_read<f32x4>(st);
      st_delta = lds_read<f32x4>(st + 256);
    }
    const float p = fast_exp2(__builtin_fmaf(s[b][e], qs_or_1, -st_lse[e % 4]));
    s[b][e] = p;
    dp[b][e] = p * (dp[b][e] - st_delta[e % 4]);
    if (e % 8 == 7) {
      p_op[e / 8] = pack8<T>(s[b], e / 8);
      ds_op[e / 8] = pack8<T>(dp[b], e / 8);
    }
  };
  // Half b of the queries from m0 on: of those that do not see the lane's key, and those behind the sequence (rows that share memory, as those of the
  // gradient of a sum, do not read as zeros there), S is what P of 0 comes from.
  auto hide = [&](auto half, int m0) __attribute__((always_inline)) {
    constexpr int b = decltype(half)::value;
    if (!(a.causal && m0 < w0 + 31 - shift) && m0 + 32 <= si.seqlen_q && qs != 0.f) return;
    const int from = a.causal ? key - shift - m0 - 4 * hi : 0, to = si.seqlen_q - m0 - 4 * hi;      // rows of the half that see the lane's key
    const float never = qs < 0.f ? __builtin_inff() : -__builtin_inff();
#pragma unroll
    for (int e = 0; e < 16; ++e) s[b][e] = 8 * (e / 4) + e % 4 < from || 8 * (e / 4) + e % 4 >= to ? never : qs == 0.f ? 0.f : s[b][e];
  };
  // S and dP of half b of a tile, with P and dS of the half in front behind their MFMAs
  auto front = [&](auto half, auto behind) __attribute__((always_inline)) {
    constexpr int b = decltype(half)::value;
#pragma unroll
    for (int n = 0; n < kRing - 1; ++n) ring[n] = read_a(b, n);
#pragma unroll
    for (int n = 0; n < kA; ++n) {
      if (n + kRing - 1 < kA) ring[(n + kRing - 1) % kRing] = read_a(b, n + kRing - 1);
      const f32x16 none = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (n < kS) s[b] = Tr::mfma(ring[n % kRing], k[n], n == 0 ? none : s[b]);
      else dp[b] = Tr::mfma(ring[n % kRing], v[n - kS], n == kS ? none : dp[b]);
      if constexpr (decltype(behind)::value) {
#pragma unroll
        for (int e = first_of(n, 16, kA); e < first_of(n + 1, 16, kA); ++e) element(1 - b, e);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto back = [&](auto half) __attribute__((always_inline)) {
    constexpr int b = decltype(half)::value;
#pragma unroll
    for (int n = 0; n < kRing - 1; ++n) ring[n] = read_b(b, n);
#pragma unroll
    for (int n = 0; n < kB; ++n) {
      if (n + kRing - 1 < kB) ring[(n + kRing - 1) % kRing] = read_b(b, n + kRing - 1);
      const int t = n / (kB / 2), x = n % (kB / 2);
      if (x < DB) mfma_acc<T>(dv[x], ring[n % kRing], p_op[t]);
      else mfma_acc<T>(dk[x - DB], ring[n % kRing], ds_op[t]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // What P and dS lost in 16 bits, as operands: where one tile of queries is all there is the few roundings do not average out, and they go
  // through the products once more (11 sequences of up to 4 tokens: dK 1.5 times as far from 64 bits as fp32 arithmetic, dC 1.6).
  const bool twice = j1 - j0 == 1;
  auto rest = [&](auto half) __attribute__((always_inline)) {
    constexpr int b = decltype(half)::value;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[b][8 * t + e] -= (float)p_op[t][e];
        dp[b][8 * t + e] -= (float)ds_op[t][e];
      }
      p_op[t] = pack8<T>(s[b], t);
      ds_op[t] = pack8<T>(dp[b], t);
    }
  };
  using zero = std::integral_constant<int, 0>;
  using one = std::integral_constant<int, 1>;
  using yes = std::true_type;
  using no = std::false_type;
  // Tiles lie in three stages: the next one's S is formed while this one's products still read theirs.  (Behind the last half S of what a stage held
  // is formed, for nothing, rather than a way around it taken, for which the accumulators would be moved.)
  if (j0 < j1) {
    latent_meet();
    if (j0 + 1 < j1) fetch(1, j0 + 1);
    front(zero{}, no{});
  }
  for (int j = j0, stage = 0; j < j1; ++j) {
    hide(zero{}, 64 * j);
    front(one{}, yes{});
    back(zero{});
    if (twice) {
      rest(zero{});
      back(zero{});
    }
    const int by = stage == 2 ? -2 * SM::BWD_STAGE : SM::BWD_STAGE;
    onward(at_e, by);
    onward(at_r, by);
    if (j + 1 < j1) latent_meet();
    if (j + 2 < j1) fetch(stage == 0 ? 2 : stage - 1, j + 2);
    hide(one{}, 64 * j + 32);
    front(zero{}, yes{});
    back(one{});
    if (twice) {
      rest(one{});
      back(one{});
    }
    onward(at_t, by);
    onward(at_c, by);
    at_stats += by;
    stage = stage == 2 ? 0 : stage + 1;
  }
  latent_meet();
  settle(dk);
  settle(dv);
  store_rows<T, DB>(dk, a.sm_scale, row_at<T>(a.dk, a.sdk, si, h, (int64_t)si.k_start + w0), a.sdk.s, keys, a.e, lane, own);
  store_rows<T, DB>(dv, 1.0f, row_at<T>(a.dv, a.sdv, si, h, (int64_t)si.k_start + w0), a.sdv.s, keys, a.ev, lane, own + kRowsOut<T, DB>);
  store_rows<float, RB>(dk + DB, 1.0f, a.part_c + (((int64_t)si.batch_index * a.heads + h) * a.part_rows + si.k_start + w0) * kLatentShared, kLatentShared, keys,
                        kLatentShared, lane, own);
}

// ---- dQ where a CU has no more than two workgroups --------------------------------------------------------------------
// As dK/dV above, with a wave's 32 rows in registers and tiles of 64 keys passing: one wave on a SIMD gets through a tile sooner than one of two, which
// is what counts where few workgroups are all there is.  delta as in latent_dq_kernel.
template <typename T, int EC>
__global__ __launch_bounds__(256, 1) void latent_dq_alone_kernel(const LatentBwdArgs a, int nseq, int tiles) {
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
  const int j1 = tiles_of(q0 + 127), see = last_key(row);
  const int see_least = __builtin_amdgcn_readfirstlane(last_key(w0));      // of the wave's rows

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
  const bool few = j1 <= kLatentFewTiles;
  float delta = 0.f, lse = __builtin_inff();
  if (row < si.seqlen_q) lse = a.lse[lse_offset(si, h, a.heads) + row] * kLog2e;
  if (!few) {
    op_t out[KE];
    const int place = smem0 + SM::STAGE + wave * SM::WAVE_V;      // (in the next stage)
    fetch_rows<EC>(row_at<T>(a.out, a.so, si, h, (int64_t)si.q_start + w0), (int)a.so.s * 2, rows, lane, 0, a.ev, place);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    take_rows<T, EC>(out, lane, place);
#pragma unroll
    for (int k = 0; k < KE; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) delta += (float)out[k][i] * (float)dout[k][i];
  }
  const float qs = a.sm_scale * kLog2e, qs_or_1 = qs == 0.f ? 1.f : qs;
  constexpr int kS = KE + KR, kA = kS + KE, kB = 2 * (DB + RB), kRing = 6;      // MFMAs of S, of both; of the product with dS; operands on their way
  // addresses of the operands in the stages of S and of the product (fa_latent_cache.h)
  int at_e[8], at_r[KR], at_t[8], at_c[4];
  static_assert(KE <= 8 && DB <= 4, "a tile's row is one period of the swizzle");
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    at_e[i] = smem0 + (Swz<EC>::row_base(lane) ^ (i % KE << 5));
    at_t[i] = smem0 + (Swz<EC>::tr_base(lane, i >> 2) ^ ((i & 3) % DB << 6));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    at_r[i] = smem0 + SM::C_OFF + (Swz<kLatentShared>::row_base(lane) ^ (i << 5));
    at_c[i] = smem0 + SM::C_OFF + (Swz<kLatentShared>::tr_base(lane, i >> 1) ^ ((i & 1) << 6));
  }
  auto onward = [&](auto& at, int by) __attribute__((always_inline)) {
#pragma unroll
    for (auto& x : at) x += by;
    arrived(at);
  };
  op_t ring[kRing], ds_op[2];
  f32x16 s[2], dp[2];
  // operand n of the products of S and dP of half b of a tile: K, the shared part, V
  auto read_a = [&](int b, int n) __attribute__((always_inline)) {
    if (n < KE) return lds_read<op_t>(at_e[n] + b * 32 * Swz<EC>::ROWB);
    if (n < kS) return lds_read<op_t>(at_r[n - KE] + b * 32 * Swz<kLatentShared>::ROWB);
    return lds_read<op_t>(at_e[n - kS] + SM::V_OFF + b * 32 * Swz<EC>::ROWB);
  };
  // of dQ, 16 keys after the other
  auto read_b = [&](int b, int n) __attribute__((always_inline)) {
    const int t = 2 * b + n / (kB / 2), x = n % (kB / 2);
    const int off = t * 16 * (x < DB ? Swz<EC>::ROWB : Swz<kLatentShared>::ROWB);
    const int lo = (x < DB ? at_t[x % DB] : at_c[x - DB]) + off, up = (x < DB ? at_t[4 + x % DB] : at_c[2 + x - DB]) + off;
    return __builtin_shufflevector(__builtin_bit_cast(typename Tr::q4_t, lds_read_tr_at(lo)), __builtin_bit_cast(typename Tr::q4_t, lds_read_tr_at(up)), 0, 1, 2, 3, 4, 5, 6, 7);
  };
  // Half b of the keys from n0 on: of those that a row does not see, S is what P of 0 comes from.
  auto hide = [&](auto half, int n0) __attribute__((always_inline)) {
    constexpr int b = decltype(half)::value;
    if (n0 + 31 <= see_least && qs != 0.f) return;
    const int limit = see - n0 - 4 * hi;
    const float never = qs < 0.f ? __builtin_inff() : -__builtin_inff();
#pragma unroll
    for (int e = 0; e < 16; ++e) s[b][e] = 8 * (e / 4) + e % 4 > limit ? never : qs == 0.f ? 0.f : s[b][e];
  };
  // P and dS of element e of the lane's 16 in s[b] and dp[b]
  auto element = [&](int b, int e) __attribute__((always_inline)) {
    s[b][e] = fast_exp2(__builtin_fmaf(s[b][e], qs_or_1, -lse)) * (dp[b][e] - delta);
    if (e % 8 == 7) ds_op[e / 8] = pack8<T>(s[b], e / 8);
  };
  // S and dP of half b of a tile, with dS of the half in front behind their MFMAs
  auto front = [&](auto half, auto behind) __attribute__((always_inline)) {
    constexpr int b = decltype(half)::value;
#pragma unroll
    for (int n = 0; n < kRing - 1; ++n) ring[n] = read_a(b, n);
#pragma unroll
    for (int n = 0; n < kA; ++n) {
      if (n + kRing - 1 < kA) ring[(n + kRing - 1) % kRing] = read_a(b, n + kRing - 1);
      const f32x16 none = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (n < kS) s[b] = Tr::mfma(ring[n % kRing], q[n], n == 0 ? none : s[b]);
      else dp[b] = Tr::mfma(ring[n % kRing], dout[n - kS], n == kS ? none : dp[b]);
      if constexpr (decltype(behind)::value) {
#pragma unroll
        for (int e = first_of(n, 16, kA); e < first_of(n + 1, 16, kA); ++e) element(1 - b, e);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  using zero = std::integral_constant<int, 0>;
  using one = std::integral_constant<int, 1>;
  using yes = std::true_type;
  using no = std::false_type;
  int stage = 0;      // of the tile that comes next
  auto step_of = [&]() { return stage == 2 ? -2 * SM::STAGE : SM::STAGE; };
  if (few) {
    for (int j = 0; j < j1; ++j) {
      latent_meet();
      fetch(stage == 2 ? 0 : stage + 1, j + 1 < j1 ? j + 1 : 0);
      front(zero{}, no{});
      front(one{}, no{});
      hide(zero{}, 64 * j);
      hide(one{}, 64 * j + 32);
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) delta = __builtin_fmaf(fast_exp2(__builtin_fmaf(s[b][e], qs_or_1, -lse)), dp[b][e], delta);
      onward(at_e, step_of());
      onward(at_r, step_of());
      onward(at_t, step_of());
      onward(at_c, step_of());
      stage = stage == 2 ? 0 : stage + 1;
    }
  }
  delta = cross_sum(delta);
  if (row < si.seqlen_q && hi == 0) {
    const int64_t at = lse_offset(si, h, a.heads) + row;
    a.stat_lse[at] = lse;
    a.stat_delta[at] = delta;
  }
  // (accumulators are written as asm, fa_wide.h, so that S and dP lie in vector registers, where the exponentials are)
  f32x16 dq[DB + RB];
#pragma unroll
  for (int b = 0; b < DB + RB; ++b) acc_zero<T>(dq[b]);
  auto back = [&](auto half) __attribute__((always_inline)) {
    constexpr int b = decltype(half)::value;
#pragma unroll
    for (int n = 0; n < kRing - 1; ++n) ring[n] = read_b(b, n);
#pragma unroll
    for (int n = 0; n < kB; ++n) {
      if (n + kRing - 1 < kB) ring[(n + kRing - 1) % kRing] = read_b(b, n + kRing - 1);
      mfma_acc<T>(dq[n % (kB / 2)], ring[n % kRing], ds_op[n / (kB / 2)]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // (what dS lost in 16 bits, where few keys do not average it out: latent_dkdv_kernel)
  const bool twice = j1 == 1;
  auto rest = [&](auto half) __attribute__((always_inline)) {
    constexpr int b = decltype(half)::value;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[b][e] -= (float)ds_op[e / 8][e % 8];
#pragma unroll
    for (int t = 0; t < 2; ++t) ds_op[t] = pack8<T>(s[b], t);
  };
  if (j1 > 0) {
    latent_meet();
    if (j1 > 1) fetch(stage == 2 ? 0 : stage + 1, 1);
    front(zero{}, no{});
  }
  for (int j = 0; j < j1; ++j) {
    hide(zero{}, 64 * j);
    front(one{}, yes{});
    back(zero{});
    if (twice) {
      rest(zero{});
      back(zero{});
    }
    const int by = step_of();
    onward(at_e, by);
    onward(at_r, by);
    if (j + 1 < j1) latent_meet();
    if (j + 2 < j1) fetch(stage == 0 ? 2 : stage - 1, j + 2);
    hide(one{}, 64 * j + 32);
    front(zero{}, yes{});
    back(one{});
    if (twice) {
      rest(one{});
      back(one{});
    }
    onward(at_t, by);
    onward(at_c, by);
    stage = stage == 2 ? 0 : stage + 1;
  }
  latent_meet();
  settle(dq);
  T* to = row_at<T>(a.dq, a.sdq, si, h, (int64_t)si.q_start + w0);
  store_rows<T, DB>(dq, a.sm_scale, to, a.sdq.s, rows, a.e, lane, own);
  store_rows<T, RB>(dq + DB, a.sm_scale, to + a.e, a.sdq.s, rows, a.r, lane, own + kRowsOut<T, DB>);
}

// Whether a sequence has row n of packed keys, as latent_seq holds them: the last one that starts no later, if it goes so far.
__device__ __forceinline__ bool latent_has_key(const LatentArgs& a, int n) {
  auto hold = [&](int x) { return x < 0 ? 0 : x < a.rows_k ? x : a.rows_k; };
  int z = 0;
  for (int left = a.seq.num_seqlens; left > 1;) {
    const int half = left / 2;
    if (hold(a.seq.cu_k[z + half]) <= n) z += half;
    left -= half;
  }
  const int start = hold(a.seq.cu_k[z]), end = hold(a.seq.cu_k[z + 1]);
  return n >= start && n < end && n - start < a.seq.max_seqlen_k;
}

// dC: the heads' parts added in their order, four columns a lane; packed rows of no sequence, which have no parts, stay as they are
template <typename T>
__global__ __launch_bounds__(256) void latent_dc_kernel(const LatentBwdArgs a, int64_t keys) {
  const int64_t at = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
  const int64_t b = at / keys, n = at % keys;
  const int col = threadIdx.x % 16 * 4;
  if (b >= a.batch || col >= a.r || (a.seq.num_seqlens != 0 && !latent_has_key(a, (int)n))) return;
  const float* from = a.part_c + (b * a.heads * a.part_rows + n) * kLatentShared + col;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int h = 0; h < a.heads; ++h) sum += *reinterpret_cast<const f32x4*>(from + (int64_t)h * a.part_rows * kLatentShared);
  typename Traits<T>::q4_t y;
#pragma unroll
  for (int r = 0; r < 4; ++r) y[r] = Traits<T>::cvt(sum[r] * a.sm_scale);
  *reinterpret_cast<typename Traits<T>::q4_t*>(reinterpret_cast<T*>(a.dc) + b * a.dc_z + n * a.dc_s + col) = y;
}

template <typename T, int EC> hipError_t launch_latent_keys(const LatentBwdArgs& args, hipStream_t s) {
  static std::atomic<uint64_t> done{0};
  const int nseq = nseq_of(args.seq, args.batch), tiles = (args.seq.max_seqlen_k + 127) / 128;
  if (nseq == 0 || tiles == 0) return hipSuccess;
  LatentBwdArgs a = args;
  a.group = latent_group(nseq * a.heads, tiles);
  hipError_t e = allow_large_lds(reinterpret_cast<const void*>(&latent_dkdv_kernel<T, EC>), LatentSmem<EC>::BWD_BYTES, done);
  if (e != hipSuccess) return e;
  if (a.heads > 0)
    hipLaunchKernelGGL((latent_dkdv_kernel<T, EC>), dim3((unsigned)(nseq * a.heads * tiles)), dim3(256), LatentSmem<EC>::BWD_BYTES, s, a, nseq, tiles);
  hipLaunchKernelGGL((latent_dc_kernel<T>), dim3((unsigned)((a.batch * a.part_rows + 15) / 16)), dim3(256), 0, s, a, a.part_rows);
  return hipGetLastError();
}

template <typename T, int EC> hipError_t launch_latent_dq_alone(const LatentBwdArgs& args, hipStream_t s) {
  static std::atomic<uint64_t> done{0};
  const int nseq = nseq_of(args.seq, args.batch), tiles = (args.seq.max_seqlen_q + 127) / 128;
  if (nseq * args.heads == 0 || tiles == 0) return hipSuccess;
  LatentBwdArgs a = args;
  a.group = latent_group(nseq * a.heads, tiles);
  hipError_t e = allow_large_lds(reinterpret_cast<const void*>(&latent_dq_alone_kernel<T, EC>), LatentSmem<EC>::DQ_BYTES, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((latent_dq_alone_kernel<T, EC>), dim3((unsigned)(nseq * a.heads * tiles)), dim3(256), LatentSmem<EC>::DQ_BYTES, s, a, nseq, tiles);
  return hipGetLastError();
}

}  // namespace fa
