// Attention with a sliding window and a few first tokens that stay visible (sinks): gfx950, MFMA 32x32x16.
//
// Query i of a sequence of n_q queries and n_k keys stands at p = i + n_k - n_q and sees key c iff
//   c <= p  and  (c > p - window  or  c < sinks).
// Forward and dQ are fwd_item and dq_item with kSinks: their tiles are the window's and, in front of those, the tiles that hold
// sinks only.  dK and dV of the window are dkdv_item's.  What is left is here: dK and dV of the first `sinks` keys, which all
// queries see.
//
// One workgroup of the window's kernel per 128 keys would make the first one loop over all queries while the others loop over
// window + 128 of them, with 124 of its 128 keys idle for 4 sinks.  So these keys are computed on their own, 32 at a time (one MFMA
// operand), the queries of all q-heads of the group cut into pieces of equal length.  A block of sinks that is one piece is
// finished there; the fp32 sums of several pieces are added by a second kernel.  Both overwrite what the window's kernel wrote for
// these keys (dK and dV are rounded once):
//   S  (queries x keys) = Q K^T, P = exp2(S c - L), dP = dO V^T, dS = P (dP - delta)
//   dV^T (d x keys) += dO^T P,   dK^T (d x keys) += Q^T dS
// Each of the four waves takes 32-query steps of its own through a private LDS area (Q and dO rows, swizzled, read by rows and
// transposed), so that the loop has no barrier; the next step's rows are in flight meanwhile.
// What bounds it: one read of Q and dO (4 D bytes a query against 8 D 32 MFMA operations), of which a wave has 16 KB in flight: Hq 32 Hk 8
// S8192 D128 134 MB in 38 us, the sums 5.  Two steps ahead instead of one need all registers and are no faster (41 -> 44 us).
#pragma once
#include "fa_bwd_impl.h"
#include "fa_fwd_impl.h"

namespace fa {

template <int D>
struct SinkSmem {      // per wave: Q and dO rows; L and -delta.  The waves' sums meet where the rows were
  static constexpr int TILE_BYTES = 32 * D * 2;
  static constexpr int STAT_OFF = 2 * TILE_BYTES;
  static constexpr int WAVE_BYTES = STAT_OFF + 256;
  static constexpr int SUM_BYTES = 2 * 32 * D * 4;      // dK and dV of 32 keys
  static constexpr int BYTES = 4 * WAVE_BYTES;
  static_assert(BYTES >= 2 * SUM_BYTES, "the sums of two waves fit");
};

// Sequences of different lengths: the steps of all blocks of 32 sinks as one list, by K/V head, block, sequence, q-head of the
// group and 32 queries, and a workgroup's piece is `length` of them, wherever a sequence ends.  The table of EvenWalk says where they
// start.  (Pieces that end with their sequence are more than the chip takes at once: 16 sequences of up to 6000 tokens, Hq 16 Hk 4
// D128, 17 sinks: 113 us and 6 for the sums; this 80 and 7.  Where all are alike it would cost 3 us more.)
struct SinkList {
  EvenWalk even;
  int group;
  int per_block, steps, length;
  __device__ __forceinline__ SinkList(const SinkBwdArgs& a, int* lds, int tid) {
    group = a.hq / a.hk;
    even.template init<256>(lds, a.seq, nseq_of(a.seq, a.batch), (a.seq.max_seqlen_q + 31) / 32, 1, 1, 32, false, 0, tid);
    even.hi = even.total;
    per_block = even.total * group;
    steps = per_block * a.hk * ((a.sinks + 31) / 32);
    length = (steps + a.sink_pieces - 1) / a.sink_pieces;
  }
  __device__ __forceinline__ int start(int head_block, int z) const {
    return head_block * per_block + (even.table ? __builtin_amdgcn_readfirstlane(even.table[z]) : z * even.num_tiles) * group;
  }
};

// four columns of a key's finished dK or dV; `e` as in sum_at below
template <typename T, int D>
__device__ __forceinline__ void sink_store(const SinkBwdArgs& a, const SeqInfo& si, int hk, int n0, int e, f32x4 acc) {
  const int lane = e % 64, g = e / 64 % 4, db = e / 256 % (D / 32), which = e / (SinkSmem<D>::SUM_BYTES / 32);
  const int key = n0 + (lane & 31), col = 32 * db + 8 * g + 4 * (lane >> 5);
  if (key >= si.seqlen_k || key >= a.sinks || col >= (which ? a.head_dim_v : a.head_dim)) return;
  const Strides3& st = which ? a.sdv : a.sdk;
  const float f = which ? 1.0f : a.sm_scale;
  vec<T, 4> t4;
#pragma unroll
  for (int r = 0; r < 4; ++r) t4[r] = Traits<T>::cvt(acc[r] * f);
  *reinterpret_cast<vec<T, 4>*>(reinterpret_cast<T*>(which ? a.dv : a.dk) + (int64_t)si.batch_index * st.z + (int64_t)hk * st.h +
                                (int64_t)(si.k_start + key) * st.s + col) = t4;
}

template <typename T, int D, int kPad, bool kList>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256))) __attribute__((amdgpu_waves_per_eu(D == 64 ? 2 : 1, D == 64 ? 2 : 1)))
void sink_dkdv_kernel(const SinkBwdArgs a) {
  extern __shared__ __attribute__((aligned(kSwzAlign))) char smem_raw[];
  using Tr = Traits<T>;
  using op_t = typename Tr::op_t;
  using SM = SinkSmem<D>;
  constexpr int DC = kPad ? kPad : D;
  constexpr int KS = DC / 16, DB = DC / 32;
  constexpr int LPR = D / 8, RPI = 64 / LPR, CH = 32 / RPI;      // lanes per row, rows per access, accesses

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, c = lane & 31, hi = lane >> 5;
  const int d_qk = kPad ? a.head_dim : D, d_v = kPad ? a.head_dim_v : D;
  const int blocks = (a.sinks + 31) / 32, group = a.hq / a.hk;
  char* area = smem_raw + wave * SM::WAVE_BYTES;
  float* stat = reinterpret_cast<float*>(area + SM::STAT_OFF);

  // kList: the workgroup's piece of the list; else one of a.sink_parts pieces of a block
  std::conditional_t<kList, SinkList, int> list = [&] {
    if constexpr (kList) return SinkList(a, reinterpret_cast<int*>(smem_raw + SM::BYTES), tid);
    else return 0;
  }();
  int pos = 0, stop = 1;
  if constexpr (kList) {
    pos = blockIdx.x * list.length;
    stop = pos + list.length < list.steps ? pos + list.length : list.steps;
  }
  while (pos < stop) {
    int z, head_block, t0, t1;
    bool from_start, to_end;
    if constexpr (kList) {
      int head, tile;
      head_block = pos / list.per_block;
      list.even.at((pos - head_block * list.per_block) / group, z, head, tile);
      const int lo = list.start(head_block, z), hi_ = list.start(head_block, z + 1), to = stop < hi_ ? stop : hi_;
      t0 = pos - lo;
      t1 = to - lo;
      from_start = t0 == 0;
      to_end = to == hi_;
      pos = to;
    } else {
      const int nseq = nseq_of(a.seq, a.batch);
      const int part = blockIdx.x % a.sink_parts, item = blockIdx.x / a.sink_parts;
      z = item % nseq;
      head_block = item / nseq;
      t0 = part * a.sink_steps;
      t1 = t0 + a.sink_steps;
      from_start = to_end = a.sink_parts == 1;
      pos = stop;
    }
    const int hk = head_block / blocks, n0 = head_block % blocks * 32;
    const SeqInfo si = get_seq(a.seq, z);
    const int keys = a.sinks < si.seqlen_k ? a.sinks : si.seqlen_k;
    if (n0 >= keys) continue;

    // the lane's key, and the first query that sees it
    const int key = n0 + c, key_c = key < keys ? key : keys - 1;
    const int shift = si.seqlen_k - si.seqlen_q;
    const int q_lo = key < keys ? (key - shift > 0 ? key - shift : 0) : 0x7fffffff;
    op_t kreg[KS], vreg[KS];
    {
      const T* kp = reinterpret_cast<const T*>(a.k) + (int64_t)si.batch_index * a.sk.z + (int64_t)hk * a.sk.h + (int64_t)(si.k_start + key_c) * a.sk.s;
      const T* vp = reinterpret_cast<const T*>(a.v) + (int64_t)si.batch_index * a.sv.z + (int64_t)hk * a.sv.h + (int64_t)(si.k_start + key_c) * a.sv.s;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        kreg[k] = op_t{};
        vreg[k] = op_t{};
        if (16 * k + 8 * hi < d_qk) kreg[k] = *reinterpret_cast<const op_t*>(kp + 16 * k + 8 * hi);
        if (16 * k + 8 * hi < d_v) vreg[k] = *reinterpret_cast<const op_t*>(vp + 16 * k + 8 * hi);
      }
    }

    // the steps, which the waves take in turn
    const int per_head = (si.seqlen_q + 31) / 32;
    t1 = t1 < per_head * group ? t1 : per_head * group;

    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) { dk[db][i] = 0.f; dv[db][i] = 0.f; }
    const float qk_scale = a.sm_scale * kLog2e;
    const int row_a = Swz<D>::row_base(lane), tr_a0 = Swz<D>::tr_base(lane, 0), tr_a1 = Swz<D>::tr_base(lane, 1);
    const int r0 = lane / LPR, ch0 = lane % LPR;
    const int q_row = (int)a.sq.s * 2, do_row = (int)a.sdo.s * 2;
    const int qvoff = ch0 * 8 < d_qk ? r0 * q_row + ch0 * 16 : kVoffOutOfRange;
    const int dovoff = ch0 * 8 < d_v ? r0 * do_row + ch0 * 16 : kVoffOutOfRange;

    op_t qn[CH], don[CH];
    float stat_n = 0.f;
    int q_at = 0;
    auto load = [&](int t) {
      const int h = hk * group + t / per_head;
      q_at = t % per_head * 32;
      const int rows = si.seqlen_q - q_at < 32 ? si.seqlen_q - q_at : 32;
      const auto qrs = wave_rsrc(reinterpret_cast<const T*>(a.q) + (int64_t)si.batch_index * a.sq.z + (int64_t)h * a.sq.h +
                                     (int64_t)(si.q_start + q_at) * a.sq.s, (rows - 1) * q_row + d_qk * 2);
      const auto dors = wave_rsrc(reinterpret_cast<const T*>(a.dout) + (int64_t)si.batch_index * a.sdo.z + (int64_t)h * a.sdo.h +
                                      (int64_t)(si.q_start + q_at) * a.sdo.s, (rows - 1) * do_row + d_v * 2);
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        qn[i] = __builtin_bit_cast(op_t, __builtin_amdgcn_raw_buffer_load_b128(qrs, qvoff, i * RPI * q_row, 0));
        don[i] = __builtin_bit_cast(op_t, __builtin_amdgcn_raw_buffer_load_b128(dors, dovoff, i * RPI * do_row, 0));
      }
      // lanes below 32: L, above: delta.  A query past the sequence gets L = inf, so that its P is 0
      const int64_t at = lse_offset(si, h, a.hq) + q_at;
      const auto lrs = wave_rsrc(a.lse + at, rows * 4);
      const auto drs = wave_rsrc(a.delta + at, rows * 4);
      const float l = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(lrs, c * 4, 0, 0));
      const float d = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(drs, c * 4, 0, 0));
      stat_n = hi ? -d : c < rows ? l * kRcpLn2 : __builtin_inff();
    };

    int t = t0 + wave;
    if (t < t1) load(t);
    for (; t < t1; t += 4) {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int at = Swz<D>::addr(r0 + i * RPI, ch0);
        *reinterpret_cast<op_t*>(area + at) = qn[i];
        *reinterpret_cast<op_t*>(area + SM::TILE_BYTES + at) = don[i];
      }
      stat[lane] = stat_n;
      const int q0 = q_at;
      if (t + 4 < t1) load(t + 4);
      // (the areas are the wave's own, and its LDS operations run in order: what remains is to keep the compiler's order)
      __builtin_amdgcn_wave_barrier();
      f32x16 s, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 d4 = *reinterpret_cast<const f32x4*>(stat + 32 + 8 * g + 4 * hi);
#pragma unroll
        for (int r = 0; r < 4; ++r) dp[4 * g + r] = d4[r];      // dP starts at -delta
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) s = Tr::mfma(swz_read_row<T, D>(area, row_a, k, 0), kreg[k], s);
#pragma unroll
      for (int k = 0; k < KS; ++k) dp = Tr::mfma(swz_read_row<T, D>(area + SM::TILE_BYTES, row_a, k, 0), vreg[k], dp);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 l4 = *reinterpret_cast<const f32x4*>(stat + 8 * g + 4 * hi);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = __builtin_fmaf(s[4 * g + r], qk_scale, -l4[r]);
          s[4 * g + r] = q0 + 8 * g + 4 * hi + r >= q_lo ? fast_exp2(x) : 0.f;
          dp[4 * g + r] *= s[4 * g + r];
        }
      }
      const op_t p0 = pack8<T>(s, 0), p1 = pack8<T>(s, 1), s0 = pack8<T>(dp, 0), s1 = pack8<T>(dp, 1);
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        dv[db] = Tr::mfma(swz_read_tr<T, D>(area + SM::TILE_BYTES, tr_a0, tr_a1, 0, db), p0, dv[db]);
        dk[db] = Tr::mfma(swz_read_tr<T, D>(area, tr_a0, tr_a1, 0, db), s0, dk[db]);
      }
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        dv[db] = Tr::mfma(swz_read_tr<T, D>(area + SM::TILE_BYTES, tr_a0, tr_a1, 1, db), p1, dv[db]);
        dk[db] = Tr::mfma(swz_read_tr<T, D>(area, tr_a0, tr_a1, 1, db), s1, dk[db]);
      }
      __builtin_amdgcn_wave_barrier();
    }

    // ---- the four waves' sums: two in LDS, the other two onto them, both out as one -----------------------------
    // (as the lanes hold them: dK then dV, [32 columns][4 columns of 8][lane])
    auto sum_at = [&](int w, int which, int db, int g) {
      return reinterpret_cast<f32x4*>(smem_raw + w * SM::SUM_BYTES) + ((which * (D / 32) + db) * 4 + g) * 64 + lane;
    };
    __syncthreads();
#pragma unroll
    for (int round = 0; round < 2; ++round) {
      if (wave / 2 == round) {
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            f32x4 x = {dk[db][4 * g], dk[db][4 * g + 1], dk[db][4 * g + 2], dk[db][4 * g + 3]};
            f32x4 y = {dv[db][4 * g], dv[db][4 * g + 1], dv[db][4 * g + 2], dv[db][4 * g + 3]};
            f32x4 *xp = sum_at(wave & 1, 0, db, g), *yp = sum_at(wave & 1, 1, db, g);
            *xp = round ? *xp + x : x;
            *yp = round ? *yp + y : y;
          }
      }
      __syncthreads();
    }
    // (a piece of the list holds at most one block that began in front of it and one that goes on behind it)
    f32x4* out = reinterpret_cast<f32x4*>(a.sink_ws) + (kList ? 2 * (int64_t)blockIdx.x + (from_start ? 1 : 0) : (int64_t)blockIdx.x) * (SM::SUM_BYTES / 16);
    const f32x4* in = reinterpret_cast<const f32x4*>(smem_raw);
#pragma unroll
    for (int e = tid; e < SM::SUM_BYTES / 16; e += 256) {
      const f32x4 x = in[e] + in[e + SM::SUM_BYTES / 16];
      if (from_start && to_end) sink_store<T, D>(a, si, hk, n0, e, x);
      else if ((e & 31) < keys - n0 && (DC == D || e / 256 % (D / 32) < DB)) out[e] = x;      // (only keys that are there)
    }
    __syncthreads();
  }
}

// Adds up the blocks that are several pieces: four columns of a key's dK or dV per thread.
template <typename T, int D, bool kList>
static __global__ __launch_bounds__(256) void sink_sum_kernel(const SinkBwdArgs a) {
  extern __shared__ int table[];
  constexpr int SUMS = SinkSmem<D>::SUM_BYTES / 16, PER = SUMS / 256;      // workgroups for a key block
  const int e = blockIdx.x % PER * 256 + threadIdx.x, item = blockIdx.x / PER, nseq = nseq_of(a.seq, a.batch);
  const int z = item % nseq, head_block = item / nseq, blocks = (a.sinks + 31) / 32;
  const f32x4* p = reinterpret_cast<const f32x4*>(a.sink_ws) + e;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  if constexpr (kList) {
    const SinkList list(a, table, threadIdx.x);
    const int lo = list.start(head_block, z), hi = list.start(head_block, z + 1);
    if (lo == hi) return;      // (no query: the window's kernel wrote zeros)
    const int first = lo / list.length, last = (hi - 1) / list.length;
    if (first == last) return;
    p += 2 * (int64_t)first * SUMS;
    acc = p[SUMS];
#pragma unroll 8
    for (int i = 1; i <= last - first; ++i) acc += p[(int64_t)i * 2 * SUMS];
  } else {
    p += (int64_t)item * a.sink_parts * SUMS;
#pragma unroll 8
    for (int i = 0; i < a.sink_parts; ++i) acc += p[(int64_t)i * SUMS];
  }
  sink_store<T, D>(a, get_seq(a.seq, z), head_block / blocks, head_block % blocks * 32, e, acc);
}

// ---- launchers ------------------------------------------------------------------------------------------------
// a.half_tiles, a.splits and the scratch pointers are the caller's
template <typename T, int D, int kPad>
hipError_t launch_fwd_sinks(const SinkFwdArgs& a, hipStream_t stream) {
  const int half = a.half_tiles, waves = half ? 4 : 8;
  static_assert(FwdTile<T, D, true>::BM == 256, "eight waves");
  SinkFwdArgs b = a;
  b.head_shift = sink_head_shift(a.hq, a.hk, waves);
  const int BM = waves * 32 >> b.head_shift, nseq = nseq_of(a.seq, a.batch);
  b.num_m_tiles = (a.seq.max_seqlen_q + BM - 1) / BM;
  b.num_zh = nseq * a.hq;
  const TileWork w = tile_work(nseq * (a.hq >> b.head_shift), 1, b.num_m_tiles * (a.splits > 1 ? a.splits : 1));
  const dim3 grid((unsigned)(kNumXcd * tile_workers(w.items_per_xcd, a.num_cu, half ? half : 1)));
  using Half = FwdHalfTile<D>;
  using Whole = FwdTile<T, D, true>;
  if (a.splits > 1) {
    b.part_group = 1; b.part_block = BM; b.part_rows = BM; b.row_blocks = b.num_m_tiles;
    if (half) return launch_fwd_variant<T, D, true, false, false, kPad, true, false, Half, false, true>(b, grid, stream);
    return launch_fwd_variant<T, D, true, false, false, kPad, true, false, Whole, false, true>(b, grid, stream);
  }
  if (half) return launch_fwd_variant<T, D, true, false, false, kPad, false, false, Half, false, true>(b, grid, stream);
  return launch_fwd_variant<T, D, true, false, false, kPad, false, false, Whole, false, true>(b, grid, stream);
}

// dK and dV of the window's keys, and over them those of the sinks
template <typename T, int D, int kPad>
hipError_t launch_dkdv_sinks(const SinkBwdArgs& a, hipStream_t stream) {
  hipError_t e = a.wide ? hipSuccess : launch_dkdv_form<T, D, kPad, true, false, false, false, false, kBiasAny, true>(a, stream);
  const int items = bwd_nseq(a) * a.hk * ((a.sinks + 31) / 32);
  if (e != hipSuccess || items == 0 || a.seq.max_seqlen_k <= 0) return e;
  constexpr int sum_groups = SinkSmem<D>::SUM_BYTES / 16 / 256;
  if (a.sink_pieces > 0) {
    e = launch_with_lds<sink_dkdv_kernel<T, D, kPad, true>>(dim3((unsigned)a.sink_pieces), 256, SinkSmem<D>::BYTES + kLevelBytes, stream, a);
    return e != hipSuccess ? e : launch_with_lds<sink_sum_kernel<T, D, true>>(dim3((unsigned)(items * sum_groups)), 256, kLevelBytes, stream, a);
  }
  e = launch_with_lds<sink_dkdv_kernel<T, D, kPad, false>>(dim3((unsigned)(items * a.sink_parts)), 256, SinkSmem<D>::BYTES, stream, a);
  return e != hipSuccess || a.sink_parts == 1 ? e : launch_with_lds<sink_sum_kernel<T, D, false>>(dim3((unsigned)(items * sum_groups)), 256, 0, stream, a);
}

}  // namespace fa
