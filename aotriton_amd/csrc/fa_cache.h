// Attention of drafted tokens over a cache of pages: gfx950, MFMA 32x32x16.
#pragma once
#include "fa_cache_args.h"
#include "fa_device.h"

namespace fa {

// What a work item needs of its sequence.
struct TreeSeq {
  int32_t length, end;           // filled slots; slots with the drafted tokens, as far as the table goes (0: the sequence is not there)
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, int z) {
  const int n = a.cache.lengths[z];
  const int64_t room = (int64_t)a.cache.columns << a.cache.page_shift, end = (int64_t)n + a.tokens;
  TreeSeq s;
  s.length = n;
  s.end = n < 0 ? 0 : (int)(end < room ? end : room);
  return s;
}

// Ancestors (and self) of the drafted tokens: a lane's token is its own number.  parent[t] < t or -1; anything else means that the
// token is not there, and neither is what hangs on it.  Walks of 1, 2, 4, ... steps are put together in six rounds.
struct TreeNode {
  uint64_t kin;                  // 0: not there
  int32_t depth;
};
__device__ __forceinline__ uint64_t shfl64(uint64_t x, int lane) {
  return (uint64_t)(uint32_t)__shfl((int)(uint32_t)(x >> 32), lane) << 32 | (uint32_t)__shfl((int)(uint32_t)x, lane);
}
__device__ __forceinline__ TreeNode tree_nodes(const TreeArgs& a, int z, int length, int lane, uint64_t& there) {
  TreeNode n;
  const bool token = lane < a.tokens;
  if (a.parents == nullptr) {
    n.kin = token ? ~0ull >> (63 - lane) : 0;
    n.depth = lane;
    there = a.tokens < 64 ? (1ull << a.tokens) - 1 : ~0ull;
  } else {
    int up = -2;
    if (token) up = a.parents[(int64_t)z * a.parents_row + lane];
    const bool ok = up >= -1 && up < lane;
    if (!ok) up = -1;
    n.kin = 1ull << lane;
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      const int from = up < 0 ? lane : up;
      const uint64_t kin = shfl64(n.kin, from);
      const int next = __shfl(up, from);
      if (up >= 0) { n.kin |= kin; up = next; }
    }
    n.depth = __builtin_popcountll(n.kin) - 1;
    const uint64_t valid = __builtin_amdgcn_ballot_w64(ok);
    if ((n.kin & ~valid) != 0) n.kin = 0;
    there = __builtin_amdgcn_ballot_w64(n.kin != 0);
  }
  // ancestors that a window leaves behind (deep trees under a short window only)
  if (a.window > 0 && __builtin_amdgcn_ballot_w64(n.kin != 0 && n.depth >= a.window) != 0)
    for (int j = 0; j < a.tokens; ++j) {
      const int d = __builtin_amdgcn_readlane(n.depth, j);
      if (n.depth - d >= a.window && length + d >= a.sinks) n.kin &= ~(1ull << j);
    }
  return n;
}

// A sequence's pages: `at` is scalar, and the table is read through the scalar cache (a kernel does not write it).
struct PageTable {
  const __attribute__((address_space(4))) int32_t* row;
  int32_t columns, pages, shift;
  __device__ __forceinline__ PageTable(const CacheArgs& c, int z)
      : row((const __attribute__((address_space(4))) int32_t*)(c.table + (int64_t)z * c.table_row)), columns(c.columns), pages(c.pages), shift(c.page_shift) {}
  __device__ __forceinline__ int page_of(int slot) const {      // negative: not there
    const int col = slot >> shift;
    if (col < 0 || col >= columns) return -1;
    const int p = row[col];
    return p < pages ? p : -1;
  }
};

// The blocks of 32 slots that a sequence's rows may see: those that hold sinks, then those of the window (without one: all).
struct TreeBlocks {
  int win_lo, all_lo;            // first slot that some row, that every row sees by its window
  int sinks, first, front, blocks;
  __device__ __forceinline__ TreeBlocks(const TreeArgs& a, const TreeSeq& seq) {
    win_lo = all_lo = 0;
    if (a.window > 0) {
      win_lo = seq.length - a.window + 1 > 0 ? seq.length - a.window + 1 : 0;
      all_lo = seq.length + a.tokens - a.window > 0 ? seq.length + a.tokens - a.window : 0;
    }
    const int last = seq.end > 0 ? (seq.end - 1) / 32 : -1;
    first = win_lo / 32;
    sinks = a.window > 0 ? a.sinks : 0;
    front = sinks < first * 32 ? (sinks + 31) / 32 : first;
    blocks = last >= first ? front + last - first + 1 : 0;
  }
  __device__ __forceinline__ int block_of(int i) const { return i < front ? i : first + i - front; }
  // every row sees all of these slots, as far as their pages are there
  __device__ __forceinline__ bool whole(const TreeSeq& seq, int n0, int n) const {
    return n0 + n <= seq.length && (n0 >= all_lo || n0 + n <= sinks);
  }
  // some row sees slot n: what lies in the others may be inf or NaN
  __device__ __forceinline__ bool seen(const TreeSeq& seq, uint64_t there, int n) const {
    const int j = n - seq.length;
    return j < 0 ? (n >= win_lo || n < sinks) : j < 64 && (there >> (j & 63) & 1) != 0;
  }
  __device__ __forceinline__ int parts(const TreeArgs& a) const { return blocks > a.part_blocks ? (blocks + a.part_blocks - 1) / a.part_blocks : 1; }
};

// What a packed row sees.
struct TreeRow {
  uint64_t kin;
  int m_lo, m_sink;              // of the filled slots [m_lo, length) and those below m_sink
  bool alive;
  __device__ __forceinline__ TreeRow(const TreeArgs& a, const TreeSeq& seq, const TreeNode& node, uint64_t there, int token) {
    kin = shfl64(node.kin, token);
    const int depth = __shfl(node.depth, token);
    alive = (there >> token & 1) != 0;
    m_lo = !alive ? 0x7fffffff : a.window > 0 ? seq.length + depth - a.window + 1 : 0;
    m_sink = alive && a.window > 0 ? a.sinks : 0;
    if (!alive) kin = 0;
  }
  __device__ __forceinline__ bool sees(const TreeSeq& seq, int n) const {
    const int j = n - seq.length;
    return j < 0 ? (n >= m_lo || n < m_sink) : j < 64 && (kin >> (j & 63) & 1) != 0;
  }
};

// ---- few rows: 32 packed (token, q-head) rows of one K/V head x one part of its keys per workgroup -----------------------
// As fwd_rows_kernel: the waves take blocks of 32 slots in turn, each with an online softmax of its own; they meet in LDS, the parts
// in combine_rows_kernel.  K and V are read once per 32 rows, and what bounds it is HBM.  The blocks of an item are those that hold
// sinks, then those of the window (without one: all).
template <int D>
struct TreeSmem {
  static constexpr int VSTR = D + 32;                    // elements; transposing reads sweep all banks
  static constexpr int V_BYTES = 32 * VSTR * 2;          // per wave
  static constexpr int OSTR = D + 4;                     // floats per row of a wave's partial O
  static constexpr int O_BYTES = 32 * OSTR * 4;          // per wave
  static constexpr int ML_OFF = 4 * (V_BYTES > O_BYTES ? V_BYTES : O_BYTES);
  static constexpr int BYTES = ML_OFF + 4 * 32 * 8;
};

template <typename T, int D, bool kPad>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
__attribute__((amdgpu_waves_per_eu(D <= 128 ? 2 : 1, D <= 128 ? 2 : 1)))
void tree_rows_kernel(const TreeArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  using Tr = Traits<T>;
  using op_t = typename Tr::op_t;
  using q4_t = typename Tr::q4_t;
  using SM = TreeSmem<D>;
  constexpr int KS = D / 16, DB = D / 32;
  constexpr int VSTR = SM::VSTR, OSTR = SM::OSTR;
  constexpr int LPR = D / 8, RPI = 64 / LPR, CHV = 32 / RPI;      // V: lanes per row, rows per access, accesses

  // units (pair, part) go round the XCDs, the row blocks of a unit follow each other on one
  const CacheArgs& c = a.cache;
  const int xcd = blockIdx.x % kNumXcd, idx = blockIdx.x / kNumXcd;
  const int unit = (idx / a.row_blocks) * kNumXcd + xcd, rb = idx % a.row_blocks;
  const int pair = unit / a.parts, part = unit % a.parts;
  if (pair >= c.sequences * c.heads) return;
  const int z = pair / c.heads, hk = pair % c.heads, group = a.hq / c.heads;
  const TreeSeq seq = tree_seq(a, z);
  const TreeBlocks range(a, seq);
  const int parts = range.parts(a);
  if (part >= parts) return;
  const int rows = a.tokens * group, r0 = rb * 32;
  const int nrows = rows - r0 < 32 ? rows - r0 : 32;

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, col = lane & 31, hi = lane >> 5;
  const int d_qk = kPad ? c.head_dim : D, d_v = kPad ? c.head_dim_v : D;

  uint64_t there;
  const TreeNode node = tree_nodes(a, z, seq.length, lane, there);
  if (seq.end == 0) there = 0;

  // this lane's packed row: its drafted token, and what it sees
  const bool row_ok = col < nrows;
  const int pr = r0 + (row_ok ? col : nrows - 1);
  const int token = pr / group, h = hk * group + pr % group;
  const TreeRow row(a, seq, node, there, token);
  const int b0 = part * a.part_blocks, b1 = b0 + a.part_blocks < range.blocks ? b0 + a.part_blocks : range.blocks;

  // ---- Q rows as the B operand (column = packed row), straight from global memory ----------------
  op_t qreg[KS];
  {
    const T* qp = reinterpret_cast<const T*>(a.q) + (int64_t)z * a.sq.z + (int64_t)h * a.sq.h + (int64_t)token * a.sq.s + 8 * hi;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qreg[ks] = op_t{};
      if (row_ok && (!kPad || 16 * ks + 8 * hi < d_qk)) qreg[ks] = *reinterpret_cast<const op_t*>(qp + 16 * ks);
    }
  }

  const PageTable pages(c, z);
  const T* kbase = reinterpret_cast<const T*>(c.k) + (int64_t)hk * c.sk.h;
  const T* vbase = reinterpret_cast<const T*>(c.v) + (int64_t)hk * c.sv.h;
  const int slot_mask = (1 << c.page_shift) - 1;
  const int vr0 = lane / LPR, vc0 = lane % LPR;
  const bool v_col = !kPad || vc0 * 8 < d_v;
  // pages have 16 slots or more, so a block lies in two pages at most, 16 slots in one
  struct Halves { int p0, p1; };
  auto halves_of = [&](int b) {
    Halves x;
    x.p0 = pages.page_of(b * 32);
    x.p1 = pages.page_of(b * 32 + 16);
    return x;
  };
  op_t kreg[KS], vreg[CHV];
  // (a page that is not there stands aside for page 0, whose values are not used)
  auto load_block = [&](int b, Halves x) {
    const int s0 = (b * 32) & slot_mask, s1 = (b * 32 + 16) & slot_mask;
    const int64_t p0 = x.p0 < 0 ? 0 : x.p0, p1 = x.p1 < 0 ? 0 : x.p1;
    const T* k0 = kbase + p0 * c.sk.z + s0 * c.sk.s;
    const T* k1 = kbase + p1 * c.sk.z + s1 * c.sk.s;
    const T* v0 = vbase + p0 * c.sv.z + s0 * c.sv.s;
    const T* v1 = vbase + p1 * c.sv.z + s1 * c.sv.s;
    const T* kp = (col < 16 ? k0 : k1) + (col & 15) * c.sk.s + 8 * hi;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      kreg[ks] = op_t{};
      if (!kPad || 16 * ks + 8 * hi < d_qk) kreg[ks] = *reinterpret_cast<const op_t*>(kp + 16 * ks);
    }
#pragma unroll
    for (int i = 0; i < CHV; ++i) {
      const int r = vr0 + i * RPI;
      vreg[i] = op_t{};
      if (v_col) vreg[i] = *reinterpret_cast<const op_t*>((i * RPI < 16 ? v0 : v1) + (r & 15) * c.sv.s + vc0 * 8);
    }
  };

  T* vs = reinterpret_cast<T*>(smem_raw + wave * SM::V_BYTES);
  const int v_st = vr0 * VSTR + vc0 * 8;
  const T* v_ld = vs + (4 * hi + (lane & 15) / 4) * VSTR + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);      // see lds_read_tr8

  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
  float m_i = kNegBig, l_i = 0.f;      // running maximum (units of s below); this lane's half of the row sum
  const float qk_scale = a.sm_scale * kLog2e;
  const float sc = score_scale(a.sm_scale, false);
  const bool prescale = !(qk_scale > 0.f);

  int i = b0 + wave;
  Halves now{-1, -1}, next{-1, -1};
  if (i < b1) {
    now = halves_of(range.block_of(i));
    load_block(range.block_of(i), now);
    if (i + 4 < b1) next = halves_of(range.block_of(i + 4));
  }
  for (; i < b1; i += 4) {
    const int n0 = range.block_of(i) * 32;
    const bool edge = !range.whole(seq, n0, 32) || now.p0 < 0 || now.p1 < 0;
    f32x16 s;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = Tr::mfma(kreg[ks], qreg[ks], s);
    if (edge) {
      // V of slots that no row sees is 0: its probability is, and what lies there (a stale slot, a page of somebody else's, a drafted
      // token that is not there) may be inf or NaN
#pragma unroll
      for (int e = 0; e < CHV; ++e) {
        if (!range.seen(seq, there, n0 + vr0 + e * RPI) || (e * RPI < 16 ? now.p0 : now.p1) < 0) vreg[e] = op_t{};
      }
    }
#pragma unroll
    for (int e = 0; e < CHV; ++e) *reinterpret_cast<op_t*>(vs + v_st + e * RPI * VSTR) = vreg[e];
    const Halves was = now;
    if (i + 4 < b1) {
      now = next;
      load_block(range.block_of(i + 4), now);
      if (i + 8 < b1) next = halves_of(range.block_of(i + 8));
    }

    if (prescale)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] *= qk_scale;
    if (edge) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const bool seen = row.sees(seq, n0 + 8 * (e / 4) + 4 * hi + (e % 4)) && (e < 8 ? was.p0 : was.p1) >= 0;
        s[e] = seen ? s[e] : -__builtin_inff();
      }
    }

    float mx = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
    mx = cross_max(mx);
    // lazy rescaling and exp2 on differences, as in fwd_item
    const float m_cand = fmaxf(m_i, mx);
    const bool upd = (m_cand - m_i) * sc > 8.0f;
    const float m_new = upd ? m_cand : m_i;
    const float alpha = fast_exp2((m_i - m_new) * sc);
    m_i = m_new;
    float rs = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[e] = fast_exp2((s[e] - m_new) * sc);
      rs += s[e];
    }
    l_i = l_i * alpha + rs;
    if (__builtin_amdgcn_ballot_w64(upd) != 0) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[db][e] *= alpha;
    }
    const op_t p0 = pack8<T>(s, 0), p1 = pack8<T>(s, 1);
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = Tr::mfma(lds_read_tr8<T>(v_ld + db * 32, VSTR), p0, o[db]);
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = Tr::mfma(lds_read_tr8<T>(v_ld + 16 * VSTR + db * 32, VSTR), p1, o[db]);
  }

  // ---- the four waves' partial results meet in LDS --------------------------------------------
  // (a token that is not there is masked in edge blocks only; it ends without a sum, and what it summed is not looked at)
  const float l = row.alive ? cross_sum(l_i) : 0.f;
  __syncthreads();      // the V areas become the O areas
  float* ml = reinterpret_cast<float*>(smem_raw + SM::ML_OFF);
  float* ow = reinterpret_cast<float*>(smem_raw + wave * SM::O_BYTES);
  if (row_ok) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(ow + col * OSTR + 32 * db + 8 * g + 4 * hi) =
            f32x4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
    if (hi == 0) {
      ml[(wave * 32 + col) * 2] = m_i;      // (kNegBig where the wave saw no key of the row; l is 0 then)
      ml[(wave * 32 + col) * 2 + 1] = l;
    }
  }
  __syncthreads();
  constexpr int QPR = D / 4;      // pieces of four columns per row
  for (int e = tid; e < nrows * QPR; e += 256) {
    const int r = e / QPR, at = (e % QPR) * 4;
    float m = ml[r * 2];
#pragma unroll
    for (int v = 1; v < 4; ++v) m = fmaxf(m, ml[(v * 32 + r) * 2]);
    float lsum = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float f = fast_exp2((ml[(v * 32 + r) * 2] - m) * sc);
      lsum += f * ml[(v * 32 + r) * 2 + 1];
      acc += f * *reinterpret_cast<const f32x4*>(smem_raw + v * SM::O_BYTES + (r * OSTR + at) * 4);
    }
    if (parts > 1) {
      const int64_t to = ((int64_t)(pair * a.row_blocks + rb) * a.parts + part) * a.part_rows + r;
      *reinterpret_cast<f32x4*>(a.part_o + to * D + at) = acc;
      if (at == 0) {
        a.part_ml[to * 2] = m;
        a.part_ml[to * 2 + 1] = lsum;
      }
    } else {
      const int pq = (r0 + r) / group, ph = hk * group + (r0 + r) % group;
      if (at < d_v) {
        const float inv = lsum > 0.f ? 1.0f / lsum : 0.f;
        q4_t t4;
#pragma unroll
        for (int x = 0; x < 4; ++x) t4[x] = Tr::cvt(lsum > 0.f ? acc[x] * inv : 0.f);
        *reinterpret_cast<q4_t*>(reinterpret_cast<T*>(a.out) + (int64_t)z * a.so.z + (int64_t)ph * a.so.h + (int64_t)pq * a.so.s + at) = t4;
      }
      if (a.lse && at == 0) a.lse[((int64_t)z * a.hq + ph) * a.tokens + pq] = lse_of(m, sc, lsum);
    }
  }
}

// ---- the parts' sums: out = sum_i 2^((m_i - m) sc) O_i / sum_i 2^((m_i - m) sc) l_i ------------------------------------------------
// A thread takes four columns of a row, and of its parts every kSlots-th.  What bounds it is the latency of loads that miss L2 (other
// XCDs wrote them): with many parts of few rows the threads of a workgroup hold all parts of a row between them.
template <typename T, int D, int kSlots>
static __global__ __launch_bounds__(256) void tree_sum_kernel(const TreeArgs a) {
  constexpr int TPR = D / 4, ROWS = 256 / TPR / kSlots, AHEAD = 4;
  __shared__ f32x4 s_acc[kSlots > 1 ? 256 : 1];
  __shared__ float s_m[kSlots > 1 ? 256 / TPR : 1], s_l[kSlots > 1 ? 256 / TPR : 1];
  const CacheArgs& c = a.cache;
  const int chunks = (a.part_rows + ROWS - 1) / ROWS;
  const int block = blockIdx.x / chunks, pair = block / a.row_blocks, rb = block % a.row_blocks;
  const int z = pair / c.heads, hk = pair % c.heads, group = a.hq / c.heads;
  const TreeSeq seq = tree_seq(a, z);
  const int parts = TreeBlocks(a, seq).parts(a);
  if (parts <= 1) return;                              // (the whole workgroup: its results are there already)
  const int lane_row = threadIdx.x / TPR / kSlots, slot = threadIdx.x / TPR % kSlots, col = threadIdx.x % TPR * 4;
  const int r = blockIdx.x % chunks * ROWS + lane_row, pr = rb * a.row_rows + r;
  const bool ok = r < a.part_rows && pr < a.tokens * group;
  const float sc = score_scale(a.sm_scale, false);
  const int64_t at = (int64_t)block * a.parts * a.part_rows + (ok ? r : 0);
  const float* po = a.part_o + at * D + col;
  const float* pm = a.part_ml + at * 2;
  float m = kNegBig, l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = slot; i0 < parts; i0 += kSlots * AHEAD) {
    f32x4 x[AHEAD];
    vec<float, 2> ml[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = i0 + k * kSlots < parts ? i0 + k * kSlots : i0;
      ml[k] = *reinterpret_cast<const vec<float, 2>*>(pm + (int64_t)i * a.part_rows * 2);
      x[k] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(po + (int64_t)i * a.part_rows * D));
    }
    float top = m;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (i0 + k * kSlots >= parts) ml[k][1] = 0.f;
      if (ml[k][1] != 0.f) top = fmaxf(top, ml[k][0]);
    }
    const float f0 = fast_exp2((m - top) * sc);
    acc *= f0;
    l *= f0;
    m = top;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (ml[k][1] != 0.f) {                           // (a part in which the row sees nothing has sums of nothing)
        const float f = fast_exp2((ml[k][0] - m) * sc);
        l += f * ml[k][1];
        acc += f * x[k];
      }
  }
  if (kSlots > 1) {
    s_acc[threadIdx.x] = acc;
    if (col == 0) { s_m[threadIdx.x / TPR] = m; s_l[threadIdx.x / TPR] = l; }
    __syncthreads();
    if (slot != 0) return;
    float top = m;
#pragma unroll
    for (int k = 1; k < kSlots; ++k) top = fmaxf(top, s_m[lane_row * kSlots + k]);
    const float f0 = fast_exp2((m - top) * sc);
    acc *= f0;
    l *= f0;
#pragma unroll
    for (int k = 1; k < kSlots; ++k) {
      const float f = fast_exp2((s_m[lane_row * kSlots + k] - top) * sc);
      l += f * s_l[lane_row * kSlots + k];
      acc += f * s_acc[threadIdx.x + k * TPR];
    }
    m = top;
  }
  if (!ok) return;
  const int token = pr / group, h = hk * group + pr % group;
  if (col < c.head_dim_v) {
    const float inv = l > 0.f ? 1.0f / l : 0.f;
    vec<T, 4> t;
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = Traits<T>::cvt(acc[j] * inv);
    *reinterpret_cast<vec<T, 4>*>(reinterpret_cast<T*>(a.out) + (int64_t)z * a.so.z + (int64_t)h * a.so.h + (int64_t)token * a.so.s + col) = t;
  }
  if (a.lse && col == 0) a.lse[((int64_t)z * a.hq + h) * a.tokens + token] = lse_of(m, sc, l);
}

template <typename T, int D, int kSlots>
hipError_t launch_tree_sum_slots(const TreeArgs& a, hipStream_t stream) {
  constexpr int ROWS = 256 / (D / 4) / kSlots;
  const unsigned blocks = (unsigned)(a.cache.sequences * a.cache.heads * a.row_blocks);
  hipLaunchKernelGGL((tree_sum_kernel<T, D, kSlots>), dim3(blocks * ((a.part_rows + ROWS - 1) / ROWS)), dim3(256), 0, stream, a);
  return hipGetLastError();
}
// Slots of a row: as many as halve the rounds of loads while the rows alone leave the chip empty.
template <typename T, int D>
hipError_t launch_tree_sum(const TreeArgs& a, hipStream_t stream) {
  const int64_t rows = (int64_t)a.cache.sequences * a.cache.heads * a.row_blocks * a.part_rows;
  if (a.parts <= 4 || rows > 4096) return launch_tree_sum_slots<T, D, 1>(a, stream);
  return launch_tree_sum_slots<T, D, 256 / (D / 4)>(a, stream);
}

template <typename T, int D, bool kPad>
hipError_t launch_tree_rows(const TreeArgs& a, hipStream_t stream) {
  auto kern = tree_rows_kernel<T, D, kPad>;
  constexpr int smem = TreeSmem<D>::BYTES;
  if (smem > 64 * 1024) {
    static std::atomic<uint64_t> lds_set{0};
    const hipError_t e = allow_large_lds(reinterpret_cast<const void*>(kern), smem, lds_set);
    if (e != hipSuccess) return e;
  }
  const int pairs = a.cache.sequences * a.cache.heads;
  const int units = (pairs * a.parts + kNumXcd - 1) / kNumXcd;
  if (units == 0 || a.row_blocks == 0) return hipSuccess;
  hipLaunchKernelGGL(kern, dim3((unsigned)(kNumXcd * units * a.row_blocks)), dim3(256), smem, stream, a);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess || a.parts <= 1 ? e : launch_tree_sum<T, D>(a, stream);
}

}  // namespace fa
