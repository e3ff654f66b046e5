// Attention of drafted tokens over a cache of pages: gfx950, MFMA 32x32x16.
#pragma once
#include "fa_cache_args.h"
#include "fa_device.h"
#include "fa_wide.h"

namespace fa {

// What a work item needs of its sequence.
struct TreeSeq {
  int32_t length, end;           // filled slots; slots with the drafted tokens, as far as the table goes (0: the sequence is not there)
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, int z) {
  // (positions, which are up to 63 more, stay below 2^31; the table, and with it what such a sequence sees, ends at 2^29)
  const int raw = a.cache.lengths[z], n = raw < 0x7fffffff - kTreeTokens ? raw : 0x7fffffff - kTreeTokens;
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
// (the parents are asked for early, and looked at while the first keys are on their way)
__device__ __forceinline__ int tree_parent(const TreeArgs& a, int z, int lane) {
  return a.parents != nullptr && lane < a.tokens ? a.parents[(int64_t)z * a.parents_row + lane] : -2;
}
__device__ __forceinline__ TreeNode tree_nodes(const TreeArgs& a, int up, int length, int lane, uint64_t& there) {
  TreeNode n;
  const bool token = lane < a.tokens;
  if (a.parents == nullptr) {
    n.kin = token ? ~0ull >> (63 - lane) : 0;
    n.depth = lane;
    there = a.tokens < 64 ? (1ull << a.tokens) - 1 : ~0ull;
  } else {
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

// Pages of a run of 16-slot stretches, entry by entry in order: 64 of them are looked up at once, a lane each, and the 64 behind them
// are on their way.  (One at a time through the scalar cache every look-up waited for the one before: B32 4900 slots, 48 tokens 225 us instead of 205.)
template <typename SlotOf>      // the slot of an entry, -1 behind the last
struct PageRun {
  const int32_t* row;
  int32_t columns, pages, shift, lane;
  SlotOf slot_of;
  int now, next, first;          // this lane's pages (-1: not there); the first entry of `now`
  __device__ __forceinline__ int look(int entry) const {
    const int slot = slot_of(entry), col = slot >> shift;
    int p = -1;
    if (slot >= 0 && col < columns) p = row[col];
    return p < pages ? p : -1;
  }
  __device__ __forceinline__ PageRun(const CacheArgs& c, int z, int lane_, SlotOf f)
      : row(c.table + (int64_t)z * c.table_row), columns(c.columns), pages(c.pages), shift(c.page_shift), lane(lane_), slot_of(f), first(0) {
    now = look(lane);
    next = look(lane + 64);
  }
  __device__ __forceinline__ void to(int entry) {      // 0, or at most 64 after the last
    if (entry - first < 64) return;
    now = next;
    first += 64;
    next = look(first + 64 + lane);
  }
  __device__ __forceinline__ int at(int entry) const { return __builtin_amdgcn_readlane(now, entry - first); }      // negative: not there
  __device__ __forceinline__ int holes(int entry) const { return (int)(__builtin_amdgcn_ballot_w64(now < 0) >> (entry - first)); }      // a bit for each
};

// The blocks of slots that a sequence's rows may see: those that hold sinks, then those of the window (without one: all).
struct TreeBlocks {
  int win_lo, all_lo;            // first slot that some row, that every row sees by its window
  int sinks, first, front, blocks;
  __device__ __forceinline__ TreeBlocks(const TreeArgs& a, const TreeSeq& seq) {
    win_lo = all_lo = 0;
    if (a.window > 0) {
      win_lo = seq.length - a.window + 1 > 0 ? seq.length - a.window + 1 : 0;
      all_lo = seq.length + a.tokens - a.window > 0 ? seq.length + a.tokens - a.window : 0;
    }
    const int shift = a.block_shift, last = seq.end > 0 ? (seq.end - 1) >> shift : -1;
    first = win_lo >> shift;
    sinks = a.window > 0 ? a.sinks : 0;
    front = sinks < first << shift ? (sinks + (1 << shift) - 1) >> shift : first;
    // (a window that starts behind the table leaves the sinks)
    blocks = last >= first ? front + last - first + 1 : front < last + 1 ? front : last + 1;
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
};
__device__ __forceinline__ int tree_blocks(const TreeArgs& a, int z) {      // in the list of all sequences' blocks: one at least
  const int n = TreeBlocks(a, tree_seq(a, z)).blocks;
  return n > 1 ? n : 1;
}

// The list of all sequences' blocks, and its cut into pieces.  Every lane of a wave takes part in the functions.
struct TreeList {
  int64_t per, total;            // blocks of a piece, of all
  int z;                         // of seek
  int64_t start;                 // of the sequence that cut or seek was asked for
  int n, sum;                    // of the last 64 sequences that cut looked at: this lane's blocks, and the sum up to it
  __device__ __forceinline__ void look(const TreeArgs& a, int base, int lane) {
    n = base + lane < a.cache.sequences ? tree_blocks(a, base + lane) : 0;
    sum = n;
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
      const int y = __shfl_up(sum, i);
      sum += lane >= i ? y : 0;
    }
  }
  __device__ __forceinline__ void cut(const TreeArgs& a, int lane, int find) {      // find < 0: none
    total = 0;
    start = 0;
    for (int base = 0; base < a.cache.sequences; base += 64) {
      look(a, base, lane);
      if (find >= base && find < base + 64) start = total + __builtin_amdgcn_readlane(sum - n, find - base);
      total += __builtin_amdgcn_readlane(sum, 63);
    }
    const int64_t even = (total + a.workers - 1) / a.workers;
    per = even > a.least ? even : a.least;
  }
  __device__ __forceinline__ void seek(const TreeArgs& a, int lane, int64_t at) {      // the sequence of block at < total
    int64_t before = 0;
    for (int base = 0; base < a.cache.sequences; base += 64) {
      if (a.cache.sequences > 64) look(a, base, lane);
      const int all = __builtin_amdgcn_readlane(sum, 63);
      if (at < before + all) {
        const int i = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before + sum > at));
        z = base + i;
        start = before + __builtin_amdgcn_readlane(sum - n, i);
        return;
      }
      before += all;
    }
  }
};

// First row of the sums of a sequence in one of its pieces.  A piece of the list has two places: for the one sequence that
// began in front of it, and for the one that begins in it and goes on behind.
__device__ __forceinline__ int64_t tree_sums(const TreeArgs& a, int hk, int rb, int piece, int z, bool begins) {
  const int64_t block = hk * a.row_blocks + rb;
  return (a.workers > 0 ? (block * a.workers + piece) * 2 + (begins ? 1 : 0) : (block * a.cache.sequences + z) * a.parts + piece) * a.part_rows;
}

// A workgroup's items: f(sequence, head, block of rows, first block, end, whether these are all of the sequence's, piece).
template <typename F>
__device__ __forceinline__ void tree_work(const TreeArgs& a, int lane, F f) {
  // units go round the XCDs, the row blocks of one follow each other on one XCD
  const int xcd = blockIdx.x % kNumXcd, idx = blockIdx.x / kNumXcd, heads = a.cache.heads;
  const int unit = (idx / a.row_blocks) * kNumXcd + xcd, rb = idx % a.row_blocks;
  const int hk = unit % heads;
  int z, first, take, size, piece;
  int64_t at = 0, end = 1;
  TreeList list;
  if (a.workers > 0) {
    piece = unit / heads;
    if (piece >= a.workers) return;
    list.cut(a, lane, -1);
    at = piece * list.per;
    end = at + list.per < list.total ? at + list.per : list.total;
    if (at >= end) return;
    list.seek(a, lane, at);
    z = list.z;
  } else {
    // (all sequences' first pieces in front: every sequence has one, the long ones have the others)
    z = unit / heads % a.cache.sequences;
    piece = unit / heads / a.cache.sequences;
    if (piece >= a.parts) return;
  }
  for (;; ++z) {
    size = tree_blocks(a, z);
    if (a.workers > 0) {
      first = (int)(at - list.start);
      take = size - first < end - at ? size - first : (int)(end - at);
    } else {
      // (the last piece has what is left, also of a sequence that is longer than planned)
      first = piece * a.part_blocks;
      if (piece > 0 && first >= size) return;
      take = piece + 1 == a.parts || size - first < a.part_blocks ? size - first : a.part_blocks;
    }
    f(z, hk, rb, first, first + take, take == size, piece);
    at += take;
    if (at >= end) return;
    list.start += size;
    __syncthreads();      // the next item reuses the LDS areas
  }
}

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
  // Bit b: the row sees slot n0 + b.  (A test of its own for each slot: 48 tokens, B8 up to 16384 slots 76 us instead of 67, 64 tokens Hq 64
  // D64 80 instead of 64.)
  __device__ __forceinline__ uint64_t sees(const TreeSeq& seq, int n0) const {
    const int d = seq.length - n0;
    const uint64_t drafted = d >= 64 || d <= -64 ? 0 : d >= 0 ? kin << d : kin >> -d;
    return (below(d) & (~below(m_lo - n0) | below(m_sink - n0))) | drafted;
  }
  static __device__ __forceinline__ uint64_t below(int n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; }
};

// ---- few rows: 32 packed (token, q-head) rows of one K/V head x one piece of the keys per workgroup -----------------------
// As fwd_rows_kernel: the waves take blocks of 32 slots in turn, each with an online softmax of its own; they meet in LDS, the parts
// in tree_sum_kernel.  K and V are read once per 32 rows, and what bounds it is HBM (B64 up to 8192 slots, Hq 32 Hk 8 D128, one token:
// 654 MB in 129 us, in tiles 126), for short sequences the chain from the length over the page table to the rows (B1 4096 slots 8.1 us,
// 17 MB).  The blocks of an item are those that hold sinks, then those of the window (without one: all).
template <int D>
struct TreeSmem {
  static constexpr int KSTR = D + 8;                     // elements; row reads sweep all banks
  static constexpr int VSTR = D + 32;                    // the same for transposing reads
  static constexpr int V_BYTES = 32 * VSTR * 2;          // per wave: a block's K, then its V
  static constexpr int OSTR = D + 4;                     // floats per row of a wave's partial O
  static constexpr int O_BYTES = 32 * OSTR * 4;          // per wave
  static constexpr int ML_OFF = 4 * (V_BYTES > O_BYTES ? V_BYTES : O_BYTES);
  static constexpr int BYTES = ML_OFF + 4 * 32 * 8;
};

// Blocks [from, to) of sequence z; `whole`: they are all of its blocks.
template <typename T, int D, bool kPad>
__device__ __forceinline__ void tree_rows_item(const TreeArgs& a, const int z, const int hk, const int rb, const int from, const int to,
                                               const bool whole, const int piece, char* smem_raw) {
  using Tr = Traits<T>;
  using op_t = typename Tr::op_t;
  using q4_t = typename Tr::q4_t;
  using SM = TreeSmem<D>;
  constexpr int KS = D / 16, DB = D / 32;
  constexpr int KSTR = SM::KSTR, VSTR = SM::VSTR, OSTR = SM::OSTR;
  constexpr int LPR = D / 8, RPI = 64 / LPR, CH = 32 / RPI;      // lanes per row, rows per access, accesses
  const CacheArgs& c = a.cache;
  const int group = a.hq / c.heads;
  const TreeSeq seq = tree_seq(a, z);
  const TreeBlocks range(a, seq);
  const int rows = a.tokens * group, r0 = rb * 32;
  const int nrows = rows - r0 < 32 ? rows - r0 : 32;

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, col = lane & 31, hi = lane >> 5;
  const int d_qk = kPad ? c.head_dim : D, d_v = kPad ? c.head_dim_v : D;

  const int up = tree_parent(a, z, lane);
  const int b1 = to < range.blocks ? to : range.blocks;
  auto slot_of_half = [&](int e) {
    const int i = from + wave + 4 * (e >> 1);
    return i < b1 ? range.block_of(i) * 32 + 16 * (e & 1) : -1;
  };
  PageRun<decltype(slot_of_half)> pages(c, z, lane, slot_of_half);

  // this lane's packed row: its drafted token
  const bool row_ok = col < nrows;
  const int pr = r0 + (row_ok ? col : nrows - 1);
  const int token = pr / group, h = hk * group + pr % group;

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

  const T* kbase = reinterpret_cast<const T*>(c.k) + (int64_t)hk * c.sk.h;
  const T* vbase = reinterpret_cast<const T*>(c.v) + (int64_t)hk * c.sv.h;
  const int slot_mask = (1 << c.page_shift) - 1;
  const int vr0 = lane / LPR, vc0 = lane % LPR;
  const bool k_col = !kPad || vc0 * 8 < d_qk, v_col = !kPad || vc0 * 8 < d_v;
  // pages have 16 slots or more, so a block lies in two pages at most, 16 slots in one
  struct Halves { int p0, p1; };
  auto halves_of = [&](int i) {
    const int e = (i - from - wave) >> 1;
    pages.to(e);
    return Halves{pages.at(e), pages.at(e + 1)};
  };
  // K and V travel as whole rows, 16 bytes per lane and consecutive lanes along a row, and change to the operands' layouts in the wave's
  // LDS area, one after the other.  (K loaded as the operand that it is, 16 bytes of 32 rows per access, takes its cache lines a quarter at
  // a time: B64 Hq 32 Hk 8 up to 8192 slots D128 226 us instead of 193.)
  op_t kreg[CH], vreg[CH];
  const int64_t k_off = vr0 * c.sk.s + vc0 * 8, v_off = vr0 * c.sv.s + vc0 * 8;
  // (a page that is not there stands aside for page 0, whose values are not used)
  auto load_k = [&](int b, Halves x) {
    const T* p0 = kbase + (int64_t)(x.p0 < 0 ? 0 : x.p0) * c.sk.z + ((b * 32) & slot_mask) * c.sk.s;
    const T* p1 = kbase + (int64_t)(x.p1 < 0 ? 0 : x.p1) * c.sk.z + ((b * 32 + 16) & slot_mask) * c.sk.s;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      kreg[i] = op_t{};
      if (k_col) kreg[i] = *reinterpret_cast<const op_t*>((i * RPI < 16 ? p0 : p1) + (i * RPI & 15) * c.sk.s + k_off);
    }
  };
  auto load_v = [&](int b, Halves x) {
    const T* p0 = vbase + (int64_t)(x.p0 < 0 ? 0 : x.p0) * c.sv.z + ((b * 32) & slot_mask) * c.sv.s;
    const T* p1 = vbase + (int64_t)(x.p1 < 0 ? 0 : x.p1) * c.sv.z + ((b * 32 + 16) & slot_mask) * c.sv.s;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      vreg[i] = op_t{};
      if (v_col) vreg[i] = *reinterpret_cast<const op_t*>((i * RPI < 16 ? p0 : p1) + (i * RPI & 15) * c.sv.s + v_off);
    }
  };

  T* area = reinterpret_cast<T*>(smem_raw + wave * SM::V_BYTES);
  const int k_st = vr0 * KSTR + vc0 * 8, v_st = vr0 * VSTR + vc0 * 8;
  const T* k_ld = area + col * KSTR + 8 * hi;
  const T* v_ld = area + (4 * hi + (lane & 15) / 4) * VSTR + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);      // see lds_read_tr8

  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
  float m_i = kNegBig, l_i = 0.f;      // running maximum (units of s below); this lane's half of the row sum
  const float qk_scale = a.sm_scale * kLog2e;
  const float sc = score_scale(a.sm_scale, false);
  const bool prescale = !(qk_scale > 0.f);

  int i = from + wave;
  Halves now{-1, -1}, next{-1, -1};
  if (i < b1) {
    now = halves_of(i);
    load_k(range.block_of(i), now);
    load_v(range.block_of(i), now);
    if (i + 4 < b1) next = halves_of(i + 4);
  }
  uint64_t there;
  const TreeNode node = tree_nodes(a, up, seq.length, lane, there);
  if (seq.end == 0) there = 0;
  const TreeRow row(a, seq, node, there, token);
  for (; i < b1; i += 4) {
    const int n0 = range.block_of(i) * 32;
    const bool edge = !range.whole(seq, n0, 32) || now.p0 < 0 || now.p1 < 0;
    const Halves was = now;
#pragma unroll
    for (int e = 0; e < CH; ++e) *reinterpret_cast<op_t*>(area + k_st + e * RPI * KSTR) = kreg[e];
    if (i + 4 < b1) load_k(range.block_of(i + 4), next);
    op_t ka[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) ka[ks] = *reinterpret_cast<const op_t*>(k_ld + 16 * ks);
    f32x16 s;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = Tr::mfma(ka[ks], qreg[ks], s);
    if (edge) {
      // V of slots that no row sees is 0: its probability is, and what lies there (a stale slot, a page of somebody else's, a drafted
      // token that is not there) may be inf or NaN
#pragma unroll
      for (int e = 0; e < CH; ++e)
        if (!range.seen(seq, there, n0 + vr0 + e * RPI) || (e * RPI < 16 ? was.p0 : was.p1) < 0) vreg[e] = op_t{};
    }
    // (the area is the wave's own and its LDS operations run in order: K has been read)
#pragma unroll
    for (int e = 0; e < CH; ++e) *reinterpret_cast<op_t*>(area + v_st + e * RPI * VSTR) = vreg[e];
    if (i + 4 < b1) {
      now = next;
      load_v(range.block_of(i + 4), now);
      if (i + 8 < b1) next = halves_of(i + 8);
    }

    if (prescale)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] *= qk_scale;
    if (edge) {
      const uint32_t there_now = (was.p0 < 0 ? 0 : 0xffffu) | (was.p1 < 0 ? 0 : 0xffff0000u);
      const uint32_t seen = ((uint32_t)row.sees(seq, n0) & there_now) >> 4 * hi;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = (seen >> (8 * (e / 4) + e % 4) & 1) != 0 ? s[e] : -__builtin_inff();
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
  // (a token that is not there is masked in edge blocks only; it ends without a sum, and what it summed is not looked at.  Nor is its
  // maximum, which a query that may hold anything can make inf: differences of those would be NaN)
  const float l = row.alive ? cross_sum(l_i) : 0.f;
  if (!row.alive) m_i = kNegBig;
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
    if (!whole) {
      const int64_t sums = tree_sums(a, hk, rb, piece, z, from == 0) + r;
      *reinterpret_cast<f32x4*>(a.part_o + sums * D + at) = acc;
      if (at == 0) {
        a.part_ml[sums * 2] = m;
        a.part_ml[sums * 2 + 1] = lsum;
      }
    } else {
      const int pq = (r0 + r) / group, ph = hk * group + (r0 + r) % group;
      if (at < d_v) {
        const float inv = 1.0f / lsum;
        q4_t t4;
#pragma unroll
        for (int x = 0; x < 4; ++x) t4[x] = Tr::cvt(lsum == 0.f ? 0.f : acc[x] * inv);      // (a NaN stays one)
        *reinterpret_cast<q4_t*>(reinterpret_cast<T*>(a.out) + (int64_t)z * a.so.z + (int64_t)ph * a.so.h + (int64_t)pq * a.so.s + at) = t4;
      }
      if (a.lse && at == 0) a.lse[((int64_t)z * a.hq + ph) * a.tokens + pq] = lse_of(m, sc, lsum);
    }
  }
}

template <typename T, int D, bool kPad>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256)))
__attribute__((amdgpu_waves_per_eu(D <= 128 ? 2 : 1, D <= 128 ? 2 : 1)))
void tree_rows_kernel(const TreeArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  tree_work(a, threadIdx.x & 63, [&](int z, int hk, int rb, int from, int to, bool whole, int piece) __attribute__((always_inline)) {
    tree_rows_item<T, D, kPad>(a, z, hk, rb, from, to, whole, piece, smem_raw);
  });
}

// ---- many rows: 32 * NW packed rows of one K/V head x one piece of the keys per workgroup ---------------------------------------
// With 64 drafted tokens and grouped heads a K/V head has hundreds of packed rows.  The kernel above would read its K and V once per 32 of
// them (from L2) and feed one MFMA operand with each piece; here a tile of 64 slots is staged in LDS once for all waves, which own
// 32 rows each, as in fwd_item (swizzled rows, one barrier per tile).  Bound by HBM up to about 128 rows, by what the waves issue beyond: 192 rows (48 tokens, Hq 32 Hk 8 D128, B8 up to 16384 slots) take six of eight waves,
// 57 us for 159 MB and 29 GFLOP.
// Tiles go from memory into LDS without registers.  With one workgroup on a CU (256 rows) two of them are on their way: a tile is worked
// on in less time than memory takes to answer.
template <int D, int NW>
struct TreeTileSmem {
  static constexpr int ROWB = Swz<D>::ROWB, TILE_BYTES = 64 * ROWB, STAGE_BYTES = 2 * TILE_BYTES;      // K, V (swizzled)
  static constexpr int STAGES = NW == 8 ? 3 : 2;
  static constexpr int BYTES = STAGES * STAGE_BYTES;
};

template <typename T, int D, int NW, bool kPad>
__device__ __forceinline__ void tree_tile_item(const TreeArgs& a, const int z, const int hk, const int rb, const int from, const int to,
                                               const bool whole, const int piece, char* smem_raw) {
  using Tr = Traits<T>;
  using op_t = typename Tr::op_t;
  using q4_t = typename Tr::q4_t;
  using SM = TreeTileSmem<D, NW>;
  constexpr int KS = D / 16, DB = D / 32, ROWB = SM::ROWB, AHEAD = SM::STAGES - 1;
  constexpr int LPR = D / 8, RW = 64 / LPR, RPI = NW * RW, CH = 64 / RPI;      // lanes per row; rows per wave's access, per workgroup's; accesses
  static_assert(16 % RW == 0 && (RPI % 16 == 0), "a wave's access lies in 16 slots, its swizzle in all of them");

  const CacheArgs& c = a.cache;
  const int group = a.hq / c.heads;
  const TreeSeq seq = tree_seq(a, z);
  const TreeBlocks range(a, seq);
  const int rows = a.tokens * group;

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, col = lane & 31, hi = lane >> 5;
  const int d_qk = kPad ? c.head_dim : D, d_v = kPad ? c.head_dim_v : D;
  const int up = tree_parent(a, z, lane);
  const int t0 = from, t1 = to < range.blocks ? to : range.blocks;
  auto slot_of = [&](int t) { return range.block_of(t) * 64; };
  auto slot_of_quarter = [&](int e) {
    const int t = t0 + (e >> 2);
    return t < t1 ? slot_of(t) + 16 * (e & 3) : -1;
  };
  PageRun<decltype(slot_of_quarter)> table(c, z, lane, slot_of_quarter);

  // this lane's packed row (waves past the last row only stage)
  const int first_row = rb * a.row_rows + wave * 32;
  const bool active = first_row < rows;
  const bool row_ok = first_row + col < rows;
  const int pr = row_ok ? first_row + col : rows - 1;
  const int token = pr / group, h = hk * group + pr % group;
  op_t qreg[KS];
  {
    const T* qp = reinterpret_cast<const T*>(a.q) + (int64_t)z * a.sq.z + (int64_t)h * a.sq.h + (int64_t)token * a.sq.s + 8 * hi;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qreg[ks] = op_t{};
      if (row_ok && (!kPad || 16 * ks + 8 * hi < d_qk)) qreg[ks] = *reinterpret_cast<const op_t*>(qp + 16 * ks);
    }
  }

  const T* kbase = reinterpret_cast<const T*>(c.k) + (int64_t)hk * c.sk.h;
  const T* vbase = reinterpret_cast<const T*>(c.v) + (int64_t)hk * c.sv.h;
  const int slot_mask = (1 << c.page_shift) - 1;
  // strides in 32 bits (check_pages): products of two scalar instructions instead of six
  const uint32_t k_page = (uint32_t)c.sk.z, v_page = (uint32_t)c.sv.z, k_slot = (uint32_t)c.sk.s, v_slot = (uint32_t)c.sv.s;
  const int k_bytes = ((RW - 1) * (int)c.sk.s + d_qk) * 2, v_bytes = ((RW - 1) * (int)c.sv.s + d_v) * 2;
  const int rl = lane / LPR, cl = lane % LPR;      // the lane's row within a wave's access, and where its piece goes
  const int ch = cl ^ Swz<D>::f(wave * RW + rl);
  const int k_voff = !kPad || ch * 8 < d_qk ? rl * (int)c.sk.s * 2 + ch * 16 : kVoffOutOfRange;
  const int v_voff = !kPad || ch * 8 < d_v ? rl * (int)c.sv.s * 2 + ch * 16 : kVoffOutOfRange;
  // access i of this wave: rows row_of(i) .. + RW - 1 of the tile
  auto row_of = [&](int i) { return wave * RW + i * RPI; };
  const int smem0 = lds_offset(smem_raw);
  // (a page that is not there: a descriptor of nothing, which reads as zero)
  auto fetch = [&](int stage, int t) __attribute__((always_inline)) {
    const int e = (t - t0) * 4, n0 = slot_of(t);
    table.to(e);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int p = table.at(e + row_of(i) / 16), slot = (n0 + row_of(i)) & slot_mask, lds = smem0 + stage + row_of(i) * ROWB;
      const uint32_t page = p < 0 ? 0 : p;
      load_to_lds1(wave_rsrc_words(kbase + ((uint64_t)page * k_page + (uint64_t)(uint32_t)slot * k_slot), p < 0 ? 0 : k_bytes), k_voff, lds);
      load_to_lds1(wave_rsrc_words(vbase + ((uint64_t)page * v_page + (uint64_t)(uint32_t)slot * v_slot), p < 0 ? 0 : v_bytes), v_voff, lds + SM::TILE_BYTES);
    }
  };
  // stages and holes of the tile that is worked on and of those behind it
  int st[SM::STAGES], holes[AHEAD + 1];
#pragma unroll
  for (int i = 0; i < SM::STAGES; ++i) st[i] = i * SM::STAGE_BYTES;
  auto ask = [&](int i, int t) __attribute__((always_inline)) {      // for tile t, i behind the one that is worked on
    holes[i] = 0;
    if (t >= t1) return;
    fetch(st[i], t);
    holes[i] = table.holes((t - t0) * 4) & 15;
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) ask(i, t0 + i);

  uint64_t there;
  const TreeNode node = tree_nodes(a, up, seq.length, lane, there);
  if (seq.end == 0) there = 0;
  const TreeRow row(a, seq, node, there, token);
  auto is_edge = [&](int n0, int holes) { return !range.whole(seq, n0, 64) || holes != 0; };
  // The tile at n0 has landed, as far as this wave brought it (`more`: the one behind it is on its way): V of slots that no row sees
  // becomes 0, as above.
  auto landed = [&](int stage, int n0, int holes, bool more) __attribute__((always_inline)) {
    if (AHEAD == 2 && more) asm volatile("s_waitcnt vmcnt(%0)" :: "n"(2 * CH) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (is_edge(n0, holes)) {
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if (!range.seen(seq, there, n0 + row_of(i) + rl))
          *reinterpret_cast<op_t*>(smem_raw + stage + SM::TILE_BYTES + (row_of(i) + rl) * ROWB + cl * 16) = op_t{};
    }
  };
  // (no wait for what is on its way)
  auto meet = [&]() __attribute__((always_inline)) { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[db][e] = 0.f;
  float m_i = kNegBig, l_i = 0.f;
  const float qk_scale = a.sm_scale * kLog2e;
  const float sc = score_scale(a.sm_scale, false);
  const bool prescale = !(qk_scale > 0.f);
  const int row_a = Swz<D>::row_base(lane), tr_a0 = Swz<D>::tr_base(lane, 0), tr_a1 = Swz<D>::tr_base(lane, 1);

  // S^T = K Q^T with the operands read two k-steps ahead of their MFMAs; V's first operands are in flight while the softmax runs; the
  // exponentials are taken against the maximum that the rows have already, and a tile whose row sums tell that it does not do
  // goes through the full step: all as in fwd_item.
  f32x16 s[2];
  op_t va[2][DB];
  auto qk = [&](int stage) __attribute__((always_inline)) {
    const char* ks = smem_raw + stage;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[mb][e] = 0.f;
    __builtin_amdgcn_s_setprio(2);
    constexpr int kAhead = 2;
    op_t ka[kAhead + 1][2];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) ka[k][mb] = swz_read_row<T, D>(ks, row_a, k, mb);
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      if (k + kAhead < KS)
#pragma unroll
        for (int mb = 0; mb < 2; ++mb)
          ka[(k + kAhead) % (kAhead + 1)][mb] = swz_read_row<T, D>(ks, row_a, k + kAhead, mb);
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) s[mb] = Tr::mfma(ka[k % (kAhead + 1)][mb], qreg[k], s[mb]);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
  };
  auto prepare = [&](int stage, int n0, int holes, bool edge) __attribute__((always_inline)) {
    const char* vs = smem_raw + stage + SM::TILE_BYTES;
#pragma unroll
    for (int db = 0; db < DB; ++db) va[0][db] = swz_read_tr<T, D>(vs, tr_a0, tr_a1, 0, db);
    if (prescale) {
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[mb][e] *= qk_scale;
    }
    if (edge) {
      const uint64_t all = row.sees(seq, n0);
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) {
        const uint32_t there_now = (holes >> 2 * mb & 1 ? 0 : 0xffffu) | (holes >> 2 * mb & 2 ? 0 : 0xffff0000u);
        const uint32_t seen = ((uint32_t)(all >> 32 * mb) & there_now) >> 4 * hi;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[mb][e] = (seen >> (8 * (e / 4) + e % 4) & 1) != 0 ? s[mb][e] : -__builtin_inff();
      }
    }
  };
  auto finish = [&](int stage) __attribute__((always_inline)) {
    const char* vs = smem_raw + stage + SM::TILE_BYTES;
    op_t pb[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) pb[k] = pack8<T>(s[k / 2], k % 2);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(2);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k + 1 < 4)
#pragma unroll
        for (int db = 0; db < DB; ++db) va[(k + 1) & 1][db] = swz_read_tr<T, D>(vs, tr_a0, tr_a1, k + 1, db);
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] = Tr::mfma(va[k & 1][db], pb[k], o[db]);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
  };
  bool have_ref = false;      // every row of the wave has a usable maximum
  float msc = 0.f;            // m_i * sc
  auto fast_step = [&](int stage, int n0, int holes, bool edge) __attribute__((always_inline)) {
    prepare(stage, n0, holes, edge);
    float rs = 0.f;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[mb][e] = fast_exp2(__builtin_fmaf(s[mb][e], sc, -msc));
        rs += s[mb][e];
      }
    if (__builtin_amdgcn_ballot_w64(!(rs < 4096.f)) != 0) return false;      // also inf and NaN
    l_i += rs;
    finish(stage);
    return true;
  };
  auto full_step = [&](int stage, int n0, int holes, bool edge) __attribute__((always_inline)) {
    prepare(stage, n0, holes, edge);
    float mx = s[0][0];
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[mb][e]);
    mx = cross_max(mx);
    const float m_cand = fmaxf(m_i, mx);
    const bool upd = (m_cand - m_i) * sc > 8.0f;
    const float m_new = upd ? m_cand : m_i;
    const float alpha = fast_exp2((m_i - m_new) * sc);
    m_i = m_new;
    msc = m_new * sc;
    // (a row that has seen nothing yet keeps the seed, and with it the wave the full step)
    have_ref = __builtin_amdgcn_ballot_w64(!(__builtin_fabsf(msc) < 1024.f)) == 0;
    float rs = 0.f;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[mb][e] = fast_exp2((s[mb][e] - m_new) * sc);
        rs += s[mb][e];
      }
    l_i = l_i * alpha + rs;
    if (__builtin_amdgcn_ballot_w64(upd) != 0) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[db][e] *= alpha;
    }
    finish(stage);
  };

  if (t0 < t1) landed(st[0], slot_of(t0), holes[0], t0 + 1 < t1);
  meet();
  for (int t = t0; t < t1; ++t) {
    const int n0 = slot_of(t);
    ask(AHEAD, t + AHEAD);
    if (active) {
      const bool edge = is_edge(n0, holes[0]);
      qk(st[0]);
      if (!(have_ref && fast_step(st[0], n0, holes[0], edge))) {
        if (have_ref) qk(st[0]);      // (the scores are spent)
        full_step(st[0], n0, holes[0], edge);
      }
    }
    if (t + 1 < t1) landed(st[1], slot_of(t + 1), holes[1], t + 2 < t1);
    meet();
    const int done = st[0];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      st[i] = st[i + 1];
      holes[i] = holes[i + 1];
    }
    st[AHEAD] = done;
  }

  if (!active) return;
  const float l = row.alive ? cross_sum(l_i) : 0.f;
  if (!row_ok) return;
  if (!whole) {
    const int64_t sums = tree_sums(a, hk, rb, piece, z, from == 0) + wave * 32 + col;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(a.part_o + sums * D + 32 * db + 8 * g + 4 * hi) = f32x4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
    if (hi == 0) {
      a.part_ml[sums * 2] = m_i;
      a.part_ml[sums * 2 + 1] = l;
    }
    return;
  }
  const float inv = 1.0f / l;
  T* op = reinterpret_cast<T*>(a.out) + (int64_t)z * a.so.z + (int64_t)h * a.so.h + (int64_t)token * a.so.s;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      q4_t t4;
#pragma unroll
      for (int x = 0; x < 4; ++x) t4[x] = Tr::cvt(l == 0.f ? 0.f : o[db][4 * g + x] * inv);
      const int at = 32 * db + 8 * g + 4 * hi;
      if (!kPad || at < d_v) *reinterpret_cast<q4_t*>(op + at) = t4;
    }
  if (a.lse && hi == 0) a.lse[((int64_t)z * a.hq + h) * a.tokens + token] = lse_of(m_i, sc, l);
}

template <typename T, int D, int NW, bool kPad>
__global__ __attribute__((amdgpu_flat_work_group_size(NW * 64, NW * 64))) __attribute__((amdgpu_waves_per_eu(2, 2)))
void tree_tile_kernel(const TreeArgs a) {
  extern __shared__ __attribute__((aligned(kSwzAlign))) char smem_raw[];
  tree_work(a, threadIdx.x & 63, [&](int z, int hk, int rb, int from, int to, bool whole, int piece) __attribute__((always_inline)) {
    tree_tile_item<T, D, NW, kPad>(a, z, hk, rb, from, to, whole, piece, smem_raw);
  });
}

// ---- the pieces' sums: out = sum_i 2^((m_i - m) sc) O_i / sum_i 2^((m_i - m) sc) l_i -----------------------------------------------
// A thread takes four columns of a row, and of its pieces every kSlots-th.  What bounds it is the latency of loads that miss L2 (other
// XCDs wrote them): with many pieces of few rows the threads of a workgroup hold all of a row's between them.  4.0 us for 32 pieces of
// 32 heads, 8.8 for 12 MB.
template <typename T, int D, int kSlots>
static __global__ __launch_bounds__(256) void tree_sum_kernel(const TreeArgs a) {
  constexpr int TPR = D / 4, ROWS = 256 / TPR / kSlots, AHEAD = 4;
  __shared__ f32x4 s_acc[kSlots > 1 ? 256 : 1];
  __shared__ float s_m[kSlots > 1 ? 256 / TPR : 1], s_l[kSlots > 1 ? 256 / TPR : 1];
  const CacheArgs& c = a.cache;
  const int chunks = (a.part_rows + ROWS - 1) / ROWS;
  const int block = blockIdx.x / chunks, rb = block % a.row_blocks, hk = block / a.row_blocks % c.heads, z = block / a.row_blocks / c.heads;
  const int group = a.hq / c.heads;
  const int size = tree_blocks(a, z);
  int p0 = 0, parts;
  if (a.workers > 0) {
    TreeList list;
    list.cut(a, threadIdx.x & 63, z);
    p0 = (int)(list.start / list.per);
    parts = (int)((list.start + size - 1) / list.per) - p0 + 1;
  } else {
    parts = (size + a.part_blocks - 1) / a.part_blocks;
    parts = parts < a.parts ? parts : a.parts;
  }
  if (parts <= 1) return;                              // (the whole workgroup: its results are there already)
  const int lane_row = threadIdx.x / TPR / kSlots, slot = threadIdx.x / TPR % kSlots, col = threadIdx.x % TPR * 4;
  const int r = blockIdx.x % chunks * ROWS + lane_row, pr = rb * a.row_rows + r;
  const bool ok = r < a.part_rows && pr < a.tokens * group;
  const float sc = score_scale(a.sm_scale, false);
  const int64_t at = tree_sums(a, hk, rb, p0, z, true) + (ok ? r : 0);
  // (tree_sums of piece i behind that of the first: of a list 0, 1, 3, 5, ...)
  auto place = [&](int i) { return (int64_t)(a.workers > 0 && i > 0 ? 2 * i - 1 : i) * a.part_rows; };
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
      ml[k] = *reinterpret_cast<const vec<float, 2>*>(pm + place(i) * 2);
      x[k] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(po + place(i) * D));
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
    const float inv = l == 0.f ? 0.f : 1.0f / l;
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
// Slots of a row: where the rows alone leave the chip empty and a sequence may lie in many pieces.
template <typename T, int D>
hipError_t launch_tree_sum(const TreeArgs& a, hipStream_t stream) {
  const int64_t rows = (int64_t)a.cache.sequences * a.cache.heads * a.row_blocks * a.part_rows;
  if ((a.workers > 0 ? a.workers / a.cache.sequences : a.parts) <= 8 || rows > 1024) return launch_tree_sum_slots<T, D, 1>(a, stream);
  return launch_tree_sum_slots<T, D, 256 / (D / 4)>(a, stream);
}

template <auto kern>
hipError_t launch_tree_kernel(const TreeArgs& a, int threads, int smem, hipStream_t stream) {
  if (smem > 64 * 1024) {
    static std::atomic<uint64_t> lds_set{0};
    const hipError_t e = allow_large_lds(reinterpret_cast<const void*>(kern), smem, lds_set);
    if (e != hipSuccess) return e;
  }
  const int pieces = a.workers > 0 ? a.workers : a.cache.sequences * a.parts, units = (a.cache.heads * pieces + kNumXcd - 1) / kNumXcd;
  if (units == 0 || a.row_blocks == 0) return hipSuccess;
  hipLaunchKernelGGL(kern, dim3((unsigned)(kNumXcd * units * a.row_blocks)), dim3(threads), smem, stream, a);
  return hipGetLastError();
}

// a.row_rows names the kernel: 32 rows, or those of a tile
template <typename T, int D, bool kPad>
hipError_t launch_tree(const TreeArgs& a, hipStream_t stream) {
  hipError_t e = hipErrorNotSupported;
  if (a.row_rows == 32) e = launch_tree_kernel<tree_rows_kernel<T, D, kPad>>(a, 256, TreeSmem<D>::BYTES, stream);
  if constexpr (D <= 128) {
    if (a.row_rows == 128) e = launch_tree_kernel<tree_tile_kernel<T, D, 4, kPad>>(a, 256, TreeTileSmem<D, 4>::BYTES, stream);
    if (a.row_rows == 256) e = launch_tree_kernel<tree_tile_kernel<T, D, 8, kPad>>(a, 512, TreeTileSmem<D, 8>::BYTES, stream);
  }
  return e != hipSuccess || a.part_o == nullptr ? e : launch_tree_sum<T, D>(a, stream);
}

}  // namespace fa
