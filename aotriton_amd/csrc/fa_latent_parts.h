// The running softmax of the kernels in fa_latent.h and fa_latent_cache.h, and the sums of keys that are cut into parts.
#pragma once
#include "fa_device.h"
#include "fa_wide.h"

namespace fa {

// 64 words into LDS (fa_wide.h: load_to_lds)
__device__ __forceinline__ void load_word_to_lds(u32x4_t rsrc, int voff, int lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dword %1, %2, 0 offen lds" :: "s"(lds), "v"(voff), "s"(rsrc) : "m0");
}

// What was loaded is in its registers from here on.
template <typename V, int N> __device__ __forceinline__ void arrived(V (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i]));
}

// Behind the last MFMA onto the accumulators, which the compiler does not see (fa_wide.h): 16 passes and what the register file takes.
template <int DB> __device__ __forceinline__ void settle(f32x16 (&o)[DB]) {
#pragma unroll
  for (int b = 0; b < DB; ++b) asm volatile("" : "+a"(o[b]));
  asm volatile("s_nop 15\n\ts_nop 15");
#pragma unroll
  for (int b = 0; b < DB; ++b) asm volatile("" : "+a"(o[b]));
}

// Maximum and sum of a lane's row; the sum is over the lane's half of the keys until cross_sum.
// The maximum is a reference: it moves, and O with it, only where a score passes it by more than 2^kSlack (P is then up to 2^kSlack, which
// both types hold without losing a bit; sums are fp32).  O lies in accumulation registers, where a product costs three
// instructions, and after the first tiles of a row its maximum hardly moves.
struct RowSoftmax {
  static constexpr float kSlack = 8.f;
  float m, l, sc, scale;      // scores are held in units of 1 / sc to base 2; prescaled by `scale` where the call's scale is not positive
  bool prescale;
  __device__ __forceinline__ RowSoftmax(float sm_scale) : m(kNegBig), l(0.f), sc(score_scale(sm_scale, false)), scale(sm_scale * kLog2e), prescale(!(sm_scale * kLog2e > 0.f)) {}

  // s: scores of NB x 32 keys, to be P, as the MFMAs leave them but for hidden() in the place of those that the row does not see.  `rescale` takes O
  // times a factor.
  __device__ __forceinline__ float hidden() const { return prescale && scale < 0.f ? __builtin_inff() : -__builtin_inff(); }
  template <int NB, typename Rescale>
  __device__ __forceinline__ void step(f32x16 (&s)[NB], Rescale rescale) {
    if (prescale) {
      // (a scale of 0: what is hidden stays so)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[b][i] = scale == 0.f && s[b][i] == hidden() ? s[b][i] : s[b][i] * scale;
    }
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
    top = cross_max(top);
    if (__builtin_amdgcn_ballot_w64((top - m) * sc > kSlack) != 0) {
      const float to = fmaxf(m, top), alpha = fast_exp2((m - to) * sc);
      m = to;
      if (__builtin_amdgcn_ballot_w64(l != 0.f) != 0) rescale(alpha);      // (before a row's first sum O is 0)
      l *= alpha;
    }
    const float msc = m * sc;
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[b][i] = fast_exp2(__builtin_fmaf(s[b][i], sc, -msc));
        sum[i & 1] += s[b][i];
      }
    l += sum[0] + sum[1];
  }
  __device__ __forceinline__ float lse(float sum) const { return sum == 0.f ? __builtin_inff() : __builtin_fmaf(m, sc, fast_log2(sum)) * kLn2; }
};

// Part `at` of 32 rows: O^T of DB blocks of 32 columns as the lanes hold it, 16 bytes a lane in a row; maximum and sum of every row.
template <int DB>
__device__ __forceinline__ void store_part(float* part_o, float* part_ml, int64_t at, const f32x16* o, const RowSoftmax& sm, int lane) {
  float* to = part_o + at * (DB * 1024) + lane * 4;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) *reinterpret_cast<f32x4*>(to + (4 * b + g) * 256) = f32x4{o[b][4 * g], o[b][4 * g + 1], o[b][4 * g + 2], o[b][4 * g + 3]};
  const float l = cross_sum(sm.l);
  part_ml[at * 64 + lane] = lane < 32 ? sm.m : l;
}

// The parts at, at + 1, ... put together: four columns of row tid % 32, those of block db that store_part's lane tid % 64 held in group tid / 64.
template <int DB>
__device__ __forceinline__ f32x4 sum_parts(const float* part_o, const float* part_ml, int64_t at, int parts, float sm_scale, int db, int tid, float& lse) {
  const int c = tid & 31;
  const float* ml = part_ml + at * 64 + c;
  const float* from = part_o + at * (DB * 1024) + db * 1024 + tid * 4;
  const float sc = score_scale(sm_scale, false);
  float m = kNegBig;
  for (int p = 0; p < parts; ++p) m = fmaxf(m, ml[p * 64]);
  float l = 0.f;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < parts; ++p) {
    const float w = fast_exp2((ml[p * 64] - m) * sc);
    l += w * ml[p * 64 + 32];
    x += w * *reinterpret_cast<const f32x4*>(from + (int64_t)p * (DB * 1024));
  }
  lse = l == 0.f ? __builtin_inff() : __builtin_fmaf(m, sc, fast_log2(l)) * kLn2;
  return x * (l == 0.f ? 0.f : 1.0f / l);
}

}  // namespace fa
