// The list of work of attention over a cache of latent rows (fa_latent_cache.h): how many units a sequence has on it, and which block a unit belongs to.
// Compiled for host and device.  Args: LatentCacheArgs, of which the heads, the rows of a block, the shifts and the margin count.
#pragma once
#include <stdint.h>

#include "fa_intervals.h"

#define FA_LIST FA_HD_MEMBER __attribute__((always_inline)) inline

namespace fa {

// a / b of numbers that are not negative (a division of 64 bits takes a microsecond)
FA_LIST int64_t latent_div(int64_t a, int64_t b) { return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b; }

// A sequence as the list of work has it: `blocks` blocks of rows, of tiles as many as their last row sees, or some more: the blocks of a group
// (LatentCacheArgs::group_shift) have the same number, a step more than the group in front, up to all `tiles`.
struct LatentSeq {
  int32_t start, tokens, length, end;      // first row of Q, tokens, filled slots (-1: not there), slots with the new ones as far as the table goes
  int32_t blocks, tiles, filled;           // (filled: tiles in front of the first new slot)
  template <typename Args> FA_LIST int tiles_of_group(const Args& a, int g) const {
    const int64_t n = filled + ((int64_t)(g + 1) << a.step_shift);
    return n < tiles ? (int)n : tiles;
  }
  template <typename Args> FA_LIST int tiles_of(const Args& a, int block) const { return tiles_of_group(a, block >> a.group_shift); }
  // the last slot that token t sees (no sum of the two: a length may be the largest number there is)
  FA_LIST int last_slot(int t) const { return t < end - length ? length + t : end - 1; }
  // groups that have not all tiles, as far as there are blocks
  template <typename Args> FA_LIST int short_groups(const Args& a) const {
    const int n = tiles > filled ? (tiles - filled - 1) >> a.step_shift : 0, all = (blocks + (1 << a.group_shift) - 1) >> a.group_shift;
    return n < all ? n : all;
  }
  // The list counts a block's tiles and LatentCacheArgs::margin on either side of them, for what beginning and ending it takes; blocks alone where
  // they stay whole.
  template <typename Args> FA_LIST int64_t units(const Args& a) const {
    if (a.margin < 0) return blocks;
    const int64_t n = short_groups(a), over = (n << a.group_shift) - blocks;      // (the last group may be short of blocks)
    const int64_t u = (n * filled + ((n * (n + 1) / 2) << a.step_shift)) << a.group_shift, last = over > 0 ? filled + (n << a.step_shift) : tiles;
    return u - over * last + (int64_t)blocks * (2 * a.margin);
  }
  // the block with unit `rel` of the sequence, and the unit's number in it
  template <typename Args> FA_LIST int block_of(const Args& a, int64_t rel, int& unit) const {
    if (a.margin < 0) {
      unit = 0;
      return (int)rel;
    }
    const int n = short_groups(a);
    for (int g = 0; g < n; ++g) {
      const int group = 1 << a.group_shift, t = filled + ((g + 1) << a.step_shift) + 2 * a.margin, have = blocks - g * group < group ? blocks - g * group : group;
      if (rel < (int64_t)have * t) {
        const int64_t b = latent_div(rel, t);      // (a group of 1024 blocks passes 32 bits with 2^22 tiles each)
        unit = (int)(rel - b * t);
        return g * group + (int)b;
      }
      rel -= (int64_t)have * t;
    }
    const int t = tiles + 2 * a.margin;
    const int64_t b = latent_div(rel, t);
    unit = (int)(rel - b * t);
    return (n << a.group_shift) + (int)b;
  }
};

// A sequence of `tokens` rows from row `start` on behind `length` slots (negative: it is not there), with a table of `room` slots.
template <typename Args> FA_LIST LatentSeq latent_seq_of(const Args& a, int32_t start, int32_t tokens, int32_t length, int64_t room) {
  LatentSeq s;
  s.start = start;
  s.tokens = tokens;
  s.length = length < 0 ? -1 : length;
  const int64_t end = (int64_t)s.length + s.tokens;
  s.end = s.length < 0 ? 0 : (int)(end < room ? end : room);
  s.blocks = (s.tokens * a.hq + a.block_rows - 1) >> a.block_shift;
  s.tiles = s.end > 32 ? (s.end + 31) / 32 : 1;
  s.filled = s.length <= 0 ? 0 : s.length < s.end ? (s.length + 31) / 32 : s.tiles;
  return s;
}

}  // namespace fa
