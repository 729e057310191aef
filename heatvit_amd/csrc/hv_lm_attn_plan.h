// hv_lm_attn_plan.h -- which kernels an attention call takes, and how the work is cut into
// shares. Code without HIP, so that tests can run it on the host.
#pragma once

#include <cmath>
#include <cstddef>
#include <cstdint>

#include "hv_lm_paged.h"

namespace hv {

// Tiles of `tile_rows` rows that a call's sequences have at most.
inline int64_t most_tiles(int rows, int batch, int group, int tile_rows) {
  return (int64_t)rows * group / tile_rows + batch;
}

// Rows of a tile (of k_attention_few, or of k_attention_tile), and whether the tiles' work
// is cut into `workgroups` shares.
static constexpr int kFewRows = 16, kTileRows = 128;
struct Shape {
  int tile_rows, workgroups;
  bool split;
};
inline Shape shape_of(int rows, int batch, int heads, int kv_heads, int width) {
  const int group = heads / kv_heads;
  const bool few = (int64_t)rows * group <= (int64_t)batch * kFewRows;
  const int tile_rows = few ? kFewRows : kTileRows;
  const int64_t items = most_tiles(rows, batch, group, tile_rows) * kv_heads;
  return {tile_rows, width <= 128 ? 512 : 256, items < (few ? 4096 : 512)};
}
// Shares cost a launch and the partial results' way through memory (us, whole and in shares).
// Few rows: one row of 32 heads over 1024 keys in e4m3 12.5 and 17.9, 2048 18.3 and 18.8, 4096
// 30.9 and 18.8, 32768 213 and 28. Tiles: the more keys and the fewer of the card's 512
// workgroups have a tile, the better (64 rows of 32 heads over 1024 keys, 24 items: 30.3 and
// 34.5, 2048 54 and 40; 1024 rows, 264 items, over 2048 64 and 68, 4096 116 and 102; a prompt
// of 1536, 392 items, 38 and 59).
// The rule holds at heads of 64 and of 256 too (a prompt of 1024 17.7 and 32.7, 39 and 44; of
// 4096, 8 heads, 55 and 50, 132 and 119; 128 rows of 32 and of 16 heads over 4096 69 and 33, 167
// and 52). most_keys: of the longest sequence, by keys_of_table or keys_of_packed.
inline bool worth_sharing(const Shape &shape, int rows, int batch, int kv_heads, int group,
                          int64_t most_keys) {
  if (shape.tile_rows == kFewRows) return most_keys > 2048;
  return most_keys * (512 - most_tiles(rows, batch, group, shape.tile_rows) * kv_heads) > 1 << 19;
}

// Keys of the longest sequence, as far as the host knows: what the caller says, or
// of a cache what a row of its table has room for. Where that is far more than the sequences have,
// a call in shares pays for parts that it does not have (us, said and not said, with a
// table of 131072 keys: a prompt of 512 over 32 heads 18 and 41, 8 rows over up to 1000 keys 12 and
// 23, one over 1000 13.7 and 17.4).
inline int64_t keys_of_table(int said, int64_t room) { return said ? said : room; }
// Of packed sequences twice their mean, as lengths spread evenly from none on have; their sum would
// cut many short ones (us, whole and in shares: 8 prompts of 512 and 4 heads of 128 16.4 and 36.7,
// 200 of 16 and 8 heads 22 and 32, 16 of 100 over one head of keys 12 and 44), their mean leave
// spread ones whole (8 rows of 16 heads on 4 of 128 over 400, 800, .. 3200 keys 32 and 20). Where
// one is longer still the caller has to say so (over 4000 and seven times 100 40 and 21).
inline int64_t keys_of_packed(int said, int64_t all, int batch) {
  const int64_t twice = 2 * ((all + batch - 1) / batch);
  return said ? said : twice < all ? twice : all;
}

// Tiles of a short sequence run on one XCD, whose L2 then has their keys once. Workgroup b runs on
// XCD b % 8: with a multiple of eight heads of keys a head's tiles meet there by themselves;
// otherwise each XCD takes the tiles of a run of the list, all heads' of as many tiles as a
// sequence has, four at most. (us, without runs and with them: 256 sequences of 197 tokens and 3
// heads of 64, two tiles, 31.5 and 28.7; of 577, five tiles, 130.8 and 128.0; of 400, causal,
// 64.1 and 61.2. Long causal sequences gain nothing, as their neighbours run at the same time
// anyway, and lose where the longest tiles come in runs: 8192 tokens and 4 heads of 128 525 and
// 543.) 0: no runs.
inline int run_of(const Shape &shape, int rows, int batch, int kv_heads, int group) {
  const int64_t tiles = ((int64_t)rows * group + (int64_t)batch * shape.tile_rows - 1) /
                        ((int64_t)batch * shape.tile_rows);
  if (shape.split || kv_heads % 8 == 0 || tiles < 2 || tiles > 8) return 0;
  return (int)(tiles < 4 ? tiles : 4) * kv_heads;
}
// The place in the list of workgroup b of a launch of a multiple of eight runs.
HV_HD int place_of(int b, int run) {
  const int turn = b / 8 / run;
  return (turn * 8 + b % 8) * run + b / 8 - turn * run;
}

// Two partial results a workgroup, of a tile that an earlier one began and of one that a later
// one ends: for each row the reference, the sum of the terms and the sums relative to it.
inline int slot_floats_of(const Shape &shape, int width) { return shape.tile_rows * (width + 2); }
inline size_t workspace_of(const Shape &shape, int width) {
  return shape.split ? (size_t)shape.workgroups * (8 * slot_floats_of(shape, width) + 32) : 0;
}

// What a sequence's tiles cost, in sixteenths of a tile of keys: tile i (of `count`) first +
// step (i + 1). Sums over a launch's tiles, 4096 at most where shares are taken, fit 32 bits,
// but for offsets that run backwards, whose sequences overlap: numbers that left 32 bits then
// still give tiles, parts and shares that there are.
static constexpr int kCostlyTiles = 1 << 14;  // of keys: more count as so many
struct Cost {
  int first, step, count;
  HV_HD int before(int i) const { return first * i + step * (i * (i + 1) / 2); }
  HV_HD int all() const { return before(count); }
  // The tile that a cost in [0, all()) lies in.
  HV_HD int tile_at(int at) const {
    const float f = first + .5f * step;
    int i = step ? (int)((sqrtf(f * f + 2.f * step * at) - f) / step) : at / first;
    i = clamp_to(i, 0, count - 1);
    while (i > 0 && before(i) > at) --i;
    while (i < count - 1 && before(i + 1) <= at) ++i;
    return i;
  }
};

// Shares of a launch's cost, n of them of four tiles of keys at least: the first `more` are one
// longer than the others.
struct Shares {
  int n, each, more;
  HV_HD Shares(int cost, int workgroups) {
    n = clamp_to(cost / 64, 1, workgroups);
    each = cost / n;
    more = cost - each * n;
  }
  HV_HD int start(int i) const { return each * i + (i < more ? i : more); }
  HV_HD int of(int at) const {
    const int longer = more * (each + 1);
    return at < longer ? at / (each + 1) : more + (at - longer) / each;
  }
  // How many shares, from `share` on, have a part of a tile whose cost ends at `end`.
  HV_HD int parts(int share, int end) const {
    return clamp_to(of(end - 1) - share + 1, 1, n - share);
  }
};

// How many of a tile's n tiles of keys lie before `at` of its cost.
HV_HD int tiles_at(int n, int at, int cost) {
  return (int)fminf(fmaxf((float)n * ((float)at / (float)cost), 0.f), (float)n);
}

}  // namespace hv
