// hv_lm_attn.h -- what the attention kernels share: their arguments, where
// their keys come from, and a row by a wavefront.
#pragma once

#include <type_traits>

#include "hv_lm.h"
#include "hv_lm_paged.h"

namespace hv {

struct LmAttnArgs {
  const void *q;
  void *out;
  float *lse;
  const void *k, *v;
  const int8_t *k_exps, *v_exps;
  const int32_t *starts, *k_starts, *table, *lengths;
  int64_t q_ld, q_head_ld, out_ld, out_head_ld;
  int64_t k_ld, k_head_ld, v_ld, v_head_ld;  // packed keys
  int64_t table_ld;
  int rows, k_rows, batch, heads, kv_heads, group, width, causal, window;
  PageMap map;
  float scale;  // of q.k, to a power of two: scale log2(e)
};

// Where a sequence's rows and keys are. keys -1: its table has no room for them.
struct Sequence {
  int first, count, keys, k_first;
  const int32_t *table;
};

template <bool PAGED>
__device__ __forceinline__ Sequence sequence_of(const LmAttnArgs &a, int b) {
  const SeqRows r = seq_rows(a.starts, b, a.rows);
  if (PAGED)
    return {r.first, r.count, paged_keys(a.map, a.lengths[b]), 0, a.table + b * a.table_ld};
  const SeqRows k = a.k_starts ? seq_rows(a.k_starts, b, a.k_rows) : seq_rows(a.starts, b, a.k_rows);
  return {r.first, r.count, k.count, k.first, nullptr};
}

// Two e4m3 values of a word (the low or the high ones) times 2^e, in 16 bits.
template <typename T>
struct Pair8;
template <>
struct Pair8<bf16> {
  typedef v2bf type;
  static __device__ __forceinline__ type of(int word, float scale, bool high) {
    return high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, true)
                : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, false);
  }
};
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
template <>
struct Pair8<f16> {
  typedef v2h type;
  static __device__ __forceinline__ type of(int word, float scale, bool high) {
    return high ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, scale, true)
                : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, scale, false);
  }
};

// 2^e of an exponent in [-127, 127], NaN for -128. (The conversion's factor is
// taken by its exponent alone, which 2^-127 still has.)
__device__ __forceinline__ float factor_of(int e) {
  return __builtin_bit_cast(float, e == -128 ? 0x7FC00000 : (e + 127) << 23);
}

// Tiles of `tile_rows` rows that a call's sequences have at most.
inline int64_t most_tiles(int rows, int batch, int group, int tile_rows) {
  return (int64_t)rows * group / tile_rows + batch;
}
// Parts of them that there are at most where the keys are cut into about `target`
// workgroups' work.
inline int64_t most_slots(int64_t tiles, int kv_heads, int target) {
  return (tiles + (target + kv_heads - 1) / kv_heads) * kv_heads;
}

// Rows of a tile (of k_attention_few, or of k_attention_tile), and whether the keys
// are cut into parts.
static constexpr int kFewRows = 16, kTileRows = 128;
struct Shape {
  int tile_rows, target;
  bool split;
};
inline Shape shape_of(int rows, int batch, int heads, int kv_heads) {
  const int group = heads / kv_heads;
  const bool few = (int64_t)rows * group <= (int64_t)batch * kFewRows;
  const int tile_rows = few ? kFewRows : kTileRows, target = few ? 1024 : 512;
  const int64_t items = most_tiles(rows, batch, group, tile_rows) * kv_heads;
  return {tile_rows, target, items < (few ? 4 * target : target)};
}
inline size_t workspace_of(int rows, int batch, int heads, int kv_heads, int width) {
  const Shape shape = shape_of(rows, batch, heads, kv_heads);
  if (!shape.split) return 0;
  const int64_t slots = most_slots(most_tiles(rows, batch, heads / kv_heads, shape.tile_rows),
                                   kv_heads, shape.target);
  return (size_t)slots * shape.tile_rows * (width * 4 + 8);
}

// The kernels of either type. The workspace is looked at here.
int attend_f16(const LmAttnArgs &a, bool paged, bool q8, void *workspace, size_t bytes, hipStream_t s);
int attend_bf16(const LmAttnArgs &a, bool paged, bool q8, void *workspace, size_t bytes,
                hipStream_t s);

// What a launch's parts of the keys are: every sequence's keys in parts of so many
// tiles of 64 that all of them together are about `target` workgroups' work.
struct Split {
  float *o;    // [slots][rows of a tile][width], sums relative to m
  float2 *ml;  // [slots][rows of a tile]: m, and the sum of the terms
  int target;
};

static constexpr int kKeys = 64;         // of a tile
static constexpr int kMinPartTiles = 4;  // of a part, at least

__device__ __forceinline__ int key_tiles(int keys) {
  return keys > 0 ? (int)(((int64_t)keys + kKeys - 1) / kKeys) : 0;
}

// A workgroup's work: a tile of a sequence's rows (of a key head's group: token r /
// group, head r % group of it) over a part of the tiles of 64 keys that they see.
struct Work {
  Sequence s;
  int keys;     // that the sequence has, 0 where its table has no room
  int n_rows;   // s.count * group
  int r0;       // the tile's first row
  int t0, t1;   // tiles of keys
  int last;     // the last key that the rows see, -1: none
  int part, used;  // of the tile's parts; used 0: no work
  int slot;     // of the tile's first part, among all items
};

// Work `index` of a launch of THREADS threads a workgroup, found by all of them: sequences'
// tiles, the last ones first (which see the most keys), each by its parts.
template <int THREADS, bool PAGED, bool SPLIT>
__device__ __forceinline__ Work locate(const LmAttnArgs &a, int tile_rows, int target, int index) {
  __shared__ int64_t all[THREADS / 64];
  __shared__ int sums[THREADS / 64], found[8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto tiles_of = [&](const Sequence &s) {
    return (int)(((int64_t)s.count * a.group + tile_rows - 1) / tile_rows);
  };
  auto sequence = [&](int b) { return b < a.batch ? sequence_of<PAGED>(a, b) : Sequence{}; };
  Sequence s = sequence(a.batch == 1 ? 0 : tid);
  int part_len = 1 << 26;  // tiles of a part
  if (SPLIT) {
    int64_t work = (int64_t)tiles_of(s) * key_tiles(s.keys);
    if (a.batch > 1) {
      for (int b = tid + THREADS; b < a.batch; b += THREADS) {
        const Sequence t = sequence(b);
        work += (int64_t)tiles_of(t) * key_tiles(t.keys);
      }
#pragma unroll
      for (int o = 1; o < 64; o *= 2) work += __shfl_xor(work, o);
      if (lane == 0) all[wave] = work;
      __syncthreads();
      work = 0;
#pragma unroll
      for (int w = 0; w < THREADS / 64; ++w) work += all[w];
    }
    const int64_t n = (work * a.kv_heads + target - 1) / target;
    part_len = (int)max((int64_t)kMinPartTiles, min(n, (int64_t)part_len));
  }
  auto parts_of = [&](const Sequence &t) {
    return SPLIT ? max(1, (key_tiles(t.keys) + part_len - 1) / part_len) : 1;
  };
  int rest = index, before = 0;
  if (a.batch == 1) {
    if (index >= tiles_of(s) * parts_of(s)) return {};
  } else {
    for (int base = 0;; base += THREADS) {
      if (base >= a.batch) return {};
      if (base) s = sequence(base + tid);
      const int mine = tiles_of(s) * parts_of(s);
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 64; o *= 2) {
        const int t = __shfl_up(upto, o);
        if (lane >= o) upto += t;
      }
      if (lane == 63) sums[wave] = upto;
      if (tid == 0) found[0] = -1;
      __syncthreads();
      int total = 0;
#pragma unroll
      for (int w = 0; w < THREADS / 64; ++w) {
        if (w < wave) upto += sums[w];
        total += sums[w];
      }
      upto += before;
      if (index < upto && index >= upto - mine) {
        found[0] = base + tid;
        found[1] = upto - mine;
        found[2] = s.first;
        found[3] = s.count;
        found[4] = s.keys;
        found[5] = s.k_first;
      }
      __syncthreads();
      const int b = __builtin_amdgcn_readfirstlane(found[0]);
      if (b >= 0) {
        before = __builtin_amdgcn_readfirstlane(found[1]);
        s = {__builtin_amdgcn_readfirstlane(found[2]), __builtin_amdgcn_readfirstlane(found[3]),
             __builtin_amdgcn_readfirstlane(found[4]), __builtin_amdgcn_readfirstlane(found[5]),
             PAGED ? a.table + b * a.table_ld : nullptr};
        rest = index - before;
        break;
      }
      before += total;
      __syncthreads();
    }
  }
  Work w;
  w.s = s;
  w.keys = max(s.keys, 0);
  w.n_rows = s.count * a.group;
  const int parts = parts_of(s);
  w.r0 = (tiles_of(s) - 1 - rest / parts) * tile_rows;
  w.part = rest % parts;
  w.slot = before + rest - w.part;
  const Seen first = seen_by(w.r0 / a.group, s.count, w.keys, a.causal, a.window);
  const Seen final = seen_by(min(w.r0 + tile_rows - 1, w.n_rows - 1) / a.group, s.count, w.keys,
                             a.causal, a.window);
  w.last = final.to - 1;
  w.t0 = first.from / kKeys;
  w.t1 = max(w.t0, key_tiles(final.to));
  w.used = 1;
  if (SPLIT) {
    w.used = max(1, (w.t1 - w.t0 + part_len - 1) / part_len);
    w.t0 += w.part * part_len;
    w.t1 = min(w.t1, w.t0 + part_len);
    if (w.part >= w.used) w.used = 0;
  }
  return w;
}

}  // namespace hv
