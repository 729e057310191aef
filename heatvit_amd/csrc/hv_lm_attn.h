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

// Workgroups that keep the card busy: two a CU.
static constexpr int kTarget = 512;

// Tiles that a call's sequences have at most, and whether their keys are cut into parts:
// where the tiles alone would leave CUs idle.
inline int64_t most_tiles(int rows, int batch, int group, int tile_rows) {
  return (int64_t)rows * group / tile_rows + batch;
}
inline int64_t most_slots(int64_t tiles, int kv_heads) {
  return (tiles + (kTarget + kv_heads - 1) / kv_heads) * kv_heads;
}
struct Shape {
  int tile_rows;
  bool split;
};
inline Shape shape_of(int rows, int batch, int heads, int kv_heads) {
  const int64_t tiles = most_tiles(rows, batch, heads / kv_heads, 128);
  return {128, tiles * kv_heads < kTarget};
}
inline size_t workspace_of(int rows, int batch, int heads, int kv_heads, int width) {
  const Shape shape = shape_of(rows, batch, heads, kv_heads);
  if (!shape.split) return 0;
  const int64_t slots =
      most_slots(most_tiles(rows, batch, heads / kv_heads, shape.tile_rows), kv_heads);
  return (size_t)slots * shape.tile_rows * (width * 4 + 8);
}

// The kernels of either type. The workspace is looked at here.
int attend_f16(const LmAttnArgs &a, bool paged, bool q8, void *workspace, size_t bytes, hipStream_t s);
int attend_bf16(const LmAttnArgs &a, bool paged, bool q8, void *workspace, size_t bytes,
                hipStream_t s);

// Items of a launch: a sequence's tiles of `rows` rows (of a key head's group:
// token r / group, head r % group of it), each over `parts` parts of its keys.
struct Item {
  int b, tile, part;
  int slot;  // of all items' parts, of the first part
};

// The index-th of the items that count(b) says sequence b has, by all threads of
// the workgroup: (sequence, index in it, items before the sequence); b -1: fewer
// than that. count is asked for every sequence once.
struct Found {
  int b, rest, before;
};
template <int THREADS, typename Count>
__device__ __forceinline__ Found find_item(int batch, int index, Count count) {
  __shared__ int sums[THREADS / 64], found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (batch == 1) return {index < count(0) ? 0 : -1, index, 0};
  int before = 0;
  for (int base = 0; base < batch; base += THREADS) {
    const int b = base + tid, mine = b < batch ? count(b) : 0;
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
      found[0] = b;
      found[1] = upto - mine;
    }
    __syncthreads();
    if (found[0] >= 0) return {found[0], index - found[1], found[1]};
    before += total;
    __syncthreads();
  }
  return {-1, 0, 0};
}

// Sum of value(b) over the sequences, by all threads of the workgroup.
template <int THREADS, typename Value>
__device__ __forceinline__ int64_t sum_over(int batch, Value value) {
  __shared__ int64_t sums[THREADS / 64];
  if (batch == 1) return value(0);
  int64_t s = 0;
  for (int b = threadIdx.x; b < batch; b += THREADS) s += value(b);
#pragma unroll
  for (int o = 1; o < 64; o *= 2) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  s = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) s += sums[w];
  return s;
}

}  // namespace hv
