// hv_lm_attn.h -- what the attention kernels share: their arguments, where
// their rows and keys lie, and which tiles and shares of them a workgroup has.
#pragma once

#include <type_traits>

#include "hv_lm.h"
#include "hv_lm_attn_plan.h"
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
  int most_keys;  // of a sequence, 0: unknown
  int run;        // run_of
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
  const SeqRows k = seq_rows(a.k_starts ? a.k_starts : a.starts, b, a.k_rows);
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

// 2^e of an exponent's byte. (The conversion takes its factor by the exponent alone, which 2^-127
// still has; -128, which no write makes, has all of a NaN's exponent bits, and gives NaN.) A byte is
// taken as it was loaded: to extend its sign there would wait for it.
__device__ __forceinline__ float factor_of(int byte) {
  return __builtin_bit_cast(float, ((byte ^ 0x80) - 1) << 23);
}

// The kernels of either type. The workspace is looked at here.
int attend_f16(const LmAttnArgs &a, bool paged, bool q8, void *workspace, size_t bytes,
               hipStream_t s);
int attend_bf16(const LmAttnArgs &a, bool paged, bool q8, void *workspace, size_t bytes,
                hipStream_t s);

// Shares of a launch's work where there are too few tiles to fill the card, or where whole
// tiles would leave the last round of them on a part of it.
// A tile that a share begins and a later one ends: rows r0 .. of n_rows of a sequence's group,
// from row `first` of the call on, in the partial results 2 share + 1, 2 (share + 1), ..
struct Cut {
  int first, n_rows, r0, head, parts;  // parts 0: none
  int unused[3];
};
struct Split {
  Cut *cuts;      // [workgroups]
  float *slots;   // [2 * workgroups][slot_floats]: partial results
  int workgroups, tile_rows, slot_floats;
  // Row r of a partial result: m and the sum of the terms, and the sums relative to m.
  __device__ __forceinline__ float2 *ml(int slot, int r) const {
    return reinterpret_cast<float2 *>(slots + (int64_t)slot * slot_floats) + r;
  }
  __device__ __forceinline__ float *sums(int slot, int r, int width) const {
    return slots + (int64_t)slot * slot_floats + 2 * tile_rows + r * width;
  }
};

static constexpr int kKeys = 64;  // of a tile

__device__ __forceinline__ int key_tiles(int keys) { return keys > 0 ? (keys - 1) / kKeys + 1 : 0; }

__device__ __forceinline__ Cost cost_of(const LmAttnArgs &a, const Sequence &s, int tile_rows) {
  const int keys = max(s.keys, 0);
  const int count = (int)(((int64_t)s.count * a.group + tile_rows - 1) / tile_rows);
  // A tile costs one of keys by itself.
  auto cost = [](int seen) { return 16 * min(1 + key_tiles(seen), kCostlyTiles); };
  if (a.causal && !a.window)
    return {cost(max(keys - s.count, 0)), tile_rows / (4 * a.group), count};
  return {cost(a.window ? min(keys, a.window) : keys), 0, count};
}

// A tile of a sequence's rows (of a key head's group: token r / group, head r % group of it)
// over some of the tiles of 64 keys that they see.
struct Work {
  Sequence s;
  int keys;    // that the sequence has, 0 where its table has no room
  int n_rows;  // s.count * group
  int r0;      // the tile's first row
  int t0, t1;  // tiles of keys
  int last;    // the last key that the rows see, -1: none
  int head;    // of the keys
  int slot;    // of the partial result, -1: the result is whole
};

// A number that all lanes have, in a scalar register.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Where a launch's work lies among the sequences, by all THREADS threads of a workgroup.
template <int THREADS, bool PAGED>
struct Finder {
  const LmAttnArgs &a;
  int tile_rows;
  v4i *held;  // in LDS: sequence threadIdx.x, of more than one
  int all;    // cost of all sequences, for one head

  __device__ __forceinline__ Sequence sequence(int b) const {
    return b < a.batch ? sequence_of<PAGED>(a, b) : Sequence{};
  }
  __device__ __forceinline__ Finder(const LmAttnArgs &args, int rows, bool costs)
      : a(args), tile_rows(rows), all(0) {
    __shared__ v4i sequences[THREADS];
    __shared__ int sums[THREADS / 64];
    held = sequences;
    if (a.batch == 1) {
      if (costs) all = uniform(cost_of(a, sequence(0), tile_rows).all());
      return;
    }
    const Sequence first = sequence(threadIdx.x);
    held[threadIdx.x] = v4i{first.first, first.count, first.keys, first.k_first};
    if (!costs) return;
    all = cost_of(a, first, tile_rows).all();
    for (int b = threadIdx.x + THREADS; b < a.batch; b += THREADS)
      all += cost_of(a, sequence(b), tile_rows).all();
#pragma unroll
    for (int o = 1; o < 64; o *= 2) all += __shfl_xor(all, o);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = all;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) all += sums[w];
    all = uniform(all);
  }

  // The sequence whose part of the sums of count(sequence) `at` lies in, and what is before
  // it. False: none.
  template <typename Count>
  __device__ __forceinline__ bool find(int at, Count count, Sequence &s, int &before) const {
    before = 0;
    if (a.batch == 1) {
      s = sequence(0);
      return at < count(s);
    }
    __shared__ int sums[THREADS / 64], found[6];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int base = 0; base < a.batch; base += THREADS) {
      Sequence t;
      if (base) {
        t = sequence(base + threadIdx.x);
      } else {
        const v4i x = held[threadIdx.x];
        t = {x[0], x[1], x[2], x[3], nullptr};
      }
      const int n = count(t);
      int upto = n;
#pragma unroll
      for (int o = 1; o < 64; o *= 2) {
        const int x = __shfl_up(upto, o);
        if (lane >= o) upto += x;
      }
      __syncthreads();
      if (lane == 63) sums[wave] = upto;
      if (threadIdx.x == 0) found[0] = -1;
      __syncthreads();
      int total = 0;
#pragma unroll
      for (int w = 0; w < THREADS / 64; ++w) {
        if (w < wave) upto += sums[w];
        total += sums[w];
      }
      const int from = before + upto - n;
      if (at >= from && at < from + n) {
        found[0] = base + threadIdx.x;
        found[1] = from;
        found[2] = t.first;
        found[3] = t.count;
        found[4] = t.keys;
        found[5] = t.k_first;
      }
      __syncthreads();
      const int b = uniform(found[0]);
      if (b >= 0) {
        before = uniform(found[1]);
        s = {uniform(found[2]), uniform(found[3]), uniform(found[4]), uniform(found[5]),
             PAGED ? a.table + b * a.table_ld : nullptr};
        return true;
      }
      before += uniform(total);
    }
    return false;
  }

  // Tile `tile` of a sequence, over all keys that its rows see.
  __device__ __forceinline__ Work work_of(const Sequence &s, int tile, int head) const {
    Work w;
    w.s = s;
    w.keys = max(s.keys, 0);
    w.n_rows = s.count * a.group;
    w.r0 = tile * tile_rows;
    w.head = head;
    w.slot = -1;
    const Seen first = seen_by(w.r0 / a.group, s.count, w.keys, a.causal, a.window);
    const Seen final = seen_by(min(w.r0 + tile_rows - 1, w.n_rows - 1) / a.group, s.count, w.keys,
                               a.causal, a.window);
    w.last = final.to - 1;
    w.t0 = first.from / kKeys;
    w.t1 = max(w.t0, key_tiles(final.to));
    return w;
  }
  // Tile `index` of all sequences', the last ones of each first, which see the most keys.
  // False: there are fewer.
  __device__ __forceinline__ bool whole(int index, int head, Work &w) const {
    Sequence s;
    int before;
    if (!find(index, [&](const Sequence &t) { return cost_of(a, t, tile_rows).count; }, s, before))
      return false;
    w = work_of(s, cost_of(a, s, tile_rows).count - 1 - (index - before), head);
    return true;
  }
  // The tile that `at` of all heads' cost lies in, whose own starts at `from`.
  __device__ __forceinline__ bool at(int at, Work &w, int &from, int &cost) const {
    const int head = at / all;
    Sequence s;
    int before;
    if (!find(at - head * all, [&](const Sequence &t) { return cost_of(a, t, tile_rows).all(); }, s,
              before))
      return false;
    before += head * all;
    const Cost c = cost_of(a, s, tile_rows);
    const int tile = c.tile_at(at - before);
    from = before + c.before(tile);
    cost = c.first + c.step * (tile + 1);
    w = work_of(s, tile, head);
    return true;
  }
};

// The same work, its numbers in scalar registers.
__device__ __forceinline__ void make_uniform(Work &w) {
  int *const n[] = {&w.s.first, &w.s.count, &w.s.keys, &w.s.k_first, &w.keys, &w.n_rows, &w.r0,
                    &w.t0,      &w.t1,      &w.last,   &w.head,      &w.slot};
#pragma unroll
  for (int i = 0; i < 12; ++i) *n[i] = uniform(*n[i]);
  const uint64_t table = (uint64_t)w.s.table;
  w.s.table = (const int32_t *)((uint64_t)(unsigned)uniform((int)(table >> 32)) << 32 |
                                (unsigned)uniform((int)table));
}

// The work of a workgroup: one tile, or a share of all tiles' cost, from which next() cuts
// what it has of one tile after another. Shares that the same XCD takes lie side by side,
// heads apart, so that they meet in its L2.
template <int THREADS, bool PAGED, bool SPLIT>
struct Walk {
  Finder<THREADS, PAGED> finder;
  const Split &split;
  int at, end, share;
  __device__ __forceinline__ Shares shares() const {
    return Shares(finder.all * finder.a.kv_heads, split.workgroups);
  }
  __device__ __forceinline__ Walk(const LmAttnArgs &a, const Split &parts, int tile_rows)
      : finder(a, tile_rows, SPLIT), split(parts), at(0), end(0), share(0) {
    if (!SPLIT) return;
    const Shares all = shares();
    share = blockIdx.x;
    if (all.n == split.workgroups) share = share % 8 * (split.workgroups / 8) + share / 8;
    if (threadIdx.x == 0) split.cuts[share] = Cut{};
    if (share >= all.n || finder.all <= 0) return;
    at = uniform(all.start(share));
    end = uniform(all.start(share + 1));
  }
  __device__ __forceinline__ bool next(Work &w) {
    if (!SPLIT) {
      const int kv_heads = finder.a.kv_heads;
      const int run = finder.a.run, at = run ? place_of(blockIdx.x, run) : (int)blockIdx.x;
      const bool some = finder.whole(at / kv_heads, at % kv_heads, w);
      make_uniform(w);
      return some;
    }
    int from, cost;
    if (at >= end || !finder.at(at, w, from, cost)) return false;
    const int t0 = w.t0, n = w.t1 - t0;
    const bool starts = at == from, ends = end >= from + cost;
    if (!starts) w.t0 = t0 + tiles_at(n, at - from, cost);
    if (!ends) w.t1 = max(w.t0, t0 + tiles_at(n, end - from, cost));
    if (!starts || !ends) w.slot = 2 * share + starts;
    if (starts && !ends && threadIdx.x == 0)
      split.cuts[share] =
          Cut{w.s.first, w.n_rows, w.r0, w.head, shares().parts(share, from + cost), {}};
    const int then = ends ? from + cost : end;
    if (then <= at) return false;  // offsets that run backwards: sums past 32 bits
    at = uniform(then);
    make_uniform(w);
    return true;
  }
};

// Whether one of the pages of keys first .. last is not in the cache, by `threads` threads
// (each those of some). A tile's loads begin at a multiple of 64 keys, where pages that a
// window has left behind may be gone: where they met a missing page, those that a row sees are
// looked through once more. (To look at each page's place as it is loaded instead took 3 % of 4 x
// 512 rows over a cache, 204 and 210 us.)
__device__ __forceinline__ bool missing_page(const LmAttnArgs &a, const int32_t *table, int first,
                                             int last, int thread, int threads) {
  if (first > last) return false;
  for (int p = (first >> a.map.shift) + thread; p <= last >> a.map.shift; p += threads)
    if ((unsigned)table[p] >= (unsigned)a.map.pages) return true;
  return false;
}

// The thread's number, found again wherever it is asked for: what hangs on it in one stretch of
// a kernel is not held in registers all through the others.
__device__ __forceinline__ int thread_again() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

}  // namespace hv
