// hv_lm_attn_tile.h -- the attention kernels, for the file of each element type.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(scale log2(e) q.k_j - m),  m the largest
#pragma once

#include "hv_lm_attn.h"

namespace hv {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));

template <typename T>
struct Mma;
template <>
struct Mma<bf16> {
  typedef v8bf frag;
  static __device__ __forceinline__ v16f wide(frag a, frag b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<f16> {
  typedef v8h frag;
  static __device__ __forceinline__ v16f wide(frag a, frag b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

// a and b after a's upper half and b's lower half of lanes have changed places.
__device__ __forceinline__ v2i halves(int a, int b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  return v2i{(int)r[0], (int)r[1]};
}
__device__ __forceinline__ void halves(float v, float &lower, float &upper) {
  const v2i r = halves(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v));
  const int lo = r[0], hi = r[1];
  lower = __builtin_bit_cast(float, lo);
  upper = __builtin_bit_cast(float, hi);
}
__device__ __forceinline__ float max_of_halves(float v) {
  float lower, upper;
  halves(v, lower, upper);
  return fmaxf(lower, upper);
}
__device__ __forceinline__ float sum_of_halves(float v) {
  float lower, upper;
  halves(v, lower, upper);
  return lower + upper;
}

// Four 16-bit values of a column of LDS, of the four rows that the lane's group
// of sixteen reads: lane 4 r + c of it gives the address of row r's elements
// 4 c .. 4 c + 3 of sixteen, lane i gets element i of the four rows.
__device__ __forceinline__ v4s read_column(const void *p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) v4s *)(__attribute__((address_space(3))) void *)p);
}

static constexpr int kKeys = 64;         // of a tile
static constexpr int kMinPartTiles = 4;  // of a part, at least

// Where 16-byte chunk c of a tile's row lies in that row, so that the reads of
// a tile meet no bank twice: of keys, one chunk of 32 rows at a time; of
// values, four chunks of four rows.
template <int DP>
__device__ __forceinline__ int k_place(int row, int c) {
  return c ^ (DP == 64 ? row >> 1 & 7 : row & 15);
}
template <int DP>
__device__ __forceinline__ int v_place(int row, int c) {
  return c ^ (DP == 64 ? (row >> 1 & 1) * 4 : (row & 3) * 4);
}

// 16 bytes a lane from memory straight to LDS, the wavefront's lanes one after
// another from `to` on (the same in all lanes).
__device__ __forceinline__ void to_lds(const void *from, void *to) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) void *)from,
      (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}

// What is loaded behind a head's width.
static __device__ const v4i kZeros[1] = {};

// Keys and values of a workgroup's tile, loaded by NW wavefronts.
template <typename T, int DP, bool PAGED, bool Q8, int NW>
struct TileLoader {
  // A unit is what a wavefront loads at once: 1 KiB of the source.
  static constexpr int kChunks = Q8 ? DP / 16 : DP / 8;  // 16-byte chunks of a row's source
  static constexpr int kRowsOf = 64 / kChunks, kUnits = kKeys / kRowsOf / NW;
  static_assert(kUnits * NW * kRowsOf == kKeys, "whole units");
  const LmAttnArgs &a;
  const Sequence &s;
  int head, lane, wave, last;  // last: the last key that is there
  int page[kUnits];
  int chunk[kUnits];
  bool bad;
  v4i held[Q8 ? 2 * kUnits : 1];
  int exps[Q8 ? 2 * kUnits : 1];

  __device__ __forceinline__ int row_of(int u) const {
    return (u * NW + wave) * kRowsOf + lane / kChunks;
  }
  __device__ __forceinline__ TileLoader(const LmAttnArgs &args, const Sequence &seq, int h, int last_key)
      : a(args), s(seq), head(h), lane(threadIdx.x & 63),
        wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), last(last_key), bad(false) {}
  // The pages of tile t's keys, which the loads of it need.
  __device__ __forceinline__ void find(int t) {
    if (!PAGED) return;
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
      page[u] = s.table[min(t * kKeys + row_of(u), last) >> a.map.shift];
  }
  // Tile t on its way into k and v (Q8: into registers).
  __device__ __forceinline__ void load(int t, T *k, T *v) {
    const int chunks = Q8 ? a.width / 16 : a.width / 8, c = lane % kChunks;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int row = row_of(u), key = min(t * kKeys + row, last);
      int64_t at_k, at_v;
      if (PAGED) {
        const bool none = (unsigned)page[u] >= (unsigned)a.map.pages;
        bad |= none;
        at_k = cache_row(a.map, a.kv_heads, none ? 0 : page[u], head, key);
        if (Q8) {
          exps[2 * u] = a.k_exps[at_k];
          exps[2 * u + 1] = a.v_exps[at_k];
        }
        at_k = at_v = at_k * a.width;
      } else {
        const int64_t r = (int64_t)s.k_first + key;
        at_k = r * a.k_ld + head * a.k_head_ld;
        at_v = r * a.v_ld + head * a.v_head_ld;
      }
      if (Q8) {
        const int64_t off = at_k + min(c, chunks - 1) * 16;
        held[2 * u] = *reinterpret_cast<const v4i *>((const uint8_t *)a.k + off);
        held[2 * u + 1] = *reinterpret_cast<const v4i *>((const uint8_t *)a.v + off);
      } else {
        const int kc = k_place<DP>(row, c), vc = v_place<DP>(row, c);
        to_lds(kc < chunks ? (const T *)a.k + at_k + kc * 8 : (const T *)kZeros,
               k + (u * NW + wave) * 512);
        to_lds(vc < chunks ? (const T *)a.v + at_v + vc * 8 : (const T *)kZeros,
               v + (u * NW + wave) * 512);
      }
    }
  }
  // Q8: what `load` brought, into k and v.
  __device__ __forceinline__ void put(T *k, T *v) {
    if (!Q8) return;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int row = row_of(u), c = lane % kChunks * 2;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const v4i w = held[2 * u + which];
        const float f = factor_of(exps[2 * u + which]);
        typename Pair8<T>::type x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[2 * i] = Pair8<T>::of(w[i], f, false);
          x[2 * i + 1] = Pair8<T>::of(w[i], f, true);
        }
        if (c * 8 >= a.width)
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = typename Pair8<T>::type{};
        T *to = (which ? v : k) + row * DP;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int at = which ? v_place<DP>(row, c + i) : k_place<DP>(row, c + i);
          __builtin_memcpy(to + at * 8, x + 4 * i, 16);
        }
      }
    }
  }
};

// What a launch's parts of the keys are: every sequence's keys in parts of so many
// tiles of 64 that all of them together are about `target` workgroups' work.
struct Split {
  float *o;    // [slots][rows of a tile][width], sums relative to m
  float2 *ml;  // [slots][rows of a tile]
  int target;
};

template <bool PAGED>
__device__ __forceinline__ int tiles_of(const LmAttnArgs &a, int b, int tile_rows) {
  const int64_t n = (int64_t)seq_rows(a.starts, b, a.rows).count * a.group;
  return (int)((n + tile_rows - 1) / tile_rows);
}
__device__ __forceinline__ int key_tiles(int keys) { return keys > 0 ? (keys + kKeys - 1) / kKeys : 0; }

// Tiles of 64 keys of a part.
template <bool PAGED, int THREADS>
__device__ __forceinline__ int part_tiles(const LmAttnArgs &a, int tile_rows, int target) {
  const int64_t all = sum_over<THREADS>(a.batch, [&](int b) {
    return (int64_t)tiles_of<PAGED>(a, b, tile_rows) * key_tiles(sequence_of<PAGED>(a, b).keys);
  });
  const int64_t n = (all * a.kv_heads + target - 1) / target;
  return (int)max((int64_t)kMinPartTiles, min(n, (int64_t)1 << 26));
}
__device__ __forceinline__ int parts_of(int keys, int part) {
  return max(1, (key_tiles(keys) + part - 1) / part);
}

// NW x 32 rows by all keys that they see (SPLIT: by a part of them), 64 keys at
// a time through LDS, two tiles of which take turns.
//
//   S^T = K Q^T   32x32x16 MFMA: lane l has the scores of row l % 32 and of
//                 keys 8 a + 4 (l / 32) + b, so that a row's largest score and
//                 sum are its lane's own but for one exchange of halves
//   O^T += V^T P^T  where P^T, rounded, is an operand just as it lies: k slot 8 h + i
//                 of a product is key 16 s + 8 (i / 4) + 4 h + i % 4, and V^T
//                 is read from LDS by columns in that order
template <typename T, int DP, bool PAGED, bool Q8, int NW, bool SPLIT>
__global__ __launch_bounds__(64 * NW, DP <= 128 ? 2 : 1) void k_attention_tile(LmAttnArgs a,
                                                                                Split split) {
  typedef typename Mma<T>::frag frag;
  constexpr int kRows = 32 * NW, kD = DP / 32, kSteps = DP / 16, kThreads = 64 * NW;
  __shared__ __attribute__((aligned(16))) T k0[kKeys * DP];
  __shared__ __attribute__((aligned(16))) T k1[kKeys * DP];
  __shared__ __attribute__((aligned(16))) T v0[kKeys * DP];
  __shared__ __attribute__((aligned(16))) T v1[kKeys * DP];

  const int head = blockIdx.x % a.kv_heads, index = blockIdx.x / a.kv_heads;
  Found f;
  int part_len = 0;
  if (SPLIT) {
    part_len = part_tiles<PAGED, kThreads>(a, kRows, split.target);
    f = find_item<kThreads>(a.batch, index, [&](int b) {
      return tiles_of<PAGED>(a, b, kRows) * parts_of(sequence_of<PAGED>(a, b).keys, part_len);
    });
  } else {
    f = find_item<kThreads>(a.batch, index, [&](int b) { return tiles_of<PAGED>(a, b, kRows); });
  }
  if (f.b < 0) return;
  const Sequence s = sequence_of<PAGED>(a, f.b);
  const int keys = max(s.keys, 0), parts = SPLIT ? parts_of(keys, part_len) : 1;
  const int n_rows = s.count * a.group;
  // The last tiles, which see the most keys, go first.
  const int tile = tiles_of<PAGED>(a, f.b, kRows) - 1 - f.rest / parts, part = f.rest % parts;
  const int r0 = tile * kRows;
  const Seen first = seen_by(r0 / a.group, s.count, keys, a.causal, a.window);
  const Seen final = seen_by(min(r0 + kRows - 1, n_rows - 1) / a.group, s.count, keys, a.causal,
                             a.window);
  int t0 = first.from / kKeys, t1 = max(t0, key_tiles(final.to)), used = 1;
  if (SPLIT) {
    used = max(1, (t1 - t0 + part_len - 1) / part_len);
    if (part >= used) return;
    t0 += part * part_len;
    t1 = min(t1, t0 + part_len);
  }

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int w0 = r0 + wave * 32;  // the wavefront's first row
  const bool idle = w0 >= n_rows;
  const int row = min(w0 + col, n_rows - 1), token = row / a.group;
  const int q_head = head * a.group + (row - token * a.group);
  const Seen seen = seen_by(token, s.count, keys, a.causal, a.window);
  // What all, and any, of the wavefront's rows see.
  const Seen top = seen_by(min(w0, n_rows - 1) / a.group, s.count, keys, a.causal, a.window);
  const Seen end = seen_by(min(w0 + 31, n_rows - 1) / a.group, s.count, keys, a.causal, a.window);

  frag q[kSteps];
  {
    const T *from = (const T *)a.q + (int64_t)(s.first + token) * a.q_ld + q_head * a.q_head_ld;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int d = 16 * i + 8 * half;
      q[i] = d < a.width ? *reinterpret_cast<const frag *>(from + d) : frag{};
    }
  }
  TileLoader<T, DP, PAGED, Q8, NW> loader(a, s, head, final.to - 1);
  v16f o[kD];
  float m, l;

  auto meet = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x70);  // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // CAREFUL: with values that are no numbers among the tile's, of keys that
  // not all rows see. They count as zeros in the sums, and what they make of the
  // rows that do see them is found by a product of its own.
  auto compute = [&](int t, const T *k, const T *v, auto careful) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(careful)::value;
    if (idle || t * kKeys >= end.to || (t + 1) * kKeys <= top.from) return;
    v16f x[2] = {};
    const T *kr = k + col * DP;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int c = k_place<DP>(col, 2 * i + half) * 8;
      const frag a0 = *reinterpret_cast<const frag *>(kr + c);
      const frag a1 = *reinterpret_cast<const frag *>(kr + 32 * DP + c);
      x[0] = Mma<T>::wide(a0, q[i], x[0]);
      x[1] = Mma<T>::wide(a1, q[i], x[1]);
    }
    // Whether the row sees the tile's key 4 half + i.
    const unsigned below = t * kKeys + 4 * half - seen.from, span = seen.to - seen.from;
    auto sees = [&](int i) { return below + i < span; };
    if (t * kKeys < end.from || (t + 1) * kKeys > top.to) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (!sees(32 * (i / 16) + 8 * (i % 16 / 4) + i % 4)) x[i / 16][i % 16] = -__builtin_inff();
    }
    float most = x[0][0];
#pragma unroll
    for (int i = 1; i < 32; ++i) most = fmaxf(most, x[i / 16][i % 16]);
    most = max_of_halves(most) * a.scale;
    // A row's reference rises only when a score passes it by 2^8: what is summed
    // is the same but for its exponent.
    const bool rise = most > m + 8.f;
    if (__builtin_amdgcn_ballot_w64(rise)) {
      const float by = rise ? __builtin_amdgcn_exp2f(m - most) : 1.f;
      m = rise ? most : m;
      l *= by;
#pragma unroll
      for (int i = 0; i < kD; ++i) o[i] *= by;
    }
    const float ref = m == -__builtin_inff() ? 0.f : m;
    frag p[4];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i / 16][i % 16], a.scale, -ref));
      l += e;
      p[i / 8][i % 8] = (T)e;
    }
    frag seen_keys[CAREFUL ? 4 : 1];
    if (CAREFUL) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        seen_keys[i / 8][i % 8] =
            (T)(sees(32 * (i / 16) + 8 * (i % 16 / 4) + i % 4) ? 1.f : 0.f);
    }
    const int vr = 4 * half + (lane >> 2 & 3);
#pragma unroll
    for (int d = 0; d < kD; ++d) {
      const int c = v_place<DP>(vr, 4 * d + (lane >> 4 & 1) * 2 + (lane >> 1 & 1)) * 8 + (lane & 1) * 4;
      const T *vc = v + vr * DP + c;
      v16f odd = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v4s lo = read_column(vc + 16 * i * DP), hi = read_column(vc + (16 * i + 8) * DP);
        v8s both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        if (CAREFUL) {
          // 1 for a NaN, 2^7 and 2^14 for the infinities, times 1 where the row sees the key
          frag kind;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float val = (float)__builtin_bit_cast(T, (short)both[e]);
            const bool fine = fabsf(val) < __builtin_inff();
            kind[e] = (T)(fine ? 0.f : val != val ? 1.f : val > 0.f ? 128.f : 16384.f);
            if (!fine) both[e] = 0;
          }
          odd = Mma<T>::wide(kind, seen_keys[i], odd);
        }
        o[d] = Mma<T>::wide(__builtin_bit_cast(frag, both), p[i], o[d]);
      }
      if (CAREFUL) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int code = (int)odd[i];
          const float up = code >> 7 & 127 ? __builtin_inff() : 0.f;
          const float down = code >> 14 ? -__builtin_inff() : 0.f;
          o[d][i] += code & 127 ? __builtin_nanf("") : up + down;
        }
      }
    }
  };
  auto step = [&](int t, T *k, T *v, T *nk, T *nv, auto careful) __attribute__((always_inline)) {
    meet();
    if (t + 1 < t1) {
      loader.load(t + 1, nk, nv);
      loader.find(t + 2);
    }
    compute(t, k, v, careful);
    if (t + 1 < t1) loader.put(nk, nv);
  };
  auto pass = [&](auto careful) __attribute__((always_inline)) {
    m = -__builtin_inff();
    l = 0.f;
#pragma unroll
    for (int i = 0; i < kD; ++i) o[i] = v16f{};
    if (t0 >= t1) return;
    loader.find(t0);
    loader.load(t0, k0, v0);
    loader.find(t0 + 1);
    loader.put(k0, v0);
#pragma unroll 1
    for (int t = t0; t < t1; t += 2) {
      step(t, k0, v0, k1, v1, careful);
      if (t + 1 < t1) step(t + 1, k1, v1, k0, v0, careful);
    }
  };
  pass(std::false_type());
  // NaN or infinities in what was summed: from values of keys that a row may not
  // see, since 0 times those is a NaN.
  float sum = 0.f;
#pragma unroll
  for (int d = 0; d < kD; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) sum = __builtin_fmaf(o[d][i], 0.f, sum);
  if (__syncthreads_or(sum != 0.f)) pass(std::true_type());

  l = sum_of_halves(l);
  if (PAGED && __syncthreads_or(s.keys < 0 || loader.bad)) l = __builtin_nanf("");
  if (idle || w0 + col >= n_rows) return;
  if (SPLIT && used > 1) {
    const int64_t at = ((int64_t)(f.before + f.rest) * a.kv_heads + head) * kRows + wave * 32 + col;
    if (half == 0) split.ml[at] = make_float2(m, l);
    float *to = split.o + at * a.width;
#pragma unroll
    for (int d = 0; d < kD; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = 32 * d + 8 * i + 4 * half;
        const v4f x = {o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
        if (e < a.width) *reinterpret_cast<v4f *>(to + e) = x;
      }
    return;
  }
  const float by = l == 0.f ? 0.f : 1.f / l;
  if (a.lse && half == 0)
    a.lse[(int64_t)(s.first + token) * a.heads + q_head] =
        l == 0.f ? -__builtin_inff() : (m + log2f(l)) * 0.69314718055994531f;
  T *to = (T *)a.out + (int64_t)(s.first + token) * a.out_ld + q_head * a.out_head_ld;
#pragma unroll
  for (int d = 0; d < kD; ++d)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // Lanes of either half exchange fours, so that each has eight in a row.
      typedef T four __attribute__((ext_vector_type(4)));
      four lo, hi;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo[e] = (T)(o[d][8 * i + e] * by);
        hi[e] = (T)(o[d][8 * i + 4 + e] * by);
      }
      const v2i x = __builtin_bit_cast(v2i, lo), y = __builtin_bit_cast(v2i, hi);
      const v2i u = halves(x[0], y[0]), w = halves(x[1], y[1]);
      const v4i out = {u[0], w[0], u[1], w[1]};
      const int e = 32 * d + 16 * i + 8 * half;
      if (e < a.width) *reinterpret_cast<v4i *>(to + e) = out;
    }
}

// Joins the parts of a tile's rows, of one key head: sixteen rows a workgroup, a row
// to a wavefront, LANES lanes to a part of four elements a lane.
template <typename T, bool PAGED, int LANES>
__global__ __launch_bounds__(256) void k_attention_join(LmAttnArgs a, Split split, int tile_rows) {
  const int head = blockIdx.x % a.kv_heads, index = blockIdx.x / a.kv_heads;
  const int part_len = part_tiles<PAGED, 256>(a, tile_rows, split.target);
  // The parts of all tiles before this one's: items are counted in tiles here.
  const Found f =
      find_item<256>(a.batch, index, [&](int b) { return tiles_of<PAGED>(a, b, tile_rows); });
  if (f.b < 0) return;
  const Sequence s = sequence_of<PAGED>(a, f.b);
  const int keys = max(s.keys, 0), parts = parts_of(keys, part_len);
  if (parts == 1) return;
  const int64_t before = sum_over<256>(a.batch, [&](int b) {
    return b < f.b ? (int64_t)tiles_of<PAGED>(a, b, tile_rows) *
                         parts_of(sequence_of<PAGED>(a, b).keys, part_len)
                   : 0;
  });
  const int n_rows = s.count * a.group, tiles = (n_rows + tile_rows - 1) / tile_rows;
  const int tile = tiles - 1 - f.rest, r0 = tile * tile_rows;
  const Seen first = seen_by(r0 / a.group, s.count, keys, a.causal, a.window);
  const Seen final = seen_by(min(r0 + tile_rows - 1, n_rows - 1) / a.group, s.count, keys, a.causal,
                             a.window);
  const int used = (max(first.from / kKeys, key_tiles(final.to)) - first.from / kKeys + part_len - 1) /
                   part_len;
  if (used <= 1) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int e = lane % LANES * 4, sub = lane / LANES;
  for (int i = blockIdx.y * 16 + wave; i < min(tile_rows, blockIdx.y * 16 + 16); i += 4) {
    const int r = r0 + i;
    if (r >= n_rows) return;
    const int64_t at0 = ((before + (int64_t)f.rest * parts) * a.kv_heads + head) * tile_rows + i;
    const int64_t step = (int64_t)a.kv_heads * tile_rows;
    float m = -__builtin_inff(), l = 0.f;
    for (int p = lane; p < used; p += 64) m = fmaxf(m, split.ml[at0 + p * step].x);
    m = max64(m);
    const float ref = m == -__builtin_inff() ? 0.f : m;
    v4f o = {};
    for (int p0 = 0; p0 < used; p0 += 64) {
      float w = 0.f;
      if (p0 + lane < used) {
        const float2 ml = split.ml[at0 + (p0 + lane) * step];
        w = __builtin_amdgcn_exp2f(ml.x - ref);
        l = __builtin_fmaf(w, ml.y, l);
      }
      const int n = min(64, used - p0);
      for (int p = 0; p < n; p += 64 / LANES) {
        const int mine = p + sub;
        const float wp = __shfl(w, mine & 63);
        if (mine < n && e < a.width) {
          const v4f x = *reinterpret_cast<const v4f *>(split.o + (at0 + (p0 + mine) * step) * a.width + e);
#pragma unroll
          for (int k = 0; k < 4; ++k) o[k] = __builtin_fmaf(wp, x[k], o[k]);
        }
      }
    }
    l = sum64(l);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int x = LANES; x < 64; x *= 2) o[k] += __shfl_xor(o[k], x);
    const int token = r / a.group, q_head = head * a.group + r - token * a.group;
    if (a.lse && lane == 0)
      a.lse[(int64_t)(s.first + token) * a.heads + q_head] =
          l == 0.f ? -__builtin_inff() : (m + log2f(l)) * 0.69314718055994531f;
    if (sub == 0 && e < a.width) {
      const float by = l == 0.f ? 0.f : 1.f / l;
      typedef T four __attribute__((ext_vector_type(4)));
      four t;
#pragma unroll
      for (int k = 0; k < 4; ++k) t[k] = (T)(o[k] * by);
      *reinterpret_cast<four *>((T *)a.out + (int64_t)(s.first + token) * a.out_ld +
                                q_head * a.out_head_ld + e) = t;
    }
  }
}

template <typename T, bool PAGED, bool Q8, int DP>
static void attend_launch(const LmAttnArgs &a, const Split &split, const Shape &shape, hipStream_t s) {
  const int64_t tiles = most_tiles(a.rows, a.batch, a.group, shape.tile_rows);
  if (!shape.split) {
    hv_launch(k_attention_tile<T, DP, PAGED, Q8, 4, false>, dim3((unsigned)(tiles * a.kv_heads)),
              dim3(256), 0, s, a, split);
    return;
  }
  hv_launch(k_attention_tile<T, DP, PAGED, Q8, 4, true>,
            dim3((unsigned)most_slots(tiles, a.kv_heads)), dim3(256), 0, s, a, split);
  hv_launch(k_attention_join<T, PAGED, DP / 4>,
            dim3((unsigned)(tiles * a.kv_heads), (shape.tile_rows + 15) / 16), dim3(256), 0, s, a,
            split, shape.tile_rows);
}

template <typename T, bool PAGED, bool Q8>
static int attend(const LmAttnArgs &a, void *workspace, size_t bytes, hipStream_t s) {
  const Shape shape = shape_of(a.rows, a.batch, a.heads, a.kv_heads);
  Split split{};
  if (shape.split) {
    const size_t need = workspace_of(a.rows, a.batch, a.heads, a.kv_heads, a.width);
    if (!workspace || bytes < need || ((uintptr_t)workspace & 15))
      return fail(HV_EVALUE, HV_ERR_ADDRESS, "attention: a workspace of %zu bytes, %zu needed", bytes,
                  need);
    const int64_t slots =
        most_slots(most_tiles(a.rows, a.batch, a.group, shape.tile_rows), a.kv_heads);
    split.o = (float *)workspace;
    split.ml = (float2 *)(split.o + slots * shape.tile_rows * a.width);
    split.target = kTarget;
  }
  if (a.width <= 64) attend_launch<T, PAGED, Q8, 64>(a, split, shape, s);
  else if (a.width <= 128) attend_launch<T, PAGED, Q8, 128>(a, split, shape, s);
  else attend_launch<T, PAGED, Q8, 256>(a, split, shape, s);
  return check_hip(hipGetLastError(), "k_attention_tile launch");
}

template <typename T>
static int attend_any(const LmAttnArgs &a, bool paged, bool q8, void *workspace, size_t bytes,
                      hipStream_t s) {
  if (!paged) return attend<T, false, false>(a, workspace, bytes, s);
  return q8 ? attend<T, true, true>(a, workspace, bytes, s)
            : attend<T, true, false>(a, workspace, bytes, s);
}

}  // namespace hv
