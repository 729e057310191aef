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

// Keys and values of one head of a sequence, element by element.
template <typename T, bool PAGED, bool Q8>
struct HeadKeys {
  const LmAttnArgs &a;
  Sequence s;
  int head;  // of the keys

  // Row of key j: an element offset of the packed rows (of k, and of v), or a
  // row of the cache; false where its page is none.
  struct Place {
    int64_t k, v;
    bool ok;
  };
  __device__ __forceinline__ Place place(int j) const {
    if (PAGED) {
      const int page = page_of(a.map, s.table, j);
      const int64_t row = cache_row(a.map, a.kv_heads, max(page, 0), head, j);
      return {row, row, page >= 0};
    }
    const int64_t row = (int64_t)s.k_first + j;
    return {row * a.k_ld + head * a.k_head_ld, row * a.v_ld + head * a.v_head_ld, true};
  }
  // Eight elements from d on, of k (value false) or v.
  __device__ __forceinline__ void eight(const Place &p, bool value, int d, float (&x)[8]) const {
    const int64_t at = value ? p.v : p.k;
    const void *base = value ? a.v : a.k;
    if (Q8) {
      v2i w;
      __builtin_memcpy(&w, (const uint8_t *)base + at * a.width + d, 8);
      const float f = factor_of((value ? a.v_exps : a.k_exps)[at]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const auto t = Pair8<T>::of(w[i / 2], f, i % 2);
        x[2 * i] = (float)t[0];
        x[2 * i + 1] = (float)t[1];
      }
    } else {
      const auto t = Eight<T>::load((const T *)base + (PAGED ? at * a.width : at) + d, 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)t[i];
    }
  }
};

// One row of queries over keys [from, to), by a wavefront: 64 keys at a time, a
// key to a lane for the scores and eight elements to a lane for the sums. A
// key that is not seen is not read, so nothing of it is in the result.
// m and l: the largest score (to a power of two) and the sum of the terms
// relative to it; lane i < width / 8 has elements 8 i .. 8 i + 7 of the sum of
// terms times values.
struct RowState {
  float m, l, o[8];
};
template <typename T, bool PAGED, bool Q8>
__device__ RowState attend_row(const LmAttnArgs &a, const Sequence &s, int row, int head, int from,
                               int to) {
  const int lane = threadIdx.x & 63;
  const HeadKeys<T, PAGED, Q8> keys{a, s, head / a.group};
  const T *q = (const T *)a.q + row * a.q_ld + head * a.q_head_ld;
  RowState r{-__builtin_inff(), 0.f, {}};
  for (int j0 = from; j0 < to; j0 += 64) {
    const int n = min(64, to - j0), j = j0 + min(lane, n - 1);
    const auto at = keys.place(j);
    float score = 0.f;
    for (int d = 0; d < a.width; d += 8) {
      float x[8];
      keys.eight(at, false, d, x);
      const auto y = Eight<T>::load(q + d, 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) score = __builtin_fmaf(x[i], (float)y[i], score);
    }
    score = lane < n ? score * a.scale : -__builtin_inff();
    if (!at.ok) score = __builtin_nanf("");
    const float m = fmaxf(r.m, max64(score));
    const bool none = m == -__builtin_inff();  // nothing but scores of -infinity (or NaN) so far
    const float p = none ? score == score ? 0.f : score : __builtin_amdgcn_exp2f(score - m);
    const float f = none ? 1.f : __builtin_amdgcn_exp2f(r.m - m);
    r.m = m;
    r.l = r.l * f + sum64(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) r.o[i] *= f;
    for (int i = 0; i < n; ++i) {
      const float t = __shfl(p, i);
      if (t == 0.f || lane * 8 >= a.width) continue;
      float x[8];
      keys.eight(keys.place(j0 + i), true, lane * 8, x);
#pragma unroll
      for (int k = 0; k < 8; ++k) r.o[k] = __builtin_fmaf(t, x[k], r.o[k]);
    }
  }
  return r;
}

}  // namespace hv
