// hv_lm_attn_tile.h -- the attention kernels, for the file of each element type.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(scale log2(e) q.k_j - m),  m a reference near the
//   largest
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
  static __device__ __forceinline__ v4f small(frag a, frag b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<f16> {
  typedef v8h frag;
  static __device__ __forceinline__ v16f wide(frag a, frag b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ v4f small(frag a, frag b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
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

// A row's reference lies kLift under its largest score when it rises, and rises when a score is
// kRise above it, to powers of two. f16's terms are up to 2^15 so, of 65504, as its smallest
// numbers are near: a term 2^-25 of the largest would be none with a reference at the largest
// score, though the sum counts it (1000 terms of 2^-26 beside one of a value of zero, in tiles:
// nothing left of the result; so 2^-32 is lost). It costs no time.
template <typename T>
static constexpr float kLift = std::is_same<T, f16>::value ? 7.f : 0.f;
template <typename T>
static constexpr float kRise = 8.f + kLift<T>;

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

// Element d of key j's value, as the products take it.
template <typename T, bool PAGED, bool Q8>
__device__ __forceinline__ float value_at(const LmAttnArgs &a, const Sequence &s, int head, int j,
                                          int d) {
  const T *v = (const T *)a.v;
  if (!PAGED) return (float)v[((int64_t)s.k_first + j) * a.v_ld + head * a.v_head_ld + d];
  const int page = page_of(a.map, s.table, j);
  if (page < 0) return 0.f;
  const int64_t row = cache_row(a.map, a.kv_heads, page, head, j);
  if (!Q8) return (float)v[row * a.width + d];
  const auto x = Pair8<T>::of(((const uint8_t *)a.v)[row * a.width + d],
                              factor_of((uint8_t)a.v_exps[row]), false);
  return (float)x[0];
}

// Of eight values in LDS, those that are no numbers become zeros; whether there were any.
template <typename T>
__device__ __forceinline__ bool take_out(void *at) {
  typedef T eight __attribute__((ext_vector_type(8)));
  eight v = *reinterpret_cast<const eight *>(at);
  bool any = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool fine = fabsf((float)v[i]) < __builtin_inff();
    any |= !fine;
    v[i] = fine ? v[i] : (T)0.f;
  }
  if (any) *reinterpret_cast<eight *>(at) = v;
  return any;
}

// A pointer to global memory, said so to the compiler.
template <typename P>
__device__ __forceinline__ const __attribute__((address_space(1))) P *global(const P *p) {
  return (const __attribute__((address_space(1))) P *)p;
}

// Keys and values of a workgroup's tile, loaded by NW wavefronts.
template <typename T, int DP, bool PAGED, bool Q8, int NW>
struct TileLoader {
  // A unit is what a wavefront loads at once: 1 KiB of the source, up to sixteen rows from a
  // multiple of as many on, which lie in one page.
  static constexpr int kChunks = Q8 ? DP / 16 : DP / 8;  // 16-byte chunks of a row's source
  static constexpr int kRowsOf = 64 / kChunks, kUnits = kKeys / kRowsOf / NW;
  static constexpr int kBytes = Q8 ? 1 : 2;
  static constexpr int kBehind = 0x7FFFFFF0;  // an offset that no buffer has: it reads zeros
  static_assert(kUnits * NW * kRowsOf == kKeys && kRowsOf <= 16, "whole units");
  const LmAttnArgs &a;
  const Sequence &s;
  int head, lane, wave, last;  // last: the last key that is there
  int page[PAGED ? kUnits : 1];
  int k_off[kUnits], v_off[kUnits];  // a lane's, from a unit's first row on
  bool bad;
  v4i held[Q8 ? 2 * kUnits : 1];
  int exps[Q8 ? 2 * kUnits : 1];

  __device__ __forceinline__ int row_of(int u) const {
    return (u * NW + wave) * kRowsOf + lane / kChunks;
  }
  __device__ __forceinline__ TileLoader(const LmAttnArgs &args, const Sequence &seq, int h,
                                        int last_key, int tid)
      : a(args), s(seq), head(h), lane(tid & 63), wave(uniform(tid >> 6)), last(last_key),
        bad(false) {
    const int chunks = a.width * kBytes / 16, c = lane % kChunks, r = lane / kChunks;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int kc = Q8 ? c : k_place<DP>(row_of(u), c), vc = Q8 ? c : v_place<DP>(row_of(u), c);
      k_off[u] = kc < chunks ? r * k_stride() + kc * 16 : kBehind;
      v_off[u] = vc < chunks ? r * v_stride() + vc * 16 : kBehind;
    }
  }
  // Bytes from row to row.
  __device__ __forceinline__ int k_stride() const {
    return PAGED ? a.width * kBytes : (int)a.k_ld * 2;
  }
  __device__ __forceinline__ int v_stride() const {
    return PAGED ? a.width * kBytes : (int)a.v_ld * 2;
  }
  // Whether a tile's keys lie side by side: in rows of a tensor, or in one page.
  __device__ __forceinline__ bool together() const { return !PAGED || a.map.shift >= 6; }
  // The pages of tile t's keys, which the loads of it need.
  __device__ __forceinline__ void find(int t) {
    if (!PAGED) return;
    if (together()) {
      page[0] = global(s.table)[min(t * kKeys, last) >> a.map.shift];
      return;
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
      page[u] = global(s.table)[min(t * kKeys + (u * NW + wave) * kRowsOf, last) >> a.map.shift];
  }
  // Unit u of a tile, `row` of whose rows it is, from the row of key `first` on: rows behind the
  // last key read as zeros.
  __device__ __forceinline__ void load_unit(int u, int row, int64_t at, int first, T *k, T *v) {
    const int left = last - first;  // rows behind the first
    const int k_size = min(left, kKeys) * k_stride() + a.width * kBytes;
    const int v_size = min(left, kKeys) * v_stride() + a.width * kBytes;
    const uint8_t *ks = (const uint8_t *)a.k + (PAGED ? at * a.width * kBytes
                                                      : (at * a.k_ld + head * a.k_head_ld) * 2);
    const uint8_t *vs = (const uint8_t *)a.v + (PAGED ? at * a.width * kBytes
                                                      : (at * a.v_ld + head * a.v_head_ld) * 2);
    if (Q8) {
      auto buffer = [](const void *p, int size) {
        return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, size, 0x00020000);
      };
      const int r = lane / kChunks;
      const auto ke = buffer(a.k_exps + at, left + 1), ve = buffer(a.v_exps + at, left + 1);
      exps[2 * u] = __builtin_amdgcn_raw_buffer_load_b8(ke, r, row, 0);
      exps[2 * u + 1] = __builtin_amdgcn_raw_buffer_load_b8(ve, r, row, 0);
      const int k_at = row * k_stride(), v_at = row * v_stride();
      held[2 * u] = __builtin_amdgcn_raw_buffer_load_b128(buffer(ks, k_size), k_off[u], k_at, 0);
      held[2 * u + 1] =
          __builtin_amdgcn_raw_buffer_load_b128(buffer(vs, v_size), v_off[u], v_at, 0);
    } else {
      auto to_lds = [](const void *p, int size, int lane_at, int unit_at, T *to) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, size, 0x00020000),
            (__attribute__((address_space(3))) void *)to, 16, lane_at, unit_at, 0, 0);
      };
      to_lds(ks, k_size, k_off[u], row * k_stride(), k + (u * NW + wave) * 512);
      to_lds(vs, v_size, v_off[u], row * v_stride(), v + (u * NW + wave) * 512);
    }
  }
  // The row of a key, which starts a tile or a unit.
  __device__ __forceinline__ int64_t place(int key, int page_of_it) {
    if (!PAGED) return (int64_t)s.k_first + key;
    const int p = uniform(page_of_it);
    const bool none = (unsigned)p >= (unsigned)a.map.pages;
    bad |= none;
    return cache_row(a.map, a.kv_heads, none ? 0 : p, head, key);
  }
  // Tile t on its way into k and v (Q8: into registers).
  __device__ __forceinline__ void load(int t, T *k, T *v) {
    if (together()) {
      const int64_t at = place(t * kKeys, page[0]);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) load_unit(u, (u * NW + wave) * kRowsOf, at, t * kKeys, k, v);
      return;
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int first = t * kKeys + (u * NW + wave) * kRowsOf;
      // A unit behind the last key reads the last one's row again, all of whose scores are masked.
      load_unit(u, 0, place(min(first, last), page[u]), min(first, last), k, v);
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

// NW x 32 rows by all keys that they see (SPLIT: by a part of them), 64 keys at
// a time through LDS, two tiles of which take turns.
//
//   S^T = K Q^T   32x32x16 MFMA: lane l has the scores of row l % 32 and of
//                 keys 8 a + 4 (l / 32) + b, so that a row's largest score and
//                 sum are its lane's own but for one exchange of halves
//   O^T += V^T P^T  where P^T, rounded, is an operand just as it lies: k slot 8 h + i
//                 of a product is key 16 s + 8 (i / 4) + 4 h + i % 4, and V^T
//                 is read from LDS by columns in that order
//
// The matrix cores bound long prompts, with the exponentials beside them: 8192 causal tokens of
// 32 heads over 8 of 128 in bf16 take 500 to 542 us by card (1015 to 1100 TFLOP/s; a library
// product of 8192^3 reaches 1210), the matrix cores busy for 56 % of it at the 1.7 GHz that such a
// load leaves. A wavefront's 32 products of a tile take 1024 cycles, its 32 exponentials a lane
// 512 and what else it does with the scores as many; two wavefronts a SIMD, of workgroups that
// share no barrier, run one beside the other. A lone tile of keys takes 1.3 us, and a workgroup
// 7 us around its tiles: 256 sequences of 197 tokens, 3 heads of 64, 29 us, are four tiles in
// two rounds of that.
// (Terms are rounded to the type for the second product: of the result's norm 1.1e-3 in bf16,
// 1.4e-4 in f16, where the result's own rounding takes 1.6e-3 and 2.1e-4.)
template <typename T, int DP, bool PAGED, bool Q8, int NW, bool SPLIT>
__global__ __launch_bounds__(64 * NW, DP == 64 ? 3 : DP == 128 ? 2 : 1) void k_attention_tile(
    LmAttnArgs a, Split split) {
  typedef typename Mma<T>::frag frag;
  constexpr int kRows = 32 * NW, kD = DP / 32, kSteps = DP / 16, kThreads = 64 * NW;
  // The two tiles' keys and values: variables of their own where loads go straight to
  // LDS, so that the compiler sees that a read of one need not wait for loads into
  // another; one variable otherwise, whose parts share the lanes' addresses.
  constexpr int kSize = kKeys * DP, kOwn = Q8 ? 1 : kSize;
  __shared__ __attribute__((aligned(16))) T lds0[Q8 ? 4 * kSize : kSize], lds1[kOwn], lds2[kOwn],
      lds3[kOwn];
  T *const k0 = lds0, *const k1 = Q8 ? lds0 + kSize : lds1;
  T *const v0 = Q8 ? lds0 + 2 * kSize : lds2, *const v1 = Q8 ? lds0 + 3 * kSize : lds3;
  __shared__ unsigned long long odd_keys;

  Walk<kThreads, PAGED, SPLIT> walk(a, split, kRows);
  Work w;
  if (!walk.next(w)) return;
  do {
    const Sequence &s = w.s;
    const int head = w.head, keys = w.keys, n_rows = w.n_rows, r0 = w.r0, t0 = w.t0, t1 = w.t1;

    const int tid = thread_again(), lane = tid & 63, wave = uniform(tid >> 6);
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
    TileLoader<T, DP, PAGED, Q8, NW> loader(a, s, head, w.last, tid);
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
    // Values that are no numbers, of keys that not all rows see, are taken out of a
    // tile (careful), and added to the sums of the rows that do see them.
    auto take = [&](T *v) __attribute__((always_inline)) {
      if (threadIdx.x == 0) odd_keys = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < kKeys * DP / 8; i += kThreads)
        if (take_out<T>(v + 8 * i)) atomicOr(&odd_keys, 1ull << i / (DP / 8));
      __syncthreads();
    };
    auto compute = [&](int t, const T *k, const T *v, auto careful) __attribute__((always_inline)) {
      if (idle || t * kKeys >= end.to || (t + 1) * kKeys <= top.from) return;
      v16f x[2] = {};
      const T *kr = k + col * DP;
      // Keys are read four fragments ahead of their products, and values eight: the compiler
      // by itself reads one and waits for it.
      frag kf[2][4];
      auto read_keys = [&](int g) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const T *at = kr + k_place<DP>(col, 2 * (2 * g + i) + half) * 8;
          kf[g & 1][2 * i] = *reinterpret_cast<const frag *>(at);
          kf[g & 1][2 * i + 1] = *reinterpret_cast<const frag *>(at + 32 * DP);
        }
        __builtin_amdgcn_sched_barrier(0);
      };
      v4s vf[2][8];
      const int vr = 4 * half + (lane >> 2 & 3);
      // Of two runs of 32 elements, half of the tile's keys: four fragments.
      auto read_values = [&](int g) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int d = g / 2 * 2 + e;
          const T *at = v + (vr + 32 * (g % 2)) * DP +
                        v_place<DP>(vr, 4 * d + (lane >> 4 & 1) * 2 + (lane >> 1 & 1)) * 8 +
                        (lane & 1) * 4;
#pragma unroll
          for (int i = 0; i < 4; ++i) vf[g & 1][4 * e + i] = read_column(at + 8 * i * DP);
        }
        __builtin_amdgcn_sched_barrier(0);
      };
      read_keys(0);
#pragma unroll
      for (int g = 0; g < kSteps / 2; ++g) {
        if (g + 1 < kSteps / 2) read_keys(g + 1);
        else read_values(0);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          x[0] = Mma<T>::wide(kf[g & 1][2 * i], q[2 * g + i], x[0]);
          x[1] = Mma<T>::wide(kf[g & 1][2 * i + 1], q[2 * g + i], x[1]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      // Whether the row sees the tile's key 4 half + i.
      const unsigned below = t * kKeys + 4 * half - seen.from, span = seen.to - seen.from;
      auto sees = [&](int i) { return below + i < span; };
      if (t * kKeys < end.from || (t + 1) * kKeys > top.to) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (!sees(32 * (i / 16) + 8 * (i % 16 / 4) + i % 4))
            x[i / 16][i % 16] = -__builtin_inff();
      }
      float most = x[0][0];
#pragma unroll
      for (int i = 1; i < 32; ++i) most = fmaxf(most, x[i / 16][i % 16]);
      // A row's reference rises only when a score passes it by kRise: what is summed
      // is the same but for its exponent.
      if (__builtin_amdgcn_ballot_w64(most * a.scale > m + kRise<T>)) {
        most = max_of_halves(most) * a.scale;
        const bool rise = most > m + kRise<T>;
        const float by = rise ? __builtin_amdgcn_exp2f(m - (most - kLift<T>)) : 1.f;
        m = rise ? most - kLift<T> : m;
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
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int g = 0; g < kD; ++g) {
        if (g + 1 < kD) read_values(g + 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = g / 2 * 2 + i % 2, n = 4 * (i % 2) + i / 2 * 2;
          const v8s both =
              __builtin_shufflevector(vf[g & 1][n], vf[g & 1][n + 1], 0, 1, 2, 3, 4, 5, 6, 7);
          o[d] = Mma<T>::wide(__builtin_bit_cast(frag, both), p[2 * (g % 2) + i / 2], o[d]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (!decltype(careful)::value) return;
      for (uint64_t left = odd_keys; left; left &= left - 1) {
        const int j = t * kKeys + __builtin_ctzll(left);
        if (j < seen.from || j >= seen.to) continue;
        int e0 = 4 * half;
        asm volatile("" : "+v"(e0));  // found here, and not held all along
#pragma unroll
        for (int i = 0; i < 16 * kD; ++i) {
          const int e = 32 * (i / 16) + 8 * (i % 16 / 4) + e0 + i % 4;
          const float x = e < a.width ? value_at<T, PAGED, Q8>(a, s, head, j, e) : 0.f;
          o[i / 16][i % 16] += fabsf(x) < __builtin_inff() ? 0.f : x;
          asm volatile("" ::: "memory");  // one after another, in few registers
        }
      }
    };
    auto step = [&](int t, T *k, T *v, T *nk, T *nv, auto careful) __attribute__((always_inline)) {
      meet();
      if (decltype(careful)::value) take(v);
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
    // NaN or infinities in what was summed may be of keys that a row does not see,
    // since 0 times those is a NaN: once more, with care.
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16 * kD; ++i) sum = __builtin_fmaf(o[i / 16][i % 16], 0.f, sum);
    if (__syncthreads_or(sum != 0.f)) {
      pass(std::true_type());
      __syncthreads();  // before the next tile's first loads take the place of its last values
    }

    // (Again, so that it is not held all along.)
    int at_row = min(w0 + col, n_rows - 1);
    asm volatile("" : "+v"(at_row));
    const int out_token = at_row / a.group;
    const int out_head = head * a.group + at_row - out_token * a.group;
    l = sum_of_halves(l);
    if (PAGED && __syncthreads_or(s.keys < 0 || loader.bad)) {
      const int from = seen_by(r0 / a.group, s.count, keys, a.causal, a.window).from;
      const bool missing = missing_page(a, s.table, max(t0 * kKeys, from),
                                        min(t1 * kKeys - 1, w.last), threadIdx.x, kThreads);
      if (__syncthreads_or(s.keys < 0 || missing)) l = __builtin_nanf("");
    }
    if (idle || w0 + col >= n_rows) continue;
    if (SPLIT && w.slot >= 0) {
      if (half == 0) *split.ml(w.slot, wave * 32 + col) = make_float2(m, l);
      float *to = split.sums(w.slot, wave * 32 + col, a.width);
#pragma unroll
      for (int d = 0; d < kD; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = 32 * d + 8 * i + 4 * half;
          const v4f x = {o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
          if (e < a.width) *reinterpret_cast<v4f *>(to + e) = x;
        }
      continue;
    }
    const float by = l == 0.f ? 0.f : 1.f / l;
    if (a.lse && half == 0)
      a.lse[(int64_t)(s.first + out_token) * a.heads + out_head] =
          l == 0.f ? -__builtin_inff() : (m + log2f(l)) * 0.69314718055994531f;
    T *to = (T *)a.out + (int64_t)(s.first + out_token) * a.out_ld + out_head * a.out_head_ld;
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
  } while (SPLIT && walk.next(w));
}

// Where 16-byte chunk c of a row of values lies, where sixteen rows' 32 bytes are
// read by columns at a time.
template <int DP>
__device__ __forceinline__ int few_place(int row, int c) {
  return c ^ (DP == 64 ? (row >> 1 & 3) * 2 : (row & 7) * 2);
}

// Sixteen bytes of e4m3 times 2^e as two operands.
template <typename T>
__device__ __forceinline__ void wide_of(v4i w, float f, typename Mma<T>::frag (&x)[2]) {
  typename Pair8<T>::type t[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t[2 * i] = Pair8<T>::of(w[i], f, false);
    t[2 * i + 1] = Pair8<T>::of(w[i], f, true);
  }
  __builtin_memcpy(x, t, sizeof t);
}

// Sixteen rows by a part of the keys. Four wavefronts take 32 keys each in turn, for
// themselves: keys come from memory as the lanes multiply them, values go through LDS
// of the wavefront's own to be read by columns; the next 32 are on their way
// meanwhile. In the end the wavefronts' sums are joined at their common reference.
//
//   S^T = K Q^T   16x16x32 MFMA: lane l has row l % 16, keys 4 (l / 16) + i of sixteen
//   O^T += V^T P^T  with k slot 8 g + i as key 16 (i / 4) + 4 g + i % 4, as in the tiles
//
// The cache's bytes bound it: 64 sequences of 1 to 16384 keys, 8 heads of 128 in bf16 (478 MB),
// take 94 to 101 us and their join 5, 4.9 TB/s; 16 of 32768 in e4m3 (1.1 GB) 198, 5.5 TB/s. One of
// 32768 in e4m3 takes 20 and 5: 5 until the first keys are there, 5 for its share of the work,
// then four steps of 128 keys. Eight wavefronts a workgroup take as long (1024 rows' steps are
// half as many, shares' ends rounded to 256 keys: 64 short sequences 15.5, so 19.1 us).
template <typename T, int DP, bool PAGED, bool Q8, bool SPLIT>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void k_attention_few(LmAttnArgs a,
                                                                          Split split) {
  typedef typename Mma<T>::frag frag;
  constexpr int kRows = 16, kStep = 32, kD = DP / 16, kSteps = DP / 32;
  // Loads of 16 bytes a lane: of keys, sixteen keys by 4 chunks; of values, 1 KiB of rows.
  constexpr int kChunks = Q8 ? DP / 16 : DP / 8, kLoads = kChunks / 2, kRowsOf = 64 / kChunks;
  __shared__ __attribute__((aligned(16))) uint8_t lds[4 * kStep * DP * 2];
  __shared__ float2 ml[4][kRows];

  Walk<256, PAGED, SPLIT> walk(a, split, kRows);
  Work work;
  if (!walk.next(work)) return;
  do {
    const Sequence &s = work.s;
    const int head = work.head, keys = work.keys, n_rows = work.n_rows, r0 = work.r0, t0 = work.t0;
    const int last = work.last, end = min(work.t1 * kKeys, last + 1);

    const int tid = thread_again(), lane = tid & 63, wave = uniform(tid >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int row = min(r0 + col, n_rows - 1), token = row / a.group;
    const Seen seen = seen_by(token, s.count, keys, a.causal, a.window);
    // What all rows see starts at fin.from and ends at top.to.
    const Seen top = seen_by(r0 / a.group, s.count, keys, a.causal, a.window);
    const Seen fin = seen_by(min(r0 + kRows - 1, n_rows - 1) / a.group, s.count, keys, a.causal,
                             a.window);
    frag q[kSteps];
    {
      const T *from = (const T *)a.q + (int64_t)(s.first + token) * a.q_ld +
                      (head * a.group + row - token * a.group) * a.q_head_ld;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int d = Q8 ? 64 * (i / 2) + 16 * grp + 8 * (i % 2) : 32 * i + 8 * grp;
        q[i] = d < a.width ? *reinterpret_cast<const frag *>(from + d) : frag{};
      }
    }
    T *const mine = reinterpret_cast<T *>(lds) + wave * kStep * DP;
    const int width_chunks = Q8 ? a.width / 16 : a.width / 8;

    bool bad = false;
    v4i kr[2][kLoads / 2], vr[kLoads];
    int ke[2], ve[Q8 ? kLoads : 1];
    int page[2];
    // Sixteen keys from a multiple of sixteen on lie in one page.
    auto group_of = [&](int key0, int i) { return min(key0 + 16 * i, last & ~15); };
    auto find = [&](int key0) __attribute__((always_inline)) {
      if (!PAGED) return;
#pragma unroll
      for (int i = 0; i < 2; ++i) page[i] = global(s.table)[group_of(key0, i) >> a.map.shift];
    };
    auto load = [&](int key0) __attribute__((always_inline)) {
      constexpr int kSize = Q8 ? 1 : 2;
      int64_t base[2];  // the groups' first rows
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (PAGED) {
          const int p = uniform(page[i]);
          const bool none = (unsigned)p >= (unsigned)a.map.pages;
          bad |= none;
          base[i] = cache_row(a.map, a.kv_heads, none ? 0 : p, head, group_of(key0, i));
        } else {
          base[i] = (int64_t)s.k_first + group_of(key0, i);
        }
      }
      // Where chunk c of key n of sixteen lies (of the last key's, behind it), from a row on.
      auto at = [&](const void *from, int64_t ld, int64_t head_ld, int i, int n, int c) {
        const int row = min(n, last - group_of(key0, i));
        const uint8_t *p = (const uint8_t *)from;
        if (PAGED) return p + base[i] * a.width * kSize + (__umul24(row, a.width * kSize) + c * 16);
        return p + ((base[i] + row) * ld + head * head_ld) * 2 + c * 16;
      };
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int c = 0; c < kLoads / 2; ++c)
          kr[i][c] = *global((const v4i *)at(a.k, a.k_ld, a.k_head_ld, i, col,
                                             min(4 * c + grp, width_chunks - 1)));
        const int n = min(col, last - group_of(key0, i));
        if (Q8) ke[i] = *global((const uint8_t *)a.k_exps + base[i] + n);
      }
#pragma unroll
      for (int c = 0; c < kLoads; ++c) {
        const int n = c * kRowsOf + lane / kChunks, i = c * kRowsOf / 16;
        vr[c] = *global((const v4i *)at(a.v, a.v_ld, a.v_head_ld, i, n & 15,
                                        min(lane % kChunks, width_chunks - 1)));
        const int row = min(n & 15, last - group_of(key0, i));
        if (Q8) ve[c] = *global((const uint8_t *)a.v_exps + base[i] + row);
      }
    };
    // The values that came into LDS.
    auto put = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int c = 0; c < kLoads; ++c) {
        const int n = c * kRowsOf + lane / kChunks, chunk = lane % kChunks;
        if (Q8) {
          frag x[2];
          wide_of<T>(vr[c], factor_of(ve[c]), x);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            *reinterpret_cast<frag *>(mine + n * DP + few_place<DP>(n, 2 * chunk + i) * 8) = x[i];
        } else {
          *reinterpret_cast<v4i *>(mine + n * DP + few_place<DP>(n, chunk) * 8) = vr[c];
        }
      }
    };

    v4f o[kD];
    float m, l;
    auto pass = [&](auto careful) __attribute__((always_inline)) {  // as in k_attention_tile
      m = -__builtin_inff();
      l = 0.f;
#pragma unroll
      for (int i = 0; i < kD; ++i) o[i] = v4f{};
      int key0 = t0 * kKeys + wave * kStep;
      if (key0 >= end) return;
      find(key0);
      load(key0);
      find(key0 + 4 * kStep);
#pragma unroll 1
      for (; key0 < end; key0 += 4 * kStep) {
        v4f x[2] = {};
        if (a.width < DP) {  // nothing behind a head's width
#pragma unroll
          for (int c = 0; c < kLoads / 2; ++c)
            if (4 * c + grp >= width_chunks) kr[0][c] = kr[1][c] = v4i{};
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float fk = Q8 ? factor_of(ke[i]) : 0.f;
#pragma unroll
          for (int c = 0; c < kLoads / 2; ++c) {
            if (Q8) {
              frag y[2];
              wide_of<T>(kr[i][c], fk, y);
              x[i] = Mma<T>::small(y[0], q[2 * c], x[i]);
              x[i] = Mma<T>::small(y[1], q[2 * c + 1], x[i]);
            } else {
              x[i] = Mma<T>::small(__builtin_bit_cast(frag, kr[i][c]), q[c], x[i]);
            }
          }
        }
        put();
        unsigned odd = 0;
        if (decltype(careful)::value) {
#pragma unroll 1
          for (int i = lane; i < kStep * DP / 8; i += 64) {
            const bool any = take_out<T>(mine + 8 * i);
            // which of the rows that 64 lanes look at
            const uint64_t lanes = __builtin_amdgcn_ballot_w64(any);
            constexpr int kPer = DP / 8;
#pragma unroll
            for (int r = 0; r < 64 / kPer; ++r)
              if (lanes >> r * kPer & ((1ull << kPer) - 1)) odd |= 1u << ((i - lane) / kPer + r);
          }
        }
        if (key0 + 4 * kStep < end) {
          load(key0 + 4 * kStep);
          find(key0 + 8 * kStep);
        }
        const unsigned below = key0 + 4 * grp - seen.from, span = seen.to - seen.from;
        auto sees = [&](int i) { return below + (i / 4 * 16 + i % 4) < span; };
        if (key0 < fin.from || key0 + kStep > top.to) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (!sees(i)) x[i / 4][i % 4] = -__builtin_inff();
        }
        float most = x[0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) most = fmaxf(most, x[i / 4][i % 4]);
        if (__builtin_amdgcn_ballot_w64(most * a.scale > m + kRise<T>)) {
          most = fmaxf(most, __shfl_xor(most, 16));
          most = fmaxf(most, __shfl_xor(most, 32)) * a.scale;
          const bool rise = most > m + kRise<T>;
          const float by = rise ? __builtin_amdgcn_exp2f(m - (most - kLift<T>)) : 1.f;
          m = rise ? most - kLift<T> : m;
          l *= by;
#pragma unroll
          for (int i = 0; i < kD; ++i) o[i] *= by;
        }
        const float ref = m == -__builtin_inff() ? 0.f : m;
        // A term as the sum of two of the type: with few rows the rounding of one is no longer
        // averaged out, and the products cost nothing beside the loads.
        frag p, rest;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i / 4][i % 4], a.scale, -ref));
          l += e;
          p[i] = (T)e;
          rest[i] = (T)(e - (float)p[i]);
        }
        const int n = 4 * grp + (lane >> 2 & 3);
#pragma unroll
        for (int d = 0; d < kD; ++d) {
          const int c = few_place<DP>(n, 2 * d + (lane >> 1 & 1)) * 8 + (lane & 1) * 4;
          const v4s lo = read_column(mine + n * DP + c), hi = read_column(mine + (n + 16) * DP + c);
          const v8s both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
          o[d] = Mma<T>::small(__builtin_bit_cast(frag, both), rest, o[d]);
          o[d] = Mma<T>::small(__builtin_bit_cast(frag, both), p, o[d]);
        }
        for (; odd; odd &= odd - 1) {
          const int j = key0 + __builtin_ctz(odd);
          if (j < seen.from || j >= seen.to) continue;
          int e0 = 4 * grp;
          asm volatile("" : "+v"(e0));
#pragma unroll
          for (int i = 0; i < 4 * kD; ++i) {
            const int e = 16 * (i / 4) + e0 + i % 4;
            const float x = e < a.width ? value_at<T, PAGED, Q8>(a, s, head, j, e) : 0.f;
            o[i / 4][i % 4] += fabsf(x) < __builtin_inff() ? 0.f : x;
            asm volatile("" ::: "memory");
          }
        }
      }
    };
    pass(std::false_type());
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4 * kD; ++i) sum = __builtin_fmaf(o[i / 4][i % 4], 0.f, sum);
    if (__builtin_amdgcn_ballot_w64(sum != 0.f)) pass(std::true_type());

    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (PAGED && __builtin_amdgcn_ballot_w64(bad))
      bad = missing_page(a, s.table, max(t0 * kKeys, top.from), end - 1, lane, 64);
    if (PAGED && __builtin_amdgcn_ballot_w64(s.keys < 0 || bad)) l = __builtin_nanf("");
    if (grp == 0) ml[wave][col] = make_float2(m, l);
    __syncthreads();
    float all = ml[0][col].x;
#pragma unroll
    for (int w = 1; w < 4; ++w) all = fmaxf(all, ml[w][col].x);
    const float by = __builtin_amdgcn_exp2f(m - (all == -__builtin_inff() ? 0.f : all));
    // A wavefront's sums lie where its values did: [row][element], 32 bits.
    float *sums = reinterpret_cast<float *>(lds);
    constexpr int kLd = DP;
#pragma unroll
    for (int d = 0; d < kD; ++d) {
      const v4f x = o[d] * by;
      const int e = 16 * d + 4 * grp;
      *reinterpret_cast<v4f *>(sums + (wave * kRows + col) * kLd + (e ^ (col & 7) * 4)) = x;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kRows * DP / 4; i += 256) {
      const int r = i / (DP / 4), e = i % (DP / 4) * 4;
      if (r0 + r >= n_rows || e >= a.width) continue;
      float top = ml[0][r].x, total = 0.f;
#pragma unroll
      for (int w = 1; w < 4; ++w) top = fmaxf(top, ml[w][r].x);
      const float ref = top == -__builtin_inff() ? 0.f : top;
      v4f x = {};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        total = __builtin_fmaf(__builtin_amdgcn_exp2f(ml[w][r].x - ref), ml[w][r].y, total);
        x += *reinterpret_cast<const v4f *>(sums + (w * kRows + r) * kLd + (e ^ (r & 7) * 4));
      }
      if (SPLIT && work.slot >= 0) {
        if (e == 0) *split.ml(work.slot, r) = make_float2(top, total);
        *reinterpret_cast<v4f *>(split.sums(work.slot, r, a.width) + e) = x;
        continue;
      }
      const int tok = (r0 + r) / a.group, q_head = head * a.group + r0 + r - tok * a.group;
      if (a.lse && e == 0)
        a.lse[(int64_t)(s.first + tok) * a.heads + q_head] =
            total == 0.f ? -__builtin_inff() : (top + log2f(total)) * 0.69314718055994531f;
      const float inv = total == 0.f ? 0.f : 1.f / total;
      typedef T four __attribute__((ext_vector_type(4)));
      four t;
#pragma unroll
      for (int k = 0; k < 4; ++k) t[k] = (T)(x[k] * inv);
      *reinterpret_cast<four *>((T *)a.out + (int64_t)(s.first + tok) * a.out_ld +
                                q_head * a.out_head_ld + e) = t;
    }
    __syncthreads();  // before the sums make room for the next values
  } while (SPLIT && walk.next(work));
}

// Joins the parts of the tiles that are cut, sixteen rows of one a workgroup. A thread takes four
// elements of a row and every n-th part, eight on their way at a time; threads of the
// same elements are joined through LDS.
template <typename T, int DP>
__global__ __launch_bounds__(512) void k_attention_join(LmAttnArgs a, Split split) {
  constexpr int kLanes = DP / 4, kThreads = 512;
  __shared__ v4f sums[kThreads];
  __shared__ float2 mls[kThreads];
  // Neighbouring workgroups, which lie on different XCDs, take shares that are far apart:
  // those that cut a tile may be every n-th.
  const int share = blockIdx.x % 8 * (split.workgroups / 8) + blockIdx.x / 8;
  const Cut c = split.cuts[share];
  const int r0 = c.r0 + blockIdx.y * 16, rows = min(16, c.n_rows - r0);
  if (c.parts < 2 || rows <= 0) return;
  const int parts = c.parts, head = c.head;
  int span = kLanes;  // threads that take a part
  while (span < kThreads && span < rows * kLanes) span *= 2;
  const int n = kThreads / span, sub = threadIdx.x / span;
  const int e = threadIdx.x % kLanes * 4;
  for (int i0 = 0; i0 < rows; i0 += span / kLanes) {
    const int i = i0 + threadIdx.x % span / kLanes;
    const bool live = i < rows && e < a.width;
    const int row = blockIdx.y * 16 + min(i, rows - 1);
    const int el = min(e, a.width - 4);
    float m = -__builtin_inff(), l = 0.f;
    v4f o = {};
    for (int p0 = sub; p0 < parts; p0 += 8 * n) {
      float2 ml[8];
      v4f x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int p = min(p0 + u * n, parts - 1);
        const int slot = 2 * (share + p) + (p == 0);
        ml[u] = *split.ml(slot, row);
        x[u] = *reinterpret_cast<const v4f *>(split.sums(slot, row, a.width) + el);
      }
      float top = m;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (p0 + u * n >= parts) {
          ml[u] = make_float2(-__builtin_inff(), 0.f);
          x[u] = v4f{};
        }
        top = fmaxf(top, ml[u].x);
      }
      const float ref = top == -__builtin_inff() ? 0.f : top;
      const float f = __builtin_amdgcn_exp2f(m - ref);
      m = top;
      l *= f;
      o *= f;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float by = __builtin_amdgcn_exp2f(ml[u].x - ref);
        l = __builtin_fmaf(by, ml[u].y, l);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = __builtin_fmaf(by, x[u][k], o[k]);
      }
    }
    if (n > 1) {
      __syncthreads();
      sums[threadIdx.x] = o;
      mls[threadIdx.x] = make_float2(m, l);
      __syncthreads();
      if (sub == 0) {
        for (int u = 1; u < n; ++u) {
          const float2 ml = mls[threadIdx.x + u * span];
          const v4f x = sums[threadIdx.x + u * span];
          const float top = fmaxf(m, ml.x), ref = top == -__builtin_inff() ? 0.f : top;
          const float f = __builtin_amdgcn_exp2f(m - ref), g = __builtin_amdgcn_exp2f(ml.x - ref);
          m = top;
          l = l * f + ml.y * g;
#pragma unroll
          for (int k = 0; k < 4; ++k) o[k] = o[k] * f + x[k] * g;
        }
      }
    }
    if (sub || !live) continue;
    const int r = r0 + i, token = r / a.group, q_head = head * a.group + r - token * a.group;
    if (a.lse && e == 0)
      a.lse[(int64_t)(c.first + token) * a.heads + q_head] =
          l == 0.f ? -__builtin_inff() : (m + log2f(l)) * 0.69314718055994531f;
    const float by = l == 0.f ? 0.f : 1.f / l;
    typedef T four __attribute__((ext_vector_type(4)));
    four t;
#pragma unroll
    for (int k = 0; k < 4; ++k) t[k] = (T)(o[k] * by);
    *reinterpret_cast<four *>((T *)a.out + (int64_t)(c.first + token) * a.out_ld +
                              q_head * a.out_head_ld + e) = t;
  }
}

template <typename T, bool PAGED, bool Q8, int DP>
static void attend_launch(const LmAttnArgs &a, const Split &split, const Shape &shape,
                          hipStream_t s) {
  const bool few = shape.tile_rows == kFewRows;
  const unsigned items =
      (unsigned)(most_tiles(a.rows, a.batch, a.group, shape.tile_rows) * a.kv_heads);
  const unsigned unit = a.run ? 8 * a.run : 1;
  const dim3 grid(shape.split ? shape.workgroups : (items + unit - 1) / unit * unit), block(256);
  if (!shape.split) {
    if (few) hv_launch(k_attention_few<T, DP, PAGED, Q8, false>, grid, block, 0, s, a, split);
    else hv_launch(k_attention_tile<T, DP, PAGED, Q8, 4, false>, grid, block, 0, s, a, split);
    return;
  }
  if (few) hv_launch(k_attention_few<T, DP, PAGED, Q8, true>, grid, block, 0, s, a, split);
  else hv_launch(k_attention_tile<T, DP, PAGED, Q8, 4, true>, grid, block, 0, s, a, split);
  const dim3 joins(shape.workgroups, shape.tile_rows / 16);
  hv_launch(k_attention_join<T, DP>, joins, dim3(512), 0, s, a, split);
}

template <typename T, bool PAGED, bool Q8>
static int attend(LmAttnArgs a, void *workspace, size_t bytes, hipStream_t s) {
  Shape shape = shape_of(a.rows, a.batch, a.heads, a.kv_heads, a.width);
  Split split{};
  if (shape.split) {
    const size_t need = workspace_of(shape, a.width);
    if (!workspace || bytes < need || ((uintptr_t)workspace & 15))
      return fail(HV_EVALUE, HV_ERR_ADDRESS, "attention: a workspace of %zu bytes, %zu needed",
                  bytes, need);
    split.cuts = (Cut *)workspace;
    split.slots = (float *)(split.cuts + shape.workgroups);
    split.workgroups = shape.workgroups;
    split.tile_rows = shape.tile_rows;
    split.slot_floats = slot_floats_of(shape, a.width);
    const int64_t most_keys =
        PAGED ? keys_of_table(a.most_keys, (int64_t)a.map.max_pages << a.map.shift)
              : keys_of_packed(a.most_keys, a.k_rows, a.batch);
    if (!worth_sharing(shape, a.rows, a.batch, a.kv_heads, a.group, most_keys)) shape.split = false;
  }
  a.run = run_of(shape, a.rows, a.batch, a.kv_heads, a.group);
  if (a.width <= 64) attend_launch<T, PAGED, Q8, 64>(a, split, shape, s);
  else if (a.width <= 128) attend_launch<T, PAGED, Q8, 128>(a, split, shape, s);
  else attend_launch<T, PAGED, Q8, 256>(a, split, shape, s);
  return check_hip(hipGetLastError(), "k_attention launch");
}

template <typename T>
static int attend_any(const LmAttnArgs &a, bool paged, bool q8, void *workspace, size_t bytes,
                      hipStream_t s) {
  if (!paged) return attend<T, false, false>(a, workspace, bytes, s);
  return q8 ? attend<T, true, true>(a, workspace, bytes, s)
            : attend<T, true, false>(a, workspace, bytes, s);
}

}  // namespace hv
