// hv_lm.h -- what the language-model kernels share: element types, vector
// loads, lane reductions and the 8-bit formats.
#pragma once

#include "hv_internal.h"

namespace hv {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef _Float16 f16;
typedef __bf16 bf16;
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

// Eight adjacent elements: in 16-byte accesses at any element's alignment
// where all eight are there, else the first n (the rest zero).
template <typename T>
struct Eight {
  typedef T v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ v8 load(const T *p, int n) {
    v8 t = {};
    if (n == 8) {
      __builtin_memcpy(&t, p, sizeof t);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) t[i] = p[i];
    }
    return t;
  }
  static __device__ __forceinline__ void store(T *p, int n, v8 t) {
    if (n == 8) {
      __builtin_memcpy(p, &t, sizeof t);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = t[i];
    }
  }
};

// What a cache and its table have to be, for the entry points that use them.
int check_cache(const char *what, const hv_cache_desc &c, int type, int batch, int kv_heads,
                int width);

// The value of another lane of the same 16 (n lanes on, cyclically).
template <int N>
__device__ __forceinline__ int ror16(int v) {
  return __builtin_amdgcn_update_dpp(v, v, 0x120 + N, 0xf, 0xf, false);
}
template <int N>
__device__ __forceinline__ float ror16(float v) {
  return __builtin_bit_cast(float, ror16<N>(__builtin_bit_cast(int, v)));
}

// Reductions whose result every lane of the 16, or of the wavefront, has.
// Every lane has to be active.
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, ror16<8>(v));
  v = fmaxf(v, ror16<4>(v));
  v = fmaxf(v, ror16<2>(v));
  return fmaxf(v, ror16<1>(v));
}
__device__ __forceinline__ float sum16(float v) {
  v += ror16<8>(v);
  v += ror16<4>(v);
  v += ror16<2>(v);
  return v + ror16<1>(v);
}
__device__ __forceinline__ float max64(float v) {
  v = max16(v);
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float sum64(float v) {
  v = sum16(v);
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

static constexpr int kMinExp = -127;  // the matrix cores' smallest scale, 2^-127

// Smallest e >= -127 with amax <= L 2^e, L = 448 = 1.75 2^8 (e4m3) or
// 127 = 1.984375 2^6 (int8): adding the complement of L's mantissa to the
// float's bits carries into the exponent exactly when the mantissa is larger.
// An infinite amax gives 120 or 122.
template <int FMT>
__device__ __forceinline__ int block_exp(float amax) {
  const int bits = __builtin_bit_cast(int, amax);
  const int e = FMT == HV_Q_E4M3 ? ((bits + (0x7FFFFF - 0x600000)) >> 23) - 127 - 8
                                 : ((bits + (0x7FFFFF - 0x7E0000)) >> 23) - 127 - 6;
  return e < kMinExp ? kMinExp : e;
}

// Four values p 2^-e in 8 bits (round to nearest even); the products by a
// power of two are exact, or far below the smallest step.
template <int FMT>
__device__ __forceinline__ int quant4(const float *p, float inv) {
  if (FMT == HV_Q_E4M3) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(p[0] * inv, p[1] * inv, 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(p[2] * inv, p[3] * inv, r, true);
  }
  int r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float v = rintf(p[i] * inv);
    const int q = v != v ? 0 : (int)fminf(fmaxf(v, -127.f), 127.f);
    r |= (q & 0xFF) << (8 * i);
  }
  return r;
}

template <int FMT>
__device__ __forceinline__ void store_q8(uint8_t *q, int n, const float *p, float inv) {
  const v2i t = {quant4<FMT>(p, inv), quant4<FMT>(p + 4, inv)};
  Eight<uint8_t>::v8 b;
  __builtin_memcpy(&b, &t, sizeof b);
  Eight<uint8_t>::store(q, n, b);
}

}  // namespace hv
