// hv_lm.h -- what the language-model kernels share: element types, vector
// loads and lane reductions.
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

}  // namespace hv
