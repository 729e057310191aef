// hv_lm_gemm.hip -- matrix product of e4m3 rows and weights whose blocks of
// 128 carry power-of-two scales.
//
//   y[m][n] = scale[m] sum_b 2^(ea[m][b] + ew[b][n/128]) sum_(k in b) a[m][k] w[k][n] + bias[n]
//
// The block-scaled MFMA (v_mfma_scale_f32_16x16x128_f8f6f4) takes one scale
// byte (2^(byte - 127)) for each row and 32 values of k of either operand; a
// block of 128 is one MFMA whose four bytes are the same, so the scales cost
// no instruction on the accumulators, and the order of k inside a block is
// free: lane l holds k = 64 h + 16 (l / 16) .. + 15, h = 0, 1.
//
// The 8-bit matrix cores add groups of products aligned to the largest one
// and cut off what lies 2^-13 below it (measured: 1.5e-5 of the result's norm
// on normal values, whatever the length). That is a hundredth of what the
// rounding to bf16 costs and a fourteenth of f16's, so 16-bit outputs take
// them; a float32 output takes the 16-bit matrix cores instead (Exact: e4m3
// values are exact in bf16, their sums good to 7.6e-8), block by block, the
// block's power of two applied to its sum.
#include <type_traits>

#include "hv_lm.h"

namespace hv {

struct GemmF8Args {
  const uint8_t *a;
  const int8_t *a_exps;
  const uint8_t *w;  // packed, see heatvit_hip.h
  const int8_t *w_exps;
  const float *row_scale, *bias;
  void *c;
  const int32_t *m_dev;
  int64_t lda, a_exps_ld, ldc;
  int m, n, k;
  int kb, nb;  // blocks of 128 along k and n
  bool vec;    // four outputs of a row may be stored at once
};

static constexpr int kTileBytes = 64 * 128;  // 64 channels by 128 k, packed

// Operands of one block of 128 and their product: W fragment (16 channels) by
// activation fragment (16 rows), added to acc with the factor 2^(we + ae).
struct Fast {
  typedef v8i frag;
  static __device__ __forceinline__ frag of(v4i lo, v4i hi) {
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  static __device__ __forceinline__ v4f mma(const frag &w, const frag &a, v4f acc, int we, int ae) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, acc, 0, 0, 0, we + 127, 0,
                                                            ae + 127);
  }
};
struct Exact {
  struct frag {
    v8bf v[4];
  };
  static __device__ __forceinline__ frag of(v4i lo, v4i hi) {
    frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int x = i < 2 ? lo[2 * i] : hi[2 * i - 4], y = i < 2 ? lo[2 * i + 1] : hi[2 * i - 3];
      const v2bf a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, false);
      const v2bf b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, true);
      const v2bf c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, 1.f, false);
      const v2bf d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, 1.f, true);
      f.v[i] = v8bf{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
    return f;
  }
  static __device__ __forceinline__ v4f mma(const frag &w, const frag &a, v4f acc, int we, int ae) {
    v4f t = {};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], a.v[i], t, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += ldexpf(t[i], we + ae);
    return acc;
  }
};

// Four channels n .. n + 3 of row m.
template <typename T>
__device__ __forceinline__ void store4(const GemmF8Args &g, int m, int n, v4f v, float scale) {
  T *p = (T *)g.c + m * g.ldc + n;
  v *= scale;
  if (g.bias) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < g.n) v[i] += g.bias[n + i];
  }
  if (g.vec && n + 4 <= g.n) {
    typedef T v4 __attribute__((ext_vector_type(4)));
    v4 t;
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = (T)v[i];
    *reinterpret_cast<v4 *>(p) = t;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < g.n) p[i] = (T)v[i];
  }
}

// One wavefront's part of FM x 16 rows by 64 channels; the NW wavefronts of a
// workgroup take every NW-th block of k and add up through LDS. Fragments come
// straight from memory: the packed weights are in the order the lanes take
// them.
template <typename T, int FM, int NW>
__global__ __launch_bounds__(64 * NW) void k_gemm_f8_direct(GemmF8Args g) {
  typedef typename std::conditional<std::is_same<T, float>::value, Exact, Fast>::type Mma;
  const int rows = g.m_dev ? min(g.m, *g.m_dev) : g.m;
  const int m0 = blockIdx.y * (16 * FM);
  if (m0 >= rows) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, grp = lane >> 4;
  const uint8_t *w = g.w + (size_t)blockIdx.x * g.kb * kTileBytes + lane * 16;
  const uint8_t *a[FM];
  const int8_t *ae[FM];
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int64_t m = min(m0 + 16 * i + col, rows - 1);  // rows past the end repeat the last
    a[i] = g.a + m * g.lda + 16 * grp;
    ae[i] = g.a_exps + m * g.a_exps_ld;
  }
  v4f acc[FM][4] = {};
  for (int b = wave; b < g.kb; b += NW) {
    typename Mma::frag wf[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const v4i lo = *reinterpret_cast<const v4i *>(w + (size_t)b * kTileBytes + j * 2048);
      const v4i hi = *reinterpret_cast<const v4i *>(w + (size_t)b * kTileBytes + j * 2048 + 1024);
      wf[j] = Mma::of(lo, hi);
    }
    const int we = g.w_exps[(size_t)b * g.nb + blockIdx.x / 2];
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      // past the end of k: zeros
      v4i lo = {}, hi = {};
      const int k = b * 128 + 16 * grp;
      if (k < g.k) lo = *reinterpret_cast<const v4i *>(a[i] + b * 128);
      if (k + 64 < g.k) hi = *reinterpret_cast<const v4i *>(a[i] + b * 128 + 64);
      const typename Mma::frag af = Mma::of(lo, hi);
      const int e = ae[i][b];
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = Mma::mma(wf[j], af, acc[i][j], we, e);
    }
  }
  __shared__ v4f part[NW][FM * 4][64];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) part[wave][i * 4 + j][lane] = acc[i][j];
  __syncthreads();
  for (int f = wave; f < FM * 4; f += NW) {
    v4f v = part[0][f][lane];
#pragma unroll
    for (int k = 1; k < NW; ++k) v += part[k][f][lane];
    const int m = m0 + 16 * (f / 4) + col;
    const int n = blockIdx.x * 64 + 16 * grp + 4 * (f % 4);
    if (m < rows) store4<T>(g, m, n, v, g.row_scale ? g.row_scale[m] : 1.f);
  }
}

template <typename T>
static void gemm_f8_launch(const GemmF8Args &g, hipStream_t s) {
  hv_launch(k_gemm_f8_direct<T, 4, 4>, dim3((g.n + 63) / 64, (g.m + 63) / 64), dim3(256), 0, s, g);
}

}  // namespace hv

using namespace hv;

extern "C" {

size_t hv_gemm_f8_workspace_bytes(int m, int n, int k) {
  (void)m; (void)n; (void)k;
  return 0;
}

int hv_gemm_f8(const hv_gemm_f8_desc *d, void *workspace, size_t workspace_bytes,
               hv_stream_t stream) {
  (void)workspace; (void)workspace_bytes;
  clear_error();
  if (!d) return fail(HV_EVALUE, HV_ERR_ADDRESS, "gemm_f8: null descriptor");
  if (d->type != HV_T_F32 && d->type != HV_T_F16 && d->type != HV_T_BF16)
    return fail(HV_EVALUE, HV_ERR_OPCODE, "gemm_f8: bad output type %d", d->type);
  if (d->m < 0 || d->n < 1 || d->k < 1 || d->n > HV_GEMM_F8_MAX_DIM || d->k > HV_GEMM_F8_MAX_DIM ||
      d->m > HV_GEMM_F8_MAX_ROWS || d->k % 16)
    return fail(HV_EVALUE, HV_ERR_DIMENSION,
                "gemm_f8: m=%d n=%d k=%d (k a multiple of 16)", d->m, d->n, d->k);
  GemmF8Args g{};
  g.kb = (d->k + 127) / 128;
  g.nb = (d->n + 127) / 128;
  if (d->lda < d->k || d->lda % 16 || d->a_exps_ld < g.kb || d->ldc < d->n)
    return fail(HV_EVALUE, HV_ERR_DIMENSION,
                "gemm_f8: a row stride is shorter than its row, or lda no multiple of 16");
  if (d->m == 0) return HV_OK;
  if (!d->a || !d->a_exps || !d->w_packed || !d->w_exps || !d->c)
    return fail(HV_EVALUE, HV_ERR_ADDRESS, "gemm_f8: null argument");
  const int size = d->type == HV_T_F32 ? 4 : 2;
  if ((((uintptr_t)d->a | (uintptr_t)d->w_packed) & 15) || ((uintptr_t)d->c & (size - 1)) ||
      (((uintptr_t)d->row_scale | (uintptr_t)d->bias) & 3))
    return fail(HV_EVALUE, HV_ERR_ADDRESS,
                "gemm_f8: a and w_packed must be 16-byte aligned, the others to their elements");
  g.a = (const uint8_t *)d->a; g.a_exps = d->a_exps;
  g.w = (const uint8_t *)d->w_packed; g.w_exps = d->w_exps;
  g.row_scale = d->row_scale; g.bias = d->bias; g.c = d->c; g.m_dev = d->m_dev;
  g.lda = d->lda; g.a_exps_ld = d->a_exps_ld; g.ldc = d->ldc;
  g.m = d->m; g.n = d->n; g.k = d->k;
  g.vec = d->ldc % 4 == 0 && !((uintptr_t)d->c & (4 * size - 1));
  const hipStream_t s = (hipStream_t)stream;
  if (d->type == HV_T_F32) gemm_f8_launch<float>(g, s);
  else if (d->type == HV_T_F16) gemm_f8_launch<f16>(g, s);
  else gemm_f8_launch<bf16>(g, s);
  return check_hip(hipGetLastError(), "gemm_f8 launch");
}

}  // extern "C"
