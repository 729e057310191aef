// hv_lm_norm.hip -- root-mean-square norm with the residual's addition and an
// output in 8 bits with power-of-two scales.
//
//   h = round(x + residual)          the residual stream that is kept
//   scale[r] = 1 / sqrt(mean h^2 + eps)
//   p = w h,  q = round(p 2^-e),  e the smallest exponent that holds the block
//
// The norm's factor is one number a row, so it stays out of the 8 bits: q and
// e come from p alone, need no sum over the row, and are the same bits in any
// order of work; a product over q multiplies its rows by `scale` in the end.
#include "hv_lm.h"

namespace hv {

struct NormArgs {
  const void *x, *residual, *weight;
  void *residual_out;
  uint8_t *q;
  int8_t *exps;
  float *scale;
  const int32_t *rows_dev;
  int64_t x_ld, residual_ld, residual_out_ld, q_ld, exps_ld;
  int rows, width;
  float eps;
};

static constexpr int kNormBlock = 128;  // columns that share an exponent
static constexpr int kMinExp = -127;    // the matrix cores' smallest scale, 2^-127

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

template <bool VEC>
__device__ __forceinline__ void store_q8(uint8_t *q, int n, int lo, int hi) {
  if (VEC) {
    *reinterpret_cast<v2i *>(q) = v2i{lo, hi};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) q[i] = (uint8_t)((i < 4 ? lo : hi) >> (8 * (i & 3)));
  }
}

// One workgroup a row; each thread takes eight columns at a time, so a block
// of 128 is 16 adjacent lanes.
template <typename T, int FMT, bool VEC, bool ROW>
__global__ __launch_bounds__(256) void k_rms_norm_q8(NormArgs a) {
  const int rows = a.rows_dev ? min(a.rows, *a.rows_dev) : a.rows;
  const int row = blockIdx.x;
  if (row >= rows) return;
  const T *x = (const T *)a.x + row * a.x_ld;
  const T *res = a.residual ? (const T *)a.residual + row * a.residual_ld : nullptr;
  T *out = a.residual ? (T *)a.residual_out + row * a.residual_out_ld : nullptr;
  const T *w = (const T *)a.weight;
  uint8_t *q = a.q + row * a.q_ld;
  int8_t *exps = a.exps + row * a.exps_ld;
  const int tid = threadIdx.x;
  __shared__ float part[2][4];

  float sum = 0.f, amax = 0.f;
  for (int c = 0; c < a.width; c += 2048) {
    const int c0 = c + tid * 8;
    const int n = min(8, a.width - c0);
    float h[8] = {}, p[8] = {};
    if (n > 0) {
      load8<T, VEC>(x + c0, n, h);
      if (res) {
        float r[8];
        load8<T, VEC>(res + c0, n, r);
        typedef T v8 __attribute__((ext_vector_type(8)));
        v8 t;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          t[i] = (T)(h[i] + r[i]);
          h[i] = (float)t[i];
        }
        if (VEC) {
          typedef T vt __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
          for (int i = 0; i < 8; i += 16 / sizeof(T)) {
            vt s;
#pragma unroll
            for (int j = 0; j < (int)(16 / sizeof(T)); ++j) s[j] = t[i + j];
            *reinterpret_cast<vt *>(out + c0 + i) = s;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i < n) out[c0 + i] = t[i];
        }
      }
      float g[8];
      load8<T, VEC>(w + c0, n, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = h[i] * g[i];
    }
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sum = __builtin_fmaf(h[i], h[i], sum);
      m = fmaxf(m, fabsf(p[i]));
    }
    if (ROW) {
      amax = fmaxf(amax, m);
    } else {
      const int e = block_exp<FMT>(max16(m));
      const float inv = __builtin_bit_cast(float, (127 - e) << 23);
      if (n > 0) {
        store_q8<VEC>(q + c0, n, quant4<FMT>(p, inv), quant4<FMT>(p + 4, inv));
        if ((tid & 15) == 0) exps[c0 / kNormBlock] = (int8_t)e;
      }
    }
  }

  sum = sum64(sum);
  if (ROW) amax = max64(amax);
  if ((tid & 63) == 0) {
    part[0][tid >> 6] = sum;
    part[1][tid >> 6] = amax;
  }
  __syncthreads();
  if (tid == 0) {
    sum = (part[0][0] + part[0][1]) + (part[0][2] + part[0][3]);
    a.scale[row] = 1.f / sqrtf(sum / (float)a.width + a.eps);
  }
  if (!ROW) return;
  amax = fmaxf(fmaxf(part[1][0], part[1][1]), fmaxf(part[1][2], part[1][3]));
  const int e = block_exp<FMT>(amax);
  const float inv = __builtin_bit_cast(float, (127 - e) << 23);
  if (tid == 0) exps[0] = (int8_t)e;
  // Every thread reads again what it read or wrote itself.
  const T *kept = out ? out : x;
  for (int c0 = tid * 8; c0 < a.width; c0 += 2048) {
    const int n = min(8, a.width - c0);
    float h[8], g[8];
    load8<T, VEC>(kept + c0, n, h);
    load8<T, VEC>(w + c0, n, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] *= g[i];
    store_q8<VEC>(q + c0, n, quant4<FMT>(h, inv), quant4<FMT>(h + 4, inv));
  }
}

template <typename T, int FMT, bool VEC>
static void norm_launch(const NormArgs &a, bool row, hipStream_t s) {
  const dim3 grid(a.rows), block(256);
  if (row) hv_launch(k_rms_norm_q8<T, FMT, VEC, true>, grid, block, 0, s, a);
  else hv_launch(k_rms_norm_q8<T, FMT, VEC, false>, grid, block, 0, s, a);
}

template <typename T>
static void norm_launch(const NormArgs &a, int format, bool vec, bool row, hipStream_t s) {
  if (format == HV_Q_E4M3) {
    if (vec) norm_launch<T, HV_Q_E4M3, true>(a, row, s);
    else norm_launch<T, HV_Q_E4M3, false>(a, row, s);
  } else {
    if (vec) norm_launch<T, HV_Q_I8, true>(a, row, s);
    else norm_launch<T, HV_Q_I8, false>(a, row, s);
  }
}

}  // namespace hv

using namespace hv;

extern "C" int hv_rms_norm_q8(const hv_rms_norm_desc *d, hv_stream_t stream) {
  clear_error();
  if (!d) return fail(HV_EVALUE, HV_ERR_ADDRESS, "rms_norm: null descriptor");
  if (d->type != HV_T_F32 && d->type != HV_T_F16 && d->type != HV_T_BF16)
    return fail(HV_EVALUE, HV_ERR_OPCODE, "rms_norm: bad element type %d", d->type);
  if (d->format != HV_Q_E4M3 && d->format != HV_Q_I8)
    return fail(HV_EVALUE, HV_ERR_OPCODE, "rms_norm: bad output format %d", d->format);
  if (d->block != 0 && d->block != kNormBlock)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "rms_norm: block %d is neither 128 nor 0 (the row)",
                d->block);
  if (d->rows < 0 || d->width < 1 || d->width > HV_NORM_MAX_WIDTH)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "rms_norm: %d rows of %d columns", d->rows, d->width);
  if (!(d->eps >= 0.f) || d->eps > 3e38f)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "rms_norm: eps must be finite and not negative");
  const int blocks = d->block ? (d->width + kNormBlock - 1) / kNormBlock : 1;
  if (d->x_ld < d->width || d->q_ld < d->width || d->exps_ld < blocks ||
      (d->residual && (d->residual_ld < d->width || d->residual_out_ld < d->width)))
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "rms_norm: a row stride is shorter than its row");
  if (d->rows == 0) return HV_OK;
  if (!d->x || !d->weight || !d->q || !d->exps || !d->scale ||
      (d->residual == nullptr) != (d->residual_out == nullptr))
    return fail(HV_EVALUE, HV_ERR_ADDRESS, "rms_norm: null argument");
  const int size = d->type == HV_T_F32 ? 4 : 2;
  if ((((uintptr_t)d->x | (uintptr_t)d->residual | (uintptr_t)d->residual_out |
        (uintptr_t)d->weight) & (size - 1)) || ((uintptr_t)d->scale & 3))
    return fail(HV_EVALUE, HV_ERR_ADDRESS, "rms_norm: a pointer is not aligned to its elements");
  NormArgs a{};
  a.x = d->x; a.residual = d->residual; a.weight = d->weight; a.residual_out = d->residual_out;
  a.q = (uint8_t *)d->q; a.exps = d->exps; a.scale = d->scale; a.rows_dev = d->rows_dev;
  a.x_ld = d->x_ld; a.residual_ld = d->residual_ld; a.residual_out_ld = d->residual_out_ld;
  a.q_ld = d->q_ld; a.exps_ld = d->exps_ld;
  a.rows = d->rows; a.width = d->width; a.eps = d->eps;
  // 16-byte loads and 8-byte stores where every row and chunk of eight allows it.
  uintptr_t at = (uintptr_t)d->x | (uintptr_t)d->residual | (uintptr_t)d->residual_out |
                 (uintptr_t)d->weight | (uintptr_t)(d->x_ld * size);
  if (d->residual) at |= (uintptr_t)(d->residual_ld * size) | (uintptr_t)(d->residual_out_ld * size);
  const bool vec = d->width % 8 == 0 && !(at & 15) &&
                   !(((uintptr_t)d->q | (uintptr_t)d->q_ld) & 7);
  const hipStream_t s = (hipStream_t)stream;
  if (d->type == HV_T_F32) norm_launch<float>(a, d->format, vec, d->block == 0, s);
  else if (d->type == HV_T_F16) norm_launch<f16>(a, d->format, vec, d->block == 0, s);
  else norm_launch<bf16>(a, d->format, vec, d->block == 0, s);
  return check_hip(hipGetLastError(), "k_rms_norm_q8 launch");
}
