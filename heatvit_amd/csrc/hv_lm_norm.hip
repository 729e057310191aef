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
//
// HBM bounds it: 16384 x 8192 bf16 with a residual (950 MB) take 166 us, 4096 x
// 5120 f16 with one exponent a row (147 MB, the row read again from the L2)
// 33 us, 5.7 and 4.4 TB/s. One row of 4096 takes 2.5 us, 1003 x 1000 f32 3.9:
// a load's latency, the reduction and the stores.
#include <type_traits>

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
  float eps, low;  // low: under it a sum of squares has lost bits that eps does not hide
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

template <int FMT>
__device__ __forceinline__ void store_q8(uint8_t *q, int n, const float *p, float inv) {
  const v2i t = {quant4<FMT>(p, inv), quant4<FMT>(p + 4, inv)};
  Eight<uint8_t>::v8 b;
  __builtin_memcpy(&b, &t, sizeof b);
  Eight<uint8_t>::store(q, n, b);
}

// LANES threads a row (16: sixteen rows a workgroup, 64: four, else one); each
// takes eight columns at a time, so a block of 128 is 16 adjacent lanes.
template <typename T, int FMT, bool ROW, int LANES>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void k_rms_norm_q8(NormArgs a) {
  constexpr int kRows = LANES < 256 ? 256 / LANES : 1, kWaves = LANES / 64;
  const int rows = a.rows_dev ? min(a.rows, *a.rows_dev) : a.rows;
  const int tid = threadIdx.x % LANES;
  // Of a wavefront with several rows, lanes past the last row repeat it and
  // write nothing: its other lanes need them active.
  const int64_t mine = (int64_t)blockIdx.x * kRows + threadIdx.x / LANES;
  if (LANES >= 64 ? mine >= rows : (int64_t)blockIdx.x * kRows >= rows) return;
  const bool live = mine < rows;
  const int64_t row = live ? mine : rows - 1;
  const T *x = (const T *)a.x + row * a.x_ld;
  const T *res = a.residual ? (const T *)a.residual + row * a.residual_ld : nullptr;
  T *out = a.residual ? (T *)a.residual_out + row * a.residual_out_ld : nullptr;
  const T *w = (const T *)a.weight;
  typedef typename Eight<T>::v8 v8;
  uint8_t *q = a.q + row * a.q_ld;
  int8_t *exps = a.exps + row * a.exps_ld;
  float sum = 0.f, amax = 0.f;
  for (int c = 0; c < a.width; c += LANES * 8) {
    const int c0 = c + tid * 8;
    const int n = min(8, a.width - c0);
    float h[8] = {}, p[8] = {};
    if (n > 0) {
      v8 t = Eight<T>::load(x + c0, n);
      const v8 g = Eight<T>::load(w + c0, n);
      if (res) {
        const v8 r = Eight<T>::load(res + c0, n);
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = (T)((float)t[i] + (float)r[i]);
        if (live) Eight<T>::store(out + c0, n, t);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h[i] = (float)t[i];
        p[i] = h[i] * (float)g[i];
      }
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
      if (n > 0 && live) {
        store_q8<FMT>(q + c0, n, p, inv);
        if ((tid & 15) == 0) exps[c0 / kNormBlock] = (int8_t)e;
      }
    }
  }

  if (LANES == 16) {
    sum = sum16(sum);
    if (ROW) amax = max16(amax);
  } else {
    sum = sum64(sum);
    if (ROW) amax = max64(amax);
  }
  if (LANES > 64) {
    __shared__ float part[2][kWaves > 0 ? kWaves : 1];
    if ((tid & 63) == 0) {
      part[0][tid >> 6] = sum;
      part[1][tid >> 6] = amax;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) amax = fmaxf(amax, part[1][w]);
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += part[0][w];
  }
  const T *kept = out ? out : x;
  // Squares above float32's numbers, or below its normal ones where eps does
  // not hide that, are summed again in 64 bits, by the row's first wavefront.
  // (A float16's never are.)
  constexpr int kAgain = LANES < 64 ? LANES : 64;
  if (tid < kAgain) {
    if (!std::is_same<T, f16>::value && (sum < a.low || sum >= 0x1p120f)) {
      double again = 0.;
      for (int c0 = tid * 8; c0 < a.width; c0 += kAgain * 8) {
        const v8 t = Eight<T>::load(kept + c0, min(8, a.width - c0));
#pragma unroll
        for (int i = 0; i < 8; ++i) again += (double)(float)t[i] * (double)(float)t[i];
      }
#pragma unroll
      for (int o = 1; o < kAgain; o *= 2) again += __shfl_xor(again, o);
      if (live && tid == 0) a.scale[row] = (float)(1. / sqrt(again / a.width + (double)a.eps));
    } else if (live && tid == 0) {
      a.scale[row] = 1.f / sqrtf(sum / (float)a.width + a.eps);
    }
  }
  if (!ROW || !live) return;
  const int e = block_exp<FMT>(amax);
  const float inv = __builtin_bit_cast(float, (127 - e) << 23);
  if (tid == 0) exps[0] = (int8_t)e;
  // Every thread reads again what it read or wrote itself.
  for (int c0 = tid * 8; c0 < a.width; c0 += LANES * 8) {
    const int n = min(8, a.width - c0);
    const v8 t = Eight<T>::load(kept + c0, n), g = Eight<T>::load(w + c0, n);
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = (float)t[i] * (float)g[i];
    store_q8<FMT>(q + c0, n, p, inv);
  }
}

template <typename T, int FMT, int LANES>
static void norm_launch(const NormArgs &a, bool row, hipStream_t s) {
  constexpr int kRows = LANES < 256 ? 256 / LANES : 1;
  const dim3 grid((unsigned)(((int64_t)a.rows + kRows - 1) / kRows));
  const dim3 block(LANES < 256 ? 256 : LANES);
  if (row) hv_launch(k_rms_norm_q8<T, FMT, true, LANES>, grid, block, 0, s, a);
  else hv_launch(k_rms_norm_q8<T, FMT, false, LANES>, grid, block, 0, s, a);
}

// Threads a row (us by 16, 64, 256 and 1024): many short rows want few, since
// a workgroup of idle threads costs as much as one at work (65536 x 64 bf16
// 9.1, 22.4, 55, 190; 50432 x 192 13.5, 18.5, 44, 150; 16384 x 768 17.7, 17.0,
// 19.5, 53; 8192 x 2048 32.2, 26.5, 25.0, 41), long rows and few rows many,
// whose loads are then on their way at once (16384 x 8192 228, 185, 174, 164;
// 32 x 8192 50, 14.1, 5.2, 3.6; 512 x 4096 32.7, 9.6, 5.0, 4.9). A launch has
// less than 2^32 threads.
template <typename T, int FMT>
static void norm_launch(const NormArgs &a, bool row, hipStream_t s) {
  const bool few = a.rows <= 512;
  if (a.width <= (few ? 128 : 512)) return norm_launch<T, FMT, 16>(a, row, s);
  if (a.width <= (few ? 512 : 1024)) return norm_launch<T, FMT, 64>(a, row, s);
  if (a.width <= (few ? 2048 : 8191) || a.rows >= 1 << 22)
    return norm_launch<T, FMT, 256>(a, row, s);
  norm_launch<T, FMT, 1024>(a, row, s);
}

template <typename T>
static void norm_launch(const NormArgs &a, int format, bool row, hipStream_t s) {
  if (format == HV_Q_E4M3) norm_launch<T, HV_Q_E4M3>(a, row, s);
  else norm_launch<T, HV_Q_I8>(a, row, s);
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
  if (d->rows < 0 || d->rows > HV_LM_MAX_ROWS || d->width < 1 ||
      d->width > HV_NORM_MAX_WIDTH)
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
  a.low = d->eps < 0x1p-100f ? (0x1p-100f - d->eps) * (float)d->width : 0.f;
  const hipStream_t s = (hipStream_t)stream;
  if (d->type == HV_T_F32) norm_launch<float>(a, d->format, d->block == 0, s);
  else if (d->type == HV_T_F16) norm_launch<f16>(a, d->format, d->block == 0, s);
  else norm_launch<bf16>(a, d->format, d->block == 0, s);
  return check_hip(hipGetLastError(), "k_rms_norm_q8 launch");
}
