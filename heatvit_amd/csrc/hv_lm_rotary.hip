// hv_lm_rotary.hip -- norms of the heads of queries and keys and the rotation
// by their positions, in one pass.
//
//   y = x / sqrt(mean x^2 + eps) * w           over a head (w NULL: y = x)
//   (a, b) -> s (a cos t - b sin t, a sin t + b cos t),  t = position * freq
//
// A pair's angle is taken in turns in 64 bits and reduced there, since a
// float32 angle of a far position has lost the turn it lies in; what is left
// of a turn is a float32 to half a step. All heads of a token share its angles:
// a workgroup computes those of its tokens once and keeps them in LDS.
#include <type_traits>

#include "hv_lm.h"

namespace hv {

struct RotaryArgs {
  const void *x[2], *weight[2];  // queries, keys
  void *out[2];
  const int32_t *positions;
  const float *freqs;
  const int32_t *rows_dev;
  int64_t ld[2], head_ld[2], out_ld[2], out_head_ld[2];
  int rows, heads[2], width, pairs, interleaved;
  int tokens;  // of a workgroup
  float eps, scale, inv_width, low;  // low: under it a sum of squares has lost bits
};

static constexpr int kMaxPairs = HV_ROTARY_MAX_WIDTH / 2;

// Sum over LANES lanes side by side, which all of them get.
template <int LANES>
__device__ __forceinline__ float sum_of(float v) {
  auto moved = [](float x, auto ctrl) {
    const int b = __builtin_bit_cast(int, x);
    return __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(b, b, decltype(ctrl)::value, 0xf, 0xf, false));
  };
  v += moved(v, std::integral_constant<int, 0xB1>());                  // lane ^ 1
  v += moved(v, std::integral_constant<int, 0x4E>());                  // lane ^ 2
  if (LANES > 4) v += moved(v, std::integral_constant<int, 0x141>());  // 7 - lane, of eight
  if (LANES > 8) v += moved(v, std::integral_constant<int, 0x140>());  // 15 - lane, of sixteen
  if (LANES > 16) v += __shfl_xor(v, 16);
  if (LANES > 32) v += __shfl_xor(v, 32);
  return v;
}

// LANES lanes a head; each takes 16 of its elements as two runs of eight: the
// two halves of eight pairs (or eight interleaved pairs), or what follows the
// rotated part.
template <typename T, int LANES>
__global__ __launch_bounds__(256) void k_rotary_qk(RotaryArgs a) {
  constexpr int kGroups = 256 / LANES;
  typedef typename Eight<T>::v8 v8;
  extern __shared__ float2 turn[];  // [tokens][pairs]
  const int rows = a.rows_dev ? min(a.rows, *a.rows_dev) : a.rows;
  const int64_t row0 = (int64_t)blockIdx.x * a.tokens;
  if (row0 >= rows) return;
  const int tokens = (int)min((int64_t)a.tokens, rows - row0);
  auto turns = [&]() {
    for (int i = threadIdx.x; i < tokens * a.pairs; i += 256) {
      const int t = i / a.pairs, p = i - t * a.pairs;
      const double turns =
          (double)a.positions[row0 + t] * (double)a.freqs[p] * 0.15915494309189533577;
      float sin_, cos_;
      sincospif((float)(2. * (turns - rint(turns))), &sin_, &cos_);
      turn[i] = make_float2(cos_ * a.scale, sin_ * a.scale);
    }
  };

  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int heads = a.heads[0] + a.heads[1], rotated = 2 * a.pairs;
  const int pair_lanes = (a.pairs + 7) / 8;
  const bool pair = lane < pair_lanes;
  int at[2], n[2];  // the lane's two runs
  if (pair && !a.interleaved) {
    at[0] = 8 * lane;
    at[1] = a.pairs + 8 * lane;
    n[0] = n[1] = min(8, a.pairs - 8 * lane);
  } else {
    at[0] = pair ? 16 * lane : rotated + 16 * (lane - pair_lanes);
    at[1] = at[0] + 8;
    const int left = (pair ? rotated : a.width) - at[0];
    n[0] = max(0, min(8, left));
    n[1] = max(0, min(8, left - 8));
  }
  const int items = tokens * heads;
  // Where item i's head lies, and what is loaded of it: the next one's is on its way while
  // one is worked on.
  v8 next[2];
  auto load = [&](int t, int h) {
    const int which = h >= a.heads[0], head = which ? h - a.heads[0] : h;
    const T *x = (const T *)a.x[which] + (row0 + t) * a.ld[which] + head * a.head_ld[which];
#pragma unroll
    for (int r = 0; r < 2; ++r) next[r] = n[r] > 0 ? Eight<T>::load(x + at[r], n[r]) : v8{};
  };
  const int step_t = kGroups / heads, step_h = kGroups - step_t * heads;
  int t = min(group, items - 1) / heads, h = min(group, items - 1) - t * heads;
  load(t, h);
  v8 weight[2][2] = {};  // of queries and of keys
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int r = 0; r < 2; ++r)
      if (a.weight[k] && n[r] > 0) weight[k][r] = Eight<T>::load((const T *)a.weight[k] + at[r], n[r]);
  turns();
  __syncthreads();
  // Every lane of a wavefront takes part in its reductions: a group past the
  // last item repeats it and writes nothing.
  for (int i0 = 0; i0 < items; i0 += kGroups) {
    const bool live = i0 + group < items;
    const int token = t, which = h >= a.heads[0], head = which ? h - a.heads[0] : h;
    float v[2][8];
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[r][i] = (float)next[r][i];
        sum = __builtin_fmaf(v[r][i], v[r][i], sum);
      }
    if (i0 + kGroups < items) {
      t += step_t;
      h += step_h;
      if (h >= heads) {
        h -= heads;
        ++t;
      }
      if (t >= tokens) {
        t = tokens - 1;
        h = heads - 1;
      }
      load(t, h);
    }
    if (a.weight[which]) {
      sum = sum_of<LANES>(sum);
      float f = __builtin_amdgcn_rsqf(sum * a.inv_width + a.eps);
      // Squares outside float32's normal numbers are summed again in 64 bits.
      const bool again = sum < a.low || !(sum < 0x1p120f);
      if (__builtin_amdgcn_ballot_w64(again)) {
        double s = 0.;
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int i = 0; i < 8; ++i) s += (double)v[r][i] * (double)v[r][i];
#pragma unroll
        for (int o = 1; o < LANES; o *= 2) s += __shfl_xor(s, o);
        const double d = 1. / sqrt(s / a.width + (double)a.eps);
        if (again) {
          // x f in 64 bits: f may lie outside float32's numbers where x f does not
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[r][i] = (float)((double)v[r][i] * d);
          f = 1.f;
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v[r][i] = v[r][i] * f * (float)(which ? weight[1][r][i] : weight[0][r][i]);
      }
    }
    if (pair) {
      const float2 *cs = turn + token * a.pairs + 8 * lane;
      const int count = min(8, a.pairs - 8 * lane);
      if (!a.interleaved) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 c = cs[i < count ? i : 0];
          const float p = v[0][i], q = v[1][i];
          v[0][i] = p * c.x - q * c.y;
          v[1][i] = p * c.y + q * c.x;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 c = cs[i < count ? i : 0];
          float &x0 = v[i / 4][i % 4 * 2], &x1 = v[i / 4][i % 4 * 2 + 1];
          const float p = x0, q = x1;
          x0 = p * c.x - q * c.y;
          x1 = p * c.y + q * c.x;
        }
      }
    }
    if (live) {
      T *out = (T *)a.out[which] + (row0 + token) * a.out_ld[which] + head * a.out_head_ld[which];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        v8 e;
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = (T)v[r][i];
        if (n[r] > 0) Eight<T>::store(out + at[r], n[r], e);
      }
    }
  }
}

template <typename T>
static void rotary_launch(RotaryArgs a, hipStream_t s) {
  const int lanes = (a.pairs + 7) / 8 + (a.width - 2 * a.pairs + 15) / 16;
  // Tokens a workgroup: its threads compute an angle each, while there are
  // workgroups enough.
  a.tokens = a.pairs ? max(1, min(16, 256 / a.pairs)) : 16;
  while (a.tokens > 1 && (a.rows + a.tokens - 1) / a.tokens < 1024) a.tokens /= 2;
  const dim3 grid((unsigned)((a.rows + a.tokens - 1) / a.tokens)), block(256);
  const uint32_t lds = (uint32_t)(a.tokens * a.pairs * sizeof(float2));
  if (lanes <= 4) hv_launch(k_rotary_qk<T, 4>, grid, block, lds, s, a);
  else if (lanes <= 8) hv_launch(k_rotary_qk<T, 8>, grid, block, lds, s, a);
  else if (lanes <= 16) hv_launch(k_rotary_qk<T, 16>, grid, block, lds, s, a);
  else if (lanes <= 32) hv_launch(k_rotary_qk<T, 32>, grid, block, lds, s, a);
  else hv_launch(k_rotary_qk<T, 64>, grid, block, lds, s, a);
}

}  // namespace hv

using namespace hv;

extern "C" int hv_rotary_qk(const hv_rotary_desc *d, hv_stream_t stream) {
  clear_error();
  if (!d) return fail(HV_EVALUE, HV_ERR_ADDRESS, "rotary: null descriptor");
  if (d->type != HV_T_F32 && d->type != HV_T_F16 && d->type != HV_T_BF16)
    return fail(HV_EVALUE, HV_ERR_OPCODE, "rotary: bad element type %d", d->type);
  if (d->layout != HV_ROTARY_HALF && d->layout != HV_ROTARY_INTERLEAVED)
    return fail(HV_EVALUE, HV_ERR_OPCODE, "rotary: bad layout %d", d->layout);
  if (d->rows < 0 || d->rows > HV_LM_MAX_ROWS || d->q_heads < 1 || d->k_heads < 0 ||
      d->q_heads > HV_LM_MAX_HEADS || d->k_heads > HV_LM_MAX_HEADS || d->width < 1 ||
      d->width > HV_ROTARY_MAX_WIDTH)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "rotary: %d rows of %d and %d heads of %d", d->rows,
                d->q_heads, d->k_heads, d->width);
  if (d->rotated < 0 || d->rotated > d->width || d->rotated % 2)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "rotary: %d of %d elements rotated", d->rotated,
                d->width);
  if (!(d->eps >= 0.f) || d->eps > 3e38f || !(d->scale > -3e38f) || !(d->scale < 3e38f))
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "rotary: eps or scale out of range");
  const bool keys = d->k_heads > 0;
  if (d->q_ld < 0 || d->q_head_ld < 0 || d->q_out_ld < 0 || d->q_out_head_ld < 0 || d->k_ld < 0 ||
      d->k_head_ld < 0 || d->k_out_ld < 0 || d->k_out_head_ld < 0)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "rotary: a negative stride");
  if (d->rows == 0) return HV_OK;
  if (!d->q || !d->q_out || !d->positions || (d->rotated && !d->freqs) ||
      (keys && (!d->k || !d->k_out)))
    return fail(HV_EVALUE, HV_ERR_ADDRESS, "rotary: null argument");
  const int size = d->type == HV_T_F32 ? 4 : 2;
  uintptr_t all = (uintptr_t)d->q | (uintptr_t)d->q_out | (uintptr_t)d->q_weight;
  if (keys) all |= (uintptr_t)d->k | (uintptr_t)d->k_out | (uintptr_t)d->k_weight;
  if ((all & (size - 1)) || (((uintptr_t)d->positions | (uintptr_t)d->freqs) & 3))
    return fail(HV_EVALUE, HV_ERR_ADDRESS, "rotary: a pointer is not aligned to its elements");
  RotaryArgs a{};
  a.x[0] = d->q; a.x[1] = d->k; a.weight[0] = d->q_weight; a.weight[1] = d->k_weight;
  a.out[0] = d->q_out; a.out[1] = d->k_out;
  a.positions = d->positions; a.freqs = d->freqs; a.rows_dev = d->rows_dev;
  a.ld[0] = d->q_ld; a.ld[1] = d->k_ld; a.head_ld[0] = d->q_head_ld; a.head_ld[1] = d->k_head_ld;
  a.out_ld[0] = d->q_out_ld; a.out_ld[1] = d->k_out_ld;
  a.out_head_ld[0] = d->q_out_head_ld; a.out_head_ld[1] = d->k_out_head_ld;
  a.rows = d->rows; a.heads[0] = d->q_heads; a.heads[1] = d->k_heads; a.width = d->width;
  a.pairs = d->rotated / 2; a.interleaved = d->layout == HV_ROTARY_INTERLEAVED;
  a.eps = d->eps; a.scale = d->scale; a.inv_width = 1.f / (float)d->width;
  a.low = d->eps < 0x1p-100f ? (0x1p-100f - d->eps) * (float)d->width : 0.f;
  const hipStream_t s = (hipStream_t)stream;
  if (d->type == HV_T_F32) rotary_launch<float>(a, s);
  else if (d->type == HV_T_F16) rotary_launch<f16>(a, s);
  else rotary_launch<bf16>(a, s);
  return check_hip(hipGetLastError(), "k_rotary_qk launch");
}
