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
//
// HBM bounds it: 16384 rows of 32 and 8 heads of 128 in bf16 (336 MB) take 61 us, 5.4 TB/s,
// in float32 126. One row takes 3.3 us: its loads, the angles, a barrier and the stores. What
// cost most on the way there (84 us at first): reductions through LDS and the weights loaded
// for every head (76), and registers, of which five wavefronts a SIMD leave 96 (63).
#include <type_traits>

#include "hv_lm.h"
#include "hv_lm_rotary_plan.h"

namespace hv {

struct RotaryArgs {
  const void *x[2], *weight[2];  // queries, keys
  void *out[2];
  const int32_t *positions;
  const float *freqs;
  const int32_t *rows_dev;
  int64_t ld[2], head_ld[2], out_ld[2], out_head_ld[2];
  int rows, heads[2], width, pairs, interleaved;
  int tokens[2];  // of a workgroup, of queries or of keys
  int least_exp;
  float eps, scale, inv_width, low;  // low: under it a sum of squares has lost bits
};

static constexpr int kMaxPairs = HV_ROTARY_MAX_WIDTH / 2;

// Sum, or largest, of LANES lanes side by side, which all of them get.
template <int LANES, typename Op>
__device__ __forceinline__ float all_of(float v, Op op) {
  auto moved = [](float x, auto ctrl) {
    const int b = __builtin_bit_cast(int, x);
    return __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(b, b, decltype(ctrl)::value, 0xf, 0xf, false));
  };
  v = op(v, moved(v, std::integral_constant<int, 0xB1>()));                  // lane ^ 1
  v = op(v, moved(v, std::integral_constant<int, 0x4E>()));                  // lane ^ 2
  if (LANES > 4) v = op(v, moved(v, std::integral_constant<int, 0x141>()));  // 7 - lane, of eight
  if (LANES > 8) v = op(v, moved(v, std::integral_constant<int, 0x140>()));  // 15 - lane, of 16
  if (LANES > 16) v = op(v, __shfl_xor(v, 16));
  if (LANES > 32) v = op(v, __shfl_xor(v, 32));
  return v;
}

// LANES lanes a head; each takes 16 of its elements as two runs of eight: the
// two halves of eight pairs (or eight interleaved pairs), or what follows the
// rotated part. MORE: a head of 65 lanes, of whose last one's elements 64 take one each.
template <typename T, int LANES, bool MORE>
__global__ __launch_bounds__(256, 5) void k_rotary_qk(RotaryArgs a) {
  constexpr int kGroups = 256 / LANES;
  typedef typename Eight<T>::v8 v8;
  extern __shared__ float2 turn[];  // [tokens][pairs]
  const int rows = a.rows_dev ? min(a.rows, *a.rows_dev) : a.rows;
  const int which = blockIdx.y, heads = a.heads[which];
  const int64_t row0 = (int64_t)blockIdx.x * a.tokens[which];
  if (row0 >= rows) return;
  const int tokens = (int)min((int64_t)a.tokens[which], rows - row0);
  const T *const x0 = (const T *)a.x[which] + row0 * a.ld[which];
  T *const out0 = (T *)a.out[which] + row0 * a.out_ld[which];
  const T *const w = (const T *)a.weight[which];
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
  const int rotated = 2 * a.pairs;
  const int pair_lanes = rotary_pair_lanes(a.pairs);
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
  const int more_at = rotated + 16 * (LANES - pair_lanes) + lane;
  const bool more = MORE && more_at < a.width;
  T next_more = (T)0.f;
  auto load = [&](int t, int h) {
    const T *x = x0 + t * a.ld[which] + h * a.head_ld[which];
#pragma unroll
    for (int r = 0; r < 2; ++r) next[r] = n[r] > 0 ? Eight<T>::load(x + at[r], n[r]) : v8{};
    if (more) next_more = x[more_at];
  };
  const int step_t = kGroups / heads, step_h = kGroups - step_t * heads;
  int t = min(group, items - 1) / heads, h = min(group, items - 1) - t * heads;
  load(t, h);
  v8 weight[2] = {};
#pragma unroll
  for (int r = 0; r < 2; ++r)
    if (w && n[r] > 0) weight[r] = Eight<T>::load(w + at[r], n[r]);
  const float weight_more = w && more ? (float)w[more_at] : 0.f;
  turns();
  __syncthreads();
  // Every lane of a wavefront takes part in its reductions: a group past the
  // last item repeats it and writes nothing.
  for (int i0 = 0; i0 < items; i0 += kGroups) {
    const bool live = i0 + group < items;
    const int token = t, head = h;
    float v[2][8];
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[r][i] = (float)next[r][i];
        sum = __builtin_fmaf(v[r][i], v[r][i], sum);
      }
    float v_more = (float)next_more;
    if (MORE) sum = __builtin_fmaf(v_more, v_more, sum);
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
    if (w) {
      auto add = [](float p, float q) { return p + q; };
      sum = all_of<LANES>(sum, add);
      float f = __builtin_amdgcn_rsqf(sum * a.inv_width + a.eps);
      // Squares outside float32's normal numbers are summed again, of the values times a
      // power of two, which the root of the scaled sum takes out.
      const bool again = sum < a.low || !(sum < 0x1p120f);
      if (__builtin_amdgcn_ballot_w64(again)) {
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(v[i / 8][i % 8]));
        if (MORE) most = fmaxf(most, fabsf(v_more));
        most = all_of<LANES>(most, [](float p, float q) { return fmaxf(p, q); });
        // (eps by that power squared stays a number)
        const int e = again ? max(__builtin_amdgcn_frexp_expf(most), a.least_exp) : 0;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float &x = v[i / 8][i % 8];
          x = ldexpf(x, -e);
          s = __builtin_fmaf(x, x, s);
        }
        if (MORE) {
          v_more = ldexpf(v_more, -e);
          s = __builtin_fmaf(v_more, v_more, s);
        }
        s = all_of<LANES>(s, add);
        if (again) f = __builtin_amdgcn_rsqf(s * a.inv_width + ldexpf(a.eps, -2 * e));
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[r][i] = v[r][i] * f * (float)weight[r][i];
      }
      v_more = v_more * f * weight_more;
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
      T *out = out0 + token * a.out_ld[which] + head * a.out_head_ld[which];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        v8 e;
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = (T)v[r][i];
        if (n[r] > 0) Eight<T>::store(out + at[r], n[r], e);
      }
      if (more) out[more_at] = (T)v_more;
    }
  }
}

template <typename T>
static void rotary_launch(RotaryArgs a, hipStream_t s) {
  const int lanes = rotary_lanes(a.pairs, a.width);
  // Tokens a workgroup: its threads compute an angle each, while there are
  // workgroups enough; keys, whose heads are fewer, take more of them. (4096 rows of 32 and 8
  // heads of 128 take 15.6 us by 1024 workgroups, 18.4 by 4096 of a token each; 4000 rows of
  // 20 and 20 of 100 33.3 by 1000 of four tokens, 36.2 by 400 of ten.)
  const int keys = a.heads[1] ? 1 : 0;
  int most = a.pairs ? max(1, min(16, 256 / a.pairs)) : 16;
  while (most > 1 && (a.rows + most - 1) / most < 1024) most /= 2;
  while ((a.rows + most - 1) / most > 1 << 22) most *= 2;  // a launch has less than 2^32 threads
  a.tokens[0] = a.tokens[1] = most;
  if (keys)
    a.tokens[1] = max(most, min(most * a.heads[0] / a.heads[1], min(16, 1024 / max(1, a.pairs))));
  const dim3 grid((unsigned)((a.rows + most - 1) / most), 1 + keys), block(256);
  const uint32_t lds = (uint32_t)(max(a.tokens[0], a.tokens[1]) * a.pairs * sizeof(float2));
  if (lanes <= 4) hv_launch(k_rotary_qk<T, 4, false>, grid, block, lds, s, a);
  else if (lanes <= 8) hv_launch(k_rotary_qk<T, 8, false>, grid, block, lds, s, a);
  else if (lanes <= 16) hv_launch(k_rotary_qk<T, 16, false>, grid, block, lds, s, a);
  else if (lanes <= 32) hv_launch(k_rotary_qk<T, 32, false>, grid, block, lds, s, a);
  else if (lanes <= 64) hv_launch(k_rotary_qk<T, 64, false>, grid, block, lds, s, a);
  else hv_launch(k_rotary_qk<T, 64, true>, grid, block, lds, s, a);
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
  int e = 0;
  frexpf(d->eps, &e);  // eps <= 2^e
  a.least_exp = d->eps > 0.f ? (e - 100) / 2 : -200;
  a.low = d->eps < 0x1p-100f ? (0x1p-100f - d->eps) * (float)d->width : 0.f;
  const hipStream_t s = (hipStream_t)stream;
  if (d->type == HV_T_F32) rotary_launch<float>(a, s);
  else if (d->type == HV_T_F16) rotary_launch<f16>(a, s);
  else rotary_launch<bf16>(a, s);
  return check_hip(hipGetLastError(), "k_rotary_qk launch");
}
