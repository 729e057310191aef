// hv_lm_answer.hip -- log probabilities of given tokens, entropy and the most
// probable tokens of rows of logits.
//
//   d = scale (x - max x),  S = sum e^d
//   logp(t) = d_t - log S,   H = log S - sum e^d d / S
//
// The order of the alternatives is that of the logits themselves, equal ones
// by the lower index: a 64-bit key holds the value's ordered bits above the
// complemented index, and no two keys are equal.
#include "hv_lm.h"

namespace hv {

struct AnswerArgs {
  const void *logits;
  const int32_t *tokens;
  float *logp, *entropy, *top_logp;
  int32_t *top_index;
  const int32_t *rows_dev;
  int64_t logits_ld, tokens_ld;
  int rows, width, n_tokens, top;
  float scale;
};

// Unsigned bits in the order of the values; -0 counts as 0, NaN as the largest.
__device__ __forceinline__ unsigned ordered(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const int b = __builtin_bit_cast(int, x + 0.f);
  return (unsigned)(b < 0 ? ~b : b ^ 0x80000000);
}
__device__ __forceinline__ unsigned ordered(int x) { return (unsigned)x ^ 0x80000000u; }

template <typename T>
struct Logit {
  typedef float type;  // what a logit is held in
  static __device__ __forceinline__ float lowest() { return -__builtin_inff(); }
  static __device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
  // scale (x - m); m = -inf: nothing in the row is possible
  static __device__ __forceinline__ float below(float x, float m, float scale) {
    return m == -__builtin_inff() && x == m ? m : (x - m) * scale;
  }
};
template <>
struct Logit<int> {
  typedef int type;
  static __device__ __forceinline__ int lowest() { return INT32_MIN; }
  static __device__ __forceinline__ int larger(int a, int b) { return max(a, b); }
  static __device__ __forceinline__ float below(int x, int m, float scale) {
    return -(float)((unsigned)m - (unsigned)x) * scale;
  }
};

// One workgroup a row, a pass over the row for the maximum, one for the sums
// and one for each alternative.
template <typename T>
__global__ __launch_bounds__(256) void k_log_probs(AnswerArgs a) {
  typedef Logit<T> L;
  typedef typename L::type V;
  const int rows = a.rows_dev ? min(a.rows, *a.rows_dev) : a.rows;
  const int row = blockIdx.x;
  if (row >= rows) return;
  const T *x = (const T *)a.logits + row * a.logits_ld;
  const int tid = threadIdx.x, wave = tid >> 6;
  __shared__ V wave_max[4];
  __shared__ float wave_sum[2][4];
  __shared__ u64 wave_key[4];

  V m = L::lowest();
  for (int c = tid; c < a.width; c += 256) m = L::larger(m, (V)x[c]);
  for (int o = 32; o; o >>= 1) m = L::larger(m, __shfl_xor(m, o));
  if ((tid & 63) == 0) wave_max[wave] = m;
  __syncthreads();
  m = L::larger(L::larger(wave_max[0], wave_max[1]), L::larger(wave_max[2], wave_max[3]));

  float sum = 0.f, weighted = 0.f;
  for (int c = tid; c < a.width; c += 256) {
    const float d = L::below((V)x[c], m, a.scale);
    const float e = __expf(d);
    sum += e;
    weighted += e == 0.f ? 0.f : e * d;
  }
  sum = sum64(sum);
  weighted = sum64(weighted);
  if ((tid & 63) == 0) {
    wave_sum[0][wave] = sum;
    wave_sum[1][wave] = weighted;
  }
  __syncthreads();
  sum = (wave_sum[0][0] + wave_sum[0][1]) + (wave_sum[0][2] + wave_sum[0][3]);
  weighted = (wave_sum[1][0] + wave_sum[1][1]) + (wave_sum[1][2] + wave_sum[1][3]);
  const bool none = sum == 0.f;  // every logit is -inf
  const float log_sum = logf(sum);
  if (tid == 0) a.entropy[row] = none ? 0.f : log_sum - weighted / sum;
  auto logp = [&](int t) {
    return none ? -__builtin_inff() : L::below((V)x[t], m, a.scale) - log_sum;
  };
  for (int i = tid; i < a.n_tokens; i += 256) {
    const int t = a.tokens[row * a.tokens_ld + i];
    a.logp[(size_t)row * a.n_tokens + i] =
        t < 0 ? 0.f : t >= a.width ? __builtin_nanf("") : logp(t);
  }

  u64 last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    u64 best = 0;
    for (int c = tid; c < a.width; c += 256) {
      const u64 key = (u64)ordered((V)x[c]) << 32 | (unsigned)~c;
      if (key < last && key > best) best = key;
    }
    for (int o = 32; o; o >>= 1) {
      const u64 other = __shfl_xor(best, o);
      best = other > best ? other : best;
    }
    __syncthreads();
    if ((tid & 63) == 0) wave_key[wave] = best;
    __syncthreads();
    for (int i = 0; i < 4; ++i) best = wave_key[i] > best ? wave_key[i] : best;
    last = best;
    const int t = (int)~(unsigned)best;
    if (tid == 0) {
      a.top_index[(size_t)row * a.top + k] = t;
      a.top_logp[(size_t)row * a.top + k] = logp(t);
    }
  }
}

}  // namespace hv

using namespace hv;

extern "C" {

size_t hv_log_probs_workspace_bytes(int rows, int width, int top) {
  (void)rows; (void)width; (void)top;
  return 0;
}

int hv_log_probs(const hv_log_probs_desc *d, void *workspace, size_t workspace_bytes,
                 hv_stream_t stream) {
  (void)workspace; (void)workspace_bytes;
  clear_error();
  if (!d) return fail(HV_EVALUE, HV_ERR_ADDRESS, "log_probs: null descriptor");
  if (d->type < HV_T_F32 || d->type > HV_T_I32)
    return fail(HV_EVALUE, HV_ERR_OPCODE, "log_probs: bad element type %d", d->type);
  if (d->rows < 0 || d->width < 1 || d->n_tokens < 0 || d->logits_ld < d->width ||
      (d->n_tokens && d->tokens_ld < d->n_tokens))
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "log_probs: %d rows of %d logits, %d tokens each",
                d->rows, d->width, d->n_tokens);
  if (d->top < 0 || d->top > HV_LOG_PROBS_MAX_TOP || d->top > d->width)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "log_probs: top %d outside [0, %d] or over the width",
                d->top, HV_LOG_PROBS_MAX_TOP);
  if (!(d->scale > 0.f) || d->scale > 3e38f)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "log_probs: the scale must be positive and finite");
  if (d->rows == 0) return HV_OK;
  if (!d->logits || !d->entropy || (d->n_tokens && (!d->tokens || !d->logp)) ||
      (d->top && (!d->top_logp || !d->top_index)))
    return fail(HV_EVALUE, HV_ERR_ADDRESS, "log_probs: null argument");
  const int size = d->type == HV_T_F32 || d->type == HV_T_I32 ? 4 : 2;
  if (((uintptr_t)d->logits & (size - 1)) ||
      (((uintptr_t)d->tokens | (uintptr_t)d->logp | (uintptr_t)d->entropy |
        (uintptr_t)d->top_logp | (uintptr_t)d->top_index) & 3))
    return fail(HV_EVALUE, HV_ERR_ADDRESS, "log_probs: a pointer is not aligned to its elements");
  AnswerArgs a{};
  a.logits = d->logits; a.tokens = d->tokens; a.logp = d->logp; a.entropy = d->entropy;
  a.top_logp = d->top_logp; a.top_index = d->top_index; a.rows_dev = d->rows_dev;
  a.logits_ld = d->logits_ld; a.tokens_ld = d->tokens_ld;
  a.rows = d->rows; a.width = d->width; a.n_tokens = d->n_tokens; a.top = d->top;
  a.scale = d->scale;
  const hipStream_t s = (hipStream_t)stream;
  const dim3 grid(a.rows), block(256);
  if (d->type == HV_T_F32) hv_launch(k_log_probs<float>, grid, block, 0, s, a);
  else if (d->type == HV_T_F16) hv_launch(k_log_probs<f16>, grid, block, 0, s, a);
  else if (d->type == HV_T_BF16) hv_launch(k_log_probs<bf16>, grid, block, 0, s, a);
  else hv_launch(k_log_probs<int>, grid, block, 0, s, a);
  return check_hip(hipGetLastError(), "k_log_probs launch");
}

}  // extern "C"
