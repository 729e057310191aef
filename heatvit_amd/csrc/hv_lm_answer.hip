// hv_lm_answer.hip -- log probabilities of given tokens, entropy and the most
// probable tokens of rows of logits.
//
//   d = scale (x - max x),  S = sum e^d
//   logp(t) = d_t - log S,   H = log S - sum e^d d / S
//
// The order of the alternatives is that of the logits themselves, equal ones
// by the lower index: a 64-bit key holds the value's ordered bits above the
// complemented index, and no two keys are equal.
#include <type_traits>

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
  // Rows cut into parts (parts > 1): each leaves its sums and its `top`
  // largest keys for the second kernel.
  int parts, part_width;
  struct AnswerPart *part;  // [rows][parts]
  unsigned long long *keys;  // [rows][parts][top]
};
struct AnswerPart {
  int max;  // the bits of the type the logit is held in
  float sum, weighted;
};

// Unsigned bits in the order of the values; -0 counts as 0, NaN as the largest.
__device__ __forceinline__ unsigned ordered(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const int b = __builtin_bit_cast(int, x + 0.f);
  return (unsigned)(b < 0 ? ~b : b ^ 0x80000000);
}
__device__ __forceinline__ unsigned ordered(int x) { return (unsigned)x ^ 0x80000000u; }
template <typename V>
__device__ __forceinline__ u64 key_of(V x, int at) {
  return (u64)ordered(x) << 32 | (unsigned)~at;
}
// The value of a key (of a real one, or of 0: the lowest).
__device__ __forceinline__ void key_value(u64 k, float &x) {
  const unsigned u = (unsigned)(k >> 32);
  x = k ? __builtin_bit_cast(float, u & 0x80000000u ? u ^ 0x80000000u : ~u) : -__builtin_inff();
}
__device__ __forceinline__ void key_value(u64 k, int &x) {
  x = (int)((unsigned)(k >> 32) ^ 0x80000000u);
}

template <typename T>
struct Logit {
  typedef float type;  // what a logit is held in
  // below every finite logit's place in a sum, and finite
  static __device__ __forceinline__ float lowest() { return -3.402823466e38f; }
  static __device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
  static __device__ __forceinline__ float below(float x, float m) { return x - m; }
};
template <>
struct Logit<int> {
  typedef int type;
  static __device__ __forceinline__ int lowest() { return INT32_MIN; }
  static __device__ __forceinline__ int larger(int a, int b) { return max(a, b); }
  static __device__ __forceinline__ float below(int x, int m) {
    return -(float)((unsigned)m - (unsigned)x);
  }
};

// Sum of 2^d and of 2^d d over logits, d = c (x - max), c = scale log2(e),
// and the maximum they are relative to.
template <typename T>
struct Sums {
  typedef Logit<T> L;
  typename L::type max = L::lowest();
  float sum = 0.f, weighted = 0.f;

  // Relative to a larger maximum. The factor's exponent is kept finite: with
  // it, what has no weight stays 0.
  __device__ __forceinline__ void raise(typename L::type m, float c) {
    const float d = fmaxf(L::below(max, m) * c, -1e30f);
    const float f = __builtin_amdgcn_exp2f(d);
    weighted = f * __builtin_fmaf(sum, d, weighted);
    sum *= f;
    max = m;
  }
  // d of a logit at or below the maximum; -inf and far ones weigh nothing, a
  // NaN stays one.
  __device__ __forceinline__ void add(typename L::type x, float c, bool there) {
    const float d = there ? L::below(x, max) * c : 0.f;
    const float e = there ? __builtin_amdgcn_exp2f(d) : 0.f;
    sum += e;
    weighted = __builtin_fmaf(e, fmaxf(d, -200.f), weighted);
  }
  __device__ __forceinline__ void join(const Sums &o, float c) {
    const typename L::type m = L::larger(max, o.max);
    Sums t = o;
    t.raise(m, c);
    raise(m, c);
    sum += t.sum;
    weighted += t.weighted;
  }
  __device__ __forceinline__ void join_lanes(float c) {
#pragma unroll
    for (int o = 32; o; o >>= 1) {
      Sums t;
      t.max = __shfl_xor(max, o);
      t.sum = __shfl_xor(sum, o);
      t.weighted = __shfl_xor(weighted, o);
      join(t, c);
    }
  }
};

static constexpr int kAnswerWaves = 4;
static constexpr int kMaxParts = 64;
static constexpr int kKeep = 192;  // candidates a wavefront holds

// The smallest power of two that is at least n.
__device__ __forceinline__ int pow2_from(int n) {
  return n <= 1 ? 1 : 1 << (32 - __builtin_clz(n - 1));
}

// A lower bound on the `top`-th largest of all keys, from a key of each lane,
// its own largest: lanes fall into at least `top` classes (lane mod classes),
// whose largest keys are that many different keys, the least of which bounds.
// 0 where a class has none.
__device__ __forceinline__ u64 bound_of_lanes(u64 key, int classes) {
  for (int o = 32; o; o >>= 1) {
    const u64 other = __shfl_xor(key, o);
    if (o >= classes) key = other > key ? other : key;
    else key = other < key ? other : key;
  }
  return key;
}

__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

typedef __attribute__((address_space(3))) u64 lds_u64;

// Cuts a wavefront's list of count <= kKeep keys down to its `top` largest, in
// order: a key's place is the number of larger ones. Returns the last one's
// key, 0 if there are fewer.
static __device__ __noinline__ u64 cut_list(lds_u64 *list, int count, int top) {
  const int lane = threadIdx.x & 63;
  wave_lds_fence();
  u64 mine[kKeep / 64];
  int place[kKeep / 64] = {};
#pragma unroll
  for (int i = 0; i < kKeep / 64; ++i) mine[i] = i * 64 + lane < count ? list[i * 64 + lane] : 0;
  for (int j = 0; j < count; ++j) {
    const u64 other = list[j];
#pragma unroll
    for (int i = 0; i < kKeep / 64; ++i) place[i] += other > mine[i];
  }
  wave_lds_fence();
#pragma unroll
  for (int i = 0; i < kKeep / 64; ++i)
    if (mine[i] && place[i] < top) list[place[i]] = mine[i];
  wave_lds_fence();
  return count >= top ? list[top - 1] : 0;
}

// A wavefront's candidates for the `top` largest keys: all its keys that are
// not under a bound, which rises whenever kKeep is nearly full and the list is
// cut down to `top`.
template <typename V>
struct Candidates {
  lds_u64 *list;  // kKeep
  int count, top;
  u64 bound;  // no key under it is wanted
  V value;    // its value

  __device__ __forceinline__ void set_bound(u64 b) {
    bound = b;
    key_value(b, value);
  }
  // Each lane's key where `there`, all lanes together.
  __device__ __forceinline__ void push(u64 key, bool there) {
    const bool in = there && key >= bound;
    const u64 who = __ballot(in);
    if (!who) return;
    if (in) list[count + __builtin_amdgcn_mbcnt_hi((unsigned)(who >> 32),
                                                   __builtin_amdgcn_mbcnt_lo((unsigned)who, 0))] = key;
    count += __popcll(who);
    if (count > kKeep - 64) {
      const u64 b = cut_list(list, count, top);
      if (b) set_bound(b);
      count = min(count, top);
    }
  }
};

// The `top` largest of n different keys, in order, into `out`, by a whole
// workgroup: a bound as above over its threads' largest, then the places of
// those that are not under it. `left` holds n keys.
__device__ void largest_keys(const u64 *keys, int n, int top, u64 *left, u64 *out) {
  __shared__ u64 wave_bound[kAnswerWaves];
  __shared__ int n_left;
  const int tid = threadIdx.x;
  u64 best = 0;
  for (int i = tid; i < n; i += 64 * kAnswerWaves) best = keys[i] > best ? keys[i] : best;
  const int classes = max(1, pow2_from(top) / kAnswerWaves);
  best = bound_of_lanes(best, classes);
  if ((tid & 63) == 0) wave_bound[tid >> 6] = best;
  if (tid == 0) n_left = 0;
  __syncthreads();
  for (int w = 0; w < kAnswerWaves; ++w) best = wave_bound[w] < best ? wave_bound[w] : best;
  best = best ? best : 1;  // 0 is no key
  for (int i = tid; i < n; i += 64 * kAnswerWaves)
    if (keys[i] >= best) left[atomicAdd(&n_left, 1)] = keys[i];
  __syncthreads();
  const int m = n_left;
  for (int i = tid; i < m; i += 64 * kAnswerWaves) {
    const u64 mine = left[i];
    int place = 0;
    for (int j = 0; j < m; ++j) place += left[j] > mine;
    if (place < top) out[place] = mine;
  }
  __syncthreads();
}

// The same by `top` passes over the row, for a row with a NaN or +inf in it.
template <typename T>
__device__ void largest_keys_slow(const T *x, int width, int top, u64 *out) {
  typedef typename Logit<T>::type V;
  __shared__ u64 wave_key[kAnswerWaves];
  u64 last = ~0ull;
  for (int k = 0; k < top; ++k) {
    u64 best = 0;
    for (int c = threadIdx.x; c < width; c += 64 * kAnswerWaves) {
      const u64 key = key_of((V)x[c], c);
      if (key < last && key > best) best = key;
    }
    for (int o = 32; o; o >>= 1) {
      const u64 other = __shfl_xor(best, o);
      best = other > best ? other : best;
    }
    if ((threadIdx.x & 63) == 0) wave_key[threadIdx.x >> 6] = best;
    __syncthreads();
    for (int i = 0; i < kAnswerWaves; ++i) best = wave_key[i] > best ? wave_key[i] : best;
    last = best;
    if (threadIdx.x == 0) out[k] = best;
    __syncthreads();
  }
}

// What a row gives, from its sums and its largest keys (LDS).
template <typename T>
__device__ void write_answer(const AnswerArgs &a, int64_t row, const T *x, const Sums<T> &s,
                             const u64 *best, bool slow_done) {
  typedef Logit<T> L;
  typedef typename L::type V;
  constexpr float kLn2 = 0.69314718056f;
  const int tid = threadIdx.x;
  const bool none = s.sum == 0.f;  // every logit is -inf
  const float log2_sum = log2f(s.sum), log_sum = log2_sum * kLn2;
  if (tid == 0) a.entropy[row] = none ? 0.f : (log2_sum - s.weighted / s.sum) * kLn2;
  auto logp = [&](V v) {
    return none ? -__builtin_inff() : L::below(v, s.max) * a.scale - log_sum;
  };
  for (int i = tid; i < a.n_tokens; i += 64 * kAnswerWaves) {
    const int t = a.tokens[row * a.tokens_ld + i];
    a.logp[row * a.n_tokens + i] =
        t < 0 ? 0.f : t >= a.width ? __builtin_nanf("") : logp((V)x[t]);
  }
  for (int i = tid; i < a.top; i += 64 * kAnswerWaves) {
    const int t = (int)~(unsigned)best[i];
    a.top_index[row * a.top + i] = t;
    a.top_logp[row * a.top + i] = logp((V)x[t]);
  }
}

// One workgroup a row or a part of one, in one pass: each lane keeps a running
// maximum with its sums, each wavefront the candidates for the alternatives.
template <typename T, bool TOP>
__global__ __launch_bounds__(64 * kAnswerWaves) void k_log_probs(AnswerArgs a) {
  typedef Logit<T> L;
  typedef typename L::type V;
  constexpr int E = 16 / sizeof(T), U = 4;  // logits a load, loads in a turn
  typedef T vt __attribute__((ext_vector_type(E)));
  const int rows = a.rows_dev ? min(a.rows, *a.rows_dev) : a.rows;
  const int64_t row = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  if (row >= rows) return;
  const T *x = (const T *)a.logits + row * a.logits_ld;
  const float c = a.scale * 1.44269504089f;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __shared__ u64 list[TOP ? kAnswerWaves * kKeep : 1];
  __shared__ u64 left[TOP ? kAnswerWaves * kKeep : 1];
  __shared__ u64 best[TOP ? HV_LOG_PROBS_MAX_TOP : 1];
  __shared__ V wave_max[kAnswerWaves];
  __shared__ float wave_sum[2][kAnswerWaves];
  __shared__ int n_list;

  // [lo, hi): whole loads of 16 bytes from `first` on, n of them, and up to
  // E - 1 logits on either side.
  const int lo = part * a.part_width, hi = min(a.width, lo + a.part_width);
  const int first = min(hi, lo + (int)((16 - ((uintptr_t)(x + lo) & 15)) % 16 / sizeof(T)));
  const int n = (hi - first) / E;
  const vt *xv = reinterpret_cast<const vt *>(x + first);

  Sums<T> s;
  Candidates<V> cand;
  if (TOP) {
    cand.list = (lds_u64 *)(list + wave * kKeep);
    cand.count = 0;
    cand.top = a.top;
    cand.set_bound(0);
  }
  bool begun = false;  // a bound from this wavefront's first turn
  constexpr int kTurn = 64 * kAnswerWaves * U;  // a turn's loads, the workgroup's
  const int mine_at = wave * 64 + lane;
  auto number = [&](int at, int u) { return at + u * 64 * kAnswerWaves + mine_at; };
  auto turn = [&](const vt (&v)[U], int at, auto whole) {
    // whole: all of the turn's loads are there
    constexpr bool kWhole = decltype(whole)::value;
    V high[U], m = s.max;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool there = kWhole || number(at, u) < n;
      high[u] = L::lowest();
#pragma unroll
      for (int i = 0; i < E; ++i) high[u] = L::larger(high[u], (V)v[u][i]);
      if (!there) high[u] = L::lowest();
      m = L::larger(m, high[u]);
    }
    s.raise(m, c);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool there = kWhole || number(at, u) < n;
#pragma unroll
      for (int i = 0; i < E; ++i) s.add((V)v[u][i], c, there);
    }
    if (!TOP) return;
    if (!begun) {
      begun = true;
      u64 mine = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool there = kWhole || number(at, u) < n;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const u64 key = key_of((V)v[u][i], first + number(at, u) * E + i);
          if (there && key > mine) mine = key;
        }
      }
      cand.set_bound(bound_of_lanes(mine, pow2_from(a.top)));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool there = kWhole || number(at, u) < n;
      if (!__ballot(there && high[u] >= cand.value)) continue;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (!__ballot(there && (V)v[u][i] >= cand.value)) continue;
        cand.push(key_of((V)v[u][i], first + number(at, u) * E + i), there);
      }
    }
  };
  auto fetch = [&](vt (&v)[U], int at) {
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = xv[min(number(at, u), n - 1)];
  };
  if (n > 0) {
    // the next turn's loads are on their way while one is added up
    vt now[U], next[U];
    fetch(now, 0);
    for (int at = 0; at < n; at += kTurn) {
      fetch(next, at + kTurn);
      if (at + kTurn <= n) turn(now, at, std::true_type());
      else turn(now, at, std::false_type());
#pragma unroll
      for (int u = 0; u < U; ++u) now[u] = next[u];
    }
  }
  if (wave == 0) {
    // the logits on either side of the loads, at most one a lane
    const int tail = first + n * E, before = first - lo;
    const int at = lane < before ? lo + lane : tail + lane - before;
    const bool there = at < hi;
    const V v = there ? (V)x[at] : L::lowest();
    s.raise(L::larger(s.max, v), c);
    s.add(v, c, there);
    if (TOP) cand.push(key_of(v, at), there);
  }

  s.join_lanes(c);
  if (lane == 0) {
    wave_max[wave] = s.max;
    wave_sum[0][wave] = s.sum;
    wave_sum[1][wave] = s.weighted;
  }
  if (TOP && tid == 0) n_list = 0;
  __syncthreads();
  for (int w = 1; w < kAnswerWaves; ++w) {
    Sums<T> t;
    t.max = wave_max[w];
    t.sum = wave_sum[0][w];
    t.weighted = wave_sum[1][w];
    Sums<T> mine;
    mine.max = wave_max[0];
    mine.sum = wave_sum[0][0];
    mine.weighted = wave_sum[1][0];
    if (w == 1) s = mine;
    s.join(t, c);
  }
  const bool odd = s.sum != s.sum;
  if (TOP) {
    // the wavefronts' lists one behind the other
    int total = 0;
    if (!odd || a.parts > 1) {
      int at = 0;
      if (lane == 0) at = atomicAdd(&n_list, cand.count);
      at = __shfl(at, 0);
      for (int i = lane; i < cand.count; i += 64) left[at + i] = cand.list[i];
      __syncthreads();
      total = n_list;
      if (tid < a.top) best[tid] = 0;
      __syncthreads();
      largest_keys(left, total, a.top, list, best);
    } else {
      __syncthreads();
      largest_keys_slow<T>(x, a.width, a.top, best);
    }
  }
  if (a.parts == 1) return write_answer<T>(a, row, x, s, best, odd);
  const int64_t p = row * a.parts + part;
  if (tid == 0) a.part[p] = {__builtin_bit_cast(int, s.max), s.sum, s.weighted};
  if (TOP && tid < a.top) a.keys[p * a.top + tid] = best[tid];
}

// Joins the parts of a row.
template <typename T, bool TOP>
__global__ __launch_bounds__(64 * kAnswerWaves) void k_log_probs_join(AnswerArgs a) {
  typedef typename Logit<T>::type V;
  const int rows = a.rows_dev ? min(a.rows, *a.rows_dev) : a.rows;
  const int64_t row = blockIdx.x;
  if (row >= rows) return;
  const T *x = (const T *)a.logits + row * a.logits_ld;
  __shared__ u64 left[TOP ? kMaxParts * HV_LOG_PROBS_MAX_TOP : 1];
  __shared__ u64 best[TOP ? HV_LOG_PROBS_MAX_TOP : 1];
  const int lane = threadIdx.x & 63;
  Sums<T> s;
  if (lane < a.parts) {
    const AnswerPart p = a.part[row * a.parts + lane];
    s.max = __builtin_bit_cast(V, p.max);
    s.sum = p.sum;
    s.weighted = p.weighted;
  }
  s.join_lanes(a.scale * 1.44269504089f);
  if (TOP) {
    if (s.sum != s.sum) largest_keys_slow<T>(x, a.width, a.top, best);
    else largest_keys(a.keys + row * a.parts * a.top, a.parts * a.top, a.top, left, best);
  }
  write_answer<T>(a, row, x, s, best, false);
}

// Parts of a row. A row is read by one workgroup where there are rows enough
// to keep the card busy; fewer rows are cut until kAnswerGroups workgroups
// are at work, in parts of at least kMinPart logits.
static constexpr int kAnswerGroups = 512, kMinPart = 4096;
static int answer_parts(int rows, int width, int *part_width) {
  int parts = (int)((kAnswerGroups + (int64_t)rows - 1) / (rows > 0 ? rows : 1));
  parts = parts < width / kMinPart ? parts : width / kMinPart;
  parts = parts < 1 ? 1 : parts > kMaxParts ? kMaxParts : parts;
  const int64_t w = ((int64_t)width + parts - 1) / parts;
  *part_width = parts == 1 ? width : (int)((w + 63) / 64 * 64);
  return parts == 1 ? 1 : (width + *part_width - 1) / *part_width;
}

template <typename T, bool TOP>
static void answer_launch(const AnswerArgs &a, hipStream_t s) {
  hv_launch(k_log_probs<T, TOP>, dim3((unsigned)((int64_t)a.rows * a.parts)),
            dim3(64 * kAnswerWaves), 0, s, a);
  if (a.parts > 1)
    hv_launch(k_log_probs_join<T, TOP>, dim3(a.rows), dim3(64 * kAnswerWaves), 0, s, a);
}
template <typename T>
static void answer_launch(const AnswerArgs &a, hipStream_t s) {
  if (a.top) answer_launch<T, true>(a, s);
  else answer_launch<T, false>(a, s);
}

}  // namespace hv

using namespace hv;

extern "C" {

size_t hv_log_probs_workspace_bytes(int rows, int width, int top) {
  if (rows <= 0 || width <= 0 || top < 0) return 0;
  int part_width;
  const size_t parts = answer_parts(rows, width, &part_width);
  if (parts == 1) return 0;
  return (size_t)rows * parts * (top * sizeof(u64) + sizeof(AnswerPart)) + 8;
}

int hv_log_probs(const hv_log_probs_desc *d, void *workspace, size_t workspace_bytes,
                 hv_stream_t stream) {
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
  if (!(d->scale > 0.f) || d->scale > 1e30f)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "log_probs: the scale is not in (0, 1e30]");
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
  a.parts = answer_parts(a.rows, a.width, &a.part_width);
  if (a.parts > 1) {
    if (!workspace || ((uintptr_t)workspace & 7) ||
        workspace_bytes < hv_log_probs_workspace_bytes(a.rows, a.width, a.top))
      return fail(HV_EVALUE, HV_ERR_ADDRESS, "log_probs: workspace too small or not 8-byte aligned");
    a.keys = (unsigned long long *)workspace;
    a.part = (AnswerPart *)(a.keys + (size_t)a.rows * a.parts * a.top);
  }
  const hipStream_t s = (hipStream_t)stream;
  if (d->type == HV_T_F32) answer_launch<float>(a, s);
  else if (d->type == HV_T_F16) answer_launch<f16>(a, s);
  else if (d->type == HV_T_BF16) answer_launch<bf16>(a, s);
  else answer_launch<int>(a, s);
  return check_hip(hipGetLastError(), "k_log_probs launch");
}

}  // extern "C"
