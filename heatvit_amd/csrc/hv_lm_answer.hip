// hv_lm_answer.hip -- log probabilities of given tokens, entropy and the most
// probable tokens of rows of logits.
//
//   d = scale (x - max x),  S = sum e^d
//   logp(t) = d_t - log S,   H = log S - sum e^d d / S
//
// The order of the alternatives is that of the logits themselves, equal ones
// by the lower index: a 64-bit key holds the value's ordered bits above the
// complemented index, and no two keys are equal.
//
// The logits' bytes bound it: 2048 rows of 131072 bf16 logits with five
// alternatives take 106 us, which is the rate of a large copy (4.9 TB/s); passes
// for the maximum, the sums and each alternative apart took 1984. One row of
// 131072 with 20 takes 7.1 and 4.3 us in its two kernels, 256 rows of 1000 int32
// logits with five 6.5.
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
  // x - m in halves: the type's largest and lowest numbers lie twice the largest
  // float apart.
  static constexpr float kUnit = 2.f;
  static __device__ __forceinline__ float below(float x, float m) {
    return __builtin_fmaf(x, .5f, -.5f * m);
  }
};
template <>
struct Logit<int> {
  typedef int type;
  static __device__ __forceinline__ int lowest() { return INT32_MIN; }
  static __device__ __forceinline__ int larger(int a, int b) { return max(a, b); }
  static constexpr float kUnit = 1.f;
  static __device__ __forceinline__ float below(int x, int m) {
    return -(float)((unsigned)m - (unsigned)x);
  }
};

// The largest of the wavefront's, all lanes active.
template <typename T>
__device__ __forceinline__ typename Logit<T>::type wave_max(typename Logit<T>::type v) {
  typedef Logit<T> L;
  typedef typename L::type V;
  v = L::larger(v, ror16<8>(v));
  v = L::larger(v, ror16<4>(v));
  v = L::larger(v, ror16<2>(v));
  v = L::larger(v, ror16<1>(v));
  const int bits = __builtin_bit_cast(int, v);
  auto of = [&](int lane) {
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(bits, lane));
  };
  return L::larger(L::larger(of(0), of(16)), L::larger(of(32), of(48)));
}

// What makes a below() an exponent of 2: scale log2(e), in its units.
template <typename T>
__device__ __forceinline__ float factor_of(const AnswerArgs &a) {
  return a.scale * (1.44269504089f * Logit<T>::kUnit);
}

// Sum of 2^d and of 2^d d over logits, d = c below(x, max), and the maximum
// they are relative to.
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
  // The wavefront's, in every lane.
  __device__ __forceinline__ void join_lanes(float c) {
    raise(wave_max<T>(max), c);
    sum = sum64(sum);
    weighted = sum64(weighted);
  }
};

static constexpr int kAnswerWaves = 4;
static constexpr int kMaxParts = 64;
static constexpr int kThreads = 64 * kAnswerWaves;
static constexpr int kSlots = 8;       // maxima that a thread keeps of its logits
static constexpr int kKeep = 1024;     // candidates for the alternatives

// The `top` largest of m different keys, in order: a key's place is the number
// of larger ones.
__device__ __forceinline__ void rank_keys(const u64 *keys, int m, int top, u64 *out) {
  for (int i = threadIdx.x; i < m; i += kThreads) {
    const u64 mine = keys[i];
    int place = 0, j = 0;
    for (; j + 8 <= m; j += 8) {
      u64 other[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) other[k] = keys[j + k];
#pragma unroll
      for (int k = 0; k < 8; ++k) place += other[k] > mine;
    }
    for (; j < m; ++j) place += keys[j] > mine;
    if (place < top) out[place] = mine;
  }
}

// A lower bound on the `top`-th largest of a workgroup's values, from each
// thread's largest: the `top`-th largest of 64 groups' maxima (threads of one
// lane), which takes 64 comparisons and, while `top` is well below 64, lets few
// more logits through; of all threads' for a larger one (64 groups and all
// threads: 1 row of 131072 with 9 alternatives 9.7, 11.4 us, with 32 11.4, 13.3,
// with 50 14.7, 14.6, with 64 40.2, 16.1; 2048 rows with 32 113.9, 114.1, with 50
// 125.0, 117.8).
static constexpr int kGroupsTop = 32;
template <typename T>
__device__ typename Logit<T>::type bound_of(typename Logit<T>::type best, int top) {
  typedef Logit<T> L;
  typedef typename L::type V;
  __shared__ V of_thread[kThreads];
  const int tid = threadIdx.x, lane = tid & 63;
  of_thread[tid] = best;
  __syncthreads();
  int reach = 0;  // maxima that reach this one
  if (top <= kGroupsTop) {
#pragma unroll
    for (int w = 0; w < kAnswerWaves; ++w) best = L::larger(best, of_thread[w * 64 + lane]);
    if (top == 1) return wave_max<T>(best);
    const int bits = __builtin_bit_cast(int, best);
#pragma unroll 16
    for (int i = 0; i < 64; ++i)
      reach += __builtin_bit_cast(V, __builtin_amdgcn_readlane(bits, i)) >= best;
    return wave_max<T>(reach >= top ? best : L::lowest());
  }
#pragma unroll 16
  for (int i = 0; i < kThreads; ++i) reach += of_thread[i] >= best;
  V least = wave_max<T>(reach >= top ? best : L::lowest());
  __syncthreads();
  if (lane == 0) of_thread[tid >> 6] = least;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kAnswerWaves; ++w) least = L::larger(least, of_thread[w]);
  return least;
}

// The `top` largest keys of logits [lo, hi) by as many passes over them, for a
// row with a NaN or +inf in it, or with more than kKeep logits that reach the
// bound, which takes equal ones (2048 rows of 131072 equal logits: 0.68 ms for
// the largest, 2.3 for five, 8.3 for 20).
template <typename T>
__device__ void largest_keys_slow(const T *x, int lo, int hi, int top, u64 *out) {
  typedef typename Logit<T>::type V;
  __shared__ u64 wave_key[kAnswerWaves];
  u64 last = 0;
  for (int k = 0; k < top; ++k) {
    u64 best = 0;
    for (int c = lo + threadIdx.x; c < hi; c += kThreads) {
      const u64 key = key_of((V)x[c], c);
      if ((k == 0 || key < last) && key > best) best = key;
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

// The logit of the thread's first given token, asked for before it is needed.
template <typename T>
struct Given {
  int token = -1;
  typename Logit<T>::type logit = 0;
  __device__ __forceinline__ Given(const AnswerArgs &a, int64_t row, const T *x) {
    if ((int)threadIdx.x < a.n_tokens) {
      token = a.tokens[row * a.tokens_ld + threadIdx.x];
      if (token >= 0 && token < a.width) logit = (typename Logit<T>::type)x[token];
    }
  }
};

// What a row gives, from its sums and its largest keys (LDS).
template <typename T>
__device__ void write_answer(const AnswerArgs &a, int64_t row, const T *x, const Sums<T> &s,
                             const u64 *best, const Given<T> &given) {
  typedef Logit<T> L;
  typedef typename L::type V;
  constexpr float kLn2 = 0.69314718056f;
  const int tid = threadIdx.x;
  const bool none = s.sum == 0.f;  // every logit is -inf
  const float log2_sum = log2f(s.sum), log_sum = log2_sum * kLn2;
  if (tid == 0) a.entropy[row] = none ? 0.f : (log2_sum - s.weighted / s.sum) * kLn2;
  auto logp = [&](V v) {
    return none ? -__builtin_inff() : L::below(v, s.max) * (a.scale * L::kUnit) - log_sum;
  };
  for (int i = tid; i < a.n_tokens; i += kThreads) {
    const int t = i == tid ? given.token : a.tokens[row * a.tokens_ld + i];
    const V v = i == tid ? given.logit : t >= 0 && t < a.width ? (V)x[t] : V(0);
    a.logp[row * a.n_tokens + i] = t < 0 ? 0.f : t >= a.width ? __builtin_nanf("") : logp(v);
  }
  for (int i = tid; i < a.top; i += kThreads) {
    V v;
    key_value(best[i], v);
    a.top_index[row * a.top + i] = (int)~(unsigned)best[i];
    a.top_logp[row * a.top + i] = logp(v);
  }
}

// One workgroup a row or a part of one, in one pass: each thread keeps a running
// maximum with its sums, and for the alternatives the maxima of up to kSlots
// stretches of its logits. These give a bound that the `top` largest logits are
// not under, and only the few stretches that reach it are read again (2048 x
// 131072: 106 us with five, 96 without; a list of candidates kept up with a
// rising bound in the pass itself took 145).
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) void k_log_probs(AnswerArgs a) {
  typedef Logit<T> L;
  typedef typename L::type V;
  constexpr int E = 16 / sizeof(T), U = 4;  // logits a load, loads in a turn
  typedef T vt __attribute__((ext_vector_type(E)));
  const int rows = a.rows_dev ? min(a.rows, *a.rows_dev) : a.rows;
  const int64_t row = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  if (row >= rows) return;
  const T *x = (const T *)a.logits + row * a.logits_ld;
  const float c = factor_of<T>(a);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __shared__ V slots[TOP ? kSlots * kThreads : 1];
  __shared__ u64 keys[TOP ? kKeep : 1];
  __shared__ u64 best[TOP ? HV_LOG_PROBS_MAX_TOP : 1];
  __shared__ uint16_t hits[TOP ? kSlots * kThreads : 1];
  __shared__ int n_keys, n_hits;
  __shared__ V of_wave[kAnswerWaves];
  __shared__ float wave_sum[2][kAnswerWaves];

  const Given<T> given(a.parts == 1 ? a : AnswerArgs{}, row, x);
  // [lo, hi): whole loads of 16 bytes from `first` on, n of them, and up to
  // E - 1 logits on either side.
  const int lo = part * a.part_width, hi = min(a.width, lo + a.part_width);
  const int first = min(hi, lo + (int)((16 - ((uintptr_t)(x + lo) & 15)) % 16 / sizeof(T)));
  const int n = (hi - first) / E;
  const vt *xv = reinterpret_cast<const vt *>(x + first);
  constexpr int kTurn = kThreads * U;  // a turn's loads
  const int turns = (n + kTurn - 1) / kTurn, each = (turns + kSlots - 1) / kSlots;  // turns a slot
  auto number = [&](int at, int u) { return at + u * kThreads + tid; };

  Sums<T> s;
  V high = L::lowest(), highest = L::lowest();  // this slot's, and all
  auto turn = [&](const vt (&v)[U], int at, auto whole) {
    // whole: all of the turn's loads are there
    constexpr bool kWhole = decltype(whole)::value;
    V m = L::lowest();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      V h = L::lowest();
#pragma unroll
      for (int i = 0; i < E; ++i) h = L::larger(h, (V)v[u][i]);
      m = kWhole || number(at, u) < n ? L::larger(m, h) : m;
    }
    high = L::larger(high, m);
    s.raise(L::larger(s.max, m), c);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool there = kWhole || number(at, u) < n;
#pragma unroll
      for (int i = 0; i < E; ++i) s.add((V)v[u][i], c, there);
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
    int slot = 0, left = each;
    for (int at = 0; at < n; at += kTurn) {
      fetch(next, at + kTurn);
      if (at + kTurn <= n) turn(now, at, std::true_type());
      else turn(now, at, std::false_type());
      if (TOP && (--left == 0 || at + kTurn >= n)) {
        slots[slot++ * kThreads + tid] = high;
        highest = L::larger(highest, high);
        high = L::lowest();
        left = each;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) now[u] = next[u];
    }
  }
  // the logits on either side of the loads, at most one a lane
  const int tail = first + n * E, before = first - lo;
  const int edge = lane < before ? lo + lane : tail + lane - before;
  const bool has_edge = wave == 0 && edge < hi;
  const V at_edge = has_edge ? (V)x[edge] : L::lowest();
  if (wave == 0) {
    s.raise(L::larger(s.max, at_edge), c);
    s.add(at_edge, c, has_edge);
    highest = L::larger(highest, at_edge);
  }

  s.join_lanes(c);
  if (lane == 0) {
    of_wave[wave] = s.max;
    wave_sum[0][wave] = s.sum;
    wave_sum[1][wave] = s.weighted;
  }
  if (TOP && tid == 0) n_keys = n_hits = 0;
  V bound = L::lowest();
  if (TOP) bound = bound_of<T>(highest, a.top);  // with a barrier
  else __syncthreads();
  V m = of_wave[0];
#pragma unroll
  for (int w = 1; w < kAnswerWaves; ++w) m = L::larger(m, of_wave[w]);
  s = Sums<T>();
  s.max = m;
#pragma unroll
  for (int w = 0; w < kAnswerWaves; ++w) {
    Sums<T> t;
    t.max = of_wave[w];
    t.sum = wave_sum[0][w];
    t.weighted = wave_sum[1][w];
    t.raise(m, c);
    s.sum += t.sum;
    s.weighted += t.weighted;
  }
  if (TOP) {
    auto keep = [&](V v, int at) {
      const int to = atomicAdd(&n_keys, 1);
      if (to < kKeep) keys[to] = key_of(v, at);
    };
    for (int slot = 0; slot * each < turns; ++slot)
      if (slots[slot * kThreads + tid] >= bound)
        hits[atomicAdd(&n_hits, 1)] = (uint16_t)(slot * kThreads + tid);
    __syncthreads();
    // a load of a stretch that reaches the bound for each thread
    const int loads = U * each, all = n_hits * loads;
    for (int i = tid; i < all; i += kThreads) {
      const int hit = hits[i / loads], of = i % loads;
      const int at = (hit / kThreads * each + of / U) * kTurn + of % U * kThreads + hit % kThreads;
      if (at >= n) continue;
      const vt v = xv[at];
#pragma unroll
      for (int k = 0; k < E; ++k)
        if ((V)v[k] >= bound) keep((V)v[k], first + at * E + k);
    }
    if (has_edge && at_edge >= bound) keep(at_edge, edge);
    // Fewer than `top` finite logits: -inf ones follow, by their index. The
    // first 2 top logits hold enough of them.
    if (bound <= L::lowest() && tid < 2 * a.top && lo + tid < hi) {
      const V v = (V)x[lo + tid];
      if (v < L::lowest()) keep(v, lo + tid);
    }
    if (tid < a.top) best[tid] = 0;
    __syncthreads();
    const int m = n_keys;
    if (m > kKeep || s.sum != s.sum) largest_keys_slow<T>(x, lo, hi, min(a.top, hi - lo), best);
    else rank_keys(keys, m, a.top, best);
    __syncthreads();
  }
  if (a.parts == 1) return write_answer<T>(a, row, x, s, best, given);
  const int64_t p = row * a.parts + part;
  if (tid == 0) a.part[p] = {__builtin_bit_cast(int, s.max), s.sum, s.weighted};
  if (TOP && tid < a.top) a.keys[p * a.top + tid] = best[tid];
}

// Joins the parts of a row.
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) void k_log_probs_join(AnswerArgs a) {
  typedef typename Logit<T>::type V;
  const int rows = a.rows_dev ? min(a.rows, *a.rows_dev) : a.rows;
  const int64_t row = blockIdx.x;
  if (row >= rows) return;
  const T *x = (const T *)a.logits + row * a.logits_ld;
  __shared__ u64 keys[TOP ? kMaxParts * HV_LOG_PROBS_MAX_TOP : 1];
  __shared__ u64 best[TOP ? HV_LOG_PROBS_MAX_TOP : 1];
  __shared__ int n_keys;
  const int tid = threadIdx.x, lane = tid & 63, n = a.parts * a.top;
  const u64 *from = a.keys + row * n;
  const Given<T> given(a, row, x);
  Sums<T> s;
  if (lane < a.parts) {
    const AnswerPart p = a.part[row * a.parts + lane];
    s.max = __builtin_bit_cast(V, p.max);
    s.sum = p.sum;
    s.weighted = p.weighted;
  }
  u64 bound = 1;  // keys of 0 stand where a part had fewer than `top`
  if (TOP) {
    if (tid == 0) n_keys = 0;
    // Each part's keys are in order. `each` of a part's keys are not under its
    // each-th, so the need-th largest of these bounds need * each >= top keys.
    const int each = (a.top + a.parts - 1) / a.parts, need = (a.top + each - 1) / each;
    const u64 mine = lane < a.parts ? from[lane * a.top + each - 1] : 0;
    int reach = 0;
    for (int i = 0; i < a.parts; ++i) {
      const unsigned low = __builtin_amdgcn_readlane((int)mine, i);
      const unsigned high = __builtin_amdgcn_readlane((int)(mine >> 32), i);
      reach += ((u64)high << 32 | low) >= mine;
    }
    u64 least = reach >= need ? mine : 0;
    for (int o = 32; o; o >>= 1) {
      const u64 other = __shfl_xor(least, o);
      least = other > least ? other : least;
    }
    bound = least ? least : 1;
  }
  s.join_lanes(factor_of<T>(a));
  if (TOP) {
    __syncthreads();
    for (int i = tid; i < n; i += kThreads)
      if (from[i] >= bound) keys[atomicAdd(&n_keys, 1)] = from[i];
    __syncthreads();
    if (s.sum != s.sum) largest_keys_slow<T>(x, 0, a.width, a.top, best);
    else rank_keys(keys, n_keys, a.top, best);
    __syncthreads();
  }
  write_answer<T>(a, row, x, s, best, given);
}

// Parts of a row. A row is read by one workgroup where there are rows enough
// to keep the card busy; fewer rows are cut until kAnswerGroups workgroups
// are at work, in parts of at least kMinPart logits (of 4096 and of 8192: 1 row
// of 131072 with 20 alternatives 14.6, 13.5 us; 16 rows 15.8, 14.0).
static constexpr int kAnswerGroups = 512, kMinPart = 8192;
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
            dim3(kThreads), 0, s, a);
  if (a.parts > 1)
    hv_launch(k_log_probs_join<T, TOP>, dim3(a.rows), dim3(kThreads), 0, s, a);
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
  if (d->rows < 0 || d->rows > HV_LM_MAX_ROWS || d->width < 1 ||
      d->width > HV_LOG_PROBS_MAX_WIDTH || d->n_tokens < 0 ||
      d->n_tokens > HV_LOG_PROBS_MAX_WIDTH || d->logits_ld < d->width ||
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
      return fail(HV_EVALUE, HV_ERR_ADDRESS,
                  "log_probs: workspace too small or not 8-byte aligned");
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
