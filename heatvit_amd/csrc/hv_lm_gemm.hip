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
// The 8-bit matrix cores add groups of products aligned to the largest one and
// cut off what lies 2^-13 below it. Measured, of the result's norm and whatever
// the length: 1.5e-5 on normal values, 3e-6 on values of one sign, 1e-4 with one
// channel of each block 64 times the others (of an output's sum of |a w| there
// at most 3e-4). That is a hundredth of what the rounding to bf16 costs, and a
// seventeenth with such channels; of f16's a fourteenth and a half. So 16-bit
// outputs take them; a float32 output takes the 16-bit matrix cores instead
// (Exact: e4m3 values are exact in bf16, their sums good to 1e-8 at k = 128 and
// 2e-7 at k = 4096), block by block, the block's power of two applied to its sum.
#include <type_traits>

#include "hv_lm.h"
#include "hv_lm_plan.h"

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
};

static constexpr int kTileBytes = 64 * 128;  // 64 channels by 128 k, packed

// Products of one block of 128: FN fragments of W (16 channels each) by one of
// the rows (16), added to acc with the factor 2^(we + ae - 254) of the scale
// bytes in the low bits of we and ae, or NaN where one of them is 255 (an
// exponent of -128); we is the same for the wavefront.
struct Fast {
  typedef v8i frag;
  static __device__ __forceinline__ frag of(v8i raw) { return raw; }
  template <int FN>
  static __device__ __forceinline__ void add(const frag (&w)[FN], v8i a, v4f (&acc)[FN], int we,
                                             int ae) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
      acc[j] =
          __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[j], a, acc[j], 0, 0, 0, we, 0, ae);
  }
};
struct Exact {
  static constexpr int kNoFactor = 1 << 10;  // outside what the conversion applies
  struct frag {
    v8bf v[4];
  };
  static __device__ __forceinline__ frag of(v8i raw, float scale = 1.f) {
    frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int x = raw[2 * i], y = raw[2 * i + 1];
      const v2bf a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, false);
      const v2bf b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, true);
      const v2bf c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, scale, false);
      const v2bf d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, scale, true);
      f.v[i] = v8bf{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
    return f;
  }
  // The conversion of the rows applies the factor, exactly while it stays well
  // inside bf16's exponents; what is left of a factor outside 2^-100 .. 2^100 is
  // applied to the block's sums (8192 x 8192 by k = 1024: 174 us, with every
  // factor applied to sums 183). With one fragment of W the sums are as few as
  // the rows' values, and it goes to them without the vote (48 x 14336 by 4096:
  // 20.4 us, with it 22.2).
  template <int FN>
  static __device__ __forceinline__ void add(const frag (&w)[FN], v8i raw, v4f (&acc)[FN], int we,
                                             int ae) {
    const int w8 = we & 255, a8 = ae & 255;
    const int e = max(w8, a8) == 255 ? kNoFactor : w8 + a8 - 254;
    const int in = FN > 1 ? min(max(e, -100), 100) : 0;
    const frag a = of(raw, __builtin_bit_cast(float, (in + 127) << 23));
    if (FN > 1 && __builtin_amdgcn_ballot_w64(in != e) == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[j].v[i], a.v[i], acc[j], 0, 0, 0);
    } else {
      const float from = e == kNoFactor ? __builtin_nanf("") : 0.f;
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        v4f t = {from, from, from, from};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[j].v[i], a.v[i], t, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] += ldexpf(t[i], e - in);
      }
    }
  }
};

__device__ __forceinline__ v8i join(v4i lo, v4i hi) {
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// RUN adjacent channels of row m from n on. A row may start at any element:
// wide stores need no more alignment than that.
template <typename T, int RUN>
__device__ __forceinline__ void store_run(const GemmF8Args &g, int m, int n, const float *v) {
  T *p = (T *)g.c + m * g.ldc + n;
  if (n + RUN <= g.n) {
    typedef T vt __attribute__((ext_vector_type(RUN)));
    vt t;
#pragma unroll
    for (int i = 0; i < RUN; ++i) t[i] = (T)v[i];
    __builtin_memcpy(p, &t, sizeof t);
  } else {
#pragma unroll
    for (int i = 0; i < RUN; ++i)
      if (n + i < g.n) p[i] = (T)v[i];
  }
}

// Channel of a group of 64 at which lane group grp's four of part j start: with
// parts 2 J and 2 J + 1 a lane has eight adjacent channels.
__device__ __forceinline__ int channel_of(int j, int grp) {
  return j / 2 * 32 + grp * 8 + j % 2 * 4;
}

// One lane's outputs of FM x FN fragments: rows m0 + 16 i, parts j0 .. of the
// group of 64 at n0. scale(i) and bias(n): a row's factor, a channel's addend.
template <typename T, int FM, int FN, typename Scale, typename Bias>
__device__ __forceinline__ void store_tile(const GemmF8Args &g, int rows, int m0, int n0, int j0,
                                           int grp, const v4f (&acc)[FM][FN], Scale scale,
                                           Bias bias) {
  constexpr int RUN = FN >= 2 ? 8 : 4;
  float add[FN][4];
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int k = 0; k < 4; ++k) add[j][k] = bias(n0 + channel_of(j0 + j, grp) + k);
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = m0 + 16 * i;
    if (m >= rows) continue;
    const float f = scale(i);
#pragma unroll
    for (int j = 0; j < FN; j += RUN / 4) {
      float v[RUN];
#pragma unroll
      for (int k = 0; k < RUN; ++k)
        v[k] = __builtin_fmaf(acc[i][j + k / 4][k % 4], f, add[j + k / 4][k % 4]);
      store_run<T, RUN>(g, m, n0 + channel_of(j0 + j, grp), v);
    }
  }
}

// Few rows: a workgroup takes FM x 16 rows by J parts of 16 channels of a
// group of 64, its NW wavefronts every NW-th block of k each, and adds their
// sums up through LDS in a fixed order. Fragments come straight from memory:
// the packed weights are in the order the lanes take them, each read once.
// One row by 4096 x 4096 takes 5.2 us (16.8 MB, 3.4 us at a copy's rate): a
// wavefront has four blocks, all asked for at once, so what is left over the
// bytes is one load's latency and the launch.
template <typename T, int FM, int J, int NW>
__global__ __launch_bounds__(64 * NW) void k_gemm_f8_rows(GemmF8Args g) {
  typedef typename std::conditional<std::is_same<T, float>::value, Exact, Fast>::type Mma;
  const int rows = g.m_dev ? min(g.m, *g.m_dev) : g.m;
  const int m0 = blockIdx.y * (16 * FM);
  if (m0 >= rows) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int group = blockIdx.x / (4 / J), j0 = blockIdx.x % (4 / J) * J;
  const uint8_t *w = g.w + (size_t)group * g.kb * kTileBytes + j0 * 2048 + lane * 16;
  const uint8_t *a[FM];
  const int8_t *ae[FM];
  // Odd rows load the upper halves of their lines beside even rows' lower ones:
  // rows lie whole lines apart as a rule, and one load of the same halves of 16
  // lines takes longer (16 rows by 256 channels, k = 8192: 8.2 us, so 6.7).
  const int odd = col & 1;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int64_t m = min(m0 + 16 * i + col, rows - 1);  // rows past the end repeat the last
    a[i] = g.a + m * g.lda;
    ae[i] = g.a_exps + m * g.a_exps_ld;
  }
  v4f acc[FM][J] = {};
  // Blocks b0, b0 + NW, ..: the loads of all U are on their way before the
  // first is waited for.
  auto blocks = [&](int b0, auto n_blocks) {
    constexpr int U = decltype(n_blocks)::value;
    v8i wf[U][J];
    v4i first[U][FM], second[U][FM];
    int we[U], e[U][FM];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = b0 + u * NW;
#pragma unroll
      for (int j = 0; j < J; ++j)
        wf[u][j] = join(
            *reinterpret_cast<const v4i *>(w + (size_t)b * kTileBytes + j * 2048),
            *reinterpret_cast<const v4i *>(w + (size_t)b * kTileBytes + j * 2048 + 1024));
      we[u] = g.w_exps[(size_t)b * g.nb + group / 2] + 127;
      const int k1 = b * 128 + 16 * grp + 64 * odd, k2 = k1 ^ 64;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        first[u][i] = *reinterpret_cast<const v4i *>(a[i] + (k1 < g.k ? k1 : 0));
        second[u][i] = *reinterpret_cast<const v4i *>(a[i] + (k2 < g.k ? k2 : 0));
        e[u][i] = ae[i][b] + 127;
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      typename Mma::frag wo[J];
#pragma unroll
      for (int j = 0; j < J; ++j) wo[j] = Mma::of(wf[u][j]);
      const int k = (b0 + u * NW) * 128 + 16 * grp;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        v4i x = odd ? second[u][i] : first[u][i], y = odd ? first[u][i] : second[u][i];
        if (k >= g.k) x = v4i{};  // zeros past the end of k
        if (k + 64 >= g.k) y = v4i{};
        Mma::add(wo, join(x, y), acc[i], we[u], e[u][i]);
      }
    }
  };
  constexpr int U = FM * J >= 4 ? 2 : 4;
  int b = wave;
  for (; b + (U - 1) * NW < g.kb; b += U * NW) blocks(b, std::integral_constant<int, U>());
  for (; b < g.kb; b += NW) blocks(b, std::integral_constant<int, 1>());
  __shared__ v4f part[NW][FM * J][64];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j) part[wave][i * J + j][lane] = acc[i][j];
  __syncthreads();
  for (int f = wave; f < FM * J; f += NW) {
    v4f v = part[0][f][lane];
#pragma unroll
    for (int k = 1; k < NW; ++k) v += part[k][f][lane];
    const v4f one[1][1] = {{v}};
    const int m = m0 + 16 * (f / J) + col;
    store_tile<T>(
        g, rows, m, group * 64, j0 + f % J, grp, one,
        [&](int) { return g.row_scale ? g.row_scale[m] : 1.f; },
        [&](int n) { return g.bias ? g.bias[min(n, g.n - 1)] : 0.f; });
  }
}

// 16 bytes a lane straight to LDS, the wavefront's 64 lanes one after another
// from `to` on, from base + offset + uniform of a buffer of `size` bytes (zeros
// for an offset behind it).  base, size and uniform are the same in all lanes.
__device__ __forceinline__ void buffer_to_lds(const uint8_t *base, int size, int offset,
                                              int uniform, uint8_t *to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, size, 0x00020000),
      (__attribute__((address_space(3))) void *)to, 16, offset,
      __builtin_amdgcn_readfirstlane(uniform), 0, 0);
}

// Blocks of k whose exponents a workgroup keeps in LDS at a time.
static constexpr int kExpSteps = 64;

template <int BM, int BN>
struct TileLds {
  uint8_t a[BM * 128];
  uint8_t b[BN * 128];
};

// The workgroup's tile. Tiles lie in bands of kBand along m; the eight XCDs,
// which take workgroups in turn, each get a contiguous range of them, whose
// operands meet in their L2.
template <int BM, int BN>
__device__ __forceinline__ void tile_of(const GemmF8Args &g, int &m0, int &n0) {
  constexpr int kBand = 4;
  const int tn = (g.n + BN - 1) / BN, tm = (g.m + BM - 1) / BM, total = tm * tn;
  int id = blockIdx.x;
  const int per = total / 8, rem = total % 8, x = id % 8;
  id = x * per + min(x, rem) + id / 8;
  const int band = id / (kBand * tn), in = id - band * (kBand * tn);
  const int high = min(kBand, tm - band * kBand);
  m0 = (band * kBand + in % high) * BM;
  n0 = in / high * BN;
}

// s_waitcnt: all LDS reads done, and all but the last VM loads.
constexpr int wait_loads(int vm) { return 0x70 | (vm & 15) | (vm >> 4) << 14; }

// BM x BN outputs a workgroup, WM x WN wavefronts. A block of 128 of k at a
// time goes from memory into one of S LDS stages (16 bytes a lane, straight
// to LDS):
//   rows: 128 bytes each, their 16-byte chunks at chunk ^ (row / 2 & 7), so
//         that 16 rows' reads of one chunk take each of the 64 banks once
//   weights: as they are packed, in the order the lanes take them
// A wavefront multiplies its FM row fragments one after another and reads them
// two ahead. When it has read the last one it waits for its loads of the next
// block, and a barrier tells it that everybody's are there and that nobody
// reads this stage any more: the last two fragments' products then run beside
// the reads of the next block's first fragments, and the stage is filled again
// with block b + S. Loads are spread over four fragments' products,
// because a wavefront that issues them all at once stands still until the
// memory pipeline has taken them (8192^3: all at once 502 us, spread 438).
// The exponents of kExpSteps blocks wait in LDS too: a load of theirs in the
// loop would have to wait for the stage's loads in front of it.
// The matrix cores bound a long k: 8192^3 takes 410 to 438 us by card (2.5 to 2.7
// PFLOP/s), the matrix cores busy for 64 to 68 % of it at the 1.93 GHz that such
// a load leaves. A tile's loads at the start and its stores bound a short one: 11
// us a round of 256 x 256 tiles and 1.1 a block of k (50432 x 768 by k = 192: 32.5
// us, where the stores alone take 19.3 and all but the stores 19.9). Weights alone
// bound few rows: 48 x 14336 by k = 4096 takes 12.2 us, 60 MB at a copy's rate.
template <typename T, int BM, int BN, int WM, int WN, int S>
__global__ __launch_bounds__(64 * WM * WN) void k_gemm_f8_tile(GemmF8Args g) {
  typedef typename std::conditional<std::is_same<T, float>::value, Exact, Fast>::type Mma;
  constexpr int kWaves = WM * WN, TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  constexpr int NB = (BN + 127) / 128;  // 128-column blocks of the tile
  static_assert(TN <= 64 && 64 % TN == 0 && FM % 4 == 0, "a wavefront's columns share an exponent");
  // Each stage a variable of its own: the compiler then sees that a read of one
  // need not wait for loads into another.
  static_assert(S == 2 || S == 4, "stages");
  __shared__ TileLds<BM, BN> stage0, stage1;
  __shared__ TileLds<S == 4 ? BM : 1, S == 4 ? BN : 1> stage2_, stage3_;
  auto &stage2 = reinterpret_cast<TileLds<BM, BN> &>(stage2_);
  auto &stage3 = reinterpret_cast<TileLds<BM, BN> &>(stage3_);
  __shared__ uint8_t a_exp[kExpSteps][WM][16][FM];
  __shared__ uint8_t w_exp[kExpSteps][NB];
  __shared__ float row_scale[BM], bias[BN];

  const int rows = g.m_dev ? min(g.m, *g.m_dev) : g.m;
  int m0, n0;
  tile_of<BM, BN>(g, m0, n0);
  if (m0 >= rows) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN, col = lane & 15, grp = lane >> 4;

  // Loads: wavefront `wave` takes 8 rows (1 KiB) of every kWaves x 8.
  constexpr int LA = BM / 8 / kWaves, LB = BN / 8 / kWaves;
  static_assert(LA * 8 * kWaves == BM && LB * 8 * kWaves == BN, "whole loads");
  const int last = rows - 1 - m0;  // of the tile's rows, those past it repeat it
  const uint8_t *a_base = g.a + (int64_t)m0 * g.lda;
  const int a_size = (int)(min(last, BM - 1) * g.lda + g.k);
  static_assert(kWaves % 2 == 0, "a wavefront's units of 8 rows lie alike in 16");
  const int chunk = (lane & 7) ^ (wave % 2 * 4 + (lane >> 4));
  int a_off[LA];
#pragma unroll
  for (int i = 0; i < LA; ++i)
    a_off[i] = min((i * kWaves + wave) * 8 + (lane >> 3), last) * (int)g.lda + chunk * 16;
  // The tile's groups of weights, and how far each of this wavefront's loads is
  // in them; groups past the last repeat it.
  const int groups = min(BN / 64, (g.n - 1) / 64 - n0 / 64 + 1);
  const uint8_t *w_base = g.w + (size_t)(n0 / 64) * g.kb * kTileBytes;
  int w_off[LB];
#pragma unroll
  for (int i = 0; i < LB; ++i) {
    const int kib = i * kWaves + wave;  // of the stage's BN / 8
    w_off[i] = min(kib / 8, groups - 1) * g.kb * kTileBytes + kib % 8 * 1024;
  }
  const int tail = (g.k - 1) % 128 / 16;  // the last block's last chunk of 16
  // A quarter of block b's loads; past the last block it loads that again.
  auto load = [&](TileLds<BM, BN> &s, int b, int quarter) {
    b = __builtin_amdgcn_readfirstlane(min(b, g.kb - 1));
    // behind the last of k the buffer load gives zeros
    const bool past = b == g.kb - 1 && chunk > tail;
#pragma unroll
    for (int i = 0; i < LA + LB; ++i) {
      if (i * 4 / (LA + LB) != quarter) continue;
      if (i < LA)
        buffer_to_lds(a_base, a_size, past ? 0x7FFFFFF0 : a_off[i], b * 128,
                      s.a + (i * kWaves + wave) * 1024);
      else
        buffer_to_lds(w_base, groups * g.kb * kTileBytes, lane * 16, w_off[i - LA] + b * kTileBytes,
                      s.b + ((i - LA) * kWaves + wave) * 1024);
    }
  };

  v4f acc[FM][FN] = {};
  v8i wf[2][FN], af[4];
  int we[2], ae[2][(FM + 3) / 4] = {};
  const int c0 = (grp ^ (col >> 1)) * 16;
  auto read_a = [&](const TileLds<BM, BN> &s, int i) {
    const uint8_t *p = s.a + (wm * TM + i * 16 + col) * 128;
    af[i % 4] = join(*reinterpret_cast<const v4i *>(p + c0),
                     *reinterpret_cast<const v4i *>(p + (c0 ^ 64)));
  };
  auto read_w = [&](const TileLds<BM, BN> &s, int p) {
    const uint8_t *at = s.b + wn * TN / 64 * 8192 + wn * TN % 64 / 16 * 2048 + lane * 16;
#pragma unroll
    for (int j = 0; j < FN; ++j)
      wf[p][j] = join(*reinterpret_cast<const v4i *>(at + j * 2048),
                      *reinterpret_cast<const v4i *>(at + j * 2048 + 1024));
  };
  auto read_exps = [&](int b, int p) {
    we[p] = w_exp[b % kExpSteps][wn * TN / 128];
    __builtin_memcpy(ae[p], a_exp[b % kExpSteps][wm][col], FM);
  };
  // Exponents of blocks b0 .. b0 + kExpSteps - 1 as scale bytes: 16 blocks of
  // a row at a time, at once unless that would end behind the last row's.
  const int8_t *exp_end = g.a_exps + (int64_t)(rows - 1) * g.a_exps_ld + g.kb;
  auto load_exps = [&](int b0, auto at_once) {
    constexpr int kParts = kExpSteps / 16, kEach = BM * kParts / (64 * kWaves);
    constexpr int kOnce = decltype(at_once)::value ? kEach : 1;
    static_assert(kEach * 64 * kWaves == BM * kParts, "whole loads");
#pragma unroll 1
    for (int j0 = 0; j0 < kEach; j0 += kOnce) {
      v4i v[kOnce];
#pragma unroll
      for (int j = 0; j < kOnce; ++j) {
        const int i = (j0 + j) * 64 * kWaves + tid, b = b0 + i % kParts * 16;
        const int8_t *from = g.a_exps + (int64_t)(m0 + min(i / kParts, last)) * g.a_exps_ld + b;
        const int over = (int)max((int64_t)0, from + 16 - exp_end);  // 0 .. 15, or all of it
        if (exp_end - g.a_exps >= 16) {
          // the last 16 instead, moved down
          unsigned __int128 t;
          __builtin_memcpy(&t, over < 16 ? from - over : exp_end - 16, 16);
          t = over < 16 ? t >> (8 * over) : 0;
          __builtin_memcpy(&v[j], &t, 16);
        } else {
          v[j] = v4i{};
#pragma unroll
          for (int k = 0; k < 16; ++k)
            if (b + k < g.kb) v[j][k / 4] |= (uint8_t)from[k] << (8 * (k % 4));
        }
      }
#pragma unroll
      for (int j = 0; j < kOnce; ++j) {
        const int i = (j0 + j) * 64 * kWaves + tid, r = i / kParts, b = i % kParts * 16;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          // e + 127 of four bytes at once, without a carry from one to the next
          const unsigned x = v[j][k / 4];
          a_exp[b + k][r / TM][r % 16][r % TM / 16] =
              (uint8_t)((((x & 0x7F7F7F7F) + 0x7F7F7F7F) ^ (x & 0x80808080)) >> (8 * (k % 4)));
        }
      }
    }
#pragma unroll 1
    for (int i = tid; i < kExpSteps * NB; i += 64 * kWaves) {
      const int b = min(b0 + i / NB, g.kb - 1), n = min(n0 / 128 + i % NB, g.nb - 1);
      w_exp[i / NB][i % NB] = (uint8_t)(g.w_exps[(size_t)b * g.nb + n] + 127);
    }
  };
  // This wavefront's reads are done and its loads of the next block; then
  // everybody's.
  auto meet = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(wait_loads((S - 2) * (LA + LB)));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // Block b from stage s, its fragments of W and its first two of the rows
  // already read (into half p). The stage before takes the rest of block
  // b + S - 1, this one the first half of block b + S.
  auto step = [&](int b, TileLds<BM, BN> &before, TileLds<BM, BN> &s, TileLds<BM, BN> &after,
                  int p) {
    typename Mma::frag w[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) w[j] = Mma::of(wf[p][j]);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      if (i + 2 < FM) read_a(s, i + 2);
      if (i < 2) load(before, b + S - 1, 2 + i);
      if (i == FM - 2) {
        meet();
        read_a(after, 0);
        read_w(after, 1 - p);
      }
      if (i == FM - 1) {
        read_a(after, 1);
        read_exps(b + 1, 1 - p);
      }
      if (i >= FM - 2) load(s, b + S, i - (FM - 2));
      __builtin_amdgcn_sched_barrier(0);
      Mma::add(w, af[i % 4], acc[i], we[p], (unsigned)ae[p][i / 4] >> (8 * (i % 4)));
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto next_exps = [&](int b) {
    if (b == 0 || b % kExpSteps) return;
    __syncthreads();
    load_exps(b, std::false_type());  // few registers are free here
    __syncthreads();
    read_exps(b, 0);
  };

  // Blocks 0 .. S - 2 and the first half of S - 1, which goes on in step 0.
  // Everything that the tile needs later is asked for beside them.
#pragma unroll
  for (int q = 0; q < 4; ++q) load(stage0, 0, q);
  if (S == 4) {
#pragma unroll
    for (int q = 0; q < 4; ++q) load(stage1, 1, q);
#pragma unroll
    for (int q = 0; q < 4; ++q) load(stage2, 2, q);
  }
#pragma unroll
  for (int i = tid; i < BM; i += 64 * kWaves)
    row_scale[i] = g.row_scale ? g.row_scale[m0 + min(i, last)] : 1.f;
#pragma unroll
  for (int i = tid; i < BN; i += 64 * kWaves)
    bias[i] = g.bias ? g.bias[min(n0 + i, g.n - 1)] : 0.f;
  load_exps(0, std::true_type());
  meet();
  load(S == 4 ? stage3 : stage1, S - 1, 0);
  load(S == 4 ? stage3 : stage1, S - 1, 1);
  read_w(stage0, 0);
  read_a(stage0, 0);
  read_a(stage0, 1);
  read_exps(0, 0);
  int b = 0;
  if (S == 4) {
    for (; b + 3 < g.kb; b += 4) {
      next_exps(b);
      step(b, stage3, stage0, stage1, 0);
      step(b + 1, stage0, stage1, stage2, 1);
      step(b + 2, stage1, stage2, stage3, 0);
      step(b + 3, stage2, stage3, stage0, 1);
    }
    if (b < g.kb) {
      next_exps(b);
      step(b, stage3, stage0, stage1, 0);
    }
    if (b + 1 < g.kb) step(b + 1, stage0, stage1, stage2, 1);
    if (b + 2 < g.kb) step(b + 2, stage1, stage2, stage3, 0);
  } else {
    for (; b + 1 < g.kb; b += 2) {
      next_exps(b);
      step(b, stage1, stage0, stage1, 0);
      step(b + 1, stage0, stage1, stage0, 1);
    }
    if (b < g.kb) {
      next_exps(b);
      step(b, stage1, stage0, stage1, 0);
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0070);  // the loads behind the last block

  store_tile<T>(
      g, rows, m0 + wm * TM + col, n0 + wn * TN / 64 * 64, wn * TN % 64 / 16, grp, acc,
      [&](int i) { return row_scale[wm * TM + 16 * i + col]; },
      [&](int n) { return bias[n - n0]; });
}

template <typename T, int BM, int BN, int WM, int WN, int S>
static void tile_launch(const GemmF8Args &g, hipStream_t s) {
  const int tiles = ((g.n + BN - 1) / BN) * ((g.m + BM - 1) / BM);
  hv_launch(k_gemm_f8_tile<T, BM, BN, WM, WN, S>, dim3(tiles), dim3(64 * WM * WN), 0, s, g);
}

template <typename T, int FM, int J, int NW>
static void rows_launch(const GemmF8Args &g, hipStream_t s) {
  const dim3 grid((g.n + 63) / 64 * (4 / J), (g.m + 16 * FM - 1) / (16 * FM));
  hv_launch(k_gemm_f8_rows<T, FM, J, NW>, grid, dim3(64 * NW), 0, s, g);
}

template <typename T>
static void gemm_f8_launch(const GemmF8Args &g, hipStream_t s) {
  constexpr bool kF32 = std::is_same<T, float>::value;
  const F8Kernel kernel = f8_kernel(kF32, g.m, g.n, g.lda);
  switch (kernel) {
    case F8Kernel::kRows16: return rows_launch<T, 1, 1, 8>(g, s);
    case F8Kernel::kRows16x2: return rows_launch<T, 1, 2, 8>(g, s);
    case F8Kernel::kRows32: return rows_launch<T, 2, 1, 8>(g, s);
    case F8Kernel::kTile64: return tile_launch<T, 64, 64, 1, 4, 4>(g, s);
    case F8Kernel::kTile128: return tile_launch<T, 128, 128, 2, 2, 2>(g, s);
    default: break;
  }
  if constexpr (kF32) {
    rows_launch<T, 4, 1, 8>(g, s);  // kRows64
  } else {
    if (kernel == F8Kernel::kTile128Deep) return tile_launch<T, 128, 128, 2, 2, 4>(g, s);
    tile_launch<T, 256, 256, 2, 4, 2>(g, s);  // kTile256
  }
}

}  // namespace hv

using namespace hv;

extern "C" {

int hv_gemm_f8(const hv_gemm_f8_desc *d, hv_stream_t stream) {
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
  const hipStream_t s = (hipStream_t)stream;
  if (d->type == HV_T_F32) gemm_f8_launch<float>(g, s);
  else if (d->type == HV_T_F16) gemm_f8_launch<f16>(g, s);
  else gemm_f8_launch<bf16>(g, s);
  return check_hip(hipGetLastError(), "gemm_f8 launch");
}

}  // extern "C"
