// hv_lm_cache.hip -- new keys and values into the pages of a cache.
//
// Row i of a sequence's n new rows is key length - n + i of it. In 8 bits each
// head of a token has an exponent of its own: e the smallest with |x| <= 448
// 2^e, q = round(x 2^-e), so a head is quantised by sixteen lanes that hold all
// of it, in one pass.
#include <type_traits>

#include "hv_lm.h"
#include "hv_lm_paged.h"

namespace hv {

struct CacheWriteArgs {
  const void *x[2];  // keys, values
  uint8_t *cache[2];
  int8_t *exps[2];
  const int32_t *starts, *lengths, *table;
  int64_t ld[2], head_ld[2], table_ld;
  int rows, batch, heads, width;
  PageMap map;
};

// The last sequence that starts at or before `row`, by the sixteen lanes that
// ask together (-1: none), from batch + 1 offsets: a sixteenth of what is left at a time.
__device__ __forceinline__ int find_sequence(const int32_t *starts, int batch, int row) {
  const int lane = threadIdx.x & 15, shift = threadIdx.x & 48;
  int lo = 0, left = batch + 1;
  while (true) {
    const int step = (left + 15) / 16, i = lo + lane * step;
    const bool before = lane * step < left && i <= batch && starts[i] <= row;
    const int found = __popc((unsigned)(__ballot(before) >> shift) & 0xFFFF);
    if (!found) return -1;
    lo += (found - 1) * step;
    if (step == 1) return lo;
    left = min(step, batch + 1 - lo);
  }
}

// A workgroup has kParts heads (of the keys, then of the values) in sixteen rows, which lie
// side by side in a page; a row to sixteen lanes, which load all of its heads at once.
// Memory bounds it: 16384 rows of 8 heads of 128 into e4m3 (101 MB) take 24 us, 4.2 TB/s (32 us
// with one head a workgroup, whose lanes find the rows' places for it alone). 64 rows take
// 4.6 us: offsets, length, page and rows, one load's latency after another.
static constexpr int kParts = 4;
template <typename T, bool Q8>
__global__ __launch_bounds__(256) void k_cache_write(CacheWriteArgs a) {
  typedef typename Eight<T>::v8 v8;
  const int lane = threadIdx.x & 15;
  const int part0 = blockIdx.y * kParts, parts = min(kParts, 2 * a.heads - part0);
  // Groups past the last row repeat it and write nothing.
  const int mine = blockIdx.x * 16 + threadIdx.x / 16, row = min(mine, a.rows - 1);
  v8 e[kParts][2] = {};
#pragma unroll
  for (int p = 0; p < kParts; ++p) {
    const int part = min(part0 + p, 2 * a.heads - 1), which = part >= a.heads;
    const T *x = (const T *)a.x[which] + row * a.ld[which] +
                 (which ? part - a.heads : part) * a.head_ld[which];
#pragma unroll
    for (int r = 0; r < 2; ++r)
      if (lane * 8 + r * 128 < a.width) e[p][r] = Eight<T>::load(x + lane * 8 + r * 128, 8);
  }
  int b = row, first = row, count = 1;
  if (a.starts) {
    b = find_sequence(a.starts, a.batch, row);
    if (b < 0 || b >= a.batch) return;  // before the first sequence, or behind the last
    const SeqRows s = seq_rows(a.starts, b, a.rows);
    first = s.first;
    count = s.count;
  }
  const int64_t position = (int64_t)a.lengths[b] - count + (row - first);
  const int page = page_of(a.map, a.table + b * a.table_ld, position);
  if (page < 0 || mine >= a.rows) return;
#pragma unroll
  for (int p = 0; p < kParts; ++p) {
    if (p >= parts) break;
    const int part = part0 + p, which = part >= a.heads;
    const int64_t to = cache_row(a.map, a.heads, page, which ? part - a.heads : part, position);
    if (!Q8) {
      T *out = (T *)a.cache[which] + to * a.width;
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (lane * 8 + r * 128 < a.width) Eight<T>::store(out + lane * 8 + r * 128, 8, e[p][r]);
      continue;
    }
    float v[2][8], amax = 0.f;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[r][i] = (float)e[p][r][i];
        amax = fmaxf(amax, fabsf(v[r][i]));
      }
    const int exp = block_exp<HV_Q_E4M3>(max16(amax));
    // The largest exponent of the type: 256 2^exp is past its numbers, so what
    // would round to that is 240 2^exp. Infinities stay, as NaN.
    constexpr int kTop = std::is_same<T, f16>::value ? 8 : 120;
    if (exp == kTop) {
      const float most = ldexpf(240.f, kTop);
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (fabsf(v[r][i]) > most && fabsf(v[r][i]) < __builtin_inff())
            v[r][i] = copysignf(most, v[r][i]);
    }
    const float inv = __builtin_bit_cast(float, (127 - exp) << 23);
    uint8_t *out = a.cache[which] + to * a.width;
#pragma unroll
    for (int r = 0; r < 2; ++r)
      if (lane * 8 + r * 128 < a.width) store_q8<HV_Q_E4M3>(out + lane * 8 + r * 128, 8, v[r], inv);
    if (lane == 0) a.exps[which][to] = (int8_t)exp;
  }
}

template <typename T>
static void cache_write_launch(const CacheWriteArgs &a, bool q8, hipStream_t s) {
  const dim3 grid((a.rows + 15) / 16, (2 * a.heads + kParts - 1) / kParts), block(256);
  if (q8) hv_launch(k_cache_write<T, true>, grid, block, 0, s, a);
  else hv_launch(k_cache_write<T, false>, grid, block, 0, s, a);
}

}  // namespace hv

using namespace hv;

// What a cache and its table have to be, for both that use them.
int hv::check_cache(const char *what, const hv_cache_desc &c, int type, int batch, int kv_heads,
                    int width) {
  if (c.format != HV_CACHE_SAME && c.format != HV_CACHE_E4M3)
    return fail(HV_EVALUE, HV_ERR_OPCODE, "%s: bad cache format %d", what, c.format);
  if (c.page < HV_CACHE_MIN_PAGE || c.page > HV_CACHE_MAX_PAGE || (c.page & (c.page - 1)))
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "%s: pages of %d keys", what, c.page);
  if (c.pages < 1 || c.max_pages < 0 || (int64_t)c.max_pages * c.page > HV_CACHE_MAX_KEYS ||
      c.table_ld < c.max_pages)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "%s: %d pages, a table of %d in rows of %lld", what,
                c.pages, c.max_pages, (long long)c.table_ld);
  const int unit = c.format == HV_CACHE_E4M3 ? 16 : 8;
  if (width < unit || width > HV_ATTENTION_MAX_WIDTH || width % unit)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "%s: heads of %d are no multiple of %d up to %d", what,
                width, unit, HV_ATTENTION_MAX_WIDTH);
  if (batch == 0) return HV_OK;
  if (!c.k || !c.v || !c.lengths || (c.max_pages && !c.table) ||
      (c.format == HV_CACHE_E4M3 && (!c.k_exps || !c.v_exps)))
    return fail(HV_EVALUE, HV_ERR_ADDRESS, "%s: null argument of the cache", what);
  if ((((uintptr_t)c.k | (uintptr_t)c.v) & 15) ||
      (((uintptr_t)c.table | (uintptr_t)c.lengths) & 3))
    return fail(HV_EVALUE, HV_ERR_ADDRESS, "%s: a pointer of the cache is not aligned", what);
  return HV_OK;
}

extern "C" int hv_cache_write(const hv_cache_write_desc *d, hv_stream_t stream) {
  clear_error();
  if (!d) return fail(HV_EVALUE, HV_ERR_ADDRESS, "cache_write: null descriptor");
  if (d->type != HV_T_F16 && d->type != HV_T_BF16)
    return fail(HV_EVALUE, HV_ERR_OPCODE, "cache_write: bad element type %d", d->type);
  if (d->rows < 0 || d->rows > HV_LM_MAX_ROWS || d->batch < 0 || d->batch > HV_LM_MAX_ROWS ||
      d->kv_heads < 1 || d->kv_heads > HV_LM_MAX_HEADS ||
      (int64_t)d->rows * d->kv_heads > 1 << 26)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "cache_write: %d rows of %d heads, %d sequences",
                d->rows, d->kv_heads, d->batch);
  if (!d->starts && d->rows != d->batch)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "cache_write: %d rows for one of each of %d sequences",
                d->rows, d->batch);
  const int rc = check_cache("cache_write", d->cache, d->type, d->batch, d->kv_heads, d->width);
  if (rc) return rc;
  if (d->k_ld < 0 || d->k_head_ld < 0 || d->v_ld < 0 || d->v_head_ld < 0)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "cache_write: a negative stride");
  if (d->rows == 0 || d->batch == 0 || d->cache.max_pages == 0) return HV_OK;
  if (!d->k || !d->v) return fail(HV_EVALUE, HV_ERR_ADDRESS, "cache_write: null argument");
  if ((((uintptr_t)d->k | (uintptr_t)d->v) & 1) || ((uintptr_t)d->starts & 3))
    return fail(HV_EVALUE, HV_ERR_ADDRESS, "cache_write: a pointer is not aligned to its elements");
  CacheWriteArgs a{};
  a.x[0] = d->k; a.x[1] = d->v;
  a.cache[0] = (uint8_t *)d->cache.k; a.cache[1] = (uint8_t *)d->cache.v;
  a.exps[0] = d->cache.k_exps; a.exps[1] = d->cache.v_exps;
  a.starts = d->starts; a.lengths = d->cache.lengths; a.table = d->cache.table;
  a.ld[0] = d->k_ld; a.ld[1] = d->v_ld; a.head_ld[0] = d->k_head_ld; a.head_ld[1] = d->v_head_ld;
  a.table_ld = d->cache.table_ld;
  a.rows = d->rows; a.batch = d->batch; a.heads = d->kv_heads; a.width = d->width;
  a.map = {d->cache.pages, __builtin_ctz(d->cache.page), d->cache.max_pages};
  const hipStream_t s = (hipStream_t)stream;
  const bool q8 = d->cache.format == HV_CACHE_E4M3;
  if (d->type == HV_T_F16) cache_write_launch<f16>(a, q8, s);
  else cache_write_launch<bf16>(a, q8, s);
  return check_hip(hipGetLastError(), "k_cache_write launch");
}
