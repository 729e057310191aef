// hv_lm_paged.h -- where the rows and keys of packed sequences and of a paged
// cache lie. Code without HIP, so that tests can run it on the host: whatever
// the caller's offsets, lengths and tables hold, what it returns lies inside
// the buffers or is refused.
#pragma once

#include <cstdint>

#ifdef __HIPCC__
#define HV_HD __host__ __device__ __forceinline__
#else
#define HV_HD inline
#endif

namespace hv {

HV_HD int clamp_to(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// Rows first .. first + count of sequence b of `batch`, inside [0, rows); count 0
// where the offsets run backwards. starts NULL: row b.
struct SeqRows {
  int first, count;
};
HV_HD SeqRows seq_rows(const int32_t *starts, int b, int rows) {
  if (!starts) return {b, b < rows ? 1 : 0};
  const int lo = clamp_to(starts[b], 0, rows), hi = clamp_to(starts[b + 1], 0, rows);
  return {lo, hi > lo ? hi - lo : 0};
}

// A cache of `pages` pages of 2^shift rows, a sequence's pages in a row of a
// table of max_pages entries.
struct PageMap {
  int pages, shift, max_pages;
};

// Keys that a sequence of `length` has, or -1 where the table has no room for
// them.
HV_HD int paged_keys(const PageMap &m, int length) {
  if (length <= 0) return 0;
  return length <= (int64_t)m.max_pages << m.shift ? length : -1;
}

// The page of a key, or -1: a position outside the table, a page outside the cache.
HV_HD int page_of(const PageMap &m, const int32_t *table, int64_t position) {
  if (position < 0 || position >= (int64_t)m.max_pages << m.shift) return -1;
  const int page = table[position >> m.shift];
  return page >= 0 && page < m.pages ? page : -1;
}

// Row of a page's key for one of `heads` heads in [pages][heads][2^shift] rows.
HV_HD int64_t cache_row(const PageMap &m, int heads, int page, int head, int64_t position) {
  return (((int64_t)page * heads + head) << m.shift) + (position & ((1 << m.shift) - 1));
}

// Keys [from, to) that row i of a sequence's n rows sees among `keys` of them:
// causal rows are the last n positions, and a window keeps the last `window`
// of what a row would see.
struct Seen {
  int from, to;
};
HV_HD Seen seen_by(int i, int n, int keys, bool causal, int window) {
  if (!causal) return {0, keys};
  const int64_t to64 = (int64_t)keys - n + i + 1;
  const int to = to64 < 0 ? 0 : (int)to64;
  return {window && to > window ? to - window : 0, to};
}

}  // namespace hv
