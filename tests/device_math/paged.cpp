// Where rows and keys of a paged cache lie, for the tests.
#include "hv_lm_paged.h"

using namespace hv;

extern "C" {
void seq_rows_of(const int32_t *starts, int b, int rows, int32_t *out) {
  const SeqRows r = seq_rows(starts, b, rows);
  out[0] = r.first;
  out[1] = r.count;
}
int keys_of(int pages, int shift, int max_pages, int length) {
  return paged_keys({pages, shift, max_pages}, length);
}
int page_at(int pages, int shift, int max_pages, const int32_t *table, long long position) {
  return page_of({pages, shift, max_pages}, table, position);
}
long long row_at(int pages, int shift, int heads, int page, int head, long long position) {
  return cache_row({pages, shift, 0}, heads, page, head, position);
}
void seen_at(int i, int n, int keys, int causal, int window, int32_t *out) {
  const Seen s = seen_by(i, n, keys, causal != 0, window);
  out[0] = s.from;
  out[1] = s.to;
}
}

// Which kernels a call takes.
#include "hv_lm_attn_plan.h"
extern "C" {
int attention_shape(int rows, int batch, int heads, int kv_heads, int width, long long most_keys) {
  const Shape s = shape_of(rows, batch, heads, kv_heads, width);
  const bool shares = s.split && worth_sharing(s, rows, batch, kv_heads, heads / kv_heads, most_keys);
  return (s.tile_rows == kFewRows ? 0 : 2) + shares;
}
long long attention_workspace(int rows, int batch, int heads, int kv_heads, int width) {
  return (long long)workspace_of(shape_of(rows, batch, heads, kv_heads, width), width);
}
int tile_of_cost(int first, int step, int count, int at) {
  return Cost{first, step, count}.tile_at(at);
}
int cost_before(int first, int step, int count, int tile) {
  return Cost{first, step, count}.before(tile);
}
int part_of_tiles(int n, int at, int cost) { return tiles_at(n, at, cost); }
// n, start(share), of(at), parts(share, end)
void share_numbers(int cost, int workgroups, int share, int at, int end, int32_t *out) {
  const Shares s(cost, workgroups);
  out[0] = s.n;
  out[1] = s.start(share);
  out[2] = s.of(at);
  out[3] = s.parts(share, end);
}
int attention_run(int rows, int batch, int heads, int kv_heads, int width, int split) {
  Shape s = shape_of(rows, batch, heads, kv_heads, width);
  s.split = split != 0;
  return run_of(s, rows, batch, kv_heads, heads / kv_heads);
}
int place_in_runs(int b, int run) { return place_of(b, run); }
}

// The longest sequence's keys, by what the host knows.
extern "C" {
long long table_keys(int said, long long room) { return keys_of_table(said, room); }
long long packed_keys(int said, long long all, int batch) { return keys_of_packed(said, all, batch); }
}

// Lanes of a head of the rotary kernels.
#include "hv_lm_rotary_plan.h"
extern "C" int lanes_of_head(int pairs, int width) { return rotary_lanes(pairs, width); }
