// hv_lm_attn.hip -- attention of packed sequences and over a paged cache: the entry
// points, and what they refuse.
#include "hv_lm_attn.h"

namespace hv {

static int check_rows(const char *what, const hv_attention_rows &r, bool need_starts) {
  if (r.type != HV_T_F16 && r.type != HV_T_BF16)
    return fail(HV_EVALUE, HV_ERR_OPCODE, "%s: bad element type %d", what, r.type);
  if (r.rows < 0 || r.rows > HV_LM_MAX_ROWS || r.batch < 0 || r.batch > HV_LM_MAX_ROWS ||
      r.heads < 1 || r.heads > HV_LM_MAX_HEADS || r.kv_heads < 1 || r.heads % r.kv_heads ||
      (int64_t)r.rows * r.heads > 1 << 26 || (int64_t)r.batch * r.kv_heads > 1 << 22)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "%s: %d rows of %d heads, %d of keys, %d sequences",
                what, r.rows, r.heads, r.kv_heads, r.batch);
  if (r.width < 8 || r.width > HV_ATTENTION_MAX_WIDTH || r.width % 8)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "%s: heads of %d are no multiple of 8 up to %d", what,
                r.width, HV_ATTENTION_MAX_WIDTH);
  if (r.window < 0 || (r.window && !r.causal))
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "%s: a window of %d without the causal order", what,
                r.window);
  if (r.most_keys < 0)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "%s: at most %d keys", what, r.most_keys);
  if (!(r.scale > 0.f) || r.scale > 1e30f)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "%s: scale must lie in (0, 1e30]", what);
  if (!need_starts && !r.starts && r.rows != r.batch)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "%s: %d rows for one of each of %d sequences", what,
                r.rows, r.batch);
  const int64_t ld[] = {r.q_ld, r.q_head_ld, r.out_ld, r.out_head_ld};
  for (int64_t l : ld)
    if (l < 0 || l % 8)
      return fail(HV_EVALUE, HV_ERR_DIMENSION, "%s: a stride is no multiple of 8", what);
  if (r.rows == 0 || r.batch == 0) return HV_OK;
  if (!r.q || !r.out || (need_starts && !r.starts))
    return fail(HV_EVALUE, HV_ERR_ADDRESS, "%s: null argument", what);
  if ((((uintptr_t)r.q | (uintptr_t)r.out) & 15) || (((uintptr_t)r.lse | (uintptr_t)r.starts) & 3))
    return fail(HV_EVALUE, HV_ERR_ADDRESS, "%s: a pointer is not aligned", what);
  return HV_OK;
}

static LmAttnArgs args_of(const hv_attention_rows &r) {
  LmAttnArgs a{};
  a.q = r.q; a.out = r.out; a.lse = r.lse; a.starts = r.starts;
  a.q_ld = r.q_ld; a.q_head_ld = r.q_head_ld; a.out_ld = r.out_ld; a.out_head_ld = r.out_head_ld;
  a.rows = r.rows; a.batch = r.batch; a.heads = r.heads; a.kv_heads = r.kv_heads;
  a.group = r.heads / r.kv_heads; a.width = r.width; a.causal = r.causal; a.window = r.window;
  a.most_keys = r.most_keys;
  a.scale = r.scale * 1.4426950408889634f;
  return a;
}

}  // namespace hv

using namespace hv;

extern "C" {

size_t hv_attention_workspace_bytes(int rows, int batch, int heads, int kv_heads, int width) {
  if (rows <= 0 || batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || width <= 0)
    return 0;
  return workspace_of(shape_of(rows, batch, heads, kv_heads, width), width);
}

int hv_attention(const hv_attention_desc *d, void *workspace, size_t workspace_bytes,
                 hv_stream_t stream) {
  clear_error();
  if (!d) return fail(HV_EVALUE, HV_ERR_ADDRESS, "attention: null descriptor");
  const int rc = check_rows("attention", d->rows, true);
  if (rc) return rc;
  if (d->k_rows < 0 || d->k_rows > HV_LM_MAX_ROWS || (!d->k_starts && d->k_rows != d->rows.rows))
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "attention: %d rows of keys", d->k_rows);
  const int64_t ld[] = {d->k_ld, d->k_head_ld, d->v_ld, d->v_head_ld};
  for (int64_t l : ld)
    if (l < 0 || l % 8)
      return fail(HV_EVALUE, HV_ERR_DIMENSION, "attention: a stride is no multiple of 8");
  if (d->k_ld > HV_ATTENTION_MAX_STRIDE || d->v_ld > HV_ATTENTION_MAX_STRIDE)
    return fail(HV_EVALUE, HV_ERR_DIMENSION, "attention: rows of keys or values %lld, %lld apart",
                (long long)d->k_ld, (long long)d->v_ld);
  if (d->rows.rows == 0 || d->rows.batch == 0) return HV_OK;
  if (d->k_rows && (!d->k || !d->v))
    return fail(HV_EVALUE, HV_ERR_ADDRESS, "attention: null argument");
  if ((((uintptr_t)d->k | (uintptr_t)d->v) & 15) || ((uintptr_t)d->k_starts & 3))
    return fail(HV_EVALUE, HV_ERR_ADDRESS, "attention: a pointer is not aligned");
  LmAttnArgs a = args_of(d->rows);
  a.k = d->k; a.v = d->v; a.k_starts = d->k_starts; a.k_rows = d->k_rows;
  a.k_ld = d->k_ld; a.k_head_ld = d->k_head_ld; a.v_ld = d->v_ld; a.v_head_ld = d->v_head_ld;
  const auto attend = d->rows.type == HV_T_F16 ? attend_f16 : attend_bf16;
  return attend(a, false, false, workspace, workspace_bytes, (hipStream_t)stream);
}

int hv_paged_attention(const hv_paged_attention_desc *d, void *workspace, size_t workspace_bytes,
                       hv_stream_t stream) {
  clear_error();
  if (!d) return fail(HV_EVALUE, HV_ERR_ADDRESS, "paged_attention: null descriptor");
  int rc = check_rows("paged_attention", d->rows, false);
  if (rc) return rc;
  rc = check_cache("paged_attention", d->cache, d->rows.type, d->rows.batch, d->rows.kv_heads,
                   d->rows.width);
  if (rc) return rc;
  if (d->rows.rows == 0 || d->rows.batch == 0) return HV_OK;
  LmAttnArgs a = args_of(d->rows);
  a.k = d->cache.k; a.v = d->cache.v; a.k_exps = d->cache.k_exps; a.v_exps = d->cache.v_exps;
  a.table = d->cache.table; a.lengths = d->cache.lengths; a.table_ld = d->cache.table_ld;
  a.map = {d->cache.pages, __builtin_ctz(d->cache.page), d->cache.max_pages};
  const auto attend = d->rows.type == HV_T_F16 ? attend_f16 : attend_bf16;
  return attend(a, true, d->cache.format == HV_CACHE_E4M3, workspace, workspace_bytes,
                (hipStream_t)stream);
}

}  // extern "C"
