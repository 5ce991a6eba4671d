// C-ABI layer of the operators beside the projections (rotary positions, 8-bit key/value cache, low-rank adapters):
// argument validation and dispatch to the launchers.
#include "gq_kv.h"

namespace gq {
namespace {

constexpr int64_t kLargest = (int64_t)1 << 30;

bool misaligned(const void *p, size_t a) { return ((uintptr_t)p % a) != 0; }

int check_rotary(const char *who, const gq_rotary &r, int64_t head_dim) {
  if (r.layout != GQ_ROTARY_INTERLEAVED && r.layout != GQ_ROTARY_HALF)
    return fail(GQ_ERR_UNSUPPORTED, "%s: unknown rotary layout %d", who, r.layout);
  if (r.rotary_dim < 2 || r.rotary_dim % 2 != 0 || r.rotary_dim > head_dim)
    return fail(GQ_ERR_BAD_SHAPE, "%s: rotary_dim=%d must be even, positive and at most head_dim=%lld", who, r.rotary_dim,
                (long long)head_dim);
  if (r.rotary_dim > 256) return fail(GQ_ERR_UNSUPPORTED, "%s: rotary_dim=%d exceeds 256", who, r.rotary_dim);
  if (!r.turns) return fail(GQ_ERR_NULL_POINTER, "%s: rotary.turns is NULL", who);
  if (misaligned(r.turns, 8)) return fail(GQ_ERR_MISALIGNED, "%s: rotary.turns must be 8-byte aligned", who);
  return GQ_OK;
}

// 1: proceed; 0: nothing to do; negative: refused
int check_kv(const char *who, const gq_kv_cache *cache, const gq_kv_batch *batch, KvCache &c, KvBatch &b) {
  if (!cache || !batch) return fail(GQ_ERR_NULL_POINTER, "%s: cache and batch must not be NULL", who);
  if (cache->n_blocks < 0 || cache->kv_heads < 0 || cache->head_dim < 0 || batch->sequences < 0 || batch->table_width < 0 ||
      batch->tokens < 0)
    return fail(GQ_ERR_BAD_SHAPE, "%s: negative size", who);
  if (cache->head_dim % 16 != 0 || cache->head_dim < 16 || cache->head_dim > 256)
    return fail(GQ_ERR_UNSUPPORTED, "%s: head_dim=%d must be a multiple of 16 up to 256", who, cache->head_dim);
  // (what the kernels count in 31 bits; whether a batch of these sizes fits a grid is seen to by the launchers)
  if (cache->n_blocks > kLargest || cache->kv_heads > 1024 || batch->sequences > (1 << 20) || batch->table_width > (1 << 24) ||
      batch->tokens > (1 << 24))
    return fail(GQ_ERR_UNSUPPORTED,
                "%s: more than 2^30 blocks, 1024 kv heads, 2^20 sequences, 2^24 blocks of a sequence or 2^24 rows", who);
  if (batch->tokens == 0 || batch->sequences == 0 || cache->kv_heads == 0) return 0;
  if (!batch->offsets || !batch->seq_lens || (batch->table_width > 0 && !batch->block_table))
    return fail(GQ_ERR_NULL_POINTER, "%s: offsets, seq_lens and block_table must not be NULL", who);
  if (misaligned(batch->offsets, 4) || misaligned(batch->seq_lens, 4) || misaligned(batch->block_table, 4))
    return fail(GQ_ERR_MISALIGNED, "%s: offsets, seq_lens and block_table must be 4-byte aligned", who);
  if (cache->n_blocks > 0 && (!cache->k_codes || !cache->v_codes || !cache->k_scale || !cache->v_scale))
    return fail(GQ_ERR_NULL_POINTER, "%s: the cache's arrays must not be NULL", who);
  if (misaligned(cache->k_codes, 16) || misaligned(cache->v_codes, 16) || misaligned(cache->k_scale, 4) || misaligned(cache->v_scale, 4))
    return fail(GQ_ERR_MISALIGNED, "%s: k_codes and v_codes must be 16-byte, the scales 4-byte aligned", who);
  c = KvCache{cache->k_codes, cache->v_codes, cache->k_scale, cache->v_scale, (int)cache->n_blocks, cache->kv_heads, cache->head_dim};
  b = KvBatch{batch->offsets, batch->seq_lens, batch->block_table, (int)batch->sequences, (int)batch->table_width, (int)batch->tokens};
  return 1;
}

bool bad_stride(int64_t s) { return s < 0 || s > kLargest; }

// a result that is one place of memory many times; the kernels write its rows in no order
int check_apart(const char *who, int64_t rows, int64_t stride, int64_t least) {
  return rows > 1 && stride < least ? fail(GQ_ERR_UNSUPPORTED, "%s: rows of the result lie on each other (%lld of them %lld elements apart)", who,
                                           (long long)rows, (long long)stride)
                                    : GQ_OK;
}

// 1: proceed; 0: nothing to do; negative: refused
int check_adapters(const char *who, const gq_adapters *w, int64_t rows) {
  if (!w) return fail(GQ_ERR_NULL_POINTER, "%s: adapters is NULL", who);
  if (w->n_adapters < 0 || w->rank < 0 || w->in_features < 0 || w->out_features < 0 || rows < 0)
    return fail(GQ_ERR_BAD_SHAPE, "%s: negative size (n_adapters=%lld rank=%lld in_features=%lld out_features=%lld rows=%lld)", who,
                (long long)w->n_adapters, (long long)w->rank, (long long)w->in_features, (long long)w->out_features, (long long)rows);
  if (w->rank < 1 || w->rank > 128) return fail(GQ_ERR_UNSUPPORTED, "%s: rank=%lld outside 1 ... 128", who, (long long)w->rank);
  if (w->n_adapters < 1 || w->n_adapters > 2048)
    return fail(GQ_ERR_UNSUPPORTED, "%s: n_adapters=%lld outside 1 ... 2048", who, (long long)w->n_adapters);
  if (rows > 1 << 24 || w->in_features > 1 << 20 || w->out_features > 1 << 20)
    return fail(GQ_ERR_UNSUPPORTED, "%s: more than 2^24 rows or 2^20 features", who);
  return 1;
}

int check_adapter_pointers(const char *who, const gq_adapters *w) {
  if (!w->down || !w->up || !w->scaling) return fail(GQ_ERR_NULL_POINTER, "%s: down, up and scaling must not be NULL", who);
  if (misaligned(w->down, 2) || misaligned(w->up, 2) || misaligned(w->scaling, 4))
    return fail(GQ_ERR_MISALIGNED, "%s: down and up must be 2-byte, scaling 4-byte aligned", who);
  return GQ_OK;
}

int check_workspace(const char *who, const void *workspace, int64_t bytes, int64_t need, size_t align) {
  if (need <= 0) return GQ_OK;
  if (!workspace) return fail(GQ_ERR_NULL_POINTER, "%s: workspace is NULL", who);
  if (misaligned(workspace, align)) return fail(GQ_ERR_MISALIGNED, "%s: workspace must be %d-byte aligned", who, (int)align);
  if (bytes < need) return fail(GQ_ERR_BAD_SHAPE, "%s: workspace of %lld bytes, need %lld", who, (long long)bytes, (long long)need);
  return GQ_OK;
}

}  // namespace
}  // namespace gq

extern "C" {

int gq_rotary_f16(const uint16_t *t, int64_t t_token_stride, int64_t t_head_stride, const int32_t *positions,
                  const gq_rotary *rotary, int32_t inverse, uint16_t *out, int64_t out_token_stride, int64_t out_head_stride,
                  int64_t tokens, int64_t heads, int64_t head_dim, void *stream) {
  const char *who = "gq_rotary_f16";
  if (!rotary) return gq::fail(GQ_ERR_NULL_POINTER, "%s: rotary is NULL", who);
  if (tokens < 0 || heads < 0 || head_dim < 0) return gq::fail(GQ_ERR_BAD_SHAPE, "%s: negative size", who);
  if (tokens == 0 || heads == 0 || head_dim == 0) return GQ_OK;
  if (const int rc = gq::check_rotary(who, *rotary, head_dim)) return rc;
  if (tokens > 1 << 24 || heads > 65535 || head_dim > 2048)
    return gq::fail(GQ_ERR_UNSUPPORTED, "%s: more than 2^24 tokens, 65535 heads or a head_dim over 2048", who);
  if (!t || !positions || !out) return gq::fail(GQ_ERR_NULL_POINTER, "%s: t, positions and out must not be NULL", who);
  if (gq::misaligned(t, 2) || gq::misaligned(out, 2) || gq::misaligned(positions, 4))
    return gq::fail(GQ_ERR_MISALIGNED, "%s: t and out must be 2-byte, positions 4-byte aligned", who);
  if (gq::bad_stride(t_token_stride) || gq::bad_stride(t_head_stride) || gq::bad_stride(out_token_stride) || gq::bad_stride(out_head_stride))
    return gq::fail(GQ_ERR_UNSUPPORTED, "%s: a stride is negative or exceeds 2^30", who);
  if (t == out && (t_token_stride != out_token_stride || t_head_stride != out_head_stride))
    return gq::fail(GQ_ERR_UNSUPPORTED, "%s: in place, t and out must have the same strides", who);
  if (const int rc = gq::check_apart(who, tokens, out_token_stride, 1)) return rc;
  if (const int rc = gq::check_apart(who, heads, out_head_stride, 1)) return rc;
  return gq::launch_rotary(t, t_token_stride, t_head_stride, positions, *rotary, inverse != 0, out, out_token_stride,
                           out_head_stride, tokens, heads, head_dim, (hipStream_t)stream);
}

int gq_kv_append_f16(const gq_kv_cache *cache, const gq_kv_batch *batch, const uint16_t *k, int64_t k_token_stride,
                     int64_t k_head_stride, const uint16_t *v, int64_t v_token_stride, int64_t v_head_stride,
                     const gq_rotary *rotary, void *stream) {
  const char *who = "gq_kv_append_f16";
  gq::KvCache c;
  gq::KvBatch b;
  const int rc = gq::check_kv(who, cache, batch, c, b);
  if (rc <= 0) return rc;
  if (!k || !v) return gq::fail(GQ_ERR_NULL_POINTER, "%s: k and v must not be NULL", who);
  if (gq::bad_stride(k_token_stride) || gq::bad_stride(k_head_stride) || gq::bad_stride(v_token_stride) || gq::bad_stride(v_head_stride))
    return gq::fail(GQ_ERR_UNSUPPORTED, "%s: a stride is negative or exceeds 2^30", who);
  if (gq::misaligned(k, 16) || gq::misaligned(v, 16) || (k_token_stride | k_head_stride | v_token_stride | v_head_stride) % 8 != 0)
    return gq::fail(GQ_ERR_MISALIGNED, "%s: every row of k and v must be 16-byte aligned (strides multiples of 8)", who);
  if (rotary) {
    if (const int bad = gq::check_rotary(who, *rotary, cache->head_dim)) return bad;
    if (rotary->rotary_dim % (rotary->layout == GQ_ROTARY_HALF ? 16 : 8) != 0)
      return gq::fail(GQ_ERR_UNSUPPORTED, "%s: rotary_dim=%d must be a multiple of 8 (interleaved) or 16 (half): turn the keys with gq_rotary_f16 first",
                      who, rotary->rotary_dim);
  }
  return gq::launch_kv_append(c, b, k, k_token_stride, k_head_stride, v, v_token_stride, v_head_stride, rotary, (hipStream_t)stream);
}

int gq_kv_gather_f16(const gq_kv_cache *cache, const gq_kv_batch *batch, uint16_t *k, uint16_t *v, void *stream) {
  const char *who = "gq_kv_gather_f16";
  gq::KvCache c;
  gq::KvBatch b;
  const int rc = gq::check_kv(who, cache, batch, c, b);
  if (rc <= 0) return rc;
  if (!k || !v) return gq::fail(GQ_ERR_NULL_POINTER, "%s: k and v must not be NULL", who);
  if (gq::misaligned(k, 16) || gq::misaligned(v, 16)) return gq::fail(GQ_ERR_MISALIGNED, "%s: k and v must be 16-byte aligned", who);
  if (k == v) return gq::fail(GQ_ERR_UNSUPPORTED, "%s: the results lie on each other", who);
  return gq::launch_kv_gather(c, b, k, v, (hipStream_t)stream);
}

int64_t gq_kv_attention_workspace_bytes(int64_t head_dim) {
  if (head_dim < 16 || head_dim > 256 || head_dim % 16 != 0)
    return gq::fail(GQ_ERR_UNSUPPORTED, "gq_kv_attention_workspace_bytes: head_dim=%lld must be a multiple of 16 up to 256", (long long)head_dim);
  return gq::kv_attention_workspace_bytes(head_dim);
}

int gq_kv_attention_f16(const gq_kv_cache *cache, const gq_kv_batch *batch, const uint16_t *q, int64_t q_token_stride,
                        int64_t q_head_stride, uint16_t *out, int64_t out_token_stride, int64_t out_head_stride,
                        int64_t q_heads, float scale, void *workspace, int64_t workspace_bytes, void *stream) {
  const char *who = "gq_kv_attention_f16";
  gq::KvCache c;
  gq::KvBatch b;
  const int rc = gq::check_kv(who, cache, batch, c, b);
  if (rc <= 0) return rc;
  if (q_heads <= 0 || q_heads % cache->kv_heads != 0)
    return gq::fail(GQ_ERR_BAD_SHAPE, "%s: q_heads=%lld is not a multiple of kv_heads=%d", who, (long long)q_heads, cache->kv_heads);
  if (q_heads > 65535 || q_heads * batch->tokens > gq::kLargest)
    return gq::fail(GQ_ERR_UNSUPPORTED, "%s: more than 65535 query heads or 2^30 rows of them", who);
  if (!q || !out) return gq::fail(GQ_ERR_NULL_POINTER, "%s: q and out must not be NULL", who);
  if (gq::bad_stride(q_token_stride) || gq::bad_stride(q_head_stride) || gq::bad_stride(out_token_stride) || gq::bad_stride(out_head_stride))
    return gq::fail(GQ_ERR_UNSUPPORTED, "%s: a stride is negative or exceeds 2^30", who);
  if (gq::misaligned(q, 16) || (q_token_stride | q_head_stride) % 8 != 0 || gq::misaligned(out, 2))
    return gq::fail(GQ_ERR_MISALIGNED, "%s: every row of q must be 16-byte aligned (strides multiples of 8), out 2-byte", who);
  if (const int bad = gq::check_workspace(who, workspace, workspace_bytes, gq::kv_attention_workspace_bytes(cache->head_dim), 16)) return bad;
  if (out == q)  // (a row of q is read by the workgroups of several ranges of blocks)
    return gq::fail(GQ_ERR_UNSUPPORTED, "%s: out must not be q", who);
  if (const int bad = gq::check_apart(who, b.tokens, out_token_stride, 1)) return bad;
  if (const int bad = gq::check_apart(who, q_heads, out_head_stride, 1)) return bad;
  return gq::launch_kv_attention(c, b, q, q_token_stride, q_head_stride, out, out_token_stride, out_head_stride, q_heads, scale,
                                 workspace, (hipStream_t)stream);
}

int64_t gq_adapter_plan_bytes(int64_t rows, int64_t n_adapters) {
  if (rows < 0 || n_adapters < 0) return gq::fail(GQ_ERR_BAD_SHAPE, "gq_adapter_plan_bytes: negative size");
  if (rows > 1 << 24 || n_adapters < 1 || n_adapters > 2048)
    return gq::fail(GQ_ERR_UNSUPPORTED, "gq_adapter_plan_bytes: n_adapters outside 1 ... 2048 or more than 2^24 rows");
  return gq::adapter_plan_bytes(rows, n_adapters);
}

int gq_adapter_plan(const int32_t *ids, int64_t rows, int64_t n_adapters, void *plan, int64_t plan_bytes, void *stream) {
  const char *who = "gq_adapter_plan";
  const int64_t need = gq_adapter_plan_bytes(rows, n_adapters);
  if (need < 0) return (int)need;
  if (rows == 0) return GQ_OK;
  if (!ids || !plan) return gq::fail(GQ_ERR_NULL_POINTER, "%s: ids and plan must not be NULL", who);
  if (gq::misaligned(ids, 4) || gq::misaligned(plan, 16))
    return gq::fail(GQ_ERR_MISALIGNED, "%s: ids must be 4-byte, plan 16-byte aligned", who);
  if (plan_bytes < need) return gq::fail(GQ_ERR_BAD_SHAPE, "%s: plan of %lld bytes, need %lld", who, (long long)plan_bytes, (long long)need);
  return gq::launch_adapter_plan(ids, rows, n_adapters, plan, (hipStream_t)stream);
}

int64_t gq_adapter_apply_workspace_bytes(const gq_adapters *adapters, int64_t rows) {
  const int rc = gq::check_adapters("gq_adapter_apply_workspace_bytes", adapters, rows);
  if (rc < 0) return rc;
  return rows == 0 ? 0 : gq::adapter_apply_workspace_bytes(rows, adapters->n_adapters, adapters->in_features, adapters->rank);
}

int gq_adapter_apply_f16(const gq_adapters *adapters, const void *plan, int64_t rows, const uint16_t *x, int64_t x_row_stride,
                         const uint16_t *y, int64_t y_row_stride, uint16_t *out, int64_t out_row_stride, int32_t activation,
                         void *workspace, int64_t workspace_bytes, void *stream) {
  const char *who = "gq_adapter_apply_f16";
  int rc = gq::check_adapters(who, adapters, rows);
  if (rc < 0) return rc;
  if (activation < GQ_ACT_NONE || activation > GQ_ACT_GELU_TANH)
    return gq::fail(GQ_ERR_UNSUPPORTED, "%s: unknown activation %d", who, activation);
  if (rows == 0 || adapters->out_features == 0) return GQ_OK;
  if (adapters->in_features == 0) return gq::fail(GQ_ERR_UNSUPPORTED, "%s: in_features is 0", who);
  rc = gq::check_adapter_pointers(who, adapters);
  if (rc != GQ_OK) return rc;
  if (!plan || !x || !out) return gq::fail(GQ_ERR_NULL_POINTER, "%s: plan, x and out must not be NULL", who);
  if (gq::misaligned(plan, 16) || gq::misaligned(x, 2) || gq::misaligned(y, 2) || gq::misaligned(out, 2))
    return gq::fail(GQ_ERR_MISALIGNED, "%s: plan must be 16-byte, x, y and out 2-byte aligned", who);
  if (gq::bad_stride(x_row_stride) || gq::bad_stride(y_row_stride) || gq::bad_stride(out_row_stride))
    return gq::fail(GQ_ERR_UNSUPPORTED, "%s: a stride is negative or exceeds 2^30", who);
  if (y == out && y_row_stride != out_row_stride)
    return gq::fail(GQ_ERR_UNSUPPORTED, "%s: in place, y and out must have the same stride", who);
  rc = gq::check_apart(who, rows, out_row_stride, adapters->out_features);
  if (rc != GQ_OK) return rc;
  rc = gq::check_workspace(who, workspace, workspace_bytes,
                           gq::adapter_apply_workspace_bytes(rows, adapters->n_adapters, adapters->in_features, adapters->rank), 256);
  if (rc != GQ_OK) return rc;
  return gq::launch_adapter_apply(*adapters, plan, rows, x, x_row_stride, y, y_row_stride, out, out_row_stride, activation, workspace,
                                  (hipStream_t)stream);
}

int64_t gq_adapter_grad_workspace_bytes(const gq_adapters *adapters, int64_t rows) {
  const int rc = gq::check_adapters("gq_adapter_grad_workspace_bytes", adapters, rows);
  if (rc < 0) return rc;
  return rows == 0 ? 0
                   : gq::adapter_grad_workspace_bytes(rows, adapters->n_adapters, adapters->in_features, adapters->out_features, adapters->rank);
}

int gq_adapter_grad_f16(const gq_adapters *adapters, const void *plan, int64_t rows, const uint16_t *x, int64_t x_row_stride,
                        const uint16_t *dy, int64_t dy_row_stride, const uint16_t *dx, int64_t dx_row_stride, uint16_t *dx_out,
                        int64_t dx_out_row_stride, float *d_down, float *d_up, void *workspace, int64_t workspace_bytes,
                        void *stream) {
  const char *who = "gq_adapter_grad_f16";
  int rc = gq::check_adapters(who, adapters, rows);
  if (rc < 0) return rc;
  if (rows == 0 || adapters->in_features == 0 || adapters->out_features == 0)
    return gq::fail(GQ_ERR_UNSUPPORTED, "%s: no rows or no features", who);
  rc = gq::check_adapter_pointers(who, adapters);
  if (rc != GQ_OK) return rc;
  if (!plan || !x || !dy || !dx_out || !d_down || !d_up)
    return gq::fail(GQ_ERR_NULL_POINTER, "%s: plan, x, dy, dx_out, d_down and d_up must not be NULL", who);
  if (gq::misaligned(plan, 16) || gq::misaligned(x, 2) || gq::misaligned(dy, 2) || gq::misaligned(dx, 2) || gq::misaligned(dx_out, 2) ||
      gq::misaligned(d_down, 4) || gq::misaligned(d_up, 4))
    return gq::fail(GQ_ERR_MISALIGNED, "%s: plan must be 16-byte, x, dy, dx and dx_out 2-byte, d_down and d_up 4-byte aligned", who);
  if (gq::bad_stride(x_row_stride) || gq::bad_stride(dy_row_stride) || gq::bad_stride(dx_row_stride) || gq::bad_stride(dx_out_row_stride))
    return gq::fail(GQ_ERR_UNSUPPORTED, "%s: a stride is negative or exceeds 2^30", who);
  if (dx == dx_out && dx_row_stride != dx_out_row_stride)
    return gq::fail(GQ_ERR_UNSUPPORTED, "%s: in place, dx and dx_out must have the same stride", who);
  if (dx_out == x || dx_out == dy)  // (both are read again behind it)
    return gq::fail(GQ_ERR_UNSUPPORTED, "%s: dx_out must not be x or dy", who);
  rc = gq::check_apart(who, rows, dx_out_row_stride, adapters->in_features);
  if (rc != GQ_OK) return rc;
  rc = gq::check_workspace(who, workspace, workspace_bytes,
                           gq::adapter_grad_workspace_bytes(rows, adapters->n_adapters, adapters->in_features, adapters->out_features,
                                                            adapters->rank), 256);
  if (rc != GQ_OK) return rc;
  return gq::launch_adapter_grad(*adapters, plan, rows, x, x_row_stride, dy, dy_row_stride, dx, dx_row_stride, dx_out, dx_out_row_stride,
                                 d_down, d_up, workspace, (hipStream_t)stream);
}

}  // extern "C"
