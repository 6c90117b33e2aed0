// extern "C" entry points of the key / value cache held in 4 bits (declared in
// include/zentorch_hip.h): argument validation and launch.
#include "capi_cache.hpp"
#include "mx4.hpp"

namespace {

using namespace zt;

// Of the write and the read, so that sizes in bytes fit 64 bits.
constexpr int64_t kMostTokens = (int64_t)1 << 36;

int64_t blocks_of_row(const zt_kv_cache_mxfp4 *c) { return (c->head_dim + kMxBlock - 1) / kMxBlock; }

int check_cache(const char *op, const zt_kv_cache_mxfp4 *c, int32_t dtype) {
  if (!c) return api_fail(ZT_EINVAL, "%s: null cache", op);
  if (!is_float_dt(dtype)) return api_fail(ZT_EINVAL, "%s: the other tensors must be bf16 or fp32", op);
  if (c->pages < 0 || c->heads <= 0 || c->page_size <= 0 || c->head_dim <= 0)
    return api_fail(ZT_EINVAL, "%s: need pages >= 0 and heads, page_size, head_dim > 0", op);
  if (c->head_dim % 8 || c->head_dim > 256)
    return api_fail(ZT_EUNSUPPORTED, "%s: head_dim must be a multiple of 8 up to 256, got %lld", op,
                    (long long)c->head_dim);
  if (c->pages > INT32_MAX || c->heads > 65535 || c->page_size > INT32_MAX)
    return api_fail(ZT_EUNSUPPORTED, "%s: cache sizes exceed 32 bits, or 65535 heads", op);
  for (int i = 0; i < 3; ++i)
    if (c->k_strides[i] < 0 || c->v_strides[i] < 0 || c->k_scale_strides[i] < 0 || c->v_scale_strides[i] < 0)
      return api_fail(ZT_EINVAL, "%s: cache strides must not be negative", op);
  return ZT_OK;
}

// The pointers, and the codes' rows on 16 bytes.
int check_data(const char *op, const zt_kv_cache_mxfp4 *c) {
  if (c->pages > 0 && (!c->k || !c->v || !c->k_scales || !c->v_scales))
    return api_fail(ZT_EINVAL, "%s: null cache pointer", op);
  if (!divides16(c->k, {c->k_strides[0], c->k_strides[1], c->k_strides[2]}, 1) ||
      !divides16(c->v, {c->v_strides[0], c->v_strides[1], c->v_strides[2]}, 1))
    return api_fail(ZT_EUNSUPPORTED, "%s: the cache needs 16-byte aligned rows of codes", op);
  return ZT_OK;
}

Mx4Rows rows_of(void *codes, const int64_t *ld, uint8_t *scales, const int64_t *sc_ld) {
  Mx4Rows r{static_cast<uint8_t *>(codes), scales, {}, {}};
  for (int i = 0; i < 3; ++i) r.ld[i] = ld[i], r.sc_ld[i] = sc_ld[i];
  return r;
}
Mx4Rows keys_of(const zt_kv_cache_mxfp4 *c) { return rows_of(c->k, c->k_strides, c->k_scales, c->k_scale_strides); }
Mx4Rows values_of(const zt_kv_cache_mxfp4 *c) { return rows_of(c->v, c->v_strides, c->v_scales, c->v_scale_strides); }

// The cache's four arrays.
struct CacheRows {
  Strided k, v, k_scales, v_scales;
};
CacheRows arrays_of(const zt_kv_cache_mxfp4 *c) {
  auto of = [&](const void *p, int64_t row, const int64_t *ld) {
    return Strided{p, row * blocks_of_row(c), {c->pages, c->heads, c->page_size}, {ld[0], ld[1], ld[2]}};
  };
  return {of(c->k, 16, c->k_strides), of(c->v, 16, c->v_strides), of(c->k_scales, 1, c->k_scale_strides),
          of(c->v_scales, 1, c->v_scale_strides)};
}
bool touches_cache(const Span &s, const zt_kv_cache_mxfp4 *c, std::initializer_list<Span> others) {
  const CacheRows r = arrays_of(c);
  return touches(s, others, {r.k, r.v, r.k_scales, r.v_scales});
}

}  // namespace

extern "C" {

int zt_rotary_cache_append_mxfp4(const void *q, int32_t dtype, int64_t T, int64_t H, const int64_t *q_strides,
                                 const void *k, const int64_t *k_strides, const void *v,
                                 const int64_t *v_strides, const int64_t *positions,
                                 const float *table, int64_t length, int64_t R, int64_t ld_table,
                                 int32_t interleaved, const int64_t *slots,
                                 const zt_kv_cache_mxfp4 *cache, void *q_out, zt_stream_t stream) {
  static const char *op = "zt_rotary_cache_append_mxfp4";
  if (const int rc = check_cache(op, cache, dtype)) return rc;
  const int64_t D = cache->head_dim, KV = cache->heads;
  if (const int rc = check_rotary(op, q, T, H, D, positions, table, length, R, ld_table, q_out)) return rc;
  if (!q_strides || !k_strides || !v_strides) return api_fail(ZT_EINVAL, "%s: null strides", op);
  if (H > 65535) return api_fail(ZT_EUNSUPPORTED, "%s: at most 65535 heads", op);
  if (T > kMostTokens) return api_fail(ZT_EUNSUPPORTED, "%s: too many tokens for one call", op);
  if (T == 0) return ZT_OK;
  if (!k || !v || !slots) return api_fail(ZT_EINVAL, "%s: null tensor pointer", op);
  if (const int rc = check_data(op, cache)) return rc;
  const int64_t es = dtype == ZT_DT_F32 ? 4 : 2;
  const Span out{q_out, T * H * D, es};
  if (touches_rows(out, q, T, H, D, q_strides[0], q_strides[1], es) ||
      touches_rows(out, k, T, KV, D, k_strides[0], k_strides[1], es) ||
      touches_rows(out, v, T, KV, D, v_strides[0], v_strides[1], es) ||
      touches(out, Strided{table, R * 4, {length, 1, 1}, {ld_table * 4, 0, 0}}) ||
      touches_cache(out, cache, {{positions, T, 8}, {slots, T, 8}}))
    return api_fail(ZT_EINVAL, "%s: the output overlaps an input or the cache", op);
  Mx4AppendArgs a{};
  a.q = q, a.k = k, a.v = v, a.q_out = q_out;
  for (int i = 0; i < 2; ++i) a.q_ld[i] = q_strides[i], a.k_ld[i] = k_strides[i], a.v_ld[i] = v_strides[i];
  a.keys = keys_of(cache), a.values = values_of(cache);
  a.pos = positions, a.slots = slots, a.table = table, a.length = length, a.table_ld = ld_table;
  a.pages = cache->pages, a.page_size = (int)cache->page_size;
  a.T = T, a.H = (int)H, a.KV = (int)KV, a.D = (int)D, a.R = (int)R, a.NB = (int)blocks_of_row(cache);
  a.interleaved = interleaved != 0;
  // eight elements lie within a half, and loads of 16 bytes are aligned
  const bool wide = R % (a.interleaved ? 8 : 16) == 0 && divides16(q, {q_strides[0], q_strides[1]}, es) &&
                    divides16(k, {k_strides[0], k_strides[1]}, es) &&
                    divides16(v, {v_strides[0], v_strides[1]}, es) && divides16(q_out, {}, es);
  return hip_status(launch_append_mx4(a, dtype, wide, reinterpret_cast<hipStream_t>(stream)), op);
}

int zt_cache_read_mxfp4(const zt_kv_cache_mxfp4 *cache, const int64_t *slots, int64_t n, int32_t dtype,
                        void *k_out, void *v_out, zt_stream_t stream) {
  static const char *op = "zt_cache_read_mxfp4";
  if (const int rc = check_cache(op, cache, dtype)) return rc;
  if (n < 0) return api_fail(ZT_EINVAL, "%s: need n >= 0", op);
  if (n == 0) return ZT_OK;
  if (!slots || !k_out || !v_out) return api_fail(ZT_EINVAL, "%s: null tensor pointer", op);
  if (const int rc = check_data(op, cache)) return rc;
  if (n > kMostTokens) return api_fail(ZT_EUNSUPPORTED, "%s: too many tokens for one call", op);
  const int64_t es = dtype == ZT_DT_F32 ? 4 : 2, rows = n * cache->heads * cache->head_dim;
  if (!divides16(k_out, {}, es) || !divides16(v_out, {}, es))
    return api_fail(ZT_EUNSUPPORTED, "%s: the outputs need 16-byte alignment", op);
  if (const int rc = check_apart(op, {{slots, n, 8}}, {{k_out, rows, es}, {v_out, rows, es}})) return rc;
  if (touches_cache({k_out, rows, es}, cache, {}) || touches_cache({v_out, rows, es}, cache, {}))
    return api_fail(ZT_EINVAL, "%s: an output overlaps the cache", op);
  Mx4ReadArgs a{};
  a.keys = keys_of(cache), a.values = values_of(cache);
  a.slots = slots, a.n = n, a.pages = cache->pages, a.page_size = (int)cache->page_size;
  a.KV = (int)cache->heads, a.D = (int)cache->head_dim, a.k_out = k_out, a.v_out = v_out;
  return hip_status(launch_read_mx4(a, dtype, reinterpret_cast<hipStream_t>(stream)), op);
}

// The checked arguments of an attention call, without its pointers.
static int checked_attn(const char *op, int64_t T, int64_t H, int32_t dtype, const zt_kv_cache_mxfp4 *c, int64_t S,
                        int64_t W, int64_t max_query_len, int32_t causal, int64_t window, Mx4AttnArgs *a) {
  if (const int rc = check_cache(op, c, dtype)) return rc;
  zt_kv_cache sizes{};
  sizes.dtype = dtype, sizes.pages = c->pages, sizes.heads = c->heads;
  sizes.page_size = c->page_size, sizes.head_dim = c->head_dim;
  *a = Mx4AttnArgs{};
  if (const int rc = attn_args(op, T, H, &sizes, S, W, max_query_len, causal, window, a)) return rc;
  a->NB = (int)blocks_of_row(c);
  if (T > 0 && !paged_attn_mx4_countable(*a))
    return api_fail(ZT_EUNSUPPORTED, "%s: too many tokens over too long tables for one call", op);
  return ZT_OK;
}

size_t zt_paged_attention_mxfp4_workspace_size(int64_t T, int64_t H, int32_t dtype,
                                               const zt_kv_cache_mxfp4 *cache, int64_t S, int64_t W,
                                               int64_t max_query_len) {
  Mx4AttnArgs a;
  if (checked_attn("zt_paged_attention_mxfp4_workspace_size", T, H, dtype, cache, S, W, max_query_len, 0, 0, &a))
    return 0;
  return paged_attn_mx4_workspace(a);
}

int zt_paged_attention_mxfp4(const void *q, int32_t dtype, int64_t T, int64_t H, int64_t ld_token, int64_t ld_head,
                             const zt_kv_cache_mxfp4 *cache, const int32_t *block_table, int64_t S, int64_t W,
                             const int32_t *cu_seqlens, const int32_t *context_lens, int64_t max_query_len,
                             int32_t causal, int64_t window, float scale, void *out, void *workspace,
                             size_t workspace_bytes, zt_stream_t stream) {
  static const char *op = "zt_paged_attention_mxfp4";
  Mx4AttnArgs a;
  if (const int rc = checked_attn(op, T, H, dtype, cache, S, W, max_query_len, causal, window, &a)) return rc;
  if (!std::isfinite(scale)) return api_fail(ZT_EINVAL, "%s: scale must be finite", op);
  if (T == 0) return ZT_OK;
  if (!q || !out || !cu_seqlens || (S > 0 && !context_lens) || (S * W > 0 && !block_table))
    return api_fail(ZT_EINVAL, "%s: null tensor pointer", op);
  if (const int rc = check_data(op, cache)) return rc;
  const int64_t es = dtype == ZT_DT_F32 ? 4 : 2;
  if (!divides16(q, {ld_token, ld_head}, es) || !divides16(out, {}, es))
    return api_fail(ZT_EUNSUPPORTED, "%s: query and output need 16-byte aligned rows", op);
  // the kernels count a layer's rows in units of 16 bytes, in 32 bits
  for (const int64_t *st : {cache->k_strides, cache->v_strides})
    if ((double)cache->pages * (double)st[0] + (double)cache->page_size * (double)st[2] >= 4294967295.0 * 16)
      return api_fail(ZT_EUNSUPPORTED, "%s: one head's keys or values span 64 GB and more", op);
  const size_t need = paged_attn_mx4_workspace(a);
  if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
    return api_fail(ZT_EINVAL, "%s: 16-byte aligned workspace of %zu bytes needed, %zu given", op, need,
                    workspace ? workspace_bytes : (size_t)0);
  const Span to{out, T * H * cache->head_dim, es}, scratch{workspace, (int64_t)need, 1};
  if (touches_rows(to, q, T, H, cache->head_dim, ld_token, ld_head, es) || overlap(to, scratch) ||
      touches_rows(scratch, q, T, H, cache->head_dim, ld_token, ld_head, es))
    return api_fail(ZT_EINVAL, "%s: query, output and workspace must not overlap", op);
  for (const Span &s : {to, scratch})
    if (touches_cache(s, cache, {{block_table, S * W, 4}, {cu_seqlens, S + 1, 4}, {context_lens, S, 4}}))
      return api_fail(ZT_EINVAL, "%s: output or workspace overlap the cache, the table or the lengths", op);
  a.q = q, a.q_ld[0] = ld_token, a.q_ld[1] = ld_head;
  a.k = cache->k, a.v = cache->v, a.k_sc = cache->k_scales, a.v_sc = cache->v_scales;
  for (int i = 0; i < 3; ++i) {
    a.k_ld[i] = cache->k_strides[i], a.v_ld[i] = cache->v_strides[i];
    a.k_sc_ld[i] = cache->k_scale_strides[i], a.v_sc_ld[i] = cache->v_scale_strides[i];
  }
  a.table = block_table, a.cu = cu_seqlens, a.ctx = context_lens, a.scale = scale, a.out = out;
  return hip_status(launch_paged_attn_mx4(a, workspace, reinterpret_cast<hipStream_t>(stream)), op);
}

}  // extern "C"
