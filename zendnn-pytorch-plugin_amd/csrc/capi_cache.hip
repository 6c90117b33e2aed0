// extern "C" entry points of the paged key / value cache (declared in
// include/zentorch_hip.h): argument validation and launch.
#include "capi_cache.hpp"

namespace {

using namespace zt;

// The sizes and strides of a cache (ZT_OK or the error code).
int check_cache(const char *op, const zt_kv_cache *c, bool need_data) {
  if (!c) return api_fail(ZT_EINVAL, "%s: null cache", op);
  if (!is_float_dt(c->dtype)) return api_fail(ZT_EINVAL, "%s: the cache must be bf16 or fp32", op);
  if (c->pages < 0 || c->heads <= 0 || c->page_size <= 0 || c->head_dim <= 0)
    return api_fail(ZT_EINVAL, "%s: need pages >= 0 and heads, page_size, head_dim > 0", op);
  if (c->pages > INT32_MAX || c->heads > INT32_MAX || c->page_size > INT32_MAX ||
      c->head_dim > INT32_MAX)
    return api_fail(ZT_EUNSUPPORTED, "%s: cache sizes exceed 32 bits", op);
  for (int i = 0; i < 3; ++i)
    if (c->k_strides[i] < 0 || c->v_strides[i] < 0)
      return api_fail(ZT_EINVAL, "%s: cache strides must not be negative", op);
  if (need_data && c->pages > 0 && (!c->k || !c->v))
    return api_fail(ZT_EINVAL, "%s: null cache pointer", op);
  return ZT_OK;
}

}  // namespace

extern "C" {

int zt_rotary_embedding(const void *x, int32_t dtype, int64_t T, int64_t H, int64_t D,
                        int64_t ld_token, int64_t ld_head, const int64_t *positions,
                        const float *table, int64_t length, int64_t R, int64_t ld_table,
                        int32_t interleaved, void *out, zt_stream_t stream) {
  static const char *op = "zt_rotary_embedding";
  if (!is_float_dt(dtype)) return api_fail(ZT_EINVAL, "%s: input must be bf16 or fp32", op);
  if (const int rc = check_rotary(op, x, T, H, D, positions, table, length, R, ld_table, out)) return rc;
  if (too_many(T, H, D)) return api_fail(ZT_EUNSUPPORTED, "%s: sizes exceed the grid", op);
  if (T == 0) return ZT_OK;
  const int64_t es = dtype == ZT_DT_F32 ? 4 : 2;
  zt::RotaryArgs a{};
  a.q = x, a.q_ld[0] = ld_token, a.q_ld[1] = ld_head, a.q_out = out;
  a.pos = positions, a.table = table, a.length = length, a.table_ld = ld_table;
  a.T = T, a.H = (int)H, a.KV = 0, a.D = (int)D, a.R = (int)R, a.page_size = 1;
  a.interleaved = interleaved != 0;
  const bool wide = divides16(x, {ld_token, ld_head, D, R / 2}, es) && divides16(out, {}, es);
  return hip_status(zt::launch_rotary(a, dtype, wide, reinterpret_cast<hipStream_t>(stream)), op);
}

int zt_rotary_cache_append(const void *q, int64_t T, int64_t H, const int64_t *q_strides,
                           const void *k, const int64_t *k_strides, const void *v,
                           const int64_t *v_strides, const int64_t *positions,
                           const float *table, int64_t length, int64_t R, int64_t ld_table,
                           int32_t interleaved, const int64_t *slots, const zt_kv_cache *cache,
                           void *q_out, zt_stream_t stream) {
  static const char *op = "zt_rotary_cache_append";
  if (const int rc = check_cache(op, cache, true)) return rc;
  const int64_t D = cache->head_dim, KV = cache->heads;
  if (const int rc = check_rotary(op, q, T, H, D, positions, table, length, R, ld_table, q_out)) return rc;
  if (!q_strides || !k_strides || !v_strides) return api_fail(ZT_EINVAL, "%s: null strides", op);
  if (T > 0 && (!k || !v || !slots)) return api_fail(ZT_EINVAL, "%s: null tensor pointer", op);
  if (too_many(T, H + 2 * KV, D)) return api_fail(ZT_EUNSUPPORTED, "%s: sizes exceed the grid", op);
  if (T == 0) return ZT_OK;
  const int64_t es = cache->dtype == ZT_DT_F32 ? 4 : 2;
  zt::RotaryArgs a{};
  a.q = q, a.k = k, a.v = v, a.q_out = q_out;
  a.k_cache = cache->k, a.v_cache = cache->v;
  for (int i = 0; i < 2; ++i) a.q_ld[i] = q_strides[i], a.k_ld[i] = k_strides[i], a.v_ld[i] = v_strides[i];
  for (int i = 0; i < 3; ++i) a.kc_ld[i] = cache->k_strides[i], a.vc_ld[i] = cache->v_strides[i];
  a.pos = positions, a.slots = slots, a.table = table, a.length = length, a.table_ld = ld_table;
  a.pages = cache->pages, a.page_size = (int)cache->page_size;
  a.T = T, a.H = (int)H, a.KV = (int)KV, a.D = (int)D, a.R = (int)R;
  a.interleaved = interleaved != 0;
  const bool wide =
      divides16(q, {q_strides[0], q_strides[1], D, R / 2}, es) &&
      divides16(k, {k_strides[0], k_strides[1]}, es) && divides16(v, {v_strides[0], v_strides[1]}, es) &&
      divides16(q_out, {}, es) &&
      divides16(cache->k, {cache->k_strides[0], cache->k_strides[1], cache->k_strides[2]}, es) &&
      divides16(cache->v, {cache->v_strides[0], cache->v_strides[1], cache->v_strides[2]}, es);
  return hip_status(zt::launch_rotary(a, cache->dtype, wide, reinterpret_cast<hipStream_t>(stream)), op);
}

int zt_cache_extend(const int32_t *block_table, const int32_t *context_lens,
                    const int32_t *ref_counts, const int32_t *cu_seqlens, int64_t S, int64_t W,
                    int64_t pages, int64_t page_size, int64_t T, int32_t *table_out,
                    int32_t *context_out, int32_t *refs_out, int64_t *positions, int64_t *slots,
                    zt_stream_t stream) {
  static const char *op = "zt_cache_extend";
  if (S < 0 || W < 0 || pages < 0 || page_size <= 0 || T < 0)
    return api_fail(ZT_EINVAL, "%s: need S, W, pages, T >= 0 and page_size > 0", op);
  if (S > kMaxRows) return api_fail(ZT_EUNSUPPORTED, "%s: at most %lld sequences", op, (long long)kMaxRows);
  if (W > (1 << 24) || pages > INT32_MAX || page_size > (1 << 24) || W * page_size >= (1 << 30) ||
      S * W >= (1 << 30))
    return api_fail(ZT_EUNSUPPORTED, "%s: sizes exceed 32 bits", op);
  if ((S * W > 0 && (!block_table || !table_out)) || (pages > 0 && (!ref_counts || !refs_out)) ||
      (S > 0 && (!context_lens || !context_out)) || !cu_seqlens || (T > 0 && (!positions || !slots)))
    return api_fail(ZT_EINVAL, "%s: null tensor pointer", op);
  if (const int rc = check_apart(
          op, {{block_table, S * W, 4}, {context_lens, S, 4}, {ref_counts, pages, 4}, {cu_seqlens, S + 1, 4}},
          {{table_out, S * W, 4}, {context_out, S, 4}, {refs_out, pages, 4}, {positions, T, 8}, {slots, T, 8}}))
    return rc;
  zt::ExtendArgs a{};
  a.table = block_table, a.ctx = context_lens, a.refs = ref_counts, a.cu = cu_seqlens;
  a.S = (int)S, a.W = (int)W, a.page_size = (int)page_size, a.pages = pages, a.T = T;
  a.table_out = table_out, a.ctx_out = context_out, a.refs_out = refs_out;
  a.pos_out = positions, a.slots = slots;
  return hip_status(zt::launch_cache_extend(a, reinterpret_cast<hipStream_t>(stream)), op);
}

int zt_cache_fork(const int32_t *block_table, const int32_t *context_lens,
                  const int32_t *ref_counts, const int32_t *parents, int64_t S, int64_t W,
                  int64_t pages, int64_t page_size, int32_t *table_out, int32_t *context_out,
                  int32_t *refs_out, int32_t *copies, zt_stream_t stream) {
  static const char *op = "zt_cache_fork";
  if (S < 0 || W < 0 || pages < 0 || page_size <= 0)
    return api_fail(ZT_EINVAL, "%s: need S, W, pages >= 0 and page_size > 0", op);
  if (S > kMaxRows) return api_fail(ZT_EUNSUPPORTED, "%s: at most %lld rows", op, (long long)kMaxRows);
  if (W > (1 << 24) || pages > INT32_MAX || page_size > (1 << 24) || W * page_size >= (1 << 30) ||
      S * W >= (1 << 30))
    return api_fail(ZT_EUNSUPPORTED, "%s: sizes exceed 32 bits", op);
  if ((S * W > 0 && (!block_table || !table_out)) || (pages > 0 && (!ref_counts || !refs_out)) ||
      (S > 0 && (!context_lens || !context_out || !parents || !copies)))
    return api_fail(ZT_EINVAL, "%s: null tensor pointer", op);
  if (S == 0 && pages == 0) return ZT_OK;
  if (const int rc = check_apart(
          op, {{block_table, S * W, 4}, {context_lens, S, 4}, {ref_counts, pages, 4}, {parents, S, 4}},
          {{table_out, S * W, 4}, {context_out, S, 4}, {refs_out, pages, 4}, {copies, 2 * S, 4}}))
    return rc;
  zt::ForkArgs a{};
  a.table = block_table, a.ctx = context_lens, a.refs = ref_counts, a.parents = parents;
  a.S = (int)S, a.W = (int)W, a.page_size = (int)page_size, a.pages = pages;
  a.table_out = table_out, a.ctx_out = context_out, a.refs_out = refs_out, a.copies = copies;
  return hip_status(zt::launch_cache_fork(a, reinterpret_cast<hipStream_t>(stream)), op);
}

size_t zt_cache_compact_workspace_size(int64_t pages) {
  return pages > 0 ? (size_t)pages * sizeof(int32_t) : 0;
}

int zt_cache_compact(const int32_t *block_table, int64_t entries, const int32_t *ref_counts,
                     int64_t pages, int32_t *table_out, int32_t *refs_out, int32_t *copies,
                     void *workspace, size_t workspace_bytes, zt_stream_t stream) {
  static const char *op = "zt_cache_compact";
  if (entries < 0 || pages < 0) return api_fail(ZT_EINVAL, "%s: need entries, pages >= 0", op);
  if (pages > INT32_MAX) return api_fail(ZT_EUNSUPPORTED, "%s: sizes exceed 32 bits", op);
  if ((entries > 0 && (!block_table || !table_out)) || (pages > 0 && (!ref_counts || !refs_out)) ||
      (pages > 1 && !copies))
    return api_fail(ZT_EINVAL, "%s: null tensor pointer", op);
  const size_t need = zt_cache_compact_workspace_size(pages);
  if (need && (!workspace || workspace_bytes < need))
    return api_fail(ZT_EINVAL, "%s: workspace of %zu bytes needed, %zu given", op, need,
                    workspace ? workspace_bytes : (size_t)0);
  if (entries == 0 && pages == 0) return ZT_OK;
  if (const int rc = check_apart(op, {{block_table, entries, 4}, {ref_counts, pages, 4}},
                                 {{table_out, entries, 4}, {refs_out, pages, 4}, {copies, pages / 2 * 2, 4},
                                  {workspace, (int64_t)need, 1}}))
    return rc;
  zt::CompactArgs a{};
  a.table = block_table, a.refs = ref_counts, a.entries = entries, a.pages = pages;
  a.table_out = table_out, a.refs_out = refs_out, a.copies = copies;
  a.to = static_cast<int32_t *>(workspace);
  return hip_status(zt::launch_cache_compact(a, reinterpret_cast<hipStream_t>(stream)), op);
}

int zt_cache_copy_pages(void *const *caches, int64_t n_caches, int64_t pages, int64_t page_bytes,
                        int64_t page_stride_bytes, const int32_t *copies, int64_t n_copies,
                        zt_stream_t stream) {
  static const char *op = "zt_cache_copy_pages";
  if (n_caches < 0 || pages < 0 || page_bytes < 0 || n_copies < 0)
    return api_fail(ZT_EINVAL, "%s: sizes must not be negative", op);
  if (page_stride_bytes < page_bytes)
    return api_fail(ZT_EINVAL, "%s: pages overlap (stride %lld of %lld bytes)", op,
                    (long long)page_stride_bytes, (long long)page_bytes);
  if (pages > INT32_MAX || n_copies > INT32_MAX / 64)
    return api_fail(ZT_EUNSUPPORTED, "%s: sizes exceed 32 bits", op);
  if (n_caches == 0 || pages == 0 || page_bytes == 0 || n_copies == 0) return ZT_OK;
  if (!caches || !copies) return api_fail(ZT_EINVAL, "%s: null pointer", op);
  for (int64_t i = 0; i < n_caches; ++i)
    if (!caches[i]) return api_fail(ZT_EINVAL, "%s: null cache pointer", op);
  for (int64_t i = 0; i < n_caches; i += zt::kCopyCaches) {
    zt::CopyArgs a{};
    const int n = (int)std::min<int64_t>(n_caches - i, zt::kCopyCaches);
    bool wide = page_bytes % 16 == 0 && page_stride_bytes % 16 == 0;
    for (int j = 0; j < n; ++j) {
      a.caches[j] = caches[i + j];
      wide = wide && reinterpret_cast<uintptr_t>(caches[i + j]) % 16 == 0;
    }
    a.copies = copies, a.pages = pages, a.page_stride = page_stride_bytes, a.page_bytes = page_bytes;
    const hipError_t e = zt::launch_copy_pages(a, n, n_copies, wide, reinterpret_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_status(e, op);
  }
  return ZT_OK;
}

// The checked arguments of an attention call, without its pointers.
static int checked_attn(const char *op, int64_t T, int64_t H, const zt_kv_cache *cache, int64_t S,
                        int64_t W, int64_t max_query_len, int32_t causal, int64_t window, AttnArgs *a) {
  if (const int rc = check_cache(op, cache, false)) return rc;
  if (const int rc = attn_args(op, T, H, cache, S, W, max_query_len, causal, window, a)) return rc;
  if (T > 0 && !zt::paged_attn_countable(*a))
    return api_fail(ZT_EUNSUPPORTED, "%s: too many tokens over too long tables for one call", op);
  return ZT_OK;
}

size_t zt_paged_attention_workspace_size(int64_t T, int64_t H, const zt_kv_cache *cache, int64_t S,
                                         int64_t W, int64_t max_query_len) {
  zt::AttnArgs a;
  if (checked_attn("zt_paged_attention_workspace_size", T, H, cache, S, W, max_query_len, 0, 0, &a)) return 0;
  return zt::paged_attn_workspace(a);
}

int zt_paged_attention(const void *q, int64_t T, int64_t H, int64_t ld_token, int64_t ld_head,
                       const zt_kv_cache *cache, const int32_t *block_table, int64_t S, int64_t W,
                       const int32_t *cu_seqlens, const int32_t *context_lens,
                       int64_t max_query_len, int32_t causal, int64_t window, float scale,
                       void *out, void *workspace, size_t workspace_bytes, zt_stream_t stream) {
  static const char *op = "zt_paged_attention";
  zt::AttnArgs a;
  if (const int rc = checked_attn(op, T, H, cache, S, W, max_query_len, causal, window, &a)) return rc;
  if (!std::isfinite(scale)) return api_fail(ZT_EINVAL, "%s: scale must be finite", op);
  if (T == 0) return ZT_OK;
  if (!q || !out || !cu_seqlens || (S > 0 && !context_lens) || (S * W > 0 && !block_table) ||
      (cache->pages > 0 && (!cache->k || !cache->v)))
    return api_fail(ZT_EINVAL, "%s: null tensor pointer", op);
  const int64_t es = cache->dtype == ZT_DT_F32 ? 4 : 2;
  if (!divides16(q, {ld_token, ld_head}, es) || !divides16(out, {}, es) ||
      !divides16(cache->k, {cache->k_strides[0], cache->k_strides[1], cache->k_strides[2]}, es) ||
      !divides16(cache->v, {cache->v_strides[0], cache->v_strides[1], cache->v_strides[2]}, es))
    return api_fail(ZT_EUNSUPPORTED, "%s: query, output and cache need 16-byte aligned rows", op);
  // the kernels count a layer's rows in units of 16 bytes, in 32 bits
  for (const int64_t *st : {cache->k_strides, cache->v_strides})
    if ((double)cache->pages * (double)st[0] + (double)cache->page_size * (double)st[2] >=
        4294967295.0 * (16 / es))
      return api_fail(ZT_EUNSUPPORTED, "%s: one head's keys or values span 64 GB and more", op);
  const size_t need = zt::paged_attn_workspace(a);
  if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
    return api_fail(ZT_EINVAL, "%s: 16-byte aligned workspace of %zu bytes needed, %zu given", op, need,
                    workspace ? workspace_bytes : (size_t)0);
  const Span to{out, T * H * cache->head_dim, es}, scratch{workspace, (int64_t)need, 1};
  if (touches_rows(to, q, T, H, cache->head_dim, ld_token, ld_head, es) || overlap(to, scratch) ||
      touches_rows(scratch, q, T, H, cache->head_dim, ld_token, ld_head, es))
    return api_fail(ZT_EINVAL, "%s: query, output and workspace must not overlap", op);
  auto held = [&](const void *p, const int64_t *ld) {
    return Strided{p, cache->head_dim * es, {cache->pages, cache->heads, cache->page_size}, {ld[0] * es, ld[1] * es, ld[2] * es}};
  };
  for (const Span &s : {to, scratch})
    if (touches(s, {{block_table, S * W, 4}, {cu_seqlens, S + 1, 4}, {context_lens, S, 4}},
                {held(cache->k, cache->k_strides), held(cache->v, cache->v_strides)}))
      return api_fail(ZT_EINVAL, "%s: output or workspace overlap the cache, the table or the lengths", op);
  a.q = q, a.q_ld[0] = ld_token, a.q_ld[1] = ld_head;
  a.k = cache->k, a.v = cache->v;
  for (int i = 0; i < 3; ++i) a.k_ld[i] = cache->k_strides[i], a.v_ld[i] = cache->v_strides[i];
  a.table = block_table, a.cu = cu_seqlens, a.ctx = context_lens, a.scale = scale, a.out = out;
  return hip_status(zt::launch_paged_attn(a, workspace, reinterpret_cast<hipStream_t>(stream)), op);
}

}  // extern "C"
