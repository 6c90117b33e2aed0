// The torch ops of the paged key / value cache (no reference counterpart):
// rotary positions, append, attention over the cache and the upkeep of its
// pages, on the C-ABI of include/zentorch_hip.h.  Like the other zentorch ops
// they run asynchronously on the current stream, never synchronise, and take
// their workspace from torch's caching allocator.
#include <ATen/ATen.h>
#include <torch/library.h>

#include <cmath>
#include <tuple>
#include <vector>

#include "ops_util.hpp"
#include "zentorch_hip.h"

namespace zentorch_hip {

namespace {

zt_stream_t stream_of() { return reinterpret_cast<zt_stream_t>(current_stream()); }

void check_int32(const at::Tensor &t, int64_t dim, const at::Tensor &like, const char *op,
                 const char *name) {
  check_device(t, like, op, name);
  TORCH_CHECK(t.scalar_type() == at::kInt, op, ": ", name, " must be int32, got ", t.scalar_type());
  TORCH_CHECK(t.dim() == dim, op, ": ", name, " must be ", dim, "D, got ", t.dim(), "D");
}

void check_float(const at::Tensor &t, const char *op, const char *name) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat, op, ": ", name,
              " must be bfloat16 or float32, got ", t.scalar_type());
}

// t with unit last stride, and, where `aligned`, rows on 16 bytes (a copy if need be).
at::Tensor rows_of(const at::Tensor &t, bool aligned) {
  bool ok = t.size(-1) == 1 || t.stride(-1) == 1;
  for (int64_t i = 0; ok && i < t.dim(); ++i) ok = t.stride(i) >= 0;
  if (ok && aligned) {
    ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int64_t i = 0; ok && i + 1 < t.dim(); ++i)
      ok = t.size(i) == 1 || t.stride(i) * (int64_t)t.element_size() % 16 == 0;
  }
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// A dimension of one entry may carry any stride; the kernels get 0 for it.
int64_t stride_of(const at::Tensor &t, int64_t d) { return t.size(d) == 1 ? 0 : t.stride(d); }

zt_kv_cache cache_of(const at::Tensor &k, const at::Tensor &v, const at::Tensor &like, const char *op) {
  check_device(k, like, op, "key_cache");
  check_device(v, like, op, "value_cache");
  TORCH_CHECK(k.dim() == 4, op, ": key_cache must be [pages, heads, page_size, head_dim], got ", k.dim(), "D");
  TORCH_CHECK(v.sizes() == k.sizes(), op, ": value_cache must have key_cache's shape ", k.sizes(),
              ", got ", v.sizes());
  TORCH_CHECK(k.scalar_type() == like.scalar_type() && v.scalar_type() == like.scalar_type(), op,
              ": the caches must have the input's type ", like.scalar_type(), ", got ",
              k.scalar_type(), " and ", v.scalar_type());
  TORCH_CHECK((k.size(3) == 1 || k.stride(3) == 1) && (v.size(3) == 1 || v.stride(3) == 1), op,
              ": the caches' last dimension must be dense");
  zt_kv_cache c{};
  c.k = k.data_ptr(), c.v = v.data_ptr(), c.dtype = zt_dtype_of(k);
  c.pages = k.size(0), c.heads = k.size(1), c.page_size = k.size(2), c.head_dim = k.size(3);
  for (int i = 0; i < 3; ++i) c.k_strides[i] = stride_of(k, i), c.v_strides[i] = stride_of(v, i);
  return c;
}

at::Tensor table_rows(const at::Tensor &cos_sin, const at::Tensor &like, const char *op) {
  check_device(cos_sin, like, op, "cos_sin");
  TORCH_CHECK(cos_sin.scalar_type() == at::kFloat && cos_sin.dim() == 2, op,
              ": cos_sin must be a 2D float32 tensor [length, rotated], got ",
              cos_sin.scalar_type(), " ", cos_sin.sizes());
  const at::Tensor t = rows_of(cos_sin, false);
  // rows that lie on each other (an expanded table) are laid out
  return t.size(0) > 1 && t.stride(0) < t.size(1) ? t.clone(at::MemoryFormat::Contiguous) : t;
}

at::Tensor long_1d(const at::Tensor &t, int64_t n, const at::Tensor &like, const char *op,
                   const char *name) {
  check_device(t, like, op, name);
  TORCH_CHECK(t.scalar_type() == at::kLong && t.dim() == 1 && t.size(0) == n, op, ": ", name,
              " must be int64 [", n, "], got ", t.scalar_type(), " ", t.sizes());
  return t.contiguous();
}

// The caller keeps the memory of another stream's tensors alive as for any
// torch op; these ops only use the current stream.
void check_heads(const at::Tensor &t, const char *op, const char *name) {
  TORCH_CHECK(t.dim() == 3, op, ": ", name, " must be [tokens, heads, head_dim], got ", t.dim(), "D");
}

}  // namespace

at::Tensor rotary_embedding(const at::Tensor &input, const at::Tensor &positions,
                            const at::Tensor &cos_sin, bool interleaved,
                            c10::string_view zentorch_op_name) {
  const char *op = "zentorch_rotary_embedding";
  check_device(input, input, op, "input");
  check_heads(input, op, "input");
  check_float(input, op, "input");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(input.device());
  const OpRange range{std::string(zentorch_op_name)};
  const at::Tensor pos = long_1d(positions, input.size(0), input, op, "positions");
  const at::Tensor table = table_rows(cos_sin, input, op), x = rows_of(input, false);
  at::Tensor out = at::empty(input.sizes(), input.options());
  if (out.numel() == 0) return out;
  const int rc = zt_rotary_embedding(
      x.data_ptr(), zt_dtype_of(x), x.size(0), x.size(1), x.size(2), stride_of(x, 0),
      stride_of(x, 1), pos.data_ptr<int64_t>(), table.data_ptr<float>(), table.size(0),
      table.size(1), table.size(0) > 1 ? table.stride(0) : table.size(1), interleaved,
      out.data_ptr(), stream_of());
  TORCH_CHECK(rc == ZT_OK, op, ": ", zt_last_error_string());
  return out;
}

at::Tensor rotary_cache_append(const at::Tensor &query, const at::Tensor &key,
                               const at::Tensor &value, const at::Tensor &positions,
                               const at::Tensor &cos_sin, const at::Tensor &slots,
                               at::Tensor &key_cache, at::Tensor &value_cache, bool interleaved,
                               c10::string_view zentorch_op_name) {
  const char *op = "zentorch_rotary_cache_append";
  check_device(query, query, op, "query");
  check_heads(query, op, "query");
  check_heads(key, op, "key");
  check_heads(value, op, "value");
  check_float(query, op, "query");
  check_device(key, query, op, "key");
  check_device(value, query, op, "value");
  const zt_kv_cache cache = cache_of(key_cache, value_cache, query, op);
  const int64_t T = query.size(0);
  TORCH_CHECK(query.size(2) == cache.head_dim, op, ": query's head_dim (", query.size(2),
              ") must equal the cache's (", cache.head_dim, ")");
  TORCH_CHECK(key.size(0) == T && key.size(1) == cache.heads && key.size(2) == cache.head_dim &&
                  value.sizes() == key.sizes(),
              op, ": key and value must be [", T, ", ", cache.heads, ", ", cache.head_dim, "], got ",
              key.sizes(), " and ", value.sizes());
  TORCH_CHECK(key.scalar_type() == query.scalar_type() && value.scalar_type() == query.scalar_type(),
              op, ": query, key and value must have one type");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(query.device());
  const OpRange range{std::string(zentorch_op_name)};
  const at::Tensor pos = long_1d(positions, T, query, op, "positions");
  const at::Tensor slot = long_1d(slots, T, query, op, "slots");
  const at::Tensor table = table_rows(cos_sin, query, op);
  const at::Tensor q = rows_of(query, false), k = rows_of(key, false), v = rows_of(value, false);
  at::Tensor out = at::empty(query.sizes(), query.options());
  if (T == 0) return out;
  const int64_t qs[2] = {stride_of(q, 0), stride_of(q, 1)}, ks[2] = {stride_of(k, 0), stride_of(k, 1)},
                vs[2] = {stride_of(v, 0), stride_of(v, 1)};
  const int rc = zt_rotary_cache_append(
      q.data_ptr(), T, q.size(1), qs, k.data_ptr(), ks, v.data_ptr(), vs,
      pos.data_ptr<int64_t>(), table.data_ptr<float>(), table.size(0), table.size(1),
      table.size(0) > 1 ? table.stride(0) : table.size(1), interleaved, slot.data_ptr<int64_t>(),
      &cache, out.data_ptr(), stream_of());
  TORCH_CHECK(rc == ZT_OK, op, ": ", zt_last_error_string());
  return out;
}

at::Tensor paged_attention(const at::Tensor &query, const at::Tensor &key_cache,
                           const at::Tensor &value_cache, const at::Tensor &block_table,
                           const at::Tensor &cu_seqlens, const at::Tensor &context_lens,
                           int64_t max_query_len, bool causal, int64_t window,
                           c10::optional<double> scale, c10::string_view zentorch_op_name) {
  const char *op = "zentorch_paged_attention";
  check_device(query, query, op, "query");
  check_heads(query, op, "query");
  check_float(query, op, "query");
  const zt_kv_cache cache = cache_of(key_cache, value_cache, query, op);
  TORCH_CHECK(query.size(2) == cache.head_dim, op, ": query's head_dim (", query.size(2),
              ") must equal the cache's (", cache.head_dim, ")");
  check_int32(block_table, 2, query, op, "block_table");
  check_int32(cu_seqlens, 1, query, op, "cu_seqlens");
  check_int32(context_lens, 1, query, op, "context_lens");
  const int64_t S = block_table.size(0);
  TORCH_CHECK(cu_seqlens.size(0) == S + 1 && context_lens.size(0) == S, op, ": ", S,
              " rows in block_table need ", S + 1, " cu_seqlens and ", S, " context_lens, got ",
              cu_seqlens.size(0), " and ", context_lens.size(0));
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(query.device());
  const OpRange range{std::string(zentorch_op_name)};
  const at::Tensor q = rows_of(query, true);
  const at::Tensor table = block_table.contiguous(), cu = cu_seqlens.contiguous(),
                   ctx = context_lens.contiguous();
  at::Tensor out = at::empty(query.sizes(), query.options());
  const int64_t T = q.size(0), H = q.size(1), W = table.size(1);
  const size_t ws = zt_paged_attention_workspace_size(T, H, &cache, S, W, max_query_len);
  const at::Tensor wsp = call_workspace(query, ws);
  const int rc = zt_paged_attention(
      q.data_ptr(), T, H, stride_of(q, 0), stride_of(q, 1), &cache, table.data_ptr<int32_t>(), S, W,
      cu.data_ptr<int32_t>(), ctx.data_ptr<int32_t>(), max_query_len, causal, window,
      (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)cache.head_dim)), out.data_ptr(),
      wsp.data_ptr(), ws, stream_of());
  TORCH_CHECK(rc == ZT_OK, op, ": ", zt_last_error_string());
  return out;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> cache_extend(
    const at::Tensor &block_table, const at::Tensor &context_lens, const at::Tensor &ref_counts,
    const at::Tensor &cu_seqlens, int64_t page_size, int64_t num_tokens,
    c10::string_view zentorch_op_name) {
  const char *op = "zentorch_cache_extend";
  check_int32(block_table, 2, block_table, op, "block_table");
  check_int32(context_lens, 1, block_table, op, "context_lens");
  check_int32(ref_counts, 1, block_table, op, "ref_counts");
  check_int32(cu_seqlens, 1, block_table, op, "cu_seqlens");
  const int64_t S = block_table.size(0), W = block_table.size(1), pages = ref_counts.size(0);
  TORCH_CHECK(cu_seqlens.size(0) == S + 1 && context_lens.size(0) == S, op, ": ", S,
              " rows in block_table need ", S + 1, " cu_seqlens and ", S, " context_lens, got ",
              cu_seqlens.size(0), " and ", context_lens.size(0));
  TORCH_CHECK(num_tokens >= 0, op, ": num_tokens must not be negative, got ", num_tokens);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(block_table.device());
  const OpRange range{std::string(zentorch_op_name)};
  const at::Tensor table = block_table.contiguous(), ctx = context_lens.contiguous(),
                   refs = ref_counts.contiguous(), cu = cu_seqlens.contiguous();
  at::Tensor table_out = at::empty(table.sizes(), table.options());
  at::Tensor ctx_out = at::empty({S}, ctx.options()), refs_out = at::empty({pages}, refs.options());
  at::Tensor pos = at::empty({num_tokens}, table.options().dtype(at::kLong));
  at::Tensor slots = at::empty({num_tokens}, pos.options());
  const int rc = zt_cache_extend(
      table.data_ptr<int32_t>(), ctx.data_ptr<int32_t>(), refs.data_ptr<int32_t>(),
      cu.data_ptr<int32_t>(), S, W, pages, page_size, num_tokens, table_out.data_ptr<int32_t>(),
      ctx_out.data_ptr<int32_t>(), refs_out.data_ptr<int32_t>(), pos.data_ptr<int64_t>(),
      slots.data_ptr<int64_t>(), stream_of());
  TORCH_CHECK(rc == ZT_OK, op, ": ", zt_last_error_string());
  return {table_out, ctx_out, refs_out, pos, slots};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> cache_fork(
    const at::Tensor &block_table, const at::Tensor &context_lens, const at::Tensor &ref_counts,
    const at::Tensor &parents, int64_t page_size, c10::string_view zentorch_op_name) {
  const char *op = "zentorch_cache_fork";
  check_int32(block_table, 2, block_table, op, "block_table");
  check_int32(context_lens, 1, block_table, op, "context_lens");
  check_int32(ref_counts, 1, block_table, op, "ref_counts");
  check_int32(parents, 1, block_table, op, "parents");
  const int64_t S = block_table.size(0), W = block_table.size(1), pages = ref_counts.size(0);
  TORCH_CHECK(context_lens.size(0) == S && parents.size(0) == S, op, ": ", S,
              " rows in block_table need as many context_lens and parents, got ",
              context_lens.size(0), " and ", parents.size(0));
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(block_table.device());
  const OpRange range{std::string(zentorch_op_name)};
  const at::Tensor table = block_table.contiguous(), ctx = context_lens.contiguous(),
                   refs = ref_counts.contiguous(), par = parents.contiguous();
  at::Tensor table_out = at::empty(table.sizes(), table.options());
  at::Tensor ctx_out = at::empty({S}, ctx.options()), refs_out = at::empty({pages}, refs.options());
  at::Tensor copies = at::empty({S, 2}, ctx.options());
  const int rc = zt_cache_fork(
      table.data_ptr<int32_t>(), ctx.data_ptr<int32_t>(), refs.data_ptr<int32_t>(),
      par.data_ptr<int32_t>(), S, W, pages, page_size, table_out.data_ptr<int32_t>(),
      ctx_out.data_ptr<int32_t>(), refs_out.data_ptr<int32_t>(), copies.data_ptr<int32_t>(),
      stream_of());
  TORCH_CHECK(rc == ZT_OK, op, ": ", zt_last_error_string());
  return {table_out, ctx_out, refs_out, copies};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> cache_compact(const at::Tensor &block_table,
                                                             const at::Tensor &ref_counts,
                                                             c10::string_view zentorch_op_name) {
  const char *op = "zentorch_cache_compact";
  check_int32(block_table, 2, block_table, op, "block_table");
  check_int32(ref_counts, 1, block_table, op, "ref_counts");
  const int64_t pages = ref_counts.size(0);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(block_table.device());
  const OpRange range{std::string(zentorch_op_name)};
  const at::Tensor table = block_table.contiguous(), refs = ref_counts.contiguous();
  at::Tensor table_out = at::empty(table.sizes(), table.options());
  at::Tensor refs_out = at::empty({pages}, refs.options());
  at::Tensor copies = at::empty({pages / 2, 2}, refs.options());
  const size_t ws = zt_cache_compact_workspace_size(pages);
  const at::Tensor wsp = call_workspace(table, ws);
  const int rc = zt_cache_compact(table.data_ptr<int32_t>(), table.numel(), refs.data_ptr<int32_t>(),
                                  pages, table_out.data_ptr<int32_t>(), refs_out.data_ptr<int32_t>(),
                                  copies.data_ptr<int32_t>(), wsp.data_ptr(), ws, stream_of());
  TORCH_CHECK(rc == ZT_OK, op, ": ", zt_last_error_string());
  return {table_out, refs_out, copies};
}

void cache_copy_pages(at::TensorList caches, const at::Tensor &copies,
                      c10::string_view zentorch_op_name) {
  const char *op = "zentorch_cache_copy_pages";
  check_int32(copies, 2, copies, op, "copies");
  TORCH_CHECK(copies.size(1) == 2, op, ": copies must be [n, 2] pairs (from, to), got ", copies.sizes());
  if (caches.empty()) return;
  const at::Tensor &c0 = caches[0];
  TORCH_CHECK(c0.dim() >= 2, op, ": a cache has its pages in its first dimension, got ", c0.dim(), "D");
  std::vector<void *> at;
  at.reserve(caches.size());
  for (const at::Tensor &c : caches) {
    check_device(c, copies, op, "cache");
    TORCH_CHECK(c.sizes() == c0.sizes() && c.strides() == c0.strides() &&
                    c.scalar_type() == c0.scalar_type(),
                op, ": the caches must have one shape, layout and type");
    at.push_back(c.data_ptr());
  }
  if (c0.numel() == 0) return;
  int64_t page = 1;  // elements of a page, which lie together in any order of dimensions
  for (int64_t d = 1; d < c0.dim(); ++d) page *= c0.size(d);
  TORCH_CHECK(c0.select(0, 0).is_non_overlapping_and_dense(), op, ": a page's elements must lie together");
  const int64_t stride = c0.size(0) > 1 ? c0.stride(0) : page;
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(copies.device());
  const OpRange range{std::string(zentorch_op_name)};
  const at::Tensor pairs = copies.contiguous();
  const int64_t es = c0.element_size();
  const int rc = zt_cache_copy_pages(at.data(), (int64_t)at.size(), c0.size(0), page * es, stride * es,
                                     pairs.data_ptr<int32_t>(), pairs.size(0), stream_of());
  TORCH_CHECK(rc == ZT_OK, op, ": ", zt_last_error_string());
}

}  // namespace zentorch_hip

TORCH_LIBRARY_FRAGMENT(zentorch, m) {
  m.def("zentorch_rotary_embedding(Tensor input, Tensor positions, Tensor cos_sin, *, "
        "bool interleaved=False, str zentorch_op_name="
        "'zentorch::zentorch_rotary_embedding') -> Tensor");
  m.def("zentorch_rotary_cache_append(Tensor query, Tensor key, Tensor value, Tensor positions, "
        "Tensor cos_sin, Tensor slots, Tensor(a!) key_cache, Tensor(b!) value_cache, *, "
        "bool interleaved=False, str zentorch_op_name="
        "'zentorch::zentorch_rotary_cache_append') -> Tensor");
  m.def("zentorch_paged_attention(Tensor query, Tensor key_cache, Tensor value_cache, "
        "Tensor block_table, Tensor cu_seqlens, Tensor context_lens, int max_query_len, *, "
        "bool causal=True, int window=0, float? scale=None, str zentorch_op_name="
        "'zentorch::zentorch_paged_attention') -> Tensor");
  m.def("zentorch_cache_extend(Tensor block_table, Tensor context_lens, Tensor ref_counts, "
        "Tensor cu_seqlens, int page_size, int num_tokens, *, str zentorch_op_name="
        "'zentorch::zentorch_cache_extend') -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("zentorch_cache_fork(Tensor block_table, Tensor context_lens, Tensor ref_counts, "
        "Tensor parents, int page_size, *, str zentorch_op_name="
        "'zentorch::zentorch_cache_fork') -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("zentorch_cache_compact(Tensor block_table, Tensor ref_counts, *, str zentorch_op_name="
        "'zentorch::zentorch_cache_compact') -> (Tensor, Tensor, Tensor)");
  m.def("zentorch_cache_copy_pages(Tensor(a!)[] caches, Tensor copies, *, str zentorch_op_name="
        "'zentorch::zentorch_cache_copy_pages') -> ()");
}

TORCH_LIBRARY_IMPL(zentorch, CUDA, m) {
  using namespace zentorch_hip;
  m.impl("zentorch_rotary_embedding", rotary_embedding);
  m.impl("zentorch_rotary_cache_append", rotary_cache_append);
  m.impl("zentorch_paged_attention", paged_attention);
  m.impl("zentorch_cache_extend", cache_extend);
  m.impl("zentorch_cache_fork", cache_fork);
  m.impl("zentorch_cache_compact", cache_compact);
  m.impl("zentorch_cache_copy_pages", cache_copy_pages);
}
