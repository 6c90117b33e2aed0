// The torch ops of the key / value cache held in 4 bits (no reference
// counterpart): append, read and attention, on the C-ABI of
// include/zentorch_hip.h.  The pages' upkeep is the paged cache's (ops_cache.cpp).
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <torch/library.h>

#include <cmath>
#include <tuple>

#include "ops_cache_util.hpp"
#include "zentorch_hip.h"

namespace zentorch_hip {

namespace {

zt_kv_cache_mxfp4 cache_of(const at::Tensor &k, const at::Tensor &k_scales, const at::Tensor &v,
                           const at::Tensor &v_scales, int64_t head_dim, const at::Tensor &like, const char *op) {
  const struct {
    const at::Tensor &t;
    const char *name;
  } all[] = {{k, "key_cache"}, {k_scales, "key_scales"}, {v, "value_cache"}, {v_scales, "value_scales"}};
  const int64_t blocks = (head_dim + 31) / 32;
  TORCH_CHECK(head_dim > 0, op, ": head_dim must be positive, got ", head_dim);
  for (int i = 0; i < 4; ++i) {
    const at::Tensor &t = all[i].t;
    check_device(t, like, op, all[i].name);
    TORCH_CHECK(t.scalar_type() == at::kByte, op, ": ", all[i].name, " must be uint8, got ", t.scalar_type());
    TORCH_CHECK(t.dim() == 4, op, ": ", all[i].name, " must be [pages, heads, page_size, bytes], got ", t.dim(), "D");
    TORCH_CHECK(t.size(0) == k.size(0) && t.size(1) == k.size(1) && t.size(2) == k.size(2), op, ": ", all[i].name,
                " must have key_cache's pages, heads and page_size ", k.sizes(), ", got ", t.sizes());
    const int64_t bytes = i % 2 ? blocks : 16 * blocks;
    TORCH_CHECK(t.size(3) == bytes, op, ": ", all[i].name, " must have ", bytes, " bytes a row for head_dim ",
                head_dim, ", got ", t.size(3));
    TORCH_CHECK(t.size(3) == 1 || t.stride(3) == 1, op, ": the last dimension of ", all[i].name, " must be dense");
  }
  zt_kv_cache_mxfp4 c{};
  c.k = k.data_ptr(), c.v = v.data_ptr();
  c.k_scales = k_scales.data_ptr<uint8_t>(), c.v_scales = v_scales.data_ptr<uint8_t>();
  c.pages = k.size(0), c.heads = k.size(1), c.page_size = k.size(2), c.head_dim = head_dim;
  for (int i = 0; i < 3; ++i) {
    c.k_strides[i] = stride_of(k, i), c.v_strides[i] = stride_of(v, i);
    c.k_scale_strides[i] = stride_of(k_scales, i), c.v_scale_strides[i] = stride_of(v_scales, i);
  }
  return c;
}

}  // namespace

at::Tensor rotary_cache_append_mxfp4(const at::Tensor &query, const at::Tensor &key, const at::Tensor &value,
                                     const at::Tensor &positions, const at::Tensor &cos_sin, const at::Tensor &slots,
                                     at::Tensor &key_cache, at::Tensor &key_scales, at::Tensor &value_cache,
                                     at::Tensor &value_scales, bool interleaved, c10::string_view zentorch_op_name) {
  const char *op = "zentorch_rotary_cache_append_mxfp4";
  check_device(query, query, op, "query");
  check_heads(query, op, "query");
  check_heads(key, op, "key");
  check_heads(value, op, "value");
  check_float(query, op, "query");
  check_device(key, query, op, "key");
  check_device(value, query, op, "value");
  const zt_kv_cache_mxfp4 cache =
      cache_of(key_cache, key_scales, value_cache, value_scales, query.size(2), query, op);
  const at::Tensor *written[] = {&key_cache, &key_scales, &value_cache, &value_scales};
  for (int i = 0; i < 4; ++i) {
    at::assert_no_internal_overlap(*written[i]);
    for (int j = 0; j < i; ++j) at::assert_no_overlap(*written[i], *written[j]);
  }
  const int64_t T = query.size(0);
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
  const int64_t qs[2] = {stride_of(q, 0), stride_of(q, 1)}, ks[2] = {stride_of(k, 0), stride_of(k, 1)},
                vs[2] = {stride_of(v, 0), stride_of(v, 1)};
  const int rc = zt_rotary_cache_append_mxfp4(
      q.data_ptr(), zt_dtype_of(q), T, q.size(1), qs, k.data_ptr(), ks, v.data_ptr(), vs, pos.data_ptr<int64_t>(),
      table.data_ptr<float>(), table.size(0), table.size(1), table.size(0) > 1 ? table.stride(0) : table.size(1),
      interleaved, slot.data_ptr<int64_t>(), &cache, out.data_ptr(), stream_of());
  TORCH_CHECK(rc == ZT_OK, op, ": ", zt_last_error_string());
  return out;
}

std::tuple<at::Tensor, at::Tensor> cache_read_mxfp4(const at::Tensor &key_cache, const at::Tensor &key_scales,
                                                    const at::Tensor &value_cache, const at::Tensor &value_scales,
                                                    const at::Tensor &slots, int64_t head_dim, at::ScalarType dtype,
                                                    c10::string_view zentorch_op_name) {
  const char *op = "zentorch_cache_read_mxfp4";
  const zt_kv_cache_mxfp4 cache = cache_of(key_cache, key_scales, value_cache, value_scales, head_dim, key_cache, op);
  TORCH_CHECK(dtype == at::kBFloat16 || dtype == at::kFloat, op, ": dtype must be bfloat16 or float32, got ", dtype);
  TORCH_CHECK(slots.dim() == 1, op, ": slots must be 1D, got ", slots.dim(), "D");
  const int64_t n = slots.size(0);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(key_cache.device());
  const OpRange range{std::string(zentorch_op_name)};
  const at::Tensor slot = long_1d(slots, n, key_cache, op, "slots");
  at::Tensor k = at::empty({n, cache.heads, head_dim}, key_cache.options().dtype(dtype)), v = at::empty_like(k);
  const int rc = zt_cache_read_mxfp4(&cache, slot.data_ptr<int64_t>(), n, zt_dtype_of(k), k.data_ptr(), v.data_ptr(),
                                     stream_of());
  TORCH_CHECK(rc == ZT_OK, op, ": ", zt_last_error_string());
  return {k, v};
}

at::Tensor paged_attention_mxfp4(const at::Tensor &query, const at::Tensor &key_cache, const at::Tensor &key_scales,
                                 const at::Tensor &value_cache, const at::Tensor &value_scales,
                                 const at::Tensor &block_table, const at::Tensor &cu_seqlens,
                                 const at::Tensor &context_lens, int64_t max_query_len, bool causal, int64_t window,
                                 c10::optional<double> scale, c10::string_view zentorch_op_name) {
  const char *op = "zentorch_paged_attention_mxfp4";
  check_device(query, query, op, "query");
  check_heads(query, op, "query");
  check_float(query, op, "query");
  const zt_kv_cache_mxfp4 cache =
      cache_of(key_cache, key_scales, value_cache, value_scales, query.size(2), query, op);
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
  const at::Tensor table = block_table.contiguous(), cu = cu_seqlens.contiguous(), ctx = context_lens.contiguous();
  at::Tensor out = at::empty(query.sizes(), query.options());
  const int64_t T = q.size(0), H = q.size(1), W = table.size(1);
  const int32_t dt = zt_dtype_of(q);
  const size_t ws = zt_paged_attention_mxfp4_workspace_size(T, H, dt, &cache, S, W, max_query_len);
  const at::Tensor wsp = call_workspace(query, ws);
  const int rc = zt_paged_attention_mxfp4(
      q.data_ptr(), dt, T, H, stride_of(q, 0), stride_of(q, 1), &cache, table.data_ptr<int32_t>(), S, W,
      cu.data_ptr<int32_t>(), ctx.data_ptr<int32_t>(), max_query_len, causal, window,
      (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)cache.head_dim)), out.data_ptr(), wsp.data_ptr(),
      ws, stream_of());
  TORCH_CHECK(rc == ZT_OK, op, ": ", zt_last_error_string());
  return out;
}

}  // namespace zentorch_hip

TORCH_LIBRARY_FRAGMENT(zentorch, m) {
  m.def("zentorch_rotary_cache_append_mxfp4(Tensor query, Tensor key, Tensor value, Tensor positions, "
        "Tensor cos_sin, Tensor slots, Tensor(a!) key_cache, Tensor(b!) key_scales, Tensor(c!) value_cache, "
        "Tensor(d!) value_scales, *, bool interleaved=False, str zentorch_op_name="
        "'zentorch::zentorch_rotary_cache_append_mxfp4') -> Tensor");
  m.def("zentorch_cache_read_mxfp4(Tensor key_cache, Tensor key_scales, Tensor value_cache, "
        "Tensor value_scales, Tensor slots, int head_dim, *, ScalarType dtype=bfloat16, str zentorch_op_name="
        "'zentorch::zentorch_cache_read_mxfp4') -> (Tensor, Tensor)");
  m.def("zentorch_paged_attention_mxfp4(Tensor query, Tensor key_cache, Tensor key_scales, "
        "Tensor value_cache, Tensor value_scales, Tensor block_table, Tensor cu_seqlens, "
        "Tensor context_lens, int max_query_len, *, bool causal=True, int window=0, float? scale=None, "
        "str zentorch_op_name='zentorch::zentorch_paged_attention_mxfp4') -> Tensor");
}

TORCH_LIBRARY_IMPL(zentorch, CUDA, m) {
  using namespace zentorch_hip;
  m.impl("zentorch_rotary_cache_append_mxfp4", rotary_cache_append_mxfp4);
  m.impl("zentorch_cache_read_mxfp4", cache_read_mxfp4);
  m.impl("zentorch_paged_attention_mxfp4", paged_attention_mxfp4);
}
