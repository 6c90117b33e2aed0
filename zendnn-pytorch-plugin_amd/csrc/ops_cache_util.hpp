// Helpers of the paged caches' torch ops (ops_cache.cpp, ops_cache_mx4.cpp).
#pragma once

#include "ops_util.hpp"

namespace zentorch_hip {

inline zt_stream_t stream_of() { return reinterpret_cast<zt_stream_t>(current_stream()); }

inline void check_int32(const at::Tensor &t, int64_t dim, const at::Tensor &like, const char *op,
                 const char *name) {
  check_device(t, like, op, name);
  TORCH_CHECK(t.scalar_type() == at::kInt, op, ": ", name, " must be int32, got ", t.scalar_type());
  TORCH_CHECK(t.dim() == dim, op, ": ", name, " must be ", dim, "D, got ", t.dim(), "D");
}

inline void check_float(const at::Tensor &t, const char *op, const char *name) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat, op, ": ", name,
              " must be bfloat16 or float32, got ", t.scalar_type());
}

// t with unit last stride, and, where `aligned`, rows on 16 bytes (a copy if need be).
inline at::Tensor rows_of(const at::Tensor &t, bool aligned) {
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
inline int64_t stride_of(const at::Tensor &t, int64_t d) { return t.size(d) == 1 ? 0 : t.stride(d); }

inline at::Tensor table_rows(const at::Tensor &cos_sin, const at::Tensor &like, const char *op) {
  check_device(cos_sin, like, op, "cos_sin");
  TORCH_CHECK(cos_sin.scalar_type() == at::kFloat && cos_sin.dim() == 2, op,
              ": cos_sin must be a 2D float32 tensor [length, rotated], got ",
              cos_sin.scalar_type(), " ", cos_sin.sizes());
  const at::Tensor t = rows_of(cos_sin, false);
  // rows that lie on each other (an expanded table) are laid out
  return t.size(0) > 1 && t.stride(0) < t.size(1) ? t.clone(at::MemoryFormat::Contiguous) : t;
}

inline at::Tensor long_1d(const at::Tensor &t, int64_t n, const at::Tensor &like, const char *op,
                   const char *name) {
  check_device(t, like, op, name);
  TORCH_CHECK(t.scalar_type() == at::kLong && t.dim() == 1 && t.size(0) == n, op, ": ", name,
              " must be int64 [", n, "], got ", t.scalar_type(), " ", t.sizes());
  return t.contiguous();
}

// The caller keeps the memory of another stream's tensors alive as for any
// torch op; these ops only use the current stream.
inline void check_heads(const at::Tensor &t, const char *op, const char *name) {
  TORCH_CHECK(t.dim() == 3, op, ": ", name, " must be [tokens, heads, head_dim], got ", t.dim(), "D");
}

}  // namespace zentorch_hip
