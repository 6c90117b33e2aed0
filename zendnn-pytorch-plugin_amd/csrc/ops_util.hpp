// Helpers of the torch ops' bodies (ops.cpp, ops_cache.cpp).
#pragma once

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <rocprofiler-sdk-roctx/roctx.h>

#include <algorithm>
#include <string>

#include "zentorch_hip.h"

namespace zentorch_hip {

inline int32_t zt_dtype_of(const at::Tensor &t) {
  switch (t.scalar_type()) {
  case at::kFloat: return ZT_DT_F32;
  case at::kBFloat16: return ZT_DT_BF16;
  case at::kHalf: return ZT_DT_F16;
  case at::kChar: return ZT_DT_S8;
  case at::kByte: return ZT_DT_U8;
  case at::kInt: return ZT_DT_S32;
  default: return ZT_DT_NONE;
  }
}

inline void check_device(const at::Tensor &t, const at::Tensor &ref, const char *op,
                  const char *name) {
  TORCH_CHECK(t.is_cuda(), op, ": ", name,
              " must be a GPU tensor (zentorch-mi355x has no CPU kernels), got ",
              t.device());
  TORCH_CHECK(t.device() == ref.device(), op, ": ", name, " is on ", t.device(),
              " but input is on ", ref.device());
}

inline hipStream_t current_stream() {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream();
}

// Device workspace of one call, from torch's stream-ordered caching
// allocator.  It is released when the call returns; the allocator hands the
// block to later work on the same stream only, and inside a HIP graph
// capture it comes from the graph's private pool, so a captured call keeps
// its own workspace on every replay.
inline at::Tensor call_workspace(const at::Tensor &like, size_t bytes) {
  return at::empty({(int64_t)std::max<size_t>(bytes, 1)}, like.options().dtype(at::kByte));
}

// The reference hands zentorch_op_name to ZenDNNL's profiler
// (MatmulUtils.hpp:763); here it names a ROCTx range around the launches,
// which rocprofv3 --marker-trace records.
struct OpRange {
  explicit OpRange(const std::string &name) { roctxRangePushA(name.c_str()); }
  ~OpRange() { roctxRangePop(); }
};

}  // namespace zentorch_hip
