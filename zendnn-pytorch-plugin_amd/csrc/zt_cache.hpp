// Launch interface of the paged key / value cache's kernels (kv_cache.hip,
// paged_attn.hip), shared with the C-ABI layer (capi_cache.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <algorithm>

#include "zt_common.hpp"

namespace zt {

// Sets the calling thread's error message and returns `code` (capi.hip).
int api_fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));

// Rows of a batch that the page kernels hold in LDS.
constexpr int64_t kMaxRows = 4096;
// Sequences of an attention call (16 bytes of LDS each).
constexpr int64_t kMaxSeqs = 1024;

// Lets a kernel take `bytes` of dynamic LDS.  A call whose size is past what
// every kernel may take (64 KB) allows the kernel's largest size, always the same:
// another thread's call to it may be between this and its launch.
inline hipError_t allow_lds(const void *kernel, size_t bytes, size_t largest) {
  if (bytes <= 64 * 1024) return hipSuccess;
  return hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)largest);
}

// Division of n <= 2^30 by a fixed d >= 1: floor(n * mul / 2^(31 + L)) with
// mul = floor(2^(31 + L) / d) + 1 and L = ceil(log2 d), which is exact for every
// n < 2^31; 2 n * mul is taken so that the high word is all that is needed.
struct FastDiv {
  uint32_t mul, shift;
};
inline FastDiv make_div(uint32_t d) {
  uint32_t L = 0;
  while ((1ull << L) < d) ++L;
  return {(uint32_t)((1ull << (31 + L)) / d + 1), L};
}
__device__ __forceinline__ uint32_t fast_div(uint32_t n, FastDiv d) {
  return __umulhi(2 * n, d.mul) >> d.shift;
}

// Inclusive prefix sum over a wave, by lane moves that cost an addition each
// (rows of 16 lanes, then the rows' last lanes on).
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);   // row_shr 1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);   // row_shr 2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);   // row_shr 4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);   // row_shr 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row 0 -> 1, 2 -> 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31 -> rows 2, 3
  return x;
}

struct RotaryArgs {
  const void *q, *k, *v;      // [T, H | KV | KV, D], unit last stride
  int64_t q_ld[2], k_ld[2], v_ld[2];  // token and head strides, elements
  void *q_out;                // [T, H, D]
  void *k_cache, *v_cache;    // strides of page, head, token
  int64_t kc_ld[3], vc_ld[3];
  const int64_t *pos, *slots;
  const float *table;         // [length, R]: cos, then sin
  int64_t length, table_ld, pages;
  int64_t T;
  int H, KV, D, R, page_size;
  bool interleaved;
  // units of 16 bytes (or of one element) per rotated row, per copied row and
  // per token, set by launch_rotary
  int row_units, copy_units, units;
};
hipError_t launch_rotary(RotaryArgs a, int dtype, bool wide, hipStream_t s);

struct ExtendArgs {
  const int32_t *table, *ctx, *refs, *cu;  // [S, W], [S], [pages], [S + 1]
  int S, W, page_size;
  int64_t pages, T;
  int32_t *table_out, *ctx_out, *refs_out;
  int64_t *pos_out, *slots;  // [T]
  FastDiv div_size, div_w;   // set by launch_cache_extend
};
hipError_t launch_cache_extend(ExtendArgs a, hipStream_t s);

struct ForkArgs {
  const int32_t *table, *ctx, *refs, *parents;
  int S, W, page_size;
  int64_t pages;
  int32_t *table_out, *ctx_out, *refs_out, *copies;  // copies [S, 2]
  FastDiv div_size, div_w;  // set by launch_cache_fork
};
hipError_t launch_cache_fork(ForkArgs a, hipStream_t s);

struct CompactArgs {
  const int32_t *table, *refs;
  int64_t entries, pages;
  int32_t *table_out, *refs_out, *copies;  // copies [pages / 2, 2]
  int32_t *to;                             // [pages] workspace
};
hipError_t launch_cache_compact(const CompactArgs &a, hipStream_t s);

constexpr int kCopyCaches = 64;  // caches of one launch
struct CopyArgs {
  void *caches[kCopyCaches];
  const int32_t *copies;
  int64_t pages, page_stride, page_bytes;  // bytes
  int parts;
};
hipError_t launch_copy_pages(CopyArgs a, int caches, int64_t pairs, bool wide, hipStream_t s);

struct AttnArgs {
  const void *q;  // [T, H, D]
  int64_t q_ld[2];
  const void *k, *v;  // strides of page, head, token
  int64_t k_ld[3], v_ld[3];
  const int32_t *table, *cu, *ctx;  // [S, W], [S + 1], [S]
  int64_t T, pages, max_q;
  int H, KV, D, S, W, page_size;
  int dtype;
  bool causal;
  int64_t window;
  float scale;
  void *out;  // [T, H, D]
  // set by launch_paged_attn
  int group;                    // H / KV
  int item_rows;                // rows of an item, which the partial results are laid out by
  FastDiv div_group, div_page;
  uint32_t k_row[2], v_row[2];  // strides of page and token in units of 16 bytes
  float *part_ml, *part_o;      // partial results: [slots][BM][2], [slots][BM][D]
  void *splits;                 // [workgroups] of Split
};
// Whether the work of such a call can be counted in 32 bits.
bool paged_attn_countable(const AttnArgs &a);
size_t paged_attn_workspace(const AttnArgs &a);
hipError_t launch_paged_attn(AttnArgs a, void *workspace, hipStream_t s);

}  // namespace zt
