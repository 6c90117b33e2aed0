// Argument checks that the C-ABI's calls on paged caches share (capi_cache.hip,
// capi_cache_mx4.hip).
#pragma once

#include <cmath>
#include <utility>

#include "zt_cache.hpp"

namespace zt {

inline int hip_status(hipError_t e, const char *what) {
  if (e == hipSuccess) return ZT_OK;
  return api_fail(ZT_EHIP, "%s: HIP error %d (%s)", what, (int)e, hipGetErrorString(e));
}

inline bool is_float_dt(int dt) { return dt == ZT_DT_F32 || dt == ZT_DT_BF16; }

inline bool divides16(const void *p, std::initializer_list<int64_t> elems, int64_t esize) {
  if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (int64_t e : elems)
    if (e * esize % 16) return false;
  return true;
}

// The page ops read their inputs while they write their outputs, from many
// workgroups: no output may lie on an input or on another output.
struct Span {
  const void *p;
  int64_t elems, size;  // of `size` bytes
};
inline bool overlap(const Span &a, const Span &b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
  return a.elems > 0 && b.elems > 0 && x < y + (uintptr_t)(b.elems * b.size) &&
         y < x + (uintptr_t)(a.elems * a.size);
}
// Whether s lies on a token's rows [H, D] of a tensor [T, H, D] (it may lie between
// two tokens', as in a wider buffer that the tensor is a slice of).
inline bool touches_rows(const Span &s, const void *x, int64_t T, int64_t H, int64_t D, int64_t ld_token,
                  int64_t ld_head, int64_t esize) {
  if (ld_token < 0 || ld_head < 0 || s.elems <= 0) return false;
  const int64_t token = ((H - 1) * ld_head + D) * esize, ld = ld_token * esize;
  const int64_t from = (int64_t)(reinterpret_cast<uintptr_t>(s.p) - reinterpret_cast<uintptr_t>(x));
  const int64_t end = from + s.elems * s.size;
  // token t's rows are at [t ld, t ld + token): the first that ends past `from`
  const int64_t t = from < token || ld == 0 ? 0 : (from - token) / ld + 1;
  return t < T && t * ld < end && t * ld + token > from;
}
// Rows of `row` bytes at every sum of its indices' strides (in bytes, not negative).
struct Strided {
  const void *p;
  int64_t row, n[3], ld[3];
};
// Whether bytes [from, end) from x's start on lie on its rows, the indices before d at
// 0.  Strides descend, so that few of an index's entries begin before `from` and reach
// past it; more than that lie on each other, and are taken as one piece.
inline bool touches_at(const Strided &x, int d, __int128 from, __int128 end) {
  __int128 inner = x.row;
  for (int i = d + 1; i < 3; ++i) inner += (__int128)(x.n[i] - 1) * x.ld[i];
  const __int128 ld = d < 3 ? x.ld[d] : 0, n = d < 3 ? x.n[d] : 1;
  if (end <= 0 || from >= inner + (n - 1) * ld) return false;
  if (d == 3 || from <= 0) return true;  // on the first row
  if (ld == 0) return touches_at(x, d + 1, from, end);
  const __int128 first = from < inner ? 0 : (from - inner) / ld + 1;
  for (__int128 i = first; i < n && i * ld < end; ++i)
    if (i - first == 64 || touches_at(x, d + 1, from - i * ld, end - i * ld)) return true;
  return false;
}
// Whether s lies on one of x's rows (it may lie between two).
inline bool touches(const Span &s, Strided x) {
  if (s.elems <= 0 || x.n[0] <= 0 || x.n[1] <= 0 || x.n[2] <= 0) return false;
  for (int i : {0, 1, 0})
    if (x.ld[i] < x.ld[i + 1]) std::swap(x.ld[i], x.ld[i + 1]), std::swap(x.n[i], x.n[i + 1]);
  const __int128 from = (__int128)reinterpret_cast<uintptr_t>(s.p) - reinterpret_cast<uintptr_t>(x.p);
  return touches_at(x, 0, from, from + (__int128)s.elems * s.size);
}
inline bool touches(const Span &s, std::initializer_list<Span> whole, std::initializer_list<Strided> rows) {
  for (const Span &x : whole)
    if (overlap(s, x)) return true;
  for (const Strided &x : rows)
    if (touches(s, x)) return true;
  return false;
}
inline int check_apart(const char *op, std::initializer_list<Span> in, std::initializer_list<Span> out) {
  for (auto o = out.begin(); o != out.end(); ++o) {
    for (const Span &i : in)
      if (overlap(*o, i)) return api_fail(ZT_EINVAL, "%s: an output overlaps an input", op);
    for (auto other = out.begin(); other != o; ++other)
      if (overlap(*o, *other)) return api_fail(ZT_EINVAL, "%s: two outputs overlap", op);
  }
  return ZT_OK;
}

inline int check_rotary(const char *op, const void *x, int64_t T, int64_t H, int64_t D,
                 const int64_t *positions, const float *table, int64_t length, int64_t R,
                 int64_t ld_table, const void *out) {
  if (T < 0 || H <= 0 || D <= 0) return api_fail(ZT_EINVAL, "%s: need T >= 0 and heads, head_dim > 0", op);
  if (R <= 0 || R % 2 || R > D)
    return api_fail(ZT_EINVAL, "%s: the table's width (%lld) must be even, positive and at most "
                    "head_dim = %lld", op, (long long)R, (long long)D);
  if (length < 0 || ld_table < R) return api_fail(ZT_EINVAL, "%s: bad table length or row stride", op);
  if (T > 0 && (!x || !positions || !out || (length > 0 && !table)))
    return api_fail(ZT_EINVAL, "%s: null tensor pointer", op);
  return ZT_OK;
}

// Grids are counted in 32 bits.
inline bool too_many(int64_t T, int64_t heads, int64_t D) {
  return heads > INT32_MAX / 4 || D > (1 << 20) || heads * D > INT32_MAX ||
         (double)T * (double)heads * (double)D >= 256.0 * 2147483647.0;
}

// The checked arguments of an attention call, without its pointers.  The caller has
// checked the cache, and whether its kernels can count the work.
inline int attn_args(const char *op, int64_t T, int64_t H, const zt_kv_cache *cache, int64_t S,
                     int64_t W, int64_t max_query_len, int32_t causal, int64_t window, AttnArgs *a) {
  if (T < 0 || H <= 0 || S < 0 || W < 0 || max_query_len < 0)
    return api_fail(ZT_EINVAL, "%s: need T, S, W, max_query_len >= 0 and heads > 0", op);
  if (H % cache->heads)
    return api_fail(ZT_EINVAL, "%s: query heads (%lld) must be a multiple of the cache's (%lld)", op,
                    (long long)H, (long long)cache->heads);
  if (cache->head_dim % 8 || cache->head_dim > 256)
    return api_fail(ZT_EUNSUPPORTED, "%s: head_dim must be a multiple of 8 up to 256, got %lld", op,
                    (long long)cache->head_dim);
  if (window < 0 || (window && !causal))
    return api_fail(ZT_EINVAL, "%s: a window (%lld) must not be negative and needs causal", op,
                    (long long)window);
  if (H > 65535 || S > kMaxSeqs || T > (1 << 24) || T * H > INT32_MAX / 2 || W > (1 << 24) ||
      cache->page_size > (1 << 24) || W * cache->page_size > (1 << 30))
    return api_fail(ZT_EUNSUPPORTED, "%s: at most 65535 heads, %lld sequences, 2^24 tokens, 2^30 / "
                    "heads rows and a table of 2^30 tokens a sequence", op, (long long)kMaxSeqs);
  *a = AttnArgs{};
  a->T = T, a->H = (int)H, a->KV = (int)cache->heads, a->D = (int)cache->head_dim;
  a->S = (int)S, a->W = (int)W, a->page_size = (int)cache->page_size, a->pages = cache->pages;
  a->dtype = cache->dtype, a->max_q = max_query_len, a->causal = causal != 0, a->window = window;
  return ZT_OK;
}

}  // namespace zt
