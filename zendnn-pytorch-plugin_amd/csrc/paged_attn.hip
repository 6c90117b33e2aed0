// Attention of a chunk of new tokens over a paged cache, for gfx950.
//
//   o_r = sum_j exp(s_rj - m_r) v_j / sum_j exp(s_rj - m_r),
//   s_rj = scale * q_r . k_j,  m_r = max_j s_rj
//
// over the cached tokens j that row r (one query token, one head) sees: with
// q new tokens of n in all, token a sits at position n - q + a and sees the
// positions up to its own (causal), and of those the last `window` (if that
// is not 0).  A row that sees none is zero.
#include "zt_cache.hpp"

namespace zt {

namespace {

template <typename T>
__device__ __forceinline__ float elem(const T *p);
template <>
__device__ __forceinline__ float elem<float>(const float *p) { return *p; }
template <>
__device__ __forceinline__ float elem<uint16_t>(const uint16_t *p) { return bf16_bits_to_f32(*p); }

// One workgroup per row: wave w takes the keys w, w + 4, .., each lane up to
// four of the head's elements, with a running maximum and sum per wave; the
// four waves' parts are joined at the end.
template <typename T>
__global__ __launch_bounds__(256) void paged_attn_row_kernel(AttnArgs a) {
  __shared__ float sm_m[4], sm_l[4], sm_o[4][256];
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int lo = 0, hi = a.S + 1;
  while (lo < hi) {
    const int m = (lo + hi) / 2;
    if (a.cu[m] > t) hi = m;
    else lo = m + 1;
  }
  const int i = lo - 1;
  int64_t begin = 0, end = 0;
  if (i >= 0 && i < a.S) {
    const int64_t n = min((int64_t)max(a.ctx[i], 0), (int64_t)a.W * a.page_size);
    const int64_t pos = n - (a.cu[i + 1] - t);
    end = a.causal ? min(pos + 1, n) : n;
    if (a.window) begin = max(pos + 1 - a.window, (int64_t)0);
  }
  const T *q = static_cast<const T *>(a.q) + t * a.q_ld[0] + h * a.q_ld[1];
  const int kvh = h / (a.H / a.KV);
  float x[4], o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c < 4; ++c) x[c] = lane + 64 * c < a.D ? elem(q + lane + 64 * c) : 0.f;
  float m = -INFINITY, l = 0.f;
  for (int64_t j = begin + wave; j < end; j += 4) {
    const int64_t col = j / a.page_size, off = j - col * a.page_size;
    const int page = a.table[(int64_t)i * a.W + col];
    if (page < 0 || page >= a.pages) continue;
    const T *k = static_cast<const T *>(a.k) + page * a.k_ld[0] + kvh * a.k_ld[1] + off * a.k_ld[2];
    const T *v = static_cast<const T *>(a.v) + page * a.v_ld[0] + kvh * a.v_ld[1] + off * a.v_ld[2];
    float s = 0.f;
    for (int c = 0; c < 4; ++c)
      if (lane + 64 * c < a.D) s += x[c] * elem(k + lane + 64 * c);
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    s *= a.scale;
    const float mn = fmaxf(m, s), f = mn == -INFINITY ? 0.f : expf(m - mn);
    const float p = mn == -INFINITY ? 0.f : expf(s - mn);
    m = mn, l = l * f + p;
    for (int c = 0; c < 4; ++c)
      if (lane + 64 * c < a.D) o[c] = o[c] * f + p * elem(v + lane + 64 * c);
  }
  if (lane == 0) sm_m[wave] = m, sm_l[wave] = l;
  for (int c = 0; c < 4; ++c) sm_o[wave][lane + 64 * c] = o[c];
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= a.D) return;
  float mm = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3])), ll = 0.f, oo = 0.f;
  for (int w = 0; w < 4; ++w) {
    const float f = sm_m[w] == -INFINITY ? 0.f : expf(sm_m[w] - mm);
    ll += f * sm_l[w], oo += f * sm_o[w][d];
  }
  store_elem(a.out, a.dtype, (t * a.H + h) * a.D + d, ll > 0.f ? oo / ll : 0.f);
}

}  // namespace

size_t paged_attn_workspace(const AttnArgs &) { return 0; }

hipError_t launch_paged_attn(const AttnArgs &a, void *, hipStream_t s) {
  const dim3 grid((unsigned)a.T, (unsigned)a.H);
  if (a.dtype == ZT_DT_BF16) paged_attn_row_kernel<uint16_t><<<grid, dim3(256), 0, s>>>(a);
  else paged_attn_row_kernel<float><<<grid, dim3(256), 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace zt
