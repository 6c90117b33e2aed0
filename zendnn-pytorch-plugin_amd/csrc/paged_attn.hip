// Attention of a chunk of new tokens over a paged cache, for gfx950: few rows
// per cache head (decoding, short chunks), and the launch of both kernels.
//
//   o_r = sum_j exp(s_rj - m_r) v_j / sum_j exp(s_rj - m_r),
//   s_rj = scale * q_r . k_j,  m_r = max_j s_rj
//
// over the cached tokens j that row r (one query token, one head) sees: with
// q new tokens of n in all, token a sits at position n - q + a and sees the
// positions up to its own (causal), and of those the last `window` (if that
// is not 0).  A row that sees none is zero.
//
// Keys come in any order of blocks, with a running maximum m and sum l:
//   m' = max(m, max_j s_j),  l' = l e^(m - m') + sum_j e^(s_j - m'),
//   o' = o e^(m - m') + sum_j e^(s_j - m') v_j,
// and two parts (m, l, o) join the same way.  Scores, weights and sums are
// fp32; exponentials are powers of two with scale * log2(e) in the exponent.
#include <cmath>

#include "attn_common.hpp"

namespace zt {

namespace {

constexpr int kRowThreads = 256;

// Keys and values are read by one workgroup only: past the caches' replacement.
__device__ __forceinline__ u32x4_t load_once(const char *p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(p));
}

__device__ __forceinline__ float max_over_groups(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum_over_groups(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// 16 NT rows of one cache head against a span of its keys.
//
// Bound by HBM: the keys and values are read once, straight to registers, and
// each CU needs some 64 KB of them in flight.  So the four waves are
// independent of each other: wave w takes every fourth strip of KS keys (32,
// or 16 in fp32: 8 KB of keys and 8 KB of values at head_dim 128), with the
// next strip's loads issued as soon as the scores have used up the keys'
// registers; they meet only at the end of an (item, head).
//
// The products are taken transposed, S^T = K Q^T and O^T = V^T P^T, on 16x16
// MFMAs with the rows as columns.  The scores' layout (lane (row, g) holds
// keys 4 g .. 4 g + 3) then is the layout in which the second product takes
// its weights, without a move between lanes, if V^T takes its keys in the
// same order.  V^T needs each lane to hold keys of one column: in fp32 plain
// LDS reads give that, in bf16 the transposing ds_read_b64_tr_b16 (lane i of
// 16 gets column i of the four rows whose pieces the 16 lanes point at).  Each
// wave passes its values through LDS of its own.
//
// bf16 weights keep the digits that one bf16 drops in a second MFMA (p = hi +
// lo): the matrix pipe is idle most of the time here.
//
// Measured (32 query and 8 cache heads of 128, bf16): two sequences of 131072
// tokens 172-173 us, 6.2 TB/s; 64 ragged ones of up to 8192 129 us, 5.9
// TB/s (a large copy reaches 4.9).  One of 777: 10.9 us, round trips to memory.
template <typename T, int DP, int NT>
__global__ __launch_bounds__(kRowThreads, DP <= 128 ? 2 : 1) void paged_attn_row_kernel(AttnArgs a) {
  using Cost = RowCost;
  constexpr bool BF = sizeof(T) == 2;
  constexpr int ES = sizeof(T);
  constexpr int BM = 16 * NT;
  constexpr int KT = BF ? 2 : 1;          // 16-key tiles of a strip
  constexpr int KS = 16 * KT;             // keys of a strip
  constexpr int UK = 4 * KS;              // keys of a unit
  constexpr int KC = DP * ES / 64;        // 16-byte pieces of a key per lane
  constexpr int CR = DP * ES / 16;        // 16-byte pieces of a row
  constexpr int NV = KS * CR / 64;        // value pieces per lane
  constexpr int VP = DP * ES + (BF ? 32 : 16);  // LDS pitch: the reads meet no bank twice
  constexpr int OP = DP + 4;              // pitch of the joined outputs, floats
  constexpr int DT = DP / 16;
  constexpr int kWaveLds = KS * VP > 16 * OP * 4 ? KS * VP : 16 * OP * 4;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  __shared__ PlanShared sh;
  __shared__ float sm_m[4][16], sm_l[4][16];
  const Batch batch(smem + 4 * kWaveLds, a.S);

  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  unsigned char *vlds = smem + wave * kWaveLds;
  const Plan plan = make_plan<kRowThreads, Cost>(a, BM, UK, batch, &sh);
  Split *split = static_cast<Split *>(a.splits) + plan.wg;
  if (tid == 0) split->rows = 0;

  const float c = score_factor(a.scale);
  const int G = a.group, C = a.D * ES / 16;  // 16-byte pieces that a row has
  const char *zero = reinterpret_cast<const char *>(kZeroRow);

  Walk<Cost> walk(plan);
  Segment seg;
  while (walk.next(a, plan, batch, BM, UK, &seg)) {
    const int h = seg.head, take = seg.take;
    const Seq s = batch.uniform(seg.seq);
    const int r0 = seg.tile * BM;
    const KeyRange kr = seg.keys;
    const Shared shared(a, s, seg.tile, BM);
    const Pages pages{a.table + (int64_t)seg.seq * a.W, kr.begin, kr.end};
    // the lane's rows: token, head, and the keys each sees
    int row_t[NT], lo[NT], hi[NT];
    bool live[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = r0 + 16 * t + n;
      row_t[t] = (int)fast_div(row, a.div_group);
      live[t] = row_t[t] < s.q;
      const int pos = s.n - s.q + row_t[t];
      hi[t] = !live[t] ? INT32_MAX : a.causal ? pos + 1 : s.n;
      lo[t] = live[t] && a.causal && a.window ? (int)max((int64_t)pos + 1 - a.window, (int64_t)0) : 0;
    }
    const int kend = (seg.b0 + seg.bb + take) * UK;
    int k0 = (seg.b0 + seg.bb) * UK + wave * KS;
    auto lookup = [&](int at) { return pages.lookup(a, at + (lane & (KS - 1))); };
    int page = lookup(k0);  // on its way while the queries are fetched
    // ---- the queries, as B operands: lane (row n, g) holds piece 4 j + g
    u32x4_t q[NT][KC];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = r0 + 16 * t + n;
      const char *src = static_cast<const char *>(a.q) +
          ((int64_t)(s.q0 + row_t[t]) * a.q_ld[0] + (h * G + row - row_t[t] * G) * a.q_ld[1]) * ES;
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        const int p = 4 * j + g;
        q[t][j] = scale_sign<T>(*reinterpret_cast<const u32x4_t *>(live[t] && p < C ? src + 16 * p : zero), a.scale);
      }
    }
    f32x4_t o[NT][DT];
    float m[NT], l[NT];
    bool missed[NT];  // the row sees a value that is not finite at an edge
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = -INFINITY, l[t] = 0.f, missed[t] = false;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[t][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    const char *kbase = static_cast<const char *>(a.k) + h * a.k_ld[1] * ES;
    const char *vbase = static_cast<const char *>(a.v) + h * a.v_ld[1] * ES;

    u32x4_t kreg[KT][KC], vreg[NV];
    uint64_t there;  // which of the strip's keys there are
    auto load = [&](int at, int page) {
      const int tok = at + (lane & (KS - 1));
      const bool ok = pages.there(a, tok, page);
      there = __ballot(ok);
      const uint32_t ko = ok ? row_offset(a, a.k_row, tok, page) : ~0u;
      const uint32_t vo = ok ? row_offset(a, a.v_row, tok, page) : ~0u;
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const uint32_t r = __shfl(ko, 16 * t + n);
        const char *src = r == ~0u ? zero : kbase + (uint64_t)r * 16;
#pragma unroll
        for (int j = 0; j < KC; ++j) {
          const int p = 4 * j + g;
          kreg[t][j] = load_once(p < C ? src + 16 * p : zero);
        }
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int idx = 64 * j + lane, row = idx / CR, p = idx % CR;
        const uint32_t r = __shfl(vo, row);
        vreg[j] = load_once(r != ~0u && p < C ? vbase + (uint64_t)r * 16 + 16 * p : zero);
      }
    };
    if (k0 < kend) load(k0, page);
    page = lookup(k0 + UK);
    for (; k0 < kend; k0 += UK) {
      uint32_t bad = 0;  // keys whose values are not finite, at an edge
      if (shared.edge(k0, KS))
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const bool is = not_finite<T>(vreg[j]);
          if (is) vreg[j] = finite_of<T>(vreg[j]);
          for (uint64_t left = __ballot(is); left; left &= left - 1)
            bad |= 1u << ((64 * j + __builtin_ctzll(left)) / CR);
        }
      // values to the wave's LDS (LDS operations of a wave keep their order)
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int idx = 64 * j + lane, row = idx / CR, p = idx % CR;
        *reinterpret_cast<u32x4_t *>(vlds + row * VP + 16 * p) = vreg[j];
      }
      // scores: lane (row n, g) gets keys 16 u + 4 g .. + 3
      f32x4_t sc[NT][KT];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < KT; ++u) {
          f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < KC; ++j) {
            if constexpr (BF) {
              acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  __builtin_bit_cast(bf16x8_t, kreg[u][j]), __builtin_bit_cast(bf16x8_t, q[t][j]), acc, 0, 0, 0);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kreg[u][j][e]),
                                                           __uint_as_float(q[t][j][e]), acc, 0, 0, 0);
            }
          }
          sc[t][u] = acc;
        }
      const uint64_t held = there;
      const bool whole = (uint32_t)held == (KS == 32 ? ~0u : 0xffffu) || (KS == 16 && (held & 0xffff) == 0xffff);
      if (k0 + UK < kend) {
        load(k0 + UK, page);
        page = lookup(k0 + 2 * UK);
      }
      // weights
      bf16x8_t ph[NT], pl[NT];
      float pf[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (bad) {
          const int from = min(max(lo[t] - k0, 0), 32), to = min(max(hi[t] - k0, 0), 32);
          const uint64_t range = (1ull << to) - (1ull << min(from, to));
          missed[t] = missed[t] || (live[t] && ((uint32_t)range & bad));
        }
        if (!whole || __ballot(lo[t] > k0 || hi[t] < k0 + KS)) {
          // bit 16 u + e of `seen`: the lane's e-th key of 16
          const int from = min(max(lo[t] - k0, 0), 32), to = min(max(hi[t] - k0, 0), 32);
          const uint64_t range = (1ull << to) - (1ull << min(from, to));
          const uint32_t seen = ((uint32_t)range & (uint32_t)held) >> (4 * g);
#pragma unroll
          for (int u = 0; u < KT; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!(seen & (1u << (16 * u + e)))) sc[t][u][e] = -INFINITY;
        }
        float mx = sc[t][0][0];
#pragma unroll
        for (int u = 0; u < KT; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sc[t][u][e]);
        mx = fmaxf(m[t], max_over_groups(mx));
        if (__ballot(mx > m[t])) {
          const float f = factor(m[t], mx, c);
          l[t] *= f;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][d][e] *= f;
          m[t] = mx;
        }
        float mc = m[t] == -INFINITY ? 0.f : m[t] * c;
        if (__ballot(is_far(mc))) {
#pragma unroll
          for (int u = 0; u < KT; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[t][u][e] -= is_far(mc) ? m[t] : 0.f;
          mc = is_far(mc) ? 0.f : mc;
        }
#pragma unroll
        for (int u = 0; u < KT; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = __builtin_amdgcn_exp2f(fmaf(sc[t][u][e], c, -mc)) * kWeight;
            l[t] += p;
            if constexpr (BF) {
              const __bf16 hi_part = (__bf16)p;
              ph[t][4 * u + e] = hi_part;
              pl[t][4 * u + e] = (__bf16)(p - (float)hi_part);
            } else {
              pf[t][e] = p;
            }
          }
      }
      // O^T += V^T P^T
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        if constexpr (BF) {
          typedef __attribute__((address_space(3))) s16x4_t *tr_ptr;
          const unsigned char *at = vlds + (4 * g + n / 4) * VP + 32 * d + 8 * (n & 3);
          const s16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)at);
          const s16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(at + 16 * VP));
          const bf16x8_t v = __builtin_bit_cast(
              bf16x8_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, ph[t], o[t][d], 0, 0, 0);
            o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pl[t], o[t][d], 0, 0, 0);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = *reinterpret_cast<const float *>(vlds + (4 * g + e) * VP + 4 * (16 * d + n));
#pragma unroll
            for (int t = 0; t < NT; ++t)
              o[t][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, pf[t][e], o[t][d], 0, 0, 0);
          }
        }
      }
    }
    // ---- join the four waves, 16 rows at a time
    const bool complete = seg.complete;
    const int64_t slot = seg.slot;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float lsum = sum_over_groups(l[t]);
      __syncthreads();  // the waves' values and the previous rows are read
      if (lane < 16) sm_m[wave][n] = m[t], sm_l[wave][n] = lsum;
#pragma unroll
      for (int d = 0; d < DT; ++d)
        *reinterpret_cast<f32x4_t *>(vlds + (n * OP + 16 * d + 4 * g) * 4) = o[t][d];
      if (__builtin_expect(__ballot(missed[t]) != 0, 0))  // the values that the wave's edges left out
        for (int k = (seg.b0 + seg.bb) * UK + wave * KS; k < kend; k += UK)
          for (int key = k; key < k + KS && shared.edge(k, KS); ++key) {
            const int at = pages.lookup(a, key);
            if (!pages.there(a, key, at) || !live[t] || key < lo[t] || key >= hi[t]) continue;
            const T *v = reinterpret_cast<const T *>(vbase + (uint64_t)row_offset(a, a.v_row, key, at) * 16);
#pragma unroll 1
            for (int col = 4 * g; col < a.D; col += 16)
#pragma unroll 1
              for (int e = 0; e < 4; ++e) {
                float x;
                if constexpr (BF) x = bf16_bits_to_f32(v[col + e]);
                else x = v[col + e];
                if (!(fabsf(x) < INFINITY)) *reinterpret_cast<float *>(vlds + (n * OP + col + e) * 4) += x;
              }
          }
      __syncthreads();
      for (int e = tid; e < 16 * DP / 4; e += kRowThreads) {
        const int row = e / (DP / 4), d = e % (DP / 4) * 4;
        const int rr = r0 + 16 * t + row;
        const int tok = (int)fast_div(rr, a.div_group);
        if (tok >= s.q || d >= a.D) continue;
        const float mm = fmaxf(fmaxf(sm_m[0][row], sm_m[1][row]), fmaxf(sm_m[2][row], sm_m[3][row]));
        float ll = 0.f;
        f32x4_t oo = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float f = factor(sm_m[w][row], mm, c);
          ll += f * sm_l[w][row];
          const f32x4_t y = *reinterpret_cast<const f32x4_t *>(smem + w * kWaveLds + (row * OP + d) * 4);
#pragma unroll
          for (int k = 0; k < 4; ++k) oo[k] += f * y[k];
        }
        if (complete) {
          const int64_t at = ((int64_t)(s.q0 + tok) * a.H + h * G + rr - tok * G) * a.D + d;
          store_out<T>(a.out, at, oo, ll > 0.f ? 1.f / ll : 0.f);
        } else {
          const int64_t pr = slot * BM + 16 * t + row;
          *reinterpret_cast<f32x4_t *>(a.part_o + pr * a.D + d) = oo;
          if (d == 0) a.part_ml[2 * pr] = mm, a.part_ml[2 * pr + 1] = ll;
        }
      }
    }
    __syncthreads();  // before the next strips' values
    if (tid == 0 && seg.bb == 0 && !complete) {
      split->slot = seg.slot, split->last = seg.last;
      split->row0 = r0, split->rows = min(BM, s.q * G - r0), split->head = h, split->q0 = s.q0;
    }
  }
  zero_rows<kRowThreads>(a, plan, BM, UK, batch);
}

// One row's parts (running maximum, sum, four outputs), K loads at a time.  A
// part whose maximum is -inf saw no key, and is all zeros, or only keys whose
// scores are NaN, and its sums are: it joins parts like it as it is, so that the
// NaN shows however the keys were cut.
template <int K>
__device__ __forceinline__ f32x4_t join_parts(const AttnArgs &a, const Split &s, int first, int row, int d,
                                              float c, float *sum) {
  const int BM = a.item_rows, last = (int)s.last;
  float m = -INFINITY, l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int w0 = first; w0 <= last; w0 += K) {
    float mw[K], lw[K];
    f32x4_t y[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {  // past the last part: that one again, weighing nothing
      const int w = min(w0 + k, last);
      const int64_t at = (w == first ? s.slot : 2 * (int64_t)w) * BM + row;
      mw[k] = w0 + k <= last ? a.part_ml[2 * at] : -INFINITY;
      lw[k] = a.part_ml[2 * at + 1];
      y[k] = *reinterpret_cast<const f32x4_t *>(a.part_o + at * a.D + d);
    }
    float mm = m;
#pragma unroll
    for (int k = 0; k < K; ++k) mm = fmaxf(mm, mw[k]);
    const float f0 = factor(m, mm, c);
    m = mm, l *= f0;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= f0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float f = factor(mw[k], mm, c);
      l += lw[k] * f;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += y[k][e] * f;
    }
  }
  *sum = l;
  return o;
}

// Joins the parts of the (item, head) that workgroup blockIdx.x of the first
// launch began and others finished.  A thread takes four outputs of a row.
// Most are cut once (two parts); a long axis with few rows in dozens.  Bound by
// its round trips (2.4 us for seven parts of 32 rows) or by the parts' bytes.
template <typename T, bool DEEP>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(AttnArgs a) {
  const Split s = static_cast<const Split *>(a.splits)[blockIdx.x];
  if (s.rows == 0) return;
  const float c = score_factor(a.scale);
  const int first = (int)blockIdx.x, d4 = a.D / 4, G = a.group;
  const int64_t parts = s.last - first;  // but one
  for (int e = blockIdx.y * 256 + threadIdx.x; e < s.rows * d4; e += gridDim.y * 256) {
    const int row = e / d4, d = (e - row * d4) * 4;
    float l;
    const f32x4_t o = parts < 2             ? join_parts<2>(a, s, first, row, d, c, &l)
                      : DEEP && parts >= 16 ? join_parts<32>(a, s, first, row, d, c, &l)
                                            : join_parts<8>(a, s, first, row, d, c, &l);
    const int rr = s.row0 + row, tok = (int)fast_div(rr, a.div_group);
    const int64_t at = ((int64_t)(s.q0 + tok) * a.H + s.head * G + rr - tok * G) * a.D + d;
    store_out<T>(a.out, at, o, l > 0.f ? 1.f / l : 0.f);
  }
}

// Workgroups of the first launch, at most: two per CU.
constexpr int kRowGrid = 512;

template <typename T, int DP, int NT>
hipError_t launch_rows(const AttnArgs &a, int grid, hipStream_t s) {
  constexpr int KS = sizeof(T) == 2 ? 32 : 16, VP = DP * (int)sizeof(T) + (sizeof(T) == 2 ? 32 : 16);
  constexpr int wave = std::max(KS * VP, 16 * (DP + 4) * 4);
  const size_t lds = 4 * wave + batch_ints(a.S) * 4, largest = 4 * wave + batch_ints(kMaxSeqs) * 4;
  if (a.item_rows != 16 * NT) return hipErrorInvalidValue;
  auto kernel = paged_attn_row_kernel<T, DP, NT>;
  const hipError_t allowed = allow_lds(reinterpret_cast<const void *>(kernel), lds, largest);
  if (allowed != hipSuccess) return allowed;
  kernel<<<grid, kRowThreads, lds, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_rows_of(const AttnArgs &a, int grid, hipStream_t s) {
  if (a.dtype == ZT_DT_BF16) {
    if (a.D <= 64) return launch_rows<uint16_t, 64, 1>(a, grid, s);
    if (a.D <= 128) return launch_rows<uint16_t, 128, 1>(a, grid, s);
    return launch_rows<uint16_t, 256, 1>(a, grid, s);
  }
  if (a.D > 128) return launch_rows<float, 256, 1>(a, grid, s);
  if (a.item_rows == 16)
    return a.D <= 64 ? launch_rows<float, 64, 1>(a, grid, s) : launch_rows<float, 128, 1>(a, grid, s);
  return a.D <= 64 ? launch_rows<float, 64, 2>(a, grid, s) : launch_rows<float, 128, 2>(a, grid, s);
}

// Rows of one cache head up to which the row kernel is taken.  Measured, row
// against tile kernel, 8 cache heads, 32 sequences of 2048 tokens, us:
//   bf16  head_dim 64:  16 rows 34 / 35   32 rows 45 / 36    64 rows 82 / 42
//         head_dim 128: 16 rows 57 / 56   32 rows 82 / 59    64 rows 153 / 65
//         head_dim 256: 16 rows 127 / 119 32 rows 169 / 121  64 rows 326 / 123
//   fp32  head_dim 64:  16 rows 54 / 92   32 rows 79 / 96    48 rows 128 / 115
//         head_dim 128: 32 rows 179 / 297 64 rows 264 / 303  80 rows 428 / 307
//         head_dim 256: 32 rows 354 / 766 48 rows 580 / 776  64 rows 669 / 778
// and at the last two's borders 4 of 32768 503 / 580 (64 rows of 128) and 1004 / 1528
// (48 of 256), 64 of 500 178 / 190 and 360 / 440, where 64 rows of 256 are 472 / 441.
// On few long sequences (4 of 32768) the row kernel gains at 16 rows in bf16 too:
// 99 against 111 us at head_dim 128.
int rows_most(const AttnArgs &a) {
  if (a.dtype == ZT_DT_BF16) return 16;
  return a.D <= 64 ? 32 : a.D <= 128 ? 64 : 48;
}
// Rows of an item of the row kernel: 16, or 32 where two times 16 share the keys.
int row_item(const AttnArgs &a, int64_t rows) {
  return a.dtype == ZT_DT_F32 && a.D <= 128 && rows > 16 ? 32 : 16;
}

struct Shape {
  bool tiles;
  int bm, grid;
};
double items_most(const AttnArgs &a, int bm) { return std::floor((double)a.T * (a.H / a.KV) / bm) + a.S; }
double blocks_most(const AttnArgs &a, bool tiles) {
  const int keys = (tiles ? 64 : 128) / (a.dtype == ZT_DT_F32 ? 2 : 1);
  return std::floor((double)a.W * a.page_size / keys) + 1;
}
Shape shape_of(const AttnArgs &a) {
  const int64_t rows = std::min(std::max<int64_t>(a.max_q, 1), a.T) * (a.H / a.KV);
  Shape p{rows > rows_most(a), row_item(a, rows), kRowGrid};
  if (p.tiles) p.bm = tile_rows(a), p.grid = tile_grid(a);
  // no more workgroups than there can be blocks
  const double most = items_most(a, p.bm) * a.KV * blocks_most(a, p.tiles);
  if (most < p.grid) p.grid = std::max((int)most, 1);
  return p;
}

}  // namespace

bool paged_attn_countable(const AttnArgs &a) {
  const Shape p = shape_of(a);
  return items_most(a, p.bm) * (blocks_most(a, p.tiles) * kTileCostMost + kTileCostLead) < 2147483647.0;
}

size_t paged_attn_workspace(const AttnArgs &a) {
  if (a.T == 0) return 0;
  const Shape p = shape_of(a);
  return parts_bytes(a, p.grid, p.bm);
}

hipError_t launch_join(const AttnArgs &a, int grid, bool deep, hipStream_t s) {
  const dim3 g(grid, std::max(a.item_rows * a.D / 1024, 1));  // a thread per four outputs
  auto go = [&](auto kernel) { kernel<<<g, 256, 0, s>>>(a); };
  if (a.dtype == ZT_DT_BF16) deep ? go(paged_attn_join_kernel<uint16_t, true>) : go(paged_attn_join_kernel<uint16_t, false>);
  else deep ? go(paged_attn_join_kernel<float, true>) : go(paged_attn_join_kernel<float, false>);
  return hipGetLastError();
}

hipError_t launch_paged_attn(AttnArgs a, void *workspace, hipStream_t s) {
  const Shape p = shape_of(a);
  a.group = a.H / a.KV;
  a.div_group = make_div(a.group), a.div_page = make_div(a.page_size);
  const int64_t per16 = a.dtype == ZT_DT_F32 ? 4 : 8;
  for (int i = 0; i < 2; ++i)
    a.k_row[i] = (uint32_t)(a.k_ld[2 * i] / per16), a.v_row[i] = (uint32_t)(a.v_ld[2 * i] / per16);
  lay_parts(&a, workspace, p.grid, p.bm);
  const hipError_t e = p.tiles ? launch_tiles(a, p.grid, s) : launch_rows_of(a, p.grid, s);
  if (e != hipSuccess) return e;
  return launch_join(a, p.grid, false, s);
}

}  // namespace zt
