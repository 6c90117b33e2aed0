// Attention of a chunk of new tokens over a paged cache held in 4 bits, for
// gfx950.  The attention's definition and its running maximum and sum are
// described in paged_attn.hip, the rows, items and spans of work in
// attn_common.hpp, the format in mx4.hpp.
#include <cmath>

#include "attn_common.hpp"
#include "mx4.hpp"

namespace zt {

namespace {

constexpr int kRowThreads = 256;
constexpr int BM = 16;  // rows of an item

__device__ __forceinline__ u32x4_t load_once(const uint8_t *p) {
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

// The upper 16 bits of two numbers, as a pair of bf16.
__device__ __forceinline__ uint32_t tops(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
__device__ __forceinline__ float top(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

// 16 rows of one cache head against a span of its keys.
//
// A code's value is a bf16 number exactly, so the products are bf16 MFMAs without
// a rounding of keys or values: fp32 queries and weights go in three bf16 parts
// (cut short, 24 digits), bf16 ones in one and weights in two (p = hi + lo).
//
// The four waves are independent, wave w on every fourth strip of 32 keys; codes
// come straight to registers, the next strip's as soon as they are unpacked.  The
// products are transposed, S^T = K Q^T and O^T = V^T P^T on 16x16 MFMAs: lane
// (key n, g) of 16 x 4 unpacks 8 codes of its key to the A operand of an MFMA.  A
// lane has 16 consecutive bytes of the key, and the queries lie in that order of
// elements.  Values are unpacked to the wave's LDS, from which the transposing
// read takes columns.
template <typename T, int DP>
__global__ __launch_bounds__(kRowThreads, 2) void mx4_row_kernel(Mx4AttnArgs a) {
  using Cost = RowCost;
  constexpr bool BF = sizeof(T) == 2;
  constexpr int QP = BF ? 1 : 3, PP = BF ? 2 : 3;  // parts of a query and of a weight
  constexpr int KS = 32, UK = 4 * KS;     // keys of a strip and of a unit
  constexpr int CR = DP / 32;             // blocks of a row: 16 bytes, one scale
  constexpr int KL = DP <= 128 ? 1 : 2;   // loads of a key per lane
  constexpr int NV = KS * CR / 64;        // blocks of values per lane
  constexpr int NS = DP / 32;             // MFMA steps over a row
  constexpr int VP = DP * 2 + 32;         // LDS pitch of a row of values
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
  const int G = a.group;
  const char *zero = reinterpret_cast<const char *>(kZeroRow);
  const uint8_t *nothing = reinterpret_cast<const uint8_t *>(kZeroRow);
  // the element that step t of the lane begins with, and the block it lies in
  auto element = [&](int t) { return DP == 64 ? 16 * g + 8 * t : 128 * (t / 4) + 32 * g + 8 * (t % 4); };
  const int kblock = DP == 64 ? g / 2 : g;
  // the lane's j-th block of values: row and block
  auto vrow = [&](int j) { return CR == 2 ? lane & 31 : 16 * (j & 1) + n; };
  auto vblock = [&](int j) { return CR == 2 ? lane >> 5 : g + 4 * (j >> 1); };

  Walk<Cost> walk(plan);
  Segment seg;
  while (walk.next(a, plan, batch, BM, UK, &seg)) {
    const int h = seg.head, take = seg.take;
    const Seq s = batch.uniform(seg.seq);
    const int r0 = seg.tile * BM;
    const KeyRange kr = seg.keys;
    const Shared shared(a, s, seg.tile, BM);
    const Pages pages{a.table + (int64_t)seg.seq * a.W, kr.begin, kr.end};
    // the lane's row: token, and the keys it sees
    const int row_t = (int)fast_div(r0 + n, a.div_group);
    const bool live = row_t < s.q;
    const int pos = s.n - s.q + row_t;
    const int hi = !live ? INT32_MAX : a.causal ? pos + 1 : s.n;
    const int lo = live && a.causal && a.window ? (int)max((int64_t)pos + 1 - a.window, (int64_t)0) : 0;
    const int kend = (seg.b0 + seg.bb + take) * UK;
    int k0 = (seg.b0 + seg.bb) * UK + wave * KS;
    auto lookup = [&](int at) { return pages.lookup(a, at + (lane & 31)); };
    int page = lookup(k0);  // on its way while the queries are fetched
    // ---- the queries, as B operands
    u32x4_t q[QP][NS];
    {
      const char *src = static_cast<const char *>(a.q) +
          ((int64_t)(s.q0 + row_t) * a.q_ld[0] + (h * G + r0 + n - row_t * G) * a.q_ld[1]) * (int64_t)sizeof(T);
#pragma unroll
      for (int t = 0; t < NS; ++t) {
        const int e = element(t);
        const char *at = live && e < a.D ? src + e * sizeof(T) : zero;
        if constexpr (BF) {
          q[0][t] = scale_sign<T>(*reinterpret_cast<const u32x4_t *>(at), a.scale);
        } else {
          float x[8];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const u32x4_t w = scale_sign<T>(reinterpret_cast<const u32x4_t *>(at)[j], a.scale);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[4 * j + i] = __uint_as_float(w[i]);
          }
#pragma unroll
          for (int p = 0; p < QP; ++p)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              q[p][t][i] = tops(x[2 * i], x[2 * i + 1]);
              x[2 * i] -= top(x[2 * i]), x[2 * i + 1] -= top(x[2 * i + 1]);
            }
        }
      }
    }
    f32x4_t o[DT];
    float m = -INFINITY, l = 0.f;
    bool missed = false;  // the row sees a value that is not finite at an edge
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const uint8_t *kbase = static_cast<const uint8_t *>(a.k) + h * a.k_ld[1];
    const uint8_t *vbase = static_cast<const uint8_t *>(a.v) + h * a.v_ld[1];
    // scales: lane x < 32 has those of key x of the strip, lane 32 + x of value x
    const uint8_t *sbase = lane < 32 ? a.k_sc + h * a.k_sc_ld[1] : a.v_sc + h * a.v_sc_ld[1];
    const int64_t s_page = lane < 32 ? a.k_sc_ld[0] : a.v_sc_ld[0], s_tok = lane < 32 ? a.k_sc_ld[2] : a.v_sc_ld[2];

    u32x4_t kreg[2][KL], vreg[NV];
    uint32_t sreg[CR];
    uint64_t there;  // which of the strip's keys there are
    auto load = [&](int at, int page) {
      const int tok = at + (lane & 31);
      const bool ok = pages.there(a, tok, page);
      there = __ballot(ok);
      const uint32_t ko = ok ? row_offset(a, a.k_row, tok, page) : ~0u;
      const uint32_t vo = ok ? row_offset(a, a.v_row, tok, page) : ~0u;
      const int off = tok - (int)fast_div(tok, a.div_page) * a.page_size;
      const uint8_t *sc = ok ? sbase + page * s_page + off * s_tok : nothing;
#pragma unroll
      for (int i = 0; i < CR; ++i) sreg[i] = i < a.NB ? sc[i] : 0u;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t r = __shfl(ko, 16 * u + n);
        const uint8_t *src = kbase + (uint64_t)r * 16;
        if constexpr (DP == 64) {
          const u32x2_t y = __builtin_nontemporal_load(
              reinterpret_cast<const u32x2_t *>(r != ~0u && kblock < a.NB ? src + 8 * g : nothing));
          kreg[u][0][0] = y[0], kreg[u][0][1] = y[1];
        } else {
#pragma unroll
          for (int i = 0; i < KL; ++i) kreg[u][i] = load_once(r != ~0u && g + 4 * i < a.NB ? src + 16 * (g + 4 * i) : nothing);
        }
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const uint32_t r = __shfl(vo, vrow(j));
        vreg[j] = load_once(r != ~0u && vblock(j) < a.NB ? vbase + (uint64_t)r * 16 + 16 * vblock(j) : nothing);
      }
    };
    if (k0 < kend) load(k0, page);
    page = lookup(k0 + UK);
    for (; k0 < kend; k0 += UK) {
      // the lane's scales as words of four
      uint32_t words[(CR + 3) / 4] = {};
#pragma unroll
      for (int i = 0; i < CR; ++i) words[i / 4] |= sreg[i] << (8 * (i % 4));
      auto scale_of = [&](int row, int i, int byte) { return (__shfl(words[i], row) >> (8 * byte)) & 255u; };
      uint32_t bad = 0;  // keys whose values are not finite, at an edge
      const bool edge = shared.edge(k0, KS);
      // values to the wave's LDS (LDS operations of a wave keep their order)
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int row = vrow(j);
        uint32_t byte = scale_of(32 + row, j >> 1, CR == 2 ? lane >> 5 : g);
        bool taken = false;
        if (edge) {
          const bool is = byte > kMxLast;
          if (is) byte = 0, taken = true;
          for (uint64_t left = __ballot(is); left; left &= left - 1)
            bad |= 1u << __shfl(row, __builtin_ctzll(left));
        }
        const float sc = mx_scale(byte);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<u32x4_t *>(vlds + row * VP + ((64 * vblock(j) + 16 * i) ^ ((row & 8) << 1))) =
              mx_values(taken ? 0u : vreg[j][i], sc);
      }
      // scores: lane (row n, g) gets keys 16 u + 4 g .. + 3
      f32x4_t sc[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
        float ks[KL];
#pragma unroll
        for (int i = 0; i < KL; ++i) ks[i] = mx_scale(scale_of(16 * u + n, i, kblock));
#pragma unroll
        for (int t = 0; t < NS; ++t) {
          const bf16x8_t k = __builtin_bit_cast(bf16x8_t, mx_values(kreg[u][t / 4][t % 4], ks[t / 4]));
#pragma unroll
          for (int p = QP - 1; p >= 0; --p)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, __builtin_bit_cast(bf16x8_t, q[p][t]), acc, 0, 0, 0);
        }
        sc[u] = acc;
      }
      const uint32_t held = (uint32_t)there;
      if (k0 + UK < kend) {
        load(k0 + UK, page);
        page = lookup(k0 + 2 * UK);
      }
      // weights
      const bool some = held != ~0u || __ballot(lo > k0 || hi < k0 + KS);
      if (some) {
        // bit 16 u + e of `seen`: the lane's e-th key of 16
        const int from = min(max(lo - k0, 0), 32), to = min(max(hi - k0, 0), 32);
        const uint32_t range = (uint32_t)((1ull << to) - (1ull << min(from, to)));
        missed = missed || (live && (range & bad));
        const uint32_t seen = (range & held) >> (4 * g);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(seen & (1u << (16 * u + e)))) sc[u][e] = -INFINITY;
      } else {
        missed = missed || (live && bad);
      }
      float mx = sc[0][0];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sc[u][e]);
      mx = fmaxf(m, max_over_groups(mx));
      if (__ballot(mx > m)) {
        const float f = factor(m, mx, c);
        l *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[d][e] *= f;
        m = mx;
      }
      float mc = m == -INFINITY ? 0.f : m * c;
      if (__ballot(is_far(mc))) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[u][e] -= is_far(mc) ? m : 0.f;
        mc = is_far(mc) ? 0.f : mc;
      }
      u32x4_t pw[PP];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          float x[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            x[i] = __builtin_amdgcn_exp2f(fmaf(sc[u][e + i], c, -mc)) * kWeight;
            l += x[i];
          }
#pragma unroll
          for (int p = 0; p < PP; ++p) {
            pw[p][2 * u + e / 2] = p + 1 < PP ? tops(x[0], x[1]) : pack_bf16x2(x[0], x[1]);
            x[0] -= top(x[0]), x[1] -= top(x[1]);
          }
        }
      // O^T += V^T P^T
      const unsigned char *at0 = vlds + (4 * g + n / 4) * VP;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        typedef __attribute__((address_space(3))) s16x4_t *tr_ptr;
        const unsigned char *at = at0 + ((32 * d + 8 * (n & 3)) ^ ((g & 2) << 3));
        const s16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)at);
        const s16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(at + 16 * VP));
        const bf16x8_t v = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int p = PP - 1; p >= 0; --p)
          o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(bf16x8_t, pw[p]), o[d], 0, 0, 0);
      }
    }
    // ---- join the four waves
    const bool complete = seg.complete;
    const float lsum = sum_over_groups(l);
    __syncthreads();  // the waves' values are read
    if (lane < 16) sm_m[wave][n] = m, sm_l[wave][n] = lsum;
#pragma unroll
    for (int d = 0; d < DT; ++d)
      *reinterpret_cast<f32x4_t *>(vlds + (n * OP + 16 * d + 4 * g) * 4) = o[d];
    if (__builtin_expect(__ballot(missed) != 0, 0))  // the values that the wave's edges left out
      for (int k = (seg.b0 + seg.bb) * UK + wave * KS; k < kend; k += UK)
        for (int key = k; key < k + KS && shared.edge(k, KS); ++key) {
          const int at = pages.lookup(a, key);
          if (!pages.there(a, key, at) || !live || key < lo || key >= hi) continue;
          const int off = key - (int)fast_div(key, a.div_page) * a.page_size;
          const uint8_t *sc = a.v_sc + h * a.v_sc_ld[1] + at * a.v_sc_ld[0] + off * a.v_sc_ld[2];
#pragma unroll 1
          for (int col = 4 * g; col < a.D; col += 16)
            if (sc[col / kMxBlock] > kMxLast)
#pragma unroll 1
              for (int e = 0; e < 4; ++e) *reinterpret_cast<float *>(vlds + (n * OP + col + e) * 4) = NAN;
        }
    __syncthreads();
    for (int e = tid; e < 16 * DP / 4; e += kRowThreads) {
      const int row = e / (DP / 4), d = e % (DP / 4) * 4;
      const int rr = r0 + row;
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
        const int64_t pr = seg.slot * BM + row;
        *reinterpret_cast<f32x4_t *>(a.part_o + pr * a.D + d) = oo;
        if (d == 0) a.part_ml[2 * pr] = mm, a.part_ml[2 * pr + 1] = ll;
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

constexpr int kRowGrid = 512;  // workgroups, at most: two per CU

template <typename T, int DP>
hipError_t launch_rows(const Mx4AttnArgs &a, int grid, hipStream_t s) {
  constexpr int wave = std::max(32 * (DP * 2 + 32), 16 * (DP + 4) * 4);
  const size_t lds = 4 * wave + batch_ints(a.S) * 4, largest = 4 * wave + batch_ints(kMaxSeqs) * 4;
  auto kernel = mx4_row_kernel<T, DP>;
  const hipError_t allowed = allow_lds(reinterpret_cast<const void *>(kernel), lds, largest);
  if (allowed != hipSuccess) return allowed;
  kernel<<<grid, kRowThreads, lds, s>>>(a);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_rows_of(const Mx4AttnArgs &a, int grid, hipStream_t s) {
  if (a.D <= 64) return launch_rows<T, 64>(a, grid, s);
  if (a.D <= 128) return launch_rows<T, 128>(a, grid, s);
  return launch_rows<T, 256>(a, grid, s);
}

struct Shape {
  bool tiles;
  int bm, grid;
};
double items_most(const Mx4AttnArgs &a, int bm) { return std::floor((double)a.T * (a.H / a.KV) / bm) + a.S; }
double blocks_most(const Mx4AttnArgs &a, bool tiles) { return std::floor((double)a.W * a.page_size / (tiles ? 64 : 128)) + 1; }
Shape shape_of(const Mx4AttnArgs &a) {
  const int64_t rows = std::min(std::max<int64_t>(a.max_q, 1), a.T) * (a.H / a.KV);
  Shape p{rows > BM, BM, kRowGrid};
  if (p.tiles) p.bm = mx4_tile_rows(), p.grid = mx4_tile_grid(a);
  // no more workgroups than there can be blocks
  const double most = items_most(a, p.bm) * a.KV * blocks_most(a, p.tiles);
  if (most < p.grid) p.grid = std::max((int)most, 1);
  return p;
}

}  // namespace

bool paged_attn_mx4_countable(const Mx4AttnArgs &a) {
  const Shape p = shape_of(a);
  return items_most(a, p.bm) * (blocks_most(a, p.tiles) * kTileCostMost + kTileCostLead) < 2147483647.0;
}

size_t paged_attn_mx4_workspace(const Mx4AttnArgs &a) {
  if (a.T == 0) return 0;
  const Shape p = shape_of(a);
  return parts_bytes(a, p.grid, p.bm);
}

hipError_t launch_paged_attn_mx4(Mx4AttnArgs a, void *workspace, hipStream_t s) {
  const Shape p = shape_of(a);
  a.group = a.H / a.KV;
  a.div_group = make_div(a.group), a.div_page = make_div(a.page_size);
  for (int i = 0; i < 2; ++i)
    a.k_row[i] = (uint32_t)(a.k_ld[2 * i] / 16), a.v_row[i] = (uint32_t)(a.v_ld[2 * i] / 16);
  lay_parts(&a, workspace, p.grid, p.bm);
  const hipError_t e = p.tiles                   ? launch_mx4_tiles(a, p.grid, s)
                       : a.dtype == ZT_DT_BF16 ? launch_rows_of<uint16_t>(a, p.grid, s)
                                               : launch_rows_of<float>(a, p.grid, s);
  if (e != hipSuccess) return e;
  return launch_join(a, p.grid, s);
}

}  // namespace zt
