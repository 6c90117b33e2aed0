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
// An item's beginning and end cost two units of 256 keys, in the trips to memory that
// nothing hides: 64 ragged sequences 49 us, with one unit 53, with three 50.
struct Mx4RowCost {
  static constexpr int kLead = 2, kMost = 1, kLeast = 1, kJoin = 0;
  static __device__ __forceinline__ int of(int) { return 1; }
};
constexpr int row_strip(int dp) { return dp <= 128 ? 64 : 32; }

// Over the four lanes of a row, 16 apart: rows of 16 lanes, then halves of the wave,
// change places, which costs no trip through LDS.
__device__ __forceinline__ float max_over_groups(float x) {
  const u32x2_t a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const u32x2_t b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_over_groups(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// 16 rows of one cache head against a span of its keys.
//
// Bound by HBM on large calls, and by its trips to memory on small ones: a key and its
// value of 128 numbers are 136 bytes, which a CU gets in 14 cycles, and unpacking,
// scores and weights of 64 of them are 430 instructions of a wave.
//
// A code's value is a bf16 number exactly, so the products are bf16 MFMAs without
// a rounding of keys or values: fp32 queries and weights go in three bf16 parts
// (cut short, 24 digits), bf16 ones in one and weights in two (p = hi + lo).
//
// The four waves are independent, wave w on every fourth strip of KS keys (64, or
// 32 past head_dim 128), whose codes come straight to registers, a part of the next
// strip's as soon as the part is unpacked.  The products are transposed, S^T = K Q^T
// and O^T = V^T P^T on 16x16 MFMAs.  Lane (n, g) of 16 x 4 has quarter g of the
// codes of keys 16 u + n, and of their values: it unpacks 8 codes of its key to the A
// operand of an MFMA, and the queries lie in that order of elements.  Values are
// unpacked to the wave's LDS, 32 keys at a time, from which the transposing read
// takes columns.
//
// A key's place is found by the lane of its number, which also has its scales.  A
// key that is not there is read from the cache's first row: its score is masked by
// selection, and its value is taken as zeros.
//
// A loop's every turn issues the same loads, past the last strip too (of the first
// row then): a load behind a branch makes each wait one for all loads in flight.
//
// Measured (32 query and 8 cache heads of 128, bf16): two sequences of 131072 tokens 60
// us (the kernel 55, 5.2 TB/s; with its ends of some 9 us taken off 6), 64 ragged ones of
// up to 8192 50, one of 777 13.  Three workgroups a CU, with registers for 168 numbers
// a lane, took 76 us on the two (61 with two then): the loads go out later.  Strips
// of 32 keys: 79 and 64.  Two moved 16-byte pieces keep LDS free of conflicts (128
// cycles a strip without).
//
// NEAR: a near cache's places (mx4.hpp) are found with a third of the instructions.
// WORDS: a row's scales are loaded together.
template <typename T, int DP, int DC, bool NEAR, bool WORDS>
__global__ __launch_bounds__(kRowThreads, 2) void mx4_row_kernel(Mx4AttnArgs a) {
  using Cost = Mx4RowCost;
  constexpr bool BF = sizeof(T) == 2;
  constexpr int QP = BF ? 1 : 3, PP = BF ? 2 : 3;  // parts of a query and of a weight
  constexpr int KS = row_strip(DP), UK = 4 * KS;   // keys of a strip and of a unit
  constexpr bool WIDE = KS == 64;         // a lane to a key, else lanes 32 .. 63 do the values' part
  constexpr int KT = KS / 16;             // 16-key tiles of a strip
  constexpr int WB = DP == 64 ? 2 : 4;    // words of a lane's piece of a row
  constexpr int KL = DP == 256 ? 2 : 1;   // pieces
  constexpr int NS = DP / 32;             // MFMA steps over a row
  constexpr int CR = DP / 32;             // blocks of a row
  constexpr int VP = DP * 2 + 32;         // LDS pitch of a row of values
  constexpr int OP = DP + 4;              // pitch of the joined outputs, floats
  constexpr int DT = DC / 16;
  constexpr int kWaveLds = 32 * VP > 16 * OP * 4 ? 32 * VP : 16 * OP * 4;
  typedef unsigned piece_t __attribute__((ext_vector_type(WB)));
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
  // the lane's i-th piece of a row: its block, and its place; a block past the row's
  // end has scale 0, and any codes
  auto block = [&](int i) { return DP == 64 ? g >> 1 : g + 4 * i; };
  uint32_t place[KL];
#pragma unroll
  for (int i = 0; i < KL; ++i) place[i] = block(i) < a.NB ? (DP == 64 ? 8 * g : 16 * (g + 4 * i)) : 0;
  // the element that step t begins with
  auto element = [&](int t) { return DP == 64 ? 16 * g + 8 * t : 128 * (t / 4) + 32 * g + 8 * (t % 4); };
  // Two pieces of 16 bytes change places in rows 4 .. 11 of 16, so that lanes that
  // write eight rows, and lanes that read four, meet no bank twice.
  const int flip_w = ((n >> 2 ^ n >> 3) & 1) << 4, flip_r = ((g ^ g >> 1) & 1) << 4;
  unsigned char *write0 = vlds + n * VP + (DP == 64 ? 32 : 64) * g + flip_w, *write1 = write0 + 16 - 2 * flip_w;
  const unsigned char *columns = vlds + (4 * g + n / 4) * VP + ((8 * (n & 3)) ^ flip_r);
  // of a byte of the lane's block in a word of scales
  const int byte_at = 8 * (block(0) & 3);
  // what the lane looks after: keys, or values
  const bool of_v = !WIDE && lane >= 32;
  const int key_lane = WIDE ? lane : lane & 31;

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
    auto lookup = [&](int at) { return pages.lookup(a, at + key_lane); };
    int page = lookup(k0);  // on its way while the queries are fetched
    // ---- the queries, on their way beside the first keys' places (what is not there is
    // read from the first query)
    constexpr int kRaw = NS * (BF ? 1 : 2);  // 16 bytes each
    u32x4_t raw[kRaw];
    {
      const char *src = static_cast<const char *>(a.q) +
          ((int64_t)(s.q0 + row_t) * a.q_ld[0] + (h * G + r0 + n - row_t * G) * a.q_ld[1]) * (int64_t)sizeof(T);
#pragma unroll
      for (int y = 0; y < kRaw; ++y) {
        const int e = BF ? element(y) : element(y / 2) + 4 * (y % 2);
        raw[y] = *reinterpret_cast<const u32x4_t *>(live && e < a.D ? src + e * sizeof(T) : static_cast<const char *>(a.q));
      }
    }
    f32x4_t o[DT];
    float m = -INFINITY, l = 0.f;
    bool missed = false;  // the row sees a value that is not finite at an edge
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const uint8_t *kbase = static_cast<const uint8_t *>(a.k) + h * a.k_ld[1];
    const uint8_t *vbase = static_cast<const uint8_t *>(a.v) + h * a.v_ld[1];
    const uint8_t *ks_base = a.k_sc + h * a.k_sc_ld[1], *vs_base = a.v_sc + h * a.v_sc_ld[1];

    // Where the strip's keys and values are, and their scales.
    uint64_t there;         // which of its keys there are
    uint32_t k_row[KT], v_row[KT];  // of the lane's pieces: bytes if NEAR, else 16 of them
    uint32_t sc[2];         // words of scales: its key's and value's, or two of the one
    auto words = [&](const uint8_t *p, int first) {
      if constexpr (WORDS) {
        if constexpr (CR == 2) return (uint32_t)*reinterpret_cast<const uint16_t *>(p);
        else return *reinterpret_cast<const uint32_t *>(p + first);
      }
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < (CR < 4 ? CR : 4); ++i) {
        const uint32_t y = p[min(first + i, a.NB - 1)];
        w |= first + i < a.NB ? y << (8 * i) : 0u;
      }
      return w;
    };
    auto locate = [&](int at, int page) {
      const int tok = at + key_lane;
      const bool ok = at < kend && pages.there(a, tok, page);
      there = __ballot(ok);
      const int pg = ok ? page : 0, off = ok ? tok - (int)fast_div(tok, a.div_page) * a.page_size : 0;
      uint32_t row, other;  // of the lane's key, and its value where the lane has both
      if constexpr (NEAR) {
        row = other = __umul24(pg, a.ld[0]) + __umul24(off, a.ld[1]);
        const uint32_t to = __umul24(pg, a.sc_ld[0]) + __umul24(off, a.sc_ld[1]);
        if constexpr (WIDE) {
          sc[0] = words(ks_base + to, 0), sc[1] = words(vs_base + to, 0);
        } else {
          const uint8_t *p = (of_v ? vs_base : ks_base) + to;
          sc[0] = words(p, 0), sc[1] = words(p, 4);
        }
      } else if constexpr (WIDE) {
        row = pg * a.k_row[0] + off * a.k_row[1], other = pg * a.v_row[0] + off * a.v_row[1];
        sc[0] = words(ks_base + pg * a.k_sc_ld[0] + off * a.k_sc_ld[2], 0);
        sc[1] = words(vs_base + pg * a.v_sc_ld[0] + off * a.v_sc_ld[2], 0);
      } else {
        row = other = pg * (of_v ? a.v_row[0] : a.k_row[0]) + off * (of_v ? a.v_row[1] : a.k_row[1]);
        const uint8_t *p = of_v ? vs_base + pg * a.v_sc_ld[0] + off * a.v_sc_ld[2]
                                : ks_base + pg * a.k_sc_ld[0] + off * a.k_sc_ld[2];
        sc[0] = words(p, 0), sc[1] = words(p, 4);
      }
#pragma unroll
      for (int u = 0; u < KT; ++u) k_row[u] = __shfl(row, 16 * u + n);
#pragma unroll
      for (int u = 0; u < KT; ++u)
        v_row[u] = NEAR ? k_row[u] : (uint32_t)__shfl(other, (WIDE ? 0 : 32) + 16 * u + n);
    };
    auto load = [&](const uint8_t *base, uint32_t row, int i) {
      const uint8_t *p = NEAR ? base + (row + place[i]) : base + (uint64_t)row * 16 + place[i];
      return __builtin_nontemporal_load(reinterpret_cast<const piece_t *>(p));
    };
    piece_t kreg[KT][KL], vreg[KT][KL];
    auto load_k = [&] {
#pragma unroll
      for (int u = 0; u < KT; ++u)
#pragma unroll
        for (int i = 0; i < KL; ++i) kreg[u][i] = load(kbase, k_row[u], i);
    };
    auto load_v = [&](int from) {  // tiles from, from + 1
#pragma unroll
      for (int u = from; u < from + 2; ++u)
#pragma unroll
        for (int i = 0; i < KL; ++i) vreg[u][i] = load(vbase, v_row[u], i);
    };
    locate(k0, page);
    load_k();
    load_v(0);
    page = lookup(k0 + UK);
#pragma unroll
    for (int u = 2; u < KT; u += 2) load_v(u);
    // ---- the queries, as B operands
    u32x4_t q[QP][NS];
#pragma unroll
    for (int y = 0; y < kRaw; ++y) {
      const bool have = live && (BF ? element(y) : element(y / 2)) < a.D;
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[y][i] = have ? raw[y][i] : 0u;
      raw[y] = scale_sign<T>(raw[y], a.scale);
    }
#pragma unroll
    for (int t = 0; t < NS; ++t) {
      if constexpr (BF) {
        q[0][t] = raw[t];
      } else {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(raw[2 * t + i / 4][i % 4]);
#pragma unroll
        for (int p = 0; p < QP; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            q[p][t][i] = tops(x[2 * i], x[2 * i + 1]);
            x[2 * i] -= top(x[2 * i]), x[2 * i + 1] -= top(x[2 * i + 1]);
          }
      }
    }
    for (; k0 < kend; k0 += UK) {
      const uint64_t held = WIDE ? there : there & 0xffffffffull;
      const bool whole = held == (WIDE ? ~0ull : 0xffffffffull);
      const bool edge = shared.edge(k0, KS);
      // The scales of this strip.  A byte past the last one becomes NaN's.  Values that
      // are not there get the least scale, which their weight of 0 makes 0, and so do
      // those of an edge that are not finite.
      uint32_t now[2] = {sc[0], sc[1]};
      uint64_t bad = 0;  // keys whose values are not finite, at an edge
      if (edge || !whole || __ballot(mx_some_past(now[0]) || mx_some_past(now[1]))) {
        bool is = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bool value = WIDE ? i == 1 : of_v;
#pragma unroll
          for (int y = 0; y < 4; ++y)
            if ((now[i] >> (8 * y) & 255u) > kMxLast) {
              const bool out = edge && value;
              is = is || out;
              now[i] = out ? now[i] & ~(255u << (8 * y)) : now[i] | (255u << (8 * y));
            }
          if (value && !((held >> key_lane) & 1)) now[i] = 0;
        }
        bad = __ballot(is) >> (WIDE ? 0 : 32) & held;
      }
      float k_scale[KT][KL], v_scale[KT][KL];
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int u = 0; u < KT; ++u)
#pragma unroll
          for (int i = 0; i < KL; ++i) {
            const uint32_t w = WIDE ? __shfl(now[v], 16 * u + n) : __shfl(now[i], 32 * v + 16 * u + n);
            (v ? v_scale : k_scale)[u][i] = __uint_as_float((w >> byte_at & 255u) << 23);
          }
      __builtin_amdgcn_sched_barrier(0);
      // 32 values to the wave's LDS (LDS operations of a wave keep their order)
      auto unpack_v = [&](int from) {
#pragma unroll
        for (int u = from; u < from + 2; ++u)
#pragma unroll
          for (int i = 0; i < KL; ++i)
#pragma unroll
            for (int y = 0; y < WB; ++y)
              *reinterpret_cast<u32x4_t *>((y & 1 ? write1 : write0) + 16 * VP * (u - from) + 32 * (y >> 1) + 256 * i) =
                  mx_values(vreg[u][i][y], v_scale[u][i]);
      };
      const int page_after = lookup(k0 + 2 * UK);
      unpack_v(0);
      // scores: lane (row n, g) gets keys 16 u + 4 g .. + 3
      f32x4_t s4[KT];
#pragma unroll
      for (int u = 0; u < KT; ++u) {
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < NS; ++t) {
          const bf16x8_t k = __builtin_bit_cast(bf16x8_t, mx_values(kreg[u][t / WB][t % WB], k_scale[u][t / WB]));
#pragma unroll
          for (int p = QP - 1; p >= 0; --p)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, __builtin_bit_cast(bf16x8_t, q[p][t]), acc, 0, 0, 0);
        }
        s4[u] = acc;
        __builtin_amdgcn_sched_barrier(0);
      }
      locate(k0 + UK, page);
      load_k();
      load_v(0);
      page = page_after;
      __builtin_amdgcn_sched_barrier(0);
      // weights
      const bool some = !whole || __ballot(lo > k0 || hi < k0 + KS);
      if (some) {
        // bit 16 u + e of `seen`: the lane's e-th key of 16
        const int from = min(max(lo - k0, 0), KS), to = min(max(hi - k0, 0), KS);
        const uint64_t below = from >= 64 ? ~0ull : (1ull << from) - 1, up = to >= 64 ? ~0ull : (1ull << to) - 1;
        const uint64_t seen = (up & ~below & held) >> (4 * g);
#pragma unroll
        for (int u = 0; u < KT; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(seen & (1ull << (16 * u + e)))) s4[u][e] = -INFINITY;
      }
      float mx = s4[0][0];
#pragma unroll
      for (int u = 0; u < KT; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s4[u][e]);
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
        for (int u = 0; u < KT; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) s4[u][e] -= is_far(mc) ? m : 0.f;
        mc = is_far(mc) ? 0.f : mc;
      }
      // The headroom goes into the exponent in bf16 (its rounding there, 2^-20, is
      // below the weights'), and is a product in fp32.
      if constexpr (BF) mc += kHeadroom;
#pragma unroll
      for (int half = 0; half < KT / 2; ++half) {
        u32x4_t pw[PP];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            float x[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              x[i] = __builtin_amdgcn_exp2f(fmaf(s4[2 * half + u][e + i], c, -mc)) * (BF ? 1.f : kWeight);
              l += x[i];
            }
#pragma unroll
            for (int p = 0; p < PP; ++p) {
              pw[p][2 * u + e / 2] = p + 1 < PP ? tops(x[0], x[1]) : pack_bf16x2(x[0], x[1]);
              x[0] -= top(x[0]), x[1] -= top(x[1]);
            }
          }
        if (half) {
          unpack_v(2 * half);
          load_v(2 * half);
        }
        // O^T += V^T P^T, columns read kAhead MFMAs before their use; the fences
        // keep the compiler from reading them all at once, which costs registers
        constexpr int kAhead = 3;
        auto read = [&](int d) {
          typedef __attribute__((address_space(3))) s16x4_t *tr_ptr;
          const unsigned char *at = columns + 32 * d;
          const s16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)at);
          const s16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(at + 16 * VP));
          return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        bf16x8_t v[kAhead];
#pragma unroll
        for (int d = 0; d < kAhead; ++d) v[d] = read(d);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
#pragma unroll
          for (int p = PP - 1; p >= 0; --p)
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[d % kAhead], __builtin_bit_cast(bf16x8_t, pw[p]), o[d], 0, 0, 0);
          if (d + kAhead < DT) v[d % kAhead] = read(d + kAhead);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (bad) {
        const int from = min(max(lo - k0, 0), KS), to = min(max(hi - k0, 0), KS);
        const uint64_t below = from >= 64 ? ~0ull : (1ull << from) - 1, up = to >= 64 ? ~0ull : (1ull << to) - 1;
        missed = missed || (live && (up & ~below & bad));
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
          const uint8_t *vs = vs_base + at * a.v_sc_ld[0] + off * a.v_sc_ld[2];
#pragma unroll 1
          for (int col = 4 * g; col < a.D; col += 16)
            if (vs[col / kMxBlock] > kMxLast)
#pragma unroll 1
              for (int e = 0; e < 4; ++e) *reinterpret_cast<float *>(vlds + (n * OP + col + e) * 4) = NAN;
        }
    __syncthreads();
    for (int e = tid; e < 16 * DC / 4; e += kRowThreads) {
      const int row = e / (DC / 4), d = e % (DC / 4) * 4;
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

template <typename T, int DP, int DC, bool NEAR, bool WORDS>
hipError_t launch_rows(const Mx4AttnArgs &a, int grid, hipStream_t s) {
  constexpr int wave = std::max(32 * (DP * 2 + 32), 16 * (DP + 4) * 4);
  const size_t lds = 4 * wave + batch_ints(a.S) * 4, largest = 4 * wave + batch_ints(kMaxSeqs) * 4;
  auto kernel = mx4_row_kernel<T, DP, DC, NEAR, WORDS>;
  const hipError_t allowed = allow_lds(reinterpret_cast<const void *>(kernel), lds, largest);
  if (allowed != hipSuccess) return allowed;
  kernel<<<grid, kRowThreads, lds, s>>>(a);
  return hipGetLastError();
}
template <typename T, bool NEAR, bool WORDS>
hipError_t launch_rows_of(const Mx4AttnArgs &a, int grid, hipStream_t s) {
  if (a.D <= 64) return launch_rows<T, 64, 64, NEAR, WORDS>(a, grid, s);
  if constexpr (!WORDS)  // three blocks
    if (a.D <= 96) return launch_rows<T, 128, 96, NEAR, false>(a, grid, s);
  if (a.D <= 128) return launch_rows<T, 128, 128, NEAR, WORDS>(a, grid, s);
  return launch_rows<T, 256, 256, NEAR, WORDS>(a, grid, s);
}
// Whether a cache is near and has its scales in words (mx4.hpp), and its strides.
void set_near(Mx4AttnArgs *a) {
  constexpr int64_t k24 = 1 << 24;
  const int64_t unit = a->NB == 2 ? 2 : 4;
  a->near = a->pages <= k24 && a->page_size <= k24;
  a->words = a->NB == (a->D <= 64 ? 2 : a->D <= 128 ? 4 : 8) &&
             reinterpret_cast<uintptr_t>(a->k_sc) % unit == 0 && reinterpret_cast<uintptr_t>(a->v_sc) % unit == 0;
  for (int i = 0; i < 3; ++i) {
    a->near = a->near && a->k_ld[i] == a->v_ld[i] && a->k_sc_ld[i] == a->v_sc_ld[i];
    if (i != 1) a->near = a->near && a->k_ld[i] < k24 && a->k_sc_ld[i] < k24;
    a->words = a->words && a->k_sc_ld[i] % unit == 0 && a->v_sc_ld[i] % unit == 0;
  }
  // the last key's last byte, from the head's first
  a->near = a->near && a->pages * a->k_ld[0] + a->page_size * a->k_ld[2] + 16 * a->NB < (1ll << 32) &&
            a->pages * a->k_sc_ld[0] + a->page_size * a->k_sc_ld[2] + a->NB < (1ll << 32);
  for (int i = 0; i < 2; ++i) a->ld[i] = (uint32_t)a->k_ld[2 * i], a->sc_ld[i] = (uint32_t)a->k_sc_ld[2 * i];
  a->step_off = 64 % a->page_size;
}
template <typename T>
hipError_t launch_rows_as(const Mx4AttnArgs &a, int grid, hipStream_t s) {
  if (!a.near) return launch_rows_of<T, false, false>(a, grid, s);
  return a.words ? launch_rows_of<T, true, true>(a, grid, s) : launch_rows_of<T, true, false>(a, grid, s);
}

struct Shape {
  bool tiles;
  int bm, grid;
};
double items_most(const Mx4AttnArgs &a, int bm) { return std::floor((double)a.T * (a.H / a.KV) / bm) + a.S; }
double blocks_most(const Mx4AttnArgs &a, bool tiles) { return std::floor((double)a.W * a.page_size / (tiles ? 64 : 4 * row_strip(a.D))) + 1; }
// Rows of one cache head up to which the row kernel is taken, 16 to an item, each of
// which reads the keys again.  Measured, row against tile kernel, 8 cache heads, 32
// sequences of 2048 tokens, us:
//   bf16  head_dim 64:  32 rows 28 / 38    48 rows 40 / 44    64 rows 43 / 44
//         head_dim 128: 32 rows 36 / 49    48 rows 56 / 56    64 rows 61 / 58
//         head_dim 256: 32 rows 68 / 110   48 rows 112 / 112  64 rows 122 / 113
//   fp32  head_dim 64:  20 rows 31 / 50    64 rows 51 / 61    96 rows 73 / 67
//         head_dim 128: 32 rows 44 / 99    64 rows 78 / 104   96 rows 112 / 110
// and 4 of 32768 in bf16 at head_dim 128: 20 rows 65 / 72, 48 rows 90 / 85.  Past
// head_dim 128 the tile kernel's fp32 operands outgrow its registers (1024 rows of one
// sequence of 2048: 73 / 252, 4096 rows 231 / 655), so there is none.
int64_t rows_most(const Mx4AttnArgs &a) {
  if (a.dtype == ZT_DT_BF16) return a.D <= 64 ? 48 : 32;
  return a.D <= 128 ? 64 : INT64_MAX;
}
Shape shape_of(const Mx4AttnArgs &a) {
  const int64_t rows = std::min(std::max<int64_t>(a.max_q, 1), a.T) * (a.H / a.KV);
  Shape p{rows > rows_most(a), BM, kRowGrid};
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
  if (a.pages == 0) a.W = 0;  // no key is there, and there is no first row to read in its place
  set_near(&a);
  lay_parts(&a, workspace, p.grid, p.bm);
  const hipError_t e = p.tiles                   ? launch_mx4_tiles(a, p.grid, s)
                       : a.dtype == ZT_DT_BF16 ? launch_rows_as<uint16_t>(a, p.grid, s)
                                               : launch_rows_as<float>(a, p.grid, s);
  if (e != hipSuccess) return e;
  return launch_join(a, p.grid, !p.tiles, s);
}

}  // namespace zt
