// Attention of a chunk of new tokens over a paged cache, for gfx950: many rows
// per cache head in fp32, head_dim up to 128, on bf16 MFMAs.  The definitions are in
// paged_attn.hip.
#include "attn_common.hpp"

namespace zt {

namespace {

// x = x1 + x2 + x3 with each part a bf16: x1 the nearest to x, x2 to x - x1, x3
// to what is left (8 of fp32's 24 digits each, so the sum is x again but for
// numbers whose last part underflows).  Two numbers at a time, packed.
struct Parts {
  uint32_t p[3];
};
__device__ __forceinline__ Parts split2(float a, float b) {
  Parts s;
  s.p[0] = pack_bf16x2(a, b);
  a -= __uint_as_float(s.p[0] << 16), b -= __uint_as_float(s.p[0] & 0xffff0000u);
  s.p[1] = pack_bf16x2(a, b);
  a -= __uint_as_float(s.p[1] << 16), b -= __uint_as_float(s.p[1] & 0xffff0000u);
  s.p[2] = pack_bf16x2(a, b);
  return s;
}

// The same for keys and values, with x1 cut short, so that it is finite where x is
// (the nearest bf16 to the last 0.2 % below fp32's largest is not): else x2 would
// be infinite too, and a weight of 0 make NaN of it.  An infinite key is x1 alone:
// the median takes the NaN that is left of it for 0.
template <bool Key>
__device__ __forceinline__ Parts split2_cached(uint32_t a, uint32_t b) {
  const uint32_t wa = a & 0xffff0000u, wb = b & 0xffff0000u;
  Parts s;
  s.p[0] = __builtin_amdgcn_perm(wb, wa, 0x07060302u);  // the two high halves
  float ra = __uint_as_float(a) - __uint_as_float(wa), rb = __uint_as_float(b) - __uint_as_float(wb);
  if constexpr (Key) {
    asm("v_med3_f32 %0, %0, 0, %0" : "+v"(ra));
    asm("v_med3_f32 %0, %0, 0, %0" : "+v"(rb));
  }
  s.p[1] = pack_bf16x2(ra, rb);
  ra -= __uint_as_float(s.p[1] << 16), rb -= __uint_as_float(s.p[1] & 0xffff0000u);
  s.p[2] = pack_bf16x2(ra, rb);
  return s;
}

// The same for a query, all parts cut short and none of them zero (bf16's smallest
// number instead, 2^-133, which adds nothing to a score): an infinite key's score
// then is infinite with the product's sign, not the NaN of infinities of both
// signs or of one times 0.  (A query of 0 against an infinite key is a NaN.)
__device__ __forceinline__ Parts split2_query(uint32_t a, uint32_t b) {
  typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
  float ra = __uint_as_float(a), rb = __uint_as_float(b);
  Parts s;
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    const uint32_t wa = __float_as_uint(ra) & 0xffff0000u, wb = __float_as_uint(rb) & 0xffff0000u;
    s.p[p] = __builtin_amdgcn_perm(wb, wa, 0x07060302u);
    ra -= __uint_as_float(wa), rb -= __uint_as_float(wb);
  }
  const auto least = __builtin_bit_cast(u16x2_t, (s.p[0] & 0x80008000u) | 0x00010001u);
#pragma unroll
  for (int p = 1; p < 3; ++p)
    s.p[p] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, s.p[p]), least));
  return s;
}

// x y without its smallest terms: x1 y1 + (x1 y2 + x2 y1) + (x2 y2 + x1 y3 + x3 y1),
// smallest first.  Where both are cut short the others are below 2^-21 of x y, 2^-24
// in the mean; where one is, below 2^-23.
__device__ __forceinline__ f32x16_t mfma_split(const u32x4_t (&x)[3], const u32x4_t (&y)[3], f32x16_t acc) {
  auto mul = [&](int i, int j) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, x[i]),
                                                  __builtin_bit_cast(bf16x8_t, y[j]), acc, 0, 0, 0);
  };
  mul(2, 0), mul(0, 2), mul(1, 1), mul(1, 0), mul(0, 1), mul(0, 0);
  return acc;
}

// A block takes nearly the same time whatever rows are live, and an item's two
// ends about one block's.
struct SplitCost {
  static constexpr int kLead = 2, kMost = 2, kLeast = kMost;
  static __device__ __forceinline__ int of(int) { return 2; }
};

// NW waves of 32 rows each against a span of the keys of one cache head, as
// paged_attn_tile.hip's kernel does it for bf16, in tiles of 32 keys.
//
// An fp32 MFMA runs at a sixteenth of the bf16 rate, so every number goes in
// three bf16 parts and a product in six MFMAs, 2.7 times as fast, with all
// but the smallest terms.  Keys and values are split once per workgroup on their
// way to LDS (global memory -> registers while a tile is worked on -> three
// planes of the next stage), queries once per item, weights as they are made.
//
// Measured: eight whole sequences of up to 500 tokens, 16 heads of 64, 55 us (fp32
// MFMAs: 75); four causal prompts of 729 to 1765 tokens, 16 heads on 4: head_dim 64 109
// us, 80 144, 128 210 (109 TFLOP/s; a large fp32 product of the library 143).  Past 128
// three planes do not fit LDS twice.
template <int DP, int DC, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_attn_split_kernel(
    AttnArgs a) {
  using Cost = SplitCost;
  constexpr int NTH = 64 * NW, BM = 32 * NW, TK = 32;
  constexpr int RB = DP * 2, CR = RB / 16, PLANE = TK * RB, STAGE = 6 * PLANE;
  constexpr int PR = DP / 4, NL = TK * PR / NTH;  // 16-byte pieces of a row; of a tile, per thread
  constexpr int NQ = DC / 16, DT = DC / 32;
  static_assert(NL >= 1 && TK * PR % NTH == 0, "the threads share a tile's pieces evenly");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  __shared__ PlanShared sh;
  __shared__ uint32_t sm_bad[3];  // keys with values that are not finite, of three tiles in turn
  const Batch batch(smem + 2 * STAGE, a.S);

  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Plan plan = make_plan<NTH, Cost>(a, BM, TK, batch, &sh);
  Split *split = static_cast<Split *>(a.splits) + plan.wg;
  if (tid == 0) split->rows = 0;

  const float c = score_factor(a.scale);
  const int G = a.group, C = a.D / 4;
  const char *zero = reinterpret_cast<const char *>(kZeroRow);
  // the same permutations of a row's 16-byte pieces as the bf16 kernel's
  auto kswz = [](int row) { return CR >= 16 ? row & 15 : row & 7; };
  auto vswz = [](int row) { return CR >= 16 ? (row & 3) << 2 : ((row >> 1) & 1) << 2; };

  Walk<Cost> walk(plan);
  Segment seg;
  while (walk.next(a, plan, batch, BM, TK, &seg)) {
    const int h = seg.head, take = seg.take;
    const Seq s = batch.uniform(seg.seq);
    const int r0 = seg.tile * BM, k_first = (seg.b0 + seg.bb) * TK;
    const Pages pages{a.table + (int64_t)seg.seq * a.W, seg.keys.begin, seg.keys.end};
    const Shared shared(a, s, seg.tile, BM);
    if (shared.differ) {
      if (tid < 3) sm_bad[tid] = 0;
      __syncthreads();
    }
    const char *kbase = static_cast<const char *>(a.k) + h * a.k_ld[1] * 4;
    const char *vbase = static_cast<const char *>(a.v) + h * a.v_ld[1] * 4;

    auto lookup = [&](int at) { return pages.lookup(a, at + n); };
    u32x4_t kreg[NL], vreg[NL];
    auto fetch = [&](int at, int page) -> uint32_t {
      const int tok = at + n;
      const bool ok = pages.there(a, tok, page);
      const uint32_t ko = ok ? row_offset(a, a.k_row, tok, page) : ~0u;
      const uint32_t vo = ok ? row_offset(a, a.v_row, tok, page) : ~0u;
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const int idx = j * NTH + tid, row = idx / PR, piece = idx % PR;
        const uint32_t kr = __shfl(ko, row), vr = __shfl(vo, row);
        kreg[j] = *reinterpret_cast<const u32x4_t *>(
            kr != ~0u && piece < C ? kbase + (uint64_t)(kr + piece) * 16 : zero);
        vreg[j] = *reinterpret_cast<const u32x4_t *>(
            vr != ~0u && piece < C ? vbase + (uint64_t)(vr + piece) * 16 : zero);
      }
      return (uint32_t)__ballot(ok);
    };
    // a piece of a row to the three planes
    auto put = [&](unsigned char *to, int swz, int row, int piece, const Parts &lo, const Parts &hi) {
      to += row * RB + 16 * ((piece / 2) ^ swz) + 8 * (piece & 1);
#pragma unroll
      for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x2_t *>(to + p * PLANE) = u32x2_t{lo.p[p], hi.p[p]};
    };
    auto keep = [&](int st, int k0, uint32_t *bad) {
      const bool edge = shared.edge(k0, TK);
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const int idx = j * NTH + tid, row = idx / PR, piece = idx % PR;
        if (__builtin_expect(edge && not_finite<float>(vreg[j]), 0)) {
          vreg[j] = finite_of<float>(vreg[j]);
          atomicOr(bad, 1u << row);
        }
        put(smem + st * STAGE, kswz(row), row, piece, split2_cached<true>(kreg[j][0], kreg[j][1]),
            split2_cached<true>(kreg[j][2], kreg[j][3]));
        put(smem + st * STAGE + 3 * PLANE, vswz(row), row, piece, split2_cached<false>(vreg[j][0], vreg[j][1]),
            split2_cached<false>(vreg[j][2], vreg[j][3]));
      }
    };
    uint32_t there = fetch(k_first, lookup(k_first));
    int page = lookup(k_first + TK);

    // ---- the wave's rows: lane (row n, half) holds columns 16 j + 8 half .. + 7
    const Rows32 rows(a, s, r0 + 32 * wave + n);
    u32x4_t q[NQ][3];
    {
      const char *src = static_cast<const char *>(a.q) +
          ((int64_t)(s.q0 + rows.token) * a.q_ld[0] + (h * G + rows.row - rows.token * G) * a.q_ld[1]) * 4;
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int p = 4 * j + 2 * half + e;
          const u32x4_t x = scale_sign<float>(
              *reinterpret_cast<const u32x4_t *>(rows.live && p < C ? src + 16 * p : zero), a.scale);
          const Parts lo = split2_query(x[0], x[1]), hi = split2_query(x[2], x[3]);
#pragma unroll
          for (int k = 0; k < 3; ++k) q[j][k][2 * e] = lo.p[k], q[j][k][2 * e + 1] = hi.p[k];
        }
    }
    f32x16_t o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    bool far = false;  // of some row of the wave
    bool missed = false;  // the row sees a value that is not finite at an edge

    keep(0, k_first, sm_bad);
    int turn = 0;  // t % 3
    for (int t = 0; t < take; ++t) {
      const int k0 = k_first + t * TK, st = t & 1;
      // every wave's part of the tile is in LDS, and the previous tile is done with
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      uint32_t there_next = 0;
      if (t + 1 < take) {
        there_next = fetch(k0 + TK, page);
        page = lookup(k0 + 2 * TK);
      }
      const int turn1 = turn == 2 ? 0 : turn + 1;
      if (shared.differ) {
        if (tid == 0) sm_bad[3 - turn - turn1] = 0;  // the tile after next's
        missed |= rows.sees_of(sm_bad[turn] & there, k0);
      }
      if (rows.see(k0, TK)) {
        const unsigned char *kt = smem + st * STAGE, *vt = kt + 3 * PLANE;
        // ---- scores; the next step's keys are read before a step's MFMAs
        f32x16_t sc;
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = 0.f;
        auto read_k = [&](int j, u32x4_t (&k)[3]) {
#pragma unroll
          for (int p = 0; p < 3; ++p)
            k[p] = *reinterpret_cast<const u32x4_t *>(kt + p * PLANE + n * RB + 16 * ((2 * j + half) ^ kswz(n)));
        };
        u32x4_t k[2][3];
        read_k(0, k[0]);
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          if (j + 1 < NQ) read_k(j + 1, k[(j + 1) & 1]);
          __builtin_amdgcn_sched_barrier(0);
          sc = mfma_split(k[j & 1], q[j], sc);
          __builtin_amdgcn_sched_barrier(0);
        }
        // ---- weights
        if (there != ~0u || !rows.see_all(k0, TK)) rows.mask(sc, k0, there);
        float mx = sc[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mx = fmaxf(mx, sc[e]);
        mx = fmaxf(mx, other_half(mx));
        // in the rows that grew only, so that no row's bits depend on another's
        const bool grown = mx != -INFINITY && (mx - m) * c > 8.f;
        if (__ballot(grown)) {
          const float f = grown ? factor(m, mx, c) : 1.f;
          l *= f;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] *= f;
          m = grown ? mx : m;
          far = __ballot(m != -INFINITY && is_far(m * c)) != 0;
        }
        float ref = m == -INFINITY ? 0.f : m * c;
        if (__builtin_expect(far, 0)) {
#pragma unroll
          for (int e = 0; e < 16; ++e) sc[e] -= is_far(ref) ? m : 0.f;
          ref = is_far(ref) ? 0.f : ref;
        }
        // ---- O^T += V^T P^T, 16 keys and 32 columns a step
        typedef __attribute__((address_space(3))) s16x4_t *tr_ptr;
        const int i16 = lane & 15, r = 4 * half + i16 / 4;
        const int piece = 2 * ((lane >> 4) & 1) + (i16 & 3) / 2;
        auto read_v = [&](int j, u32x4_t (&v)[3]) {
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            const unsigned char *at = vt + p * PLANE + (16 * (j / DT) + r) * RB +
                16 * ((4 * (j % DT) + piece) ^ vswz(r)) + 8 * (i16 & 1);
            const s16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)at);
            const s16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(at + 8 * RB));
            v[p] = __builtin_bit_cast(u32x4_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
          }
        };
        u32x4_t p[3], v[2][3];
        read_v(0, v[0]);
#pragma unroll
        for (int j = 0; j < 2 * DT; ++j) {
          if (j % DT == 0)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i = 8 * (j / DT) + 2 * e;
              const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[i], c, -ref)) * kWeight;
              const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[i + 1], c, -ref)) * kWeight;
              l += p0;
              l += p1;
              const Parts w = split2(p0, p1);
#pragma unroll
              for (int x = 0; x < 3; ++x) p[x][e] = w.p[x];
            }
          if (j + 1 < 2 * DT) read_v(j + 1, v[(j + 1) & 1]);
          __builtin_amdgcn_sched_barrier(0);
          o[j % DT] = mfma_split(v[j & 1], p, o[j % DT]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (t + 1 < take) keep(st ^ 1, k0 + TK, sm_bad + turn1);
      there = there_next;
      turn = turn1;
    }
    l += other_half(l);
    rows.store<float>(a, seg, s, BM, 32 * wave + n, o, m, l);
    if (__builtin_expect(__ballot(missed) != 0, 0))
#pragma unroll 1
      for (int col = 4 * half; col < a.D; col += 8)
        add_edges<float>(a, seg, s, BM, 32 * wave + n, col, shared, pages, vbase, k_first, k_first + take * TK, TK);
    if (tid == 0 && seg.bb == 0 && !seg.complete) {
      split->slot = seg.slot, split->last = seg.last;
      split->row0 = r0, split->rows = min(BM, s.q * G - r0), split->head = h, split->q0 = s.q0;
    }
    __syncthreads();  // the last tile is done with
  }
  zero_rows<NTH>(a, plan, BM, TK, batch);
}

template <int DP, int DC, int NW>
hipError_t launch_split_as(const AttnArgs &a, int grid, hipStream_t s) {
  const size_t tiles = 2 * 6 * (size_t)32 * DP * 2;
  const size_t lds = tiles + batch_ints(a.S) * 4, largest = tiles + batch_ints(kMaxSeqs) * 4;
  if (a.item_rows != 32 * NW) return hipErrorInvalidValue;
  auto kernel = paged_attn_split_kernel<DP, DC, NW>;
  const hipError_t allowed = allow_lds(reinterpret_cast<const void *>(kernel), lds, largest);
  if (allowed != hipSuccess) return allowed;
  kernel<<<grid, 64 * NW, lds, s>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_split(const AttnArgs &a, int grid, hipStream_t s) {
  if (a.D <= 64) return launch_split_as<64, 64, 4>(a, grid, s);
  if (a.D <= 96) return launch_split_as<128, 96, 8>(a, grid, s);
  return launch_split_as<128, 128, 8>(a, grid, s);
}

}  // namespace zt
