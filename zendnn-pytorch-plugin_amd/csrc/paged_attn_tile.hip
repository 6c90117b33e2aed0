// Attention of a chunk of new tokens over a paged cache, for gfx950: many rows
// per cache head (prompt chunks).  The definitions are in paged_attn.hip.
#include "attn_common.hpp"

namespace zt {

namespace {

// LDS byte address of a pointer into shared memory.
__device__ __forceinline__ uint32_t lds_addr(const void *p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)p;
}

// 64 lanes x 16 bytes from each lane's own address to 1 KB of LDS at `lds`
// (uniform).  Written in asm because the compiler makes every LDS read wait
// for all of its builtin's transfers in flight, those of the next tile among
// them; the waits are in wait_and_meet below.  It writes no register.
__device__ __forceinline__ void load_to_lds(const void *src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :: "v"(src), "s"(lds) : "memory", "m0");
}
// Every transfer and LDS read of this wave is over, and every wave is here.
__device__ __forceinline__ void wait_and_meet() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// The cost of a block, and of an item's beginning and end.  A block of few rows
// takes nearly as long as a full one: in bf16 it waits for its keys (1.9 against
// 2.2 us, two workgroups a CU); in fp32 (past head_dim 128, one workgroup a CU) each
// wave does its own rows' matrix operations, whatever the others have.
// An item's two ends take 5 to 6 us.  In bf16 spans have four blocks at least:
// what a part of 128 rows has to write and the join to read is four blocks'
// bytes (32 tokens of 32 heads behind 2048: 40 us without, 35 with).
template <typename T>
struct TileCost {
  static constexpr int kLead = sizeof(T) == 2 ? 15 : 7, kMost = 6, kLeast = sizeof(T) == 2 ? 4 * kMost : kMost, kJoin = 0;
  static __device__ __forceinline__ int of(int rows) {
    return sizeof(T) == 2 ? 4 + (rows + 63) / 64 : 6;
  }
};

// NW waves of 32 rows each against a span of the keys of one cache head.
//
// Bound by the matrix operations with their LDS reads, and by the transfers, whose
// writes to LDS and waits they hide only in part (figures below).  All waves share
// tiles of TK keys and values (64, or 32 in fp32) that arrive in LDS by DMA, two
// tiles deep: while one is worked on the next is on its way, with one barrier per
// tile.
//
// The products are taken transposed, S^T = K Q^T and O^T = V^T P^T, on 32x32
// MFMAs with the rows as columns: a lane holds 16 keys of one row per tile of
// 32 (keys 8 (i / 4) + 4 half + i % 4), so a row's maximum and sum stay in two
// lanes, and the scores' layout is the layout in which the second product takes
// its weights if V^T takes its keys in the same order.  Columns of V come from
// plain reads in fp32 and from the transposing ds_read_b64_tr_b16 in bf16.
//
// LDS rows are RB bytes with their 16-byte pieces permuted (by the row's low
// bits; the DMA fetches the permuted piece), so that 16 lanes reading one piece
// of 16 rows of K, or four rows of a block of V, meet no bank twice.
//
// The running maximum is only a point of reference: it follows the true one
// when that has grown by more than 2^8 in the weights, so that most tiles need
// no rescaling of the outputs.  Weights stay below 2^8, in fp32 and bf16 alike
// without loss of digits.
//
// bf16 weights are rounded once for the second product (half a step each, 2^-8,
// and independent, so the sum of n of them is off by much less); their sum is
// taken of the rounded ones, so that a row's weights still add up to one.
//
// Measured (32 query and 8 cache heads of 128, bf16): 2048 tokens behind 6144
// 264-281 us, 0.9 PFLOP/s (a large product of the library reaches 1.2 on the
// same card); copies without the transfers 231, without the exponentials 261, without
// both 218 beside 272.
template <typename T, int DP, int DC, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(DP <= 128 ? 2 : 1, DP <= 128 ? 2 : 1))) void paged_attn_tile_kernel(AttnArgs a) {
  using Cost = TileCost<T>;
  constexpr bool BF = sizeof(T) == 2;
  constexpr int ES = sizeof(T), NTH = 64 * NW, BM = 32 * NW;
  constexpr int KT = BF ? 2 : 1, TK = 32 * KT;  // keys of a tile
  constexpr int RB = DP * ES, CR = RB / 16;     // bytes and 16-byte pieces of an LDS row
  constexpr int STAGE = TK * RB;                // bytes of a tile of K (or V)
  constexpr int NI = STAGE / 1024 / NW;         // DMA instructions of a wave for it
  static_assert(NI >= 1, "every wave loads");
  constexpr int NQ = DC * ES / 32;              // 16-byte pieces of a row per lane
  constexpr int DT = DC / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  __shared__ PlanShared sh;
  __shared__ uint32_t sm_bad[NW];
  const Batch batch(smem + 4 * STAGE, a.S);

  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Plan plan = make_plan<NTH, Cost>(a, BM, TK, batch, &sh);
  Split *split = static_cast<Split *>(a.splits) + plan.wg;
  if (tid == 0) split->rows = 0;

  const float c = score_factor(a.scale);
  const int G = a.group, C = a.D * ES / 16;
  const char *zero = reinterpret_cast<const char *>(kZeroRow);
  // where a lane's pieces of K and columns of V are in a tile
  auto kswz = [](int row) { return CR >= 16 ? row & 15 : row & 7; };
  auto vswz = [](int row) {
    return !BF ? ((row >> 2) & 1) << 3 : CR >= 16 ? (row & 3) << 2 : ((row >> 1) & 1) << 2;
  };
  const uint32_t lds0 = lds_addr(smem);
  // what the lane fetches in each of its wave's transfers: row, pieces of K and V
  int part_row[NI], part_k[NI], part_v[NI];
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    const int idx = (wave * NI + j) * 64 + lane, slot = idx % CR;
    part_row[j] = idx / CR;
    part_k[j] = slot ^ kswz(part_row[j]), part_v[j] = slot ^ vswz(part_row[j]);
  }

  Walk<Cost> walk(plan);
  Segment seg;
  while (walk.next(a, plan, batch, BM, TK, &seg)) {
    const int h = seg.head, take = seg.take;
    const Seq s = batch.uniform(seg.seq);
    const int r0 = seg.tile * BM;
    const KeyRange kr = seg.keys;
    const Shared shared(a, s, seg.tile, BM);
    const Pages pages{a.table + (int64_t)seg.seq * a.W, kr.begin, kr.end};
    const char *kbase = static_cast<const char *>(a.k) + h * a.k_ld[1] * ES;
    const char *vbase = static_cast<const char *>(a.v) + h * a.v_ld[1] * ES;

    auto lookup = [&](int at) { return pages.lookup(a, at + (lane & (TK - 1))); };
    // K and V of a tile go to LDS in NI parts: offsets first, then each part's
    // pieces.  Past the segment's last tile zeros are sent, so that the parts go
    // between matrix operations without a branch (265.7 us with them against 270.2
    // with one, a chunk of 2048 tokens behind 6144).
    uint32_t ko, vo;
    bool gaps;  // some of its keys are not there
    auto offsets = [&](int at, int page, bool real) -> uint64_t {
      const int tok = at + (lane & (TK - 1));
      const bool ok = real && pages.there(a, tok, page);
      ko = ok ? row_offset(a, a.k_row, tok, page) : ~0u;
      vo = ok ? row_offset(a, a.v_row, tok, page) : ~0u;
      const uint64_t m = __ballot(ok);
      gaps = m != ~0ull || C != CR;
      return TK == 64 ? m : m & 0xffffffffull;
    };
    auto issue = [&](int j, int st) {
      const uint32_t kr16 = __shfl(ko, part_row[j]), vr16 = __shfl(vo, part_row[j]);
      const char *ks = kbase + (uint64_t)(kr16 + part_k[j]) * 16, *vs = vbase + (uint64_t)(vr16 + part_v[j]) * 16;
      if (gaps) {
        ks = kr16 != ~0u && part_k[j] < C ? ks : zero;
        vs = vr16 != ~0u && part_v[j] < C ? vs : zero;
      }
      load_to_lds(ks, lds0 + st * 2 * STAGE + (wave * NI + j) * 1024);
      load_to_lds(vs, lds0 + st * 2 * STAGE + STAGE + (wave * NI + j) * 1024);
    };
    const int k_first = (seg.b0 + seg.bb) * TK;
    uint64_t there = offsets(k_first, lookup(k_first), true);
#pragma unroll
    for (int j = 0; j < NI; ++j) issue(j, 0);
    int page = lookup(k_first + TK);

    // ---- the wave's rows: lane (row n, half) holds pieces 2 j + half of q
    const Rows32 rows(a, s, r0 + 32 * wave + n);
    u32x4_t q[NQ];
    {
      const char *src = static_cast<const char *>(a.q) +
          ((int64_t)(s.q0 + rows.token) * a.q_ld[0] + (h * G + rows.row - rows.token * G) * a.q_ld[1]) * ES;
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        const int p = 2 * j + half;
        q[j] = scale_sign<T>(*reinterpret_cast<const u32x4_t *>(rows.live && p < C ? src + 16 * p : zero), a.scale);
      }
    }
    f32x16_t o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    float m = -INFINITY, mc = 0.f, l = 0.f;
    bool far = false;  // of some row of the wave
    bool missed = false;  // the row sees a value that is not finite at an edge

    for (int t = 0; t < take; ++t) {
      const int k0 = k_first + t * TK, st = t & 1;
      wait_and_meet();  // the tile is there, and the previous one is done with
      const uint64_t there_next = offsets(k0 + TK, page, t + 1 < take);
      page = lookup(k0 + 2 * TK);
      if (__builtin_expect(shared.edge(k0, TK), 0)) {  // the waves look over TK / NW values each
        constexpr int ROWS = TK / NW, LANES = 64 / ROWS;
        unsigned char *at = smem + st * 2 * STAGE + STAGE + (wave * ROWS + lane / LANES) * RB;
        bool bad = false;
#pragma unroll
        for (int j = 0; j < CR / LANES; ++j) {
          u32x4_t *x = reinterpret_cast<u32x4_t *>(at + 16 * (j * LANES + lane % LANES));
          if (not_finite<T>(*x)) bad = true, *x = finite_of<T>(*x);
        }
        uint32_t found = 0;
        for (uint64_t left = __ballot(bad); left; left &= left - 1) found |= 1u << (__builtin_ctzll(left) / LANES);
        if (lane == 0) sm_bad[wave] = found;
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        uint64_t all = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) all |= (uint64_t)sm_bad[w] << (ROWS * w);
        missed |= rows.sees_of(all & there, k0);
      }
      if (rows.see(k0, TK)) {
        const unsigned char *kt = smem + st * 2 * STAGE, *vt = kt + STAGE;
        // ---- scores.  Keys are read kAhead operands before their use; the
        // fences keep the compiler from moving each read next to its use.
        f32x16_t sc[KT];
        {
          constexpr int kSteps = KT * NQ, kAhead = kSteps < 4 ? kSteps : 4;
          u32x4_t k[kAhead];
          auto read = [&](int j) {
            return *reinterpret_cast<const u32x4_t *>(kt + (32 * (j / NQ) + n) * RB +
                                                      16 * ((2 * (j % NQ) + half) ^ kswz(n)));
          };
#pragma unroll
          for (int j = 0; j < kAhead; ++j) k[j] = read(j);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < kSteps; ++j) {
            f32x16_t &to = sc[j / NQ];
            if (j % NQ == 0)
#pragma unroll
              for (int e = 0; e < 16; ++e) to[e] = 0.f;
            if constexpr (BF) {
              to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, k[j % kAhead]),
                                                           __builtin_bit_cast(bf16x8_t, q[j % NQ]), to, 0, 0, 0);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                to = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k[j % kAhead][e]),
                                                          __uint_as_float(q[j % NQ][e]), to, 0, 0, 0);
            }
            if (j + kAhead < kSteps) k[j % kAhead] = read(j + kAhead);
            // the next tile's transfers one at a time: all at once they hold
            // up the wave that issues them
            constexpr int kEvery = kSteps / NI;
            if (j % kEvery == kEvery / 2 && j / kEvery < NI) issue(j / kEvery, st ^ 1);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        // ---- weights
        const bool whole = there == (TK == 64 ? ~0ull : 0xffffffffull);
        if (!whole || !rows.see_all(k0, TK))
#pragma unroll
          for (int u = 0; u < KT; ++u) rows.mask(sc[u], k0 + 32 * u, (uint32_t)(there >> (32 * u)));
        float mx = sc[0][0];
#pragma unroll
        for (int u = 0; u < KT; ++u)
#pragma unroll
          for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[u][e]);
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
          mc = grown ? mx * c : mc;
          far = __ballot(is_far(mc)) != 0;
        }
        float ref = mc;
        if (__builtin_expect(far, 0)) {
#pragma unroll
          for (int u = 0; u < KT; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[u][e] -= is_far(mc) ? m : 0.f;
          ref = is_far(mc) ? 0.f : mc;
        }
        // ---- O^T += V^T P^T, a step of keys at a time (16, or one of each half
        // in fp32): beside its MFMAs go the next step's weights and the reads
        // of the operands kAhead MFMAs on.  A wave that is this far goes before
        // the SIMD's other one, so that the two take turns at matrix operations
        // and weights (a chunk of 2048 tokens behind 6144: 283 -> 276 us).
        __builtin_amdgcn_s_setprio(1);
        // The headroom goes into the exponent in bf16 (its rounding there, 2^-20,
        // is far below the weights'), and is a product in fp32.
        if constexpr (BF) ref += kHeadroom;
        auto weight = [&](int e) {
          const float p = __builtin_amdgcn_exp2f(fmaf(sc[e / 16][e % 16], c, -ref));
          return BF ? p : p * kWeight;
        };
        constexpr int kAhead = 3;
        if constexpr (BF) {
          typedef __attribute__((address_space(3))) s16x4_t *tr_ptr;
          constexpr int kKeys = 2 * KT, kSteps = kKeys * DT;
          const int i16 = lane & 15, r = 4 * half + i16 / 4;
          const int piece = 2 * ((lane >> 4) & 1) + (i16 & 3) / 2;
          auto read = [&](int j) {
            const unsigned char *at = vt + (16 * (j / DT) + r) * RB +
                16 * ((4 * (j % DT) + piece) ^ vswz(r)) + 8 * (i16 & 1);
            const s16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)at);
            const s16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(at + 8 * RB));
            return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
          };
          auto weights = [&](int k, int from, int to, u32x4_t &p) {  // pairs of step k
#pragma unroll
            for (int e = from; e < to; ++e) {
              const float p0 = weight(8 * k + 2 * e), p1 = weight(8 * k + 2 * e + 1);
              const uint32_t both = pack_bf16x2(p0, p1);
              p[e] = both;
              l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, both), bf16x2_t{1.f, 1.f}, l, false);
            }
          };
          bf16x8_t v[kAhead];
          u32x4_t p[2];
#pragma unroll
          for (int j = 0; j < kAhead; ++j) v[j] = read(j);
          weights(0, 0, 4, p[0]);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < kSteps; ++j) {
            const int k = j / DT, d = j % DT;
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[j % kAhead], __builtin_bit_cast(bf16x8_t, p[k & 1]),
                                                           o[d], 0, 0, 0);
            if (j + kAhead < kSteps) v[j % kAhead] = read(j + kAhead);
            if (k + 1 < kKeys) weights(k + 1, 4 * d / DT, 4 * (d + 1) / DT, p[(k + 1) & 1]);
            __builtin_amdgcn_sched_barrier(0);
          }
        } else {
          constexpr int kSteps = 16 * DT;
          auto read = [&](int j) {
            const int e = j / DT, r = 8 * (e / 4) + 4 * half + e % 4;
            return *reinterpret_cast<const float *>(vt + r * RB + 16 * ((8 * (j % DT) + n / 4) ^ vswz(r)) +
                                                    4 * (n & 3));
          };
          float v[kAhead], p[2];
#pragma unroll
          for (int j = 0; j < kAhead; ++j) v[j] = read(j);
          l += p[0] = weight(0);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < kSteps; ++j) {
            const int e = j / DT, d = j % DT;
            o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[j % kAhead], p[e & 1], o[d], 0, 0, 0);
            if (j + kAhead < kSteps) v[j % kAhead] = read(j + kAhead);
            if (d == 0 && e + 1 < 16) l += p[(e + 1) & 1] = weight(e + 1);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < NI; ++j) issue(j, st ^ 1);
      }
      __builtin_amdgcn_s_setprio(0);
      there = there_next;
    }
    // ---- the rows' outputs, or their part: lane (row n, half) holds columns
    // 32 d + 8 k + 4 half .. + 3
    // the zeros have come to rest: the next segment's first tile, or another
    // workgroup, takes their place
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    l += other_half(l);
    rows.store<T>(a, seg, s, BM, 32 * wave + n, o, m, l);
    if (__builtin_expect(__ballot(missed) != 0, 0))
#pragma unroll 1
      for (int col = 4 * half; col < a.D; col += 8)
        add_edges<T>(a, seg, s, BM, 32 * wave + n, col, shared, pages, vbase, k_first, k_first + take * TK, TK);
    if (tid == 0 && seg.bb == 0 && !seg.complete) {
      split->slot = seg.slot, split->last = seg.last;
      split->row0 = r0, split->rows = min(BM, s.q * G - r0), split->head = h, split->q0 = s.q0;
    }
    __syncthreads();  // the last tile is done with
  }
  zero_rows<NTH>(a, plan, BM, TK, batch);
}

template <typename T, int DP, int DC, int NW>
hipError_t launch_tiles_as(const AttnArgs &a, int grid, hipStream_t s) {
  constexpr int TK = sizeof(T) == 2 ? 64 : 32;
  const size_t tiles = 4 * (size_t)TK * DP * sizeof(T);
  const size_t lds = tiles + batch_ints(a.S) * 4, largest = tiles + batch_ints(kMaxSeqs) * 4;
  if (a.item_rows != 32 * NW) return hipErrorInvalidValue;
  auto kernel = paged_attn_tile_kernel<T, DP, DC, NW>;
  const hipError_t allowed = allow_lds(reinterpret_cast<const void *>(kernel), lds, largest);
  if (allowed != hipSuccess) return allowed;
  kernel<<<grid, 64 * NW, lds, s>>>(a);
  return hipGetLastError();
}

}  // namespace

// bf16: two workgroups of four waves a CU; past head_dim 128, where a wave's
// queries and outputs need the registers of two, one.  fp32 up to head_dim 128
// goes to the kernel of paged_attn_split.hip: two workgroups of four waves up to
// 64, then one of eight.
int tile_rows(const AttnArgs &a) { return a.dtype == ZT_DT_F32 && a.D > 64 && a.D <= 128 ? 256 : 128; }
int tile_grid(const AttnArgs &a) { return a.D <= (a.dtype == ZT_DT_F32 ? 64 : 128) ? 512 : 256; }

hipError_t launch_tiles(const AttnArgs &a, int grid, hipStream_t s) {
  if (a.dtype == ZT_DT_F32)
    return a.D <= 128 ? launch_split(a, grid, s) : launch_tiles_as<float, 256, 256, 4>(a, grid, s);
  if (a.D <= 64) return launch_tiles_as<uint16_t, 64, 64, 4>(a, grid, s);
  if (a.D <= 96) return launch_tiles_as<uint16_t, 128, 96, 4>(a, grid, s);
  if (a.D <= 128) return launch_tiles_as<uint16_t, 128, 128, 4>(a, grid, s);
  return launch_tiles_as<uint16_t, 256, 256, 4>(a, grid, s);
}

}  // namespace zt
