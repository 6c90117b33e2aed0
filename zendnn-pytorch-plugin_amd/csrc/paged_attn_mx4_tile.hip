// Attention of a chunk of new tokens over a paged cache held in 4 bits, for
// gfx950: many rows per cache head (prompt chunks).  The definitions are in
// paged_attn.hip, the format in mx4.hpp.
#include "attn_common.hpp"
#include "mx4.hpp"

namespace zt {

namespace {

// Every LDS operation of this wave is over, and every wave is here.  Loads from
// memory stay on their way: what they bring goes to this thread's registers.
__device__ __forceinline__ void meet() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// As in paged_attn_tile.hip, whose item ends and tiles these resemble.  A join is worth
// four blocks.  Measured, whole items by that rule against equal spans, us: sequences
// of one length seen whole, 8 of 500 (16 heads of 64, fp32) 37 / 44, in bf16 25 / 34,
// causal ones of 400 23 / 28, 4 of 256 (32 heads of 128) 22 / 35.  Where the rule cuts the
// items its test costs up to 0.5 us: 8 x 128 behind 384 (head_dim 64) 30.6 / 30.1, 16
// mixed 30.9 / 30.5, 3 causal ones of 500 38.3 / 37.9; one of 512 31.0 / 30.9, one of 1024
// 48.8 / 48.9.  Worth 16 or 12 it would cut the eight of 500 and the four of 256 again.
struct Mx4TileCost {
  static constexpr int kLead = 15, kMost = kTileCostMost, kLeast = 4 * kMost, kJoin = 24;
  static __device__ __forceinline__ int of(int rows) { return 4 + (rows + 63) / 64; }
};

constexpr int NW = 4, NTH = 64 * NW, BM = 32 * NW, TK = 64;

// Waves per SIMD, and so workgroups per CU: two, but for sizes whose queries and
// outputs need the registers of both (fp32, head_dim 128, 512 tokens behind 1536:
// 75 us with one, 125 with two, which spill; head_dim 96: 66 and 64).
constexpr int waves(bool bf, int dim) { return dim <= (bf ? 128 : 96) ? 2 : 1; }

// Four waves of 32 rows each against a span of the keys of one cache head.
//
// Bound by the matrix operations with the vector operations beside them.  Tiles of 64
// keys and values lie in LDS two deep: each thread has its part of the next tile's
// codes in registers, unpacks it to the other stage beside the scores' MFMAs, and then
// loads its part of the tile after that.  One barrier a tile.
//
// A code's value is a bf16 number exactly, so the products are bf16 MFMAs, unpacked
// once for the four waves, without a rounding of keys or values: bf16 queries go as
// they are and weights in one part, fp32 queries and weights in three (cut short, 24
// digits).  Scores by scaled MFMAs over the codes themselves (e2m1 by queries in two
// parts of e4m3) were 7 % faster on the chunk below and 3 % slower on 33 mixed
// sequences, but two parts under one scale to 32 numbers lose the digits of those below
// 2^-13 of the largest: with a channel 2^16 times the others, outputs were off by more than
// 0.1 where values are about 1.
//
// The running maximum, the weights and the second product are those of
// paged_attn_tile.hip, on 32x32 MFMAs, transposed.
//
// Measured (32 query and 8 cache heads of 128, bf16): 2048 tokens behind 6144 260-264 us,
// 0.92 PFLOP/s (a large product of the library reaches 1.2); copies of the kernel took 239
// without unpacking, 240 without the loads, 242 without the exponentials beside 261.
// 33 mixed sequences 53 us.  Eight whole fp32 sequences of up to 500, 16 heads of 64: 33 us.
//
// NEAR: a near cache's places (mx4.hpp) are found with a third of the instructions.
template <typename T, int DP, int DC, bool NEAR>
__global__ __launch_bounds__(NTH) __attribute__((amdgpu_waves_per_eu(waves(sizeof(T) == 2, DC), waves(sizeof(T) == 2, DC)))) void mx4_tile_kernel(Mx4AttnArgs a) {
  using Cost = Mx4TileCost;
  constexpr bool BF = sizeof(T) == 2;
  constexpr int QP = BF ? 1 : 3;                // bf16 parts of a query and of a weight
  constexpr int KT = TK / 32;                   // 32-key tiles of a tile
  constexpr int CR = DP / 32;                   // blocks of a row: 16 bytes of codes, one scale
  constexpr int RB = DP * 2, PR = RB / 16;      // bytes and 16-byte pieces of an LDS row
  constexpr int STAGE = TK * RB;                // bytes of the values of a tile, and of its keys
  constexpr int NP = 2 * TK * CR / NTH;         // blocks of a tile per thread
  constexpr int NQ = DC / 16;                   // MFMA steps over a row
  constexpr int DT = DC / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  __shared__ PlanShared sh;
  __shared__ uint64_t sm_bad[2][NW];
  const Batch batch(smem + 4 * STAGE, a.S);

  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Plan plan = make_plan<NTH, Cost>(a, BM, TK, batch, &sh);
  Split *split = static_cast<Split *>(a.splits) + plan.wg;
  if (tid == 0) split->rows = 0;

  const float c = score_factor(a.scale);
  const int G = a.group;
  // the 16-byte pieces of a row are permuted, so that 16 lanes meet no bank twice
  auto kswz = [](int row) { return PR >= 16 ? row & 15 : row & 7; };
  auto vswz = [](int row) { return PR >= 16 ? (row & 3) << 2 | ((row >> 2) & 3) : ((row >> 1) & 1) << 2; };
  // the thread's blocks of a tile: one row, the blocks of K and V
  const int part = DP == 64 ? (lane >> 4) + 4 * (wave & 1) : lane >> 4;
  const int row = DP == 64 ? 16 * (part >> 1) + (lane & 15) : 16 * wave + (lane & 15);
  auto is_v = [&](int j) { return DP == 64 ? wave >= 2 : j >= NP / 2; };
  auto block = [&](int j) { return DP == 64 ? part & 1 : part + 4 * (j % (NP / 2 > 0 ? NP / 2 : 1)); };

  Walk<Cost> walk(plan);
  Segment seg;
  while (walk.next(a, plan, batch, BM, TK, &seg)) {
    const int h = seg.head, take = seg.take;
    const Seq s = batch.uniform(seg.seq);
    const int r0 = seg.tile * BM;
    const KeyRange kr = seg.keys;
    const Shared shared(a, s, seg.tile, BM);
    const Pages pages{a.table + (int64_t)seg.seq * a.W, kr.begin, kr.end};
    const uint8_t *kbase = static_cast<const uint8_t *>(a.k) + h * a.k_ld[1];
    const uint8_t *vbase = static_cast<const uint8_t *>(a.v) + h * a.v_ld[1];
    const uint8_t *ks_base = a.k_sc + h * a.k_sc_ld[1], *vs_base = a.v_sc + h * a.v_sc_ld[1];

    auto lookup = [&](int at) { return pages.template lookup<waves(BF, DC) == 2>(a, at + lane); };
    const int k_first = (seg.b0 + seg.bb) * TK;
    // where in its page the thread's row of the next tile to be loaded is
    int row_off = k_first + row - (int)fast_div(k_first + row, a.div_page) * a.page_size;
    u32x4_t codes[NP];
    uint32_t scales[NP];
    // The thread's part of the tile at `at`, and which of its keys there are.  What is
    // not there is read from the cache's first row (no branch: it would make every
    // wait one for all loads), and gets the least scale: keys are masked by
    // selection, and a weight of 0 makes the values 0.
    auto load = [&](int at, int page, bool real) -> uint64_t {
      const bool ok = real && pages.there(a, at + lane, page);
      const uint64_t m = __ballot(ok);
      const bool mine = (m >> row) & 1;
      const int its = __shfl(page, row), pg = mine ? its : 0, off = mine ? row_off : 0;
      // the next tile's row: a tile on
      row_off += a.step_off;
      row_off -= row_off >= a.page_size ? a.page_size : 0;
      const uint32_t near = __umul24(pg, a.ld[0]) + __umul24(off, a.ld[1]);
      const uint32_t near_sc = __umul24(pg, a.sc_ld[0]) + __umul24(off, a.sc_ld[1]);
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const bool v = is_v(j);
        const int b = block(j) < a.NB ? block(j) : 0;
        if constexpr (NEAR) {
          codes[j] = *reinterpret_cast<const u32x4_t *>((v ? vbase : kbase) + (near + 16 * b));
          scales[j] = (v ? vs_base : ks_base)[near_sc + b];
          continue;
        }
        const uint32_t r = (uint32_t)pg * (v ? a.v_row[0] : a.k_row[0]) + off * (v ? a.v_row[1] : a.k_row[1]);
        codes[j] = *reinterpret_cast<const u32x4_t *>((v ? vbase : kbase) + (uint64_t)r * 16 + 16 * b);
        scales[j] = (v ? vs_base : ks_base)[pg * (v ? a.v_sc_ld[0] : a.k_sc_ld[0]) + off * (v ? a.v_sc_ld[2] : a.k_sc_ld[2]) + b];
      }
      return m;
    };
    auto settle = [&](uint64_t m) {  // the scales of a tile of which the keys m are there
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const bool have = ((m >> row) & 1) && block(j) < a.NB;
        scales[j] = have ? scales[j] : 0u;
      }
    };
    // and to LDS, a piece of 16 bytes at a time
    auto unpack = [&](int j, int i, int st) {
      const int p = 4 * block(j) + i;
      unsigned char *to = smem + st * 2 * STAGE + (is_v(j) ? 0 : STAGE) + row * RB + 16 * (p ^ (is_v(j) ? vswz(row) : kswz(row)));
      *reinterpret_cast<u32x4_t *>(to) = mx_values(codes[j][i], mx_scale(scales[j]));
    };
    // the values at an edge that are not finite, taken out
    auto take_out = [&](int st) {
      uint64_t found = 0;
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const bool bad = is_v(j) && scales[j] > kMxLast;
        if (bad) scales[j] = 0;
        for (uint64_t left = __ballot(bad); left; left &= left - 1)
          found |= 1ull << __builtin_amdgcn_readlane(row, __builtin_ctzll(left));
      }
      if (lane == 0) sm_bad[st][wave] = found;
    };
    const int first_page = lookup(k_first);

    // ---- the wave's rows, and their queries' words, on their way beside the first tile
    const Rows32 rows(a, s, r0 + 32 * wave + n);
    constexpr int kRaw = NQ * (BF ? 1 : 2);  // 16 bytes each
    auto raw_element = [&](int y) {  // that word y of the lane begins with
      return BF ? 16 * y + 8 * half : 16 * (y / 2) + 8 * half + 4 * (y % 2);
    };
    u32x4_t raw[kRaw];
    {
      const char *src = static_cast<const char *>(a.q) +
          ((int64_t)(s.q0 + rows.token) * a.q_ld[0] + (h * G + rows.row - rows.token * G) * a.q_ld[1]) * (int64_t)sizeof(T);
#pragma unroll
      for (int y = 0; y < kRaw; ++y) {
        const int e = raw_element(y);
        raw[y] = *reinterpret_cast<const u32x4_t *>(rows.live && e < a.D ? src + e * sizeof(T) : static_cast<const char *>(a.q));
      }
    }
    auto settle_raw = [&] {
#pragma unroll
      for (int y = 0; y < kRaw; ++y) {
        const bool have = rows.live && raw_element(y) < a.D;
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[y][i] = have ? raw[y][i] : 0u;
        raw[y] = scale_sign<T>(raw[y], a.scale);
      }
    };
    uint64_t there = load(k_first, first_page, true);
    int page = lookup(k_first + TK);
    u32x4_t q[QP][NQ];
    settle_raw();
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      if constexpr (BF) {
        q[0][j] = raw[j];
      } else {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(raw[2 * j + i / 4][i % 4]);
#pragma unroll
        for (int p = 0; p < QP; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            q[p][j][i] = tops(x[2 * i], x[2 * i + 1]);
            x[2 * i] -= top(x[2 * i]), x[2 * i + 1] -= top(x[2 * i + 1]);
          }
      }
    }
    settle(there);
    if (shared.edge(k_first, TK)) take_out(0);
#pragma unroll
    for (int j = 0; j < NP; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) unpack(j, i, 0);
    uint64_t there_next = load(k_first + TK, page, take > 1);
    page = lookup(k_first + 2 * TK);
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
      meet();  // the tile is there, and the previous one is done with
      if (__builtin_expect(shared.edge(k0, TK), 0)) {
        uint64_t all = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) all |= sm_bad[st][w];
        missed |= rows.sees_of(all & there, k0);
      }
      settle(there_next);
      if (__builtin_expect(shared.edge(k0 + TK, TK), 0)) take_out(st ^ 1);
      if (rows.see(k0, TK)) {
        const unsigned char *vt = smem + st * 2 * STAGE, *kt = vt + STAGE;
        f32x16_t sc[KT];
        {
          // ---- scores.  Keys are read kAhead operands before their use; the
          // fences keep the compiler from moving each read next to its use.
          constexpr int kSteps = KT * NQ, kAhead = 4;
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
#pragma unroll
            for (int p = QP - 1; p >= 0; --p)
              to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, k[j % kAhead]),
                                                           __builtin_bit_cast(bf16x8_t, q[p][j % NQ]), to, 0, 0, 0);
            if (j + kAhead < kSteps) k[j % kAhead] = read(j + kAhead);
            // the next tile's pieces, evenly
#pragma unroll
            for (int i = 4 * NP * j / kSteps; i < 4 * NP * (j + 1) / kSteps; ++i) unpack(i / 4, i % 4, st ^ 1);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        const uint64_t there_after = load(k0 + 2 * TK, page, t + 2 < take);
        page = lookup(k0 + 3 * TK);
        // ---- weights
        const bool whole = there == ~0ull;
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
        // ---- O^T += V^T P^T, 16 keys at a time: beside their MFMAs go the next
        // ones' weights and the reads of the operands kAhead MFMAs on.
        __builtin_amdgcn_s_setprio(1);
        // The headroom goes into the exponent in bf16 (its rounding there, 2^-20,
        // is far below the weights'), and is a product in fp32.
        if constexpr (BF) ref += kHeadroom;
        auto weight = [&](int e) {
          const float p = __builtin_amdgcn_exp2f(fmaf(sc[e / 16][e % 16], c, -ref));
          return BF ? p : p * kWeight;
        };
        typedef __attribute__((address_space(3))) s16x4_t *tr_ptr;
        constexpr int kAhead = 3, kKeys = 2 * KT, kSteps = kKeys * DT;
        const int i16 = lane & 15, r = 4 * half + i16 / 4;
        const int piece = 2 * ((lane >> 4) & 1) + (i16 & 3) / 2;
        auto read = [&](int j) {
          const unsigned char *at = vt + (16 * (j / DT) + r) * RB + 8 * (i16 & 1);
          const int p = 4 * (j % DT) + piece;
          const s16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(at + 16 * (p ^ vswz(r))));
          const s16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(at + 8 * RB + 16 * (p ^ vswz(r + 8))));
          return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        u32x4_t p[2][QP];
        auto weights = [&](int k, int from, int to) {  // pairs of step k
#pragma unroll
          for (int e = from; e < to; ++e) {
            float p0 = weight(8 * k + 2 * e), p1 = weight(8 * k + 2 * e + 1);
            if constexpr (BF) {
              const uint32_t both = pack_bf16x2(p0, p1);
              p[k & 1][0][e] = both;
              l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, both), bf16x2_t{1.f, 1.f}, l, false);
            } else {
              l += p0, l += p1;
#pragma unroll
              for (int y = 0; y < QP; ++y) {
                p[k & 1][y][e] = tops(p0, p1);
                p0 -= top(p0), p1 -= top(p1);
              }
            }
          }
        };
        bf16x8_t v[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) v[j] = read(j);
        weights(0, 0, 4);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
          const int k = j / DT, d = j % DT;
#pragma unroll
          for (int y = QP - 1; y >= 0; --y)
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[j % kAhead], __builtin_bit_cast(bf16x8_t, p[k & 1][y]),
                                                           o[d], 0, 0, 0);
          if (j + kAhead < kSteps) v[j % kAhead] = read(j + kAhead);
          if (k + 1 < kKeys) weights(k + 1, 4 * d / DT, 4 * (d + 1) / DT);
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        there = there_next, there_next = there_after;
      } else {
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) unpack(j, i, st ^ 1);
        there = there_next, there_next = load(k0 + 2 * TK, page, t + 2 < take);
        page = lookup(k0 + 3 * TK);
      }
    }
    // ---- the rows' outputs, or their part: lane (row n, half) holds columns
    // 32 d + 8 k + 4 half .. + 3
    l += other_half(l);
    rows.store<T>(a, seg, s, BM, 32 * wave + n, o, m, l);
    if (__builtin_expect(__ballot(missed) != 0, 0) && rows.live)
      for (int k = k_first; k < k_first + take * TK; k += TK) {
        if (!shared.edge(k, TK)) continue;
        for (int key = max(k, rows.lo); key < min(k + TK, rows.hi); ++key) {
          const int pg = pages.lookup(a, key);
          if (!pages.there(a, key, pg)) continue;
          const int off = key - (int)fast_div(key, a.div_page) * a.page_size;
          const uint8_t *vs = vs_base + pg * a.v_sc_ld[0] + off * a.v_sc_ld[2];
#pragma unroll 1
          for (int col = 4 * half; col < a.D; col += 8)
            if (vs[col / kMxBlock] > kMxLast)
#pragma unroll 1
              for (int e = 0; e < 4; ++e) {
                if (seg.complete)
                  static_cast<T *>(a.out)[((int64_t)(s.q0 + rows.token) * a.H + h * G + rows.row - rows.token * G) * a.D + col + e] =
                      BF ? (T)0x7fc0 : (T)NAN;
                else a.part_o[(seg.slot * BM + 32 * wave + n) * a.D + col + e] = NAN;
              }
        }
      }
    if (tid == 0 && seg.bb == 0 && !seg.complete) {
      split->slot = seg.slot, split->last = seg.last;
      split->row0 = r0, split->rows = min(BM, s.q * G - r0), split->head = h, split->q0 = s.q0;
    }
    __syncthreads();  // the last tile is done with
  }
  zero_rows<NTH>(a, plan, BM, TK, batch);
}

template <typename T, int DP, int DC, bool NEAR>
hipError_t launch_as(const Mx4AttnArgs &a, int grid, hipStream_t s) {
  const size_t tiles = 4 * (size_t)TK * DP * 2;
  const size_t lds = tiles + batch_ints(a.S) * 4, largest = tiles + batch_ints(kMaxSeqs) * 4;
  if (a.item_rows != BM) return hipErrorInvalidValue;
  auto kernel = mx4_tile_kernel<T, DP, DC, NEAR>;
  const hipError_t allowed = allow_lds(reinterpret_cast<const void *>(kernel), lds, largest);
  if (allowed != hipSuccess) return allowed;
  kernel<<<grid, NTH, lds, s>>>(a);
  return hipGetLastError();
}
template <typename T, bool NEAR>
hipError_t launch_of(const Mx4AttnArgs &a, int grid, hipStream_t s) {
  if (a.D <= 64) return launch_as<T, 64, 64, NEAR>(a, grid, s);
  if (a.D <= 96) return launch_as<T, 128, 96, NEAR>(a, grid, s);
  if (a.D <= 128) return launch_as<T, 128, 128, NEAR>(a, grid, s);
  if constexpr (sizeof(T) == 2) return launch_as<T, 256, 256, NEAR>(a, grid, s);
  return hipErrorInvalidValue;  // fp32 past 128: the row kernel's
}
template <typename T>
hipError_t launch_by(const Mx4AttnArgs &a, int grid, hipStream_t s) {
  return a.near ? launch_of<T, true>(a, grid, s) : launch_of<T, false>(a, grid, s);
}

}  // namespace

int mx4_tile_rows() { return BM; }
int mx4_tile_grid(const Mx4AttnArgs &a) { return 256 * waves(a.dtype == ZT_DT_BF16, a.D); }
hipError_t launch_mx4_tiles(const Mx4AttnArgs &a, int grid, hipStream_t s) {
  return a.dtype == ZT_DT_BF16 ? launch_by<uint16_t>(a, grid, s) : launch_by<float>(a, grid, s);
}

}  // namespace zt
