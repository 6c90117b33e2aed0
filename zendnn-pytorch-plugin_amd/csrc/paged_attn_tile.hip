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

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32); }

// NW waves of 32 rows each against a span of the keys of one cache head.
//
// Bound by the matrix pipes and, beside them, by the exponentials.  All waves
// share tiles of TK keys and values (64, or 32 in fp32) that arrive in LDS by
// DMA, two tiles deep: while one is worked on the next is on its way, with one
// barrier per tile.
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
// taken before the rounding.
template <typename T, int DP, int DC, int NW>
__global__ __launch_bounds__(64 * NW, NW / 4) void paged_attn_tile_kernel(AttnArgs a) {
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
  int *tile_base = reinterpret_cast<int *>(smem + 4 * STAGE);

  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Plan plan = make_plan<NTH>(a, BM, TK, tile_base, &sh);
  zero_rows<NTH>(a, plan, BM, TK, tile_base);
  Split *split = static_cast<Split *>(a.splits) + plan.wg;
  if (tid == 0) split->rows = 0;
  if (plan.todo == 0) return;

  const float c = score_factor(a.scale);
  const int G = a.group, C = a.D * ES / 16;
  const char *zero = reinterpret_cast<const char *>(kZeroRow);
  const int64_t kps = a.k_ld[0] * ES, kts = a.k_ld[2] * ES, vps = a.v_ld[0] * ES, vts = a.v_ld[2] * ES;
  // where a lane's pieces of K and columns of V are in a tile
  auto kswz = [](int row) { return CR >= 16 ? row & 15 : row & 7; };
  auto vswz = [](int row) {
    return !BF ? ((row >> 2) & 1) << 3 : CR >= 16 ? (row & 3) << 2 : ((row >> 1) & 1) << 2;
  };
  const uint32_t lds0 = lds_addr(smem);

  int64_t todo = plan.todo, unit = plan.per * plan.wg;
  const int64_t span0 = unit;
  for (int h = plan.head, x = plan.item, bb = plan.off; todo > 0; ++x, bb = 0) {
    if (x == plan.items) ++h, x = 0;
    const int i = seq_of_item(tile_base, a.S, x);
    const Seq s = seq_of(a, i);
    const int r0 = (x - tile_base[i]) * BM;
    const KeyRange kr = keys_of(a, s, x - tile_base[i], BM);
    const int nb = blocks_of(kr, TK), b0 = kr.begin / TK;
    if (nb == 0) continue;
    const int take = (int)min((int64_t)(nb - bb), todo);
    const int *table = a.table + (int64_t)i * a.W;
    const char *kbase = static_cast<const char *>(a.k) + h * a.k_ld[1] * ES;
    const char *vbase = static_cast<const char *>(a.v) + h * a.v_ld[1] * ES;

    // page of key at + (lane % TK), or -1 if no row of the item sees it
    auto lookup = [&](int at) {
      const int tok = at + (lane & (TK - 1));
      const bool in = tok >= kr.begin && tok < kr.end;
      const int page = table[in ? fast_div(tok, a.div_page) : 0];
      return in ? page : -1;
    };
    // K and V of the tile at `at` into stage `st`; returns which keys there are
    auto load = [&](int at, int page, int st) -> uint64_t {
      const int tok = at + (lane & (TK - 1));
      const bool ok = page >= 0 && page < a.pages;
      const int in_page = tok - (int)fast_div(tok, a.div_page) * a.page_size;
      const uint64_t ko = (uint64_t)(ok ? kbase + page * kps + in_page * kts : zero);
      const uint64_t vo = (uint64_t)(ok ? vbase + page * vps + in_page * vts : zero);
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int idx = (wave * NI + j) * 64 + lane, row = idx / CR, slot = idx % CR;
        const char *ks = (const char *)__shfl((unsigned long long)ko, row);
        const char *vs = (const char *)__shfl((unsigned long long)vo, row);
        const int kp = slot ^ kswz(row), vp = slot ^ vswz(row);
        load_to_lds(kp < C ? ks + 16 * kp : zero, lds0 + st * 2 * STAGE + (wave * NI + j) * 1024);
        load_to_lds(vp < C ? vs + 16 * vp : zero, lds0 + st * 2 * STAGE + STAGE + (wave * NI + j) * 1024);
      }
      const uint64_t m = __ballot(ok);
      return TK == 64 ? m : m & 0xffffffffull;
    };
    const int k_first = (b0 + bb) * TK;
    uint64_t there = load(k_first, lookup(k_first), 0), there_next = 0;
    int page = take > 1 ? lookup(k_first + TK) : -1;

    // ---- the wave's rows: lane (row n, half) holds pieces 2 j + half of q
    const int row = r0 + 32 * wave + n;
    const int row_t = (int)fast_div(row, a.div_group);
    const bool live = row_t < s.q;
    const int pos = s.n - s.q + row_t;
    const int hi = !live ? INT32_MAX : a.causal ? pos + 1 : s.n;
    const int lo = live && a.causal && a.window ? (int)max((int64_t)pos + 1 - a.window, (int64_t)0) : 0;
    // over the wave's live rows, which come first: tokens ascend with the rows
    const bool wave_live = __ballot(live) != 0;
    const int last_live = 31 - __builtin_clz((uint32_t)__ballot(live) | 1u);
    const int hi_min = __builtin_amdgcn_readlane(hi, 0), lo_min = __builtin_amdgcn_readlane(lo, 0);
    const int hi_max = __builtin_amdgcn_readlane(hi, last_live), lo_max = __builtin_amdgcn_readlane(lo, last_live);
    u32x4_t q[NQ];
    {
      const char *src = static_cast<const char *>(a.q) +
          ((int64_t)(s.q0 + row_t) * a.q_ld[0] + (h * G + row - row_t * G) * a.q_ld[1]) * ES;
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        const int p = 2 * j + half;
        q[j] = scale_sign<T>(*reinterpret_cast<const u32x4_t *>(live && p < C ? src + 16 * p : zero), a.scale);
      }
    }
    f32x16_t o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    float m = -INFINITY, l = 0.f;

    for (int t = 0; t < take; ++t) {
      const int k0 = k_first + t * TK, st = t & 1;
      wait_and_meet();  // the tile is there, and the previous one is done with
      if (t + 1 < take) {
        there_next = load(k0 + TK, page, st ^ 1);
        if (t + 2 < take) page = lookup(k0 + 2 * TK);
      }
      if (wave_live && k0 < hi_max && k0 + TK > lo_min) {
        const unsigned char *kt = smem + st * 2 * STAGE, *vt = kt + STAGE;
        // ---- scores
        f32x16_t sc[KT];
#pragma unroll
        for (int u = 0; u < KT; ++u) {
#pragma unroll
          for (int e = 0; e < 16; ++e) sc[u][e] = 0.f;
#pragma unroll
          for (int j = 0; j < NQ; ++j) {
            const u32x4_t k = *reinterpret_cast<const u32x4_t *>(
                kt + (32 * u + n) * RB + 16 * ((2 * j + half) ^ kswz(n)));
            if constexpr (BF) {
              sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                  __builtin_bit_cast(bf16x8_t, k), __builtin_bit_cast(bf16x8_t, q[j]), sc[u], 0, 0, 0);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                sc[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k[e]), __uint_as_float(q[j][e]),
                                                             sc[u], 0, 0, 0);
            }
          }
        }
        // ---- weights
        const bool whole = there == (TK == 64 ? ~0ull : 0xffffffffull);
        if (!whole || k0 + TK > hi_min || k0 < lo_max) {
#pragma unroll
          for (int u = 0; u < KT; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int k = 32 * u + 8 * (e / 4) + 4 * half + e % 4;
              if (!(there >> k & 1) || k0 + k < lo || k0 + k >= hi) sc[u][e] = -INFINITY;
            }
        }
        float mx = sc[0][0];
#pragma unroll
        for (int u = 0; u < KT; ++u)
#pragma unroll
          for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[u][e]);
        mx = fmaxf(mx, other_half(mx));
        if (__ballot(mx != -INFINITY && (mx - m) * c > 8.f)) {
          const float to = fmaxf(m, mx);
          const float f = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m * c - to * c);
          l *= f;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] *= f;
          m = to;
        }
        const float mc = m == -INFINITY ? 0.f : m * c;
#pragma unroll
        for (int u = 0; u < KT; ++u)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            sc[u][e] = __builtin_amdgcn_exp2f(fmaf(sc[u][e], c, -mc));
            l += sc[u][e];
          }
        // ---- O^T += V^T P^T
        if constexpr (BF) {
          typedef __attribute__((address_space(3))) s16x4_t *tr_ptr;
          u32x4_t p[2 * KT];
#pragma unroll
          for (int k = 0; k < 2 * KT; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              p[k][e] = pack_bf16x2(sc[k / 2][8 * (k % 2) + 2 * e], sc[k / 2][8 * (k % 2) + 2 * e + 1]);
          const int i16 = lane & 15, r = 4 * half + i16 / 4;
          const int piece = 2 * ((lane >> 4) & 1) + (i16 & 3) / 2;
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            const unsigned char *at = vt + r * RB + 16 * ((4 * d + piece) ^ vswz(r)) + 8 * (i16 & 1);
#pragma unroll
            for (int k = 0; k < 2 * KT; ++k) {
              const s16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(at + 16 * k * RB));
              const s16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(at + (16 * k + 8) * RB));
              o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                  __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7)),
                  __builtin_bit_cast(bf16x8_t, p[k]), o[d], 0, 0, 0);
            }
          }
        } else {
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int r = 8 * (e / 4) + 4 * half + e % 4;
              const float v = *reinterpret_cast<const float *>(
                  vt + r * RB + 16 * ((8 * d + n / 4) ^ vswz(r)) + 4 * (n & 3));
              o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, sc[0][e], o[d], 0, 0, 0);
            }
        }
      }
      there = there_next;
    }
    // ---- the rows' outputs, or their part: lane (row n, half) holds columns
    // 32 d + 8 k + 4 half .. + 3
    const bool complete = bb == 0 && take == nb;
    l += other_half(l);
    if (live) {
      const int64_t slot = 2 * (int64_t)plan.wg + (unit > span0 ? 1 : 0), pr = slot * BM + 32 * wave + n;
      const int64_t to = ((int64_t)(s.q0 + row_t) * a.H + h * G + row - row_t * G) * a.D;
      const float r = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int col = 32 * d + 8 * k + 4 * half;
          const f32x4_t y = {o[d][4 * k], o[d][4 * k + 1], o[d][4 * k + 2], o[d][4 * k + 3]};
          if (col >= a.D) continue;
          if (complete) store_out<T>(a.out, to + col, y, r);
          else *reinterpret_cast<f32x4_t *>(a.part_o + pr * a.D + col) = y;
        }
      if (!complete && half == 0) a.part_ml[2 * pr] = m, a.part_ml[2 * pr + 1] = l;
    }
    if (tid == 0 && bb == 0 && !complete) {
      split->u0 = unit, split->u1 = unit + nb, split->per = plan.per;
      split->row0 = r0, split->rows = min(BM, s.q * G - r0), split->head = h, split->q0 = s.q0;
    }
    todo -= take;
    unit += take;
    __syncthreads();  // the last tile is done with
  }
}

template <typename T, int DP, int DC, int NW>
hipError_t launch_tiles_as(const AttnArgs &a, int grid, hipStream_t s) {
  constexpr int TK = sizeof(T) == 2 ? 64 : 32;
  const size_t lds = 4 * (size_t)TK * DP * sizeof(T) + ((size_t)a.S + 1) * 4;
  auto kernel = paged_attn_tile_kernel<T, DP, DC, NW>;
  if (lds > 64 * 1024) {
    const hipError_t grown = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (grown != hipSuccess) return grown;
  }
  kernel<<<grid, 64 * NW, lds, s>>>(a);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_tiles_t(const AttnArgs &a, int grid, hipStream_t s) {
  if (a.D <= 64) return launch_tiles_as<T, 64, 64, 8>(a, grid, s);
  if (a.D <= 96) return launch_tiles_as<T, 128, 96, 8>(a, grid, s);
  if (a.D <= 128) return launch_tiles_as<T, 128, 128, 8>(a, grid, s);
  return launch_tiles_as<T, 256, 256, 4>(a, grid, s);
}

}  // namespace

// Past head_dim 128 a wave's queries and outputs need the registers of two.
int tile_rows(const AttnArgs &a) { return a.D <= 128 ? 256 : 128; }
int tile_grid(const AttnArgs &) { return 256; }

hipError_t launch_tiles(const AttnArgs &a, hipStream_t s) {
  return a.dtype == ZT_DT_BF16 ? launch_tiles_t<uint16_t>(a, tile_grid(a), s)
                               : launch_tiles_t<float>(a, tile_grid(a), s);
}

}  // namespace zt
