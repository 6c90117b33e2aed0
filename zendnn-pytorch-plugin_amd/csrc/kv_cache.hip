// The paged key / value cache around the quantised linears, for gfx950:
// rotary positions, appending a step's keys and values, and the upkeep of
// the cache's pages.  (The attention that reads the cache: paged_attn.hip.)
//
// All of it moves bytes: a few flops or integer operations per element, so
// each kernel is bound by HBM where the operands are large and by its launch
// where they are small.  Every value that comes from the device (positions,
// slots, page ids, lengths) is checked against its bound before it is used as
// an address, because the host cannot see it without a synchronisation.
#include "zt_cache.hpp"

namespace zt {

namespace {

// ------------------------------------------------------------------ rotary
// V consecutive elements of T as floats.
template <typename T, int V>
struct Vec;
template <>
struct Vec<uint16_t, 8> {
  static __device__ __forceinline__ void load(const uint16_t *p, float (&f)[8]) {
    const u32x4_t v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(v[i] << 16);
      f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void store(uint16_t *p, const float (&f)[8]) {
    u32x4_t v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<u32x4_t *>(p) = v;
  }
};
template <>
struct Vec<float, 4> {
  static __device__ __forceinline__ void load(const float *p, float (&f)[4]) {
    const f32x4_t v = __builtin_nontemporal_load(reinterpret_cast<const f32x4_t *>(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = v[i];
  }
  static __device__ __forceinline__ void store(float *p, const float (&f)[4]) {
    *reinterpret_cast<f32x4_t *>(p) = f32x4_t{f[0], f[1], f[2], f[3]};
  }
};
template <>
struct Vec<uint16_t, 1> {
  static __device__ __forceinline__ void load(const uint16_t *p, float (&f)[1]) {
    f[0] = bf16_bits_to_f32(p[0]);
  }
  static __device__ __forceinline__ void store(uint16_t *p, const float (&f)[1]) {
    p[0] = (uint16_t)f32_to_bf16_bits(f[0]);
  }
};
template <>
struct Vec<float, 1> {
  static __device__ __forceinline__ void load(const float *p, float (&f)[1]) { f[0] = p[0]; }
  static __device__ __forceinline__ void store(float *p, const float (&f)[1]) { p[0] = f[0]; }
};

// Pair (a, b) of frequency i at position p becomes
//   (a cos - b sin, b cos + a sin),  cos = table[p][i], sin = table[p][R/2 + i],
// in fp32, rounded once.  The pairs are (x[i], x[R/2 + i]) or, interleaved,
// (x[2i], x[2i + 1]); x[R..D) passes through.
//
// One thread takes one unit of a token's head row: V elements of each half
// (2V consecutive ones when interleaved), or V consecutive ones of the part
// that passes through.  With V elements being 16 bytes every load and store
// is one full-width instruction; inputs go past the caches' replacement (8191
// tokens of 32 + 8 + 8 heads of 128: 36.7 us, 5.6 TB/s; 39.9 without; 8 tokens:
// 3.3 us, one round trip).  V = 1 (a unit then is one pair) serves row
// parts, strides and addresses that 16 bytes do not divide.
template <typename T, int V, bool IL>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = idx / a.units;
  if (t >= a.T) return;
  int u = (int)(idx - t * a.units);
  // which of the token's rows: query heads, key heads, then value heads
  const T *src;
  T *dst;
  const int64_t p = a.pos[t];
  bool rotate = true;
  if (u < a.H * a.row_units) {
    const int h = u / a.row_units;
    u -= h * a.row_units;
    src = static_cast<const T *>(a.q) + t * a.q_ld[0] + h * a.q_ld[1];
    dst = static_cast<T *>(a.q_out) + (t * a.H + h) * a.D;
  } else {
    u -= a.H * a.row_units;
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= a.pages * a.page_size) return;  // a padding token
    const int64_t page = slot / a.page_size, off = slot - page * a.page_size;
    if (u < a.KV * a.row_units) {
      const int h = u / a.row_units;
      u -= h * a.row_units;
      src = static_cast<const T *>(a.k) + t * a.k_ld[0] + h * a.k_ld[1];
      dst = static_cast<T *>(a.k_cache) + page * a.kc_ld[0] + h * a.kc_ld[1] + off * a.kc_ld[2];
    } else {
      u -= a.KV * a.row_units;
      const int h = u / a.copy_units;
      u -= h * a.copy_units;
      src = static_cast<const T *>(a.v) + t * a.v_ld[0] + h * a.v_ld[1];
      dst = static_cast<T *>(a.v_cache) + page * a.vc_ld[0] + h * a.vc_ld[1] + off * a.vc_ld[2];
      rotate = false;
    }
  }
  const int R = a.R, half = R / 2;
  const int rot_units = IL ? R / (2 * V) : half / V;
  if (!rotate || u >= rot_units) {
    const int at = rotate ? R + (u - rot_units) * V : u * V;
    float f[V];
    Vec<T, V>::load(src + at, f);
    Vec<T, V>::store(dst + at, f);
    return;
  }
  const int i0 = u * V;  // the first of the unit's V frequencies
  const int at0 = IL ? 2 * i0 : i0, at1 = IL ? 2 * i0 + V : half + i0;
  float x0[V], x1[V], y0[V], y1[V];
  Vec<T, V>::load(src + at0, x0);
  Vec<T, V>::load(src + at1, x1);
  if (p < 0) {  // a padding token's row is passed on as it is
    Vec<T, V>::store(dst + at0, x0);
    Vec<T, V>::store(dst + at1, x1);
    return;
  }
  float c[V], s[V];
  if (p < a.length) {
    const float *row = a.table + p * a.table_ld + i0;
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = row[i], s[i] = row[half + i];
  } else {  // no such position: NaN, so that it does not pass unseen
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = s[i] = __uint_as_float(0x7fc00000u);
  }
  if constexpr (IL && V > 1) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const int j = i / 2, k = V / 2 + i / 2;
      y0[i] = x0[i] * c[j] - x0[i + 1] * s[j], y0[i + 1] = x0[i + 1] * c[j] + x0[i] * s[j];
      y1[i] = x1[i] * c[k] - x1[i + 1] * s[k], y1[i + 1] = x1[i + 1] * c[k] + x1[i] * s[k];
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) y0[i] = x0[i] * c[i] - x1[i] * s[i], y1[i] = x1[i] * c[i] + x0[i] * s[i];
  }
  Vec<T, V>::store(dst + at0, y0);
  Vec<T, V>::store(dst + at1, y1);
}

// ------------------------------------------------------------------- pages
constexpr int kBlock = 1024, kWaves = kBlock / 64;

// This wave's stores and atomics have been carried out in L2, which is where
// agent-scope atomics of the same XCD meet them (a fence would write back the
// whole L2 as well).
__device__ __forceinline__ void counts_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Exclusive prefix sum of v over the workgroup's threads; *total is the sum.
// `part` is an LDS array of kWaves ints.
__device__ __forceinline__ int block_scan(int v, int *part, int *total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int x = wave_scan(v);
  __syncthreads();  // the previous use of part is over
  if (lane == 63) part[wave] = x;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int y = part[w];
    if (w < wave) before += y;
    sum += y;
  }
  *total = sum;
  return before + x - v;
}

// A step's new tokens get their pages.  Sequence i holds have_i = ceil(ctx_i /
// size) pages and needs want_i = ceil((ctx_i + new_i) / size); need_i = want_i
// - have_i if want_i fits the table's width, else 0.  The free pages (count 0)
// are given out in ascending order, sequence by sequence: i is granted when
// want_i fits and need_1 + .. + need_i <= the number of free pages.
//
// One launch: every workgroup counts the free pages and adds up the needs by
// itself (a few bytes per page and per sequence, from L2), and then
//  * writes its share of the table and of the tokens where no new page is
//    involved, and
//  * for each free page of its own slice, whose rank among the free pages it
//    knows, finds the sequence that takes this rank by bisection over the
//    needs' running sums, and writes the page's table entry, count and slots.
// So no workgroup waits for another.  Bound by round trips to memory: what the
// steps share (lengths, needs) is read once, into LDS, and the counts four to a
// load (64 sequences of up to 8192 tokens in pages of 16: 6.7 us; 15 with
// lengths, counts and table entries read one by one from memory).
__global__ __launch_bounds__(kBlock) void cache_extend_kernel(ExtendArgs a) {
  extern __shared__ int sm[];  // end[S], ctx[S], cu[S + 1]
  __shared__ int part[kWaves], part2[kWaves];
  const int tid = threadIdx.x, S = a.S, W = a.W, size = a.page_size;
  int *end = sm, *ctx = sm + S, *cu = sm + 2 * S;
  // lengths are held to what a table row can hold (W * size < 2^30), so that
  // pages and places come from 32-bit divisions
  const int most = W * size;
  for (int i = tid; i <= S; i += kBlock) {
    cu[i] = a.cu[i];
    if (i < S) ctx[i] = max(a.ctx[i], 0);
  }
  // free pages: all, and those before this workgroup's slice
  const int64_t slice = ((a.pages + gridDim.x - 1) / gridDim.x + kBlock - 1) / kBlock * kBlock;
  const int64_t s0 = min((int64_t)blockIdx.x * slice, a.pages), s1 = min(s0 + slice, a.pages);
  int all = 0, mine = 0;  // s0 is a multiple of 4
  if (reinterpret_cast<uintptr_t>(a.refs) % 16 == 0) {
    const i32x4_t *refs = reinterpret_cast<const i32x4_t *>(a.refs);
#pragma unroll 8
    for (int64_t p = tid; p < a.pages / 4; p += kBlock) {
      const i32x4_t r = refs[p];
      const int f = (r[0] == 0) + (r[1] == 0) + (r[2] == 0) + (r[3] == 0);
      all += f;
      mine += 4 * p < s0 ? f : 0;
    }
    const int64_t p = a.pages / 4 * 4 + tid;
    if (p < a.pages) {
      const int f = a.refs[p] == 0;
      all += f;
      mine += p < s0 ? f : 0;
    }
  } else {
    for (int64_t p = tid; p < a.pages; p += kBlock) {
      const int f = a.refs[p] == 0;
      all += f;
      mine += p < s0 ? f : 0;
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) all += __shfl_xor(all, d), mine += __shfl_xor(mine, d);
  if ((tid & 63) == 0) part[tid >> 6] = all, part2[tid >> 6] = mine;
  __syncthreads();
  int free_pages = 0, rank0 = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) free_pages += part[w], rank0 += part2[w];
  auto new_of = [&](int i) { return max(cu[i + 1] - cu[i], 0); };
  auto fits = [&](int i) { return ctx[i] <= most && new_of(i) <= most - ctx[i]; };
  auto have_of = [&](int i) { return (int)fast_div(ctx[i] + size - 1, a.div_size); };
  auto want_of = [&](int i) { return (int)fast_div(ctx[i] + new_of(i) + size - 1, a.div_size); };
  // needs and their running sums
  int sum = 0;
  for (int i0 = 0; i0 < S; i0 += kBlock) {
    const int i = i0 + tid;
    const int need = i < S && fits(i) ? want_of(i) - have_of(i) : 0;
    int total;
    const int before = block_scan(need, part, &total);
    if (i < S) end[i] = sum + before + need;
    sum += total;
  }
  __syncthreads();
  auto granted = [&](int i) { return fits(i) && end[i] <= free_pages; };
  const int step = (int)gridDim.x * kBlock, first = (int)blockIdx.x * kBlock + tid;
#pragma unroll 2
  for (int64_t e = first; e < (int64_t)S * W; e += step) {
    const int i = (int)fast_div((uint32_t)e, a.div_w), col = (int)e - i * W, page = a.table[e];
    if (!(granted(i) && col >= have_of(i) && col < want_of(i))) a.table_out[e] = page;
  }
  for (int i = first; i < S; i += step) a.ctx_out[i] = granted(i) ? ctx[i] + new_of(i) : a.ctx[i];
  for (int64_t t = first; t < a.T; t += step) {
    int lo = 0, hi = S + 1;  // the first j with cu[j] > t
    while (lo < hi) {
      const int m = (lo + hi) / 2;
      if (cu[m] > t) hi = m;
      else lo = m + 1;
    }
    const int i = lo - 1;
    int64_t pos = -1, slot = -1;
    bool fresh = false;
    if (i >= 0 && i < S && granted(i)) {
      const int p = ctx[i] + (int)(t - cu[i]), col = (int)fast_div(p, a.div_size);
      pos = p;
      fresh = col >= have_of(i);
      if (!fresh) {
        const int page = a.table[(int64_t)i * W + col];
        if (page >= 0 && page < a.pages) slot = (int64_t)page * size + (p - col * size);
      }
    }
    a.pos_out[t] = pos;
    // Keeps the two stores apart: merged into one store with a chosen address,
    // they come out of the compiler (clang 22 of ROCm 7.2) with the wrong
    // address for some lanes.
    asm volatile("" ::: "memory");
    if (!fresh) a.slots[t] = slot;
  }
  for (int64_t p0 = s0; p0 < s1; p0 += kBlock) {
    const int64_t p = p0 + tid;
    const int r = p < s1 ? a.refs[p] : 1;
    int total;
    const int rank = rank0 + block_scan(r == 0, part, &total);
    rank0 += total;
    if (p >= s1) continue;
    int out = r;
    if (r == 0 && S > 0 && rank < end[S - 1]) {
      int lo = 0, hi = S - 1;  // the first i with end[i] > rank
      while (lo < hi) {
        const int m = (lo + hi) / 2;
        if (end[m] > rank) hi = m;
        else lo = m + 1;
      }
      if (granted(lo)) {
        const int c = ctx[lo], n = c + new_of(lo);
        const int col = have_of(lo) + rank - (lo ? end[lo - 1] : 0);
        a.table_out[(int64_t)lo * W + col] = (int32_t)p;
        out = 1;
        const int from = col * size, last = n - from < size ? n : from + size;
        for (int pos = max(c, from); pos < last; ++pos) {
          const int64_t t = (int64_t)cu[lo] + (pos - c);
          if (t >= 0 && t < a.T) a.slots[t] = p * size + (pos - from);
        }
      }
    }
    a.refs_out[p] = out;
  }
}

// Row i continues row parents[i] (-1: the row ends).  A parent's full pages
// are shared by its children; its partly filled last page goes to the first
// child, and every other child gets a copy of it in a free page (the lowest
// ones, in row order, counted after the ended rows gave theirs back).  A row
// that finds no free page ends: context 0, an empty table row.
//
// One workgroup: the steps depend on each other through the whole pool's
// counts, and the tables are small (64 rows of 128 pages: 33 KB each way).
// Bound by round trips to memory, so lengths and parents are kept in LDS and a
// thread takes kEach table entries at once, their loads before their uses (64
// rows of 128 pages: 13.6 us; 23.5 one entry at a time).
__global__ __launch_bounds__(kBlock) void cache_fork_kernel(ForkArgs a) {
  constexpr int kEach = 8;
  extern __shared__ int sm[];
  __shared__ int part[kWaves];
  const int tid = threadIdx.x, S = a.S, W = a.W, size = a.page_size;
  // give[r]: the r-th free page; rank[i]: which of them row i gets, -1: none
  int *children = sm, *first = sm + S, *give = sm + 2 * S, *rank = sm + 3 * S, *ctx = sm + 4 * S, *par = sm + 5 * S;
  for (int i = tid; i < S; i += kBlock) {
    const int p = a.parents[i];
    children[i] = 0, first[i] = S;
    ctx[i] = min(max(a.ctx[i], 0), W * size);
    par[i] = p >= 0 && p < S ? p : -1;
  }
#pragma unroll 4
  for (int64_t p = tid; p < a.pages; p += kBlock)
    __hip_atomic_store(a.refs_out + p, a.refs[p], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  counts_done();
  __syncthreads();
  for (int i = tid; i < S; i += kBlock)
    if (par[i] >= 0) {
      atomicAdd(&children[par[i]], 1);
      atomicMin(&first[par[i]], i);
    }
  __syncthreads();
  auto have_of = [&](int i) { return (int)fast_div(ctx[i] + size - 1, a.div_size); };
  auto partial = [&](int i) { return ctx[i] != (int)fast_div(ctx[i], a.div_size) * size; };
  auto in_pool = [&](int page) { return page >= 0 && page < a.pages; };
  const int entries = S * W;
  // the counts after every child took its parent's pages
  for (int e0 = 0; e0 < entries; e0 += kEach * kBlock) {
    int page[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) page[k] = a.table[min(e0 + k * kBlock + tid, entries - 1)];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int e = e0 + k * kBlock + tid;
      if (e >= entries || !in_pool(page[k])) continue;
      const int i = (int)fast_div(e, a.div_w), col = e - i * W, have = have_of(i);
      if (col >= have) continue;
      const bool last = partial(i) && col == have - 1;
      const int gain = (last ? (children[i] > 0) : children[i]) - 1;
      if (gain) atomicAdd(a.refs_out + page[k], gain);
    }
  }
  counts_done();
  // rows that need a page of their own
  int needs = 0;
  for (int i0 = 0; i0 < S; i0 += kBlock) {
    const int i = i0 + tid;
    int need = 0;
    if (i < S) need = par[i] >= 0 && partial(par[i]) && first[par[i]] != i;
    int total;
    const int before = block_scan(need, part, &total);
    if (i < S) rank[i] = need ? needs + before : -1;
    needs += total;
  }
  int found = 0;
  for (int64_t p0 = 0; p0 < a.pages && found < needs; p0 += kBlock) {
    const int64_t p = p0 + tid;
    const int f = p < a.pages &&
        __hip_atomic_load(a.refs_out + p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0;
    int total;
    const int r = found + block_scan(f, part, &total);
    if (f && r < needs) give[r] = (int)p;
    found += total;
  }
  __syncthreads();
  for (int i = tid; i < S; i += kBlock) {
    const int p = par[i];
    const bool lost = p >= 0 && rank[i] >= found;
    int src = -1, dst = -1;
    if (rank[i] >= 0 && !lost) {
      src = a.table[(int64_t)p * W + have_of(p) - 1];
      if (!in_pool(src)) src = -1;
      dst = give[rank[i]];
      atomicAdd(a.refs_out + dst, 1);
    }
    a.ctx_out[i] = p >= 0 && !lost ? a.ctx[p] : 0;
    a.copies[2 * i] = src;
    a.copies[2 * i + 1] = dst;
  }
  for (int e0 = 0; e0 < entries; e0 += kEach * kBlock) {
    int page[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int e = min(e0 + k * kBlock + tid, entries - 1), i = (int)fast_div(e, a.div_w);
      page[k] = a.table[(int64_t)max(par[i], 0) * W + e - i * W];
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int e = e0 + k * kBlock + tid;
      if (e >= entries) continue;
      const int i = (int)fast_div(e, a.div_w), col = e - i * W, p = par[i];
      int out = -1;
      if (p >= 0 && col < have_of(p)) {
        const bool last = partial(p) && col == have_of(p) - 1;
        if (rank[i] >= found) {  // a lost row's share of the full pages goes back
          if (!last && in_pool(page[k])) atomicSub(a.refs_out + page[k], 1);
        } else {
          out = last && rank[i] >= 0 ? give[rank[i]] : page[k];
        }
      }
      a.table_out[e] = out;
    }
  }
}

// The n pages in use move to the pool's first n: the k-th page in use from n
// on (ascending) goes to the k-th free page below n.  `to` (pages ints) is
// the new place of every page.  One workgroup, as above (2048 pages: 6 us, of 96
// with the copies that it asks for in 8 layers).
__global__ __launch_bounds__(kBlock) void cache_compact_kernel(CompactArgs a) {
  __shared__ int part[kWaves];
  const int tid = threadIdx.x;
  int used = 0, n;
  for (int64_t p = tid; p < a.pages; p += kBlock) used += a.refs[p] != 0;
  block_scan(used, part, &n);
  int srcs = 0, dsts = 0;
  for (int64_t p0 = 0; p0 < a.pages; p0 += kBlock) {
    const int64_t p = p0 + tid;
    const int r = p < a.pages ? a.refs[p] : 0;
    const int src = r != 0 && p >= n, dst = p < a.pages && r == 0 && p < n;
    int total;
    const int ks = srcs + block_scan(src, part, &total);
    srcs += total;
    const int kd = dsts + block_scan(dst, part, &total);
    dsts += total;
    if (src) a.copies[2 * ks] = (int32_t)p, a.to[p] = ks;
    if (dst) a.copies[2 * kd + 1] = (int32_t)p;
  }
  __threadfence_block();
  __syncthreads();
  for (int64_t k = srcs + tid; k < a.pages / 2; k += kBlock) a.copies[2 * k] = a.copies[2 * k + 1] = -1;
  for (int64_t p = tid; p < a.pages; p += kBlock) {
    const int r = a.refs[p];
    if (p >= n) {
      a.refs_out[p] = 0;
      if (r != 0) a.refs_out[a.copies[2 * a.to[p] + 1]] = r;
    } else if (r != 0) {
      a.refs_out[p] = r;
    }
  }
  for (int64_t e = tid; e < a.entries; e += kBlock) {
    int page = a.table[e];
    if (page >= n && page < a.pages && a.refs[page] != 0) page = a.copies[2 * a.to[page] + 1];
    a.table_out[e] = page;
  }
}

// copies[k] = (src, dst): page dst of every cache becomes page src.  Pairs
// with an id outside the pool are none.  grid (pairs x parts of a page, caches).
// Bound by HBM: 512 pages of 64 KB in 8 caches 95.6 us with the op before it,
// 5.65 TB/s read and written, past the caches' replacement (113 us without).
template <typename U>
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyArgs a) {
  const int k = blockIdx.x / a.parts, part = blockIdx.x - k * a.parts;
  const int src = a.copies[2 * k], dst = a.copies[2 * k + 1];
  if (src < 0 || dst < 0 || src >= a.pages || dst >= a.pages || src == dst) return;
  char *cache = static_cast<char *>(a.caches[blockIdx.y]);
  const U *from = reinterpret_cast<const U *>(cache + src * a.page_stride);
  U *to = reinterpret_cast<U *>(cache + dst * a.page_stride);
  const int64_t n = a.page_bytes / sizeof(U);
  // four loads in flight before the first store, which may alias for all that
  // the compiler knows
  const int step = a.parts * 256;
  for (int64_t i = part * 256 + threadIdx.x; i < n; i += 4 * step) {
    U x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = __builtin_nontemporal_load(from + (i + k * step < n ? i + k * step : i));
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k * step < n) __builtin_nontemporal_store(x[k], to + i + k * step);
  }
}

// Threads of a launch, at most: the runtime counts them in 32 bits and leaves out
// what is past those without an error.
constexpr int64_t kMostThreads = 1ll << 31;

template <typename T, int V>
hipError_t launch_rotary_v(RotaryArgs a, hipStream_t s) {
  const int64_t all = a.T, step = std::max<int64_t>(kMostThreads / a.units, 1);
  auto move = [&](const void *p, int64_t elements) { return static_cast<const T *>(p) + elements; };
  for (int64_t t = 0; t < all; t += step) {
    a.T = std::min(step, all - t);
    const dim3 grid((unsigned)((a.T * a.units + 255) / 256));
    if (a.interleaved) rotary_kernel<T, V, true><<<grid, dim3(256), 0, s>>>(a);
    else rotary_kernel<T, V, false><<<grid, dim3(256), 0, s>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    a.q = move(a.q, step * a.q_ld[0]), a.q_out = static_cast<T *>(a.q_out) + step * a.H * a.D, a.pos += step;
    if (a.KV) a.k = move(a.k, step * a.k_ld[0]), a.v = move(a.v, step * a.v_ld[0]), a.slots += step;
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_rotary(RotaryArgs a, int dtype, bool wide, hipStream_t s) {
  const int v = !wide ? 1 : dtype == ZT_DT_BF16 ? 8 : 4;
  a.copy_units = a.D / v;
  a.row_units = a.R / 2 / v + (a.D - a.R) / v;
  a.units = (a.H + a.KV) * a.row_units + a.KV * a.copy_units;
  if (dtype == ZT_DT_BF16)
    return wide ? launch_rotary_v<uint16_t, 8>(a, s) : launch_rotary_v<uint16_t, 1>(a, s);
  return wide ? launch_rotary_v<float, 4>(a, s) : launch_rotary_v<float, 1>(a, s);
}

hipError_t launch_cache_extend(ExtendArgs a, hipStream_t s) {
  // a workgroup's share: one entry, page and token per thread, on 256 CUs
  const int64_t work = std::max({a.pages, (int64_t)a.S * a.W, a.T});
  const int grid = (int)std::min<int64_t>(std::max<int64_t>((work + kBlock - 1) / kBlock, 1), 256);
  a.div_size = make_div(a.page_size), a.div_w = make_div(std::max(a.W, 1));
  cache_extend_kernel<<<grid, kBlock, (3 * (size_t)a.S + 1) * sizeof(int), s>>>(a);
  return hipGetLastError();
}

hipError_t launch_cache_fork(ForkArgs a, hipStream_t s) {
  const size_t lds = (size_t)a.S * 6 * sizeof(int);
  const hipError_t allowed =
      allow_lds(reinterpret_cast<const void *>(cache_fork_kernel), lds, kMaxRows * 6 * sizeof(int));
  if (allowed != hipSuccess) return allowed;
  a.div_size = make_div(a.page_size), a.div_w = make_div(std::max(a.W, 1));
  cache_fork_kernel<<<1, kBlock, lds, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_cache_compact(const CompactArgs &a, hipStream_t s) {
  cache_compact_kernel<<<1, kBlock, 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_copy_pages(CopyArgs a, int caches, int64_t pairs, bool wide, hipStream_t s) {
  // four loads of 16 bytes per thread
  a.parts = (int)std::min<int64_t>((a.page_bytes + 16 * 1024 - 1) / (16 * 1024), 64);
  const int64_t step = kMostThreads / 256 / a.parts;
  for (int64_t k = 0; k < pairs; k += step, a.copies += 2 * step) {
    const dim3 grid((unsigned)(std::min(step, pairs - k) * a.parts), (unsigned)caches);
    if (wide) copy_pages_kernel<u32x4_t><<<grid, dim3(256), 0, s>>>(a);
    else copy_pages_kernel<uint8_t><<<grid, dim3(256), 0, s>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace zt
