// Device helpers shared by the attention kernels (paged_attn.hip,
// paged_attn_tile.hip): which keys a tile of rows sees, and how the keys of
// all tiles are dealt out to the workgroups.
//
// A *row* is one query token of one head.  The rows of sequence i that read
// cache head h are numbered token-major: row x is token x / G, head h * G + x %
// G, with G = H / KV query heads to a cache head, so a cached key or value is
// read once for all G of them.  An *item* is a tile of BM such rows (of any
// one cache head); it needs the keys of blocks [b0, b1) of UK keys.
//
// Work is dealt out by its cost: an (item, head) costs kLead for its beginning
// and end and w for each of its blocks, and lies on a line of all of them (head
// by head, in it item by item).  Each workgroup takes an equal span of the line
// and works on the blocks that start in it.  The lengths are known on the device
// only, so each workgroup finds its span by itself.  A span may end inside an
// (item, head): its workgroups then leave partial results (running maximum, sum
// and output), which a second launch joins.  That keeps every compute unit busy
// for one long sequence as for many ragged ones.  Consecutive spans go to one
// XCD (blocks are dealt round-robin over the eight of them), so the tiles of a
// head find its keys in one L2.
#pragma once

#include "zt_cache.hpp"

namespace zt {

// log2(e) times the scale's magnitude.  The scale's sign goes to the query
// (exactly), and a scale of 0 zeroes it, so that the row maximum of the raw
// products is the maximum of the scores.
__device__ __forceinline__ float score_factor(float scale) {
  return scale == 0.f ? 1.f : fabsf(scale) * 1.4426950408889634f;
}
template <typename T>
__device__ __forceinline__ u32x4_t scale_sign(u32x4_t w, float scale) {
  const uint32_t mask = scale < 0.f ? (sizeof(T) == 2 ? 0x80008000u : 0x80000000u) : 0u;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = scale == 0.f ? 0u : w[e] ^ mask;
  return w;
}

// A weight is 2^(s c - m c), one fused operation per score s.  What the rounding
// of m c adds to the exponent is the same for all keys of a row and cancels, but
// for huge scores it is huge itself.  From |m c| = 2^10 on, s - m is taken first.
constexpr float kFar = 1024.f;
__device__ __forceinline__ bool is_far(float mc) { return fabsf(mc) >= kFar; }
// The factor that brings weights from one maximum to a larger one (1 between equal
// ones, two of -inf among them, whose difference is a NaN that the minimum drops).
// For huge ones the products' roundings are as the scores' own.
__device__ __forceinline__ float factor(float from, float to, float c) {
  return __builtin_amdgcn_exp2f(fminf(from * c - to * c, 0.f));
}

// Weights are held times 2^-16, their sums too, and the division takes it out
// again: weights go up to 2^8, and as long as those of the largest values add up
// to less than 2^16, no finite value becomes infinite on the way.  More headroom
// would take it from small values: those of 2^-110 and more keep all their digits.
constexpr int kHeadroom = 16;
constexpr float kWeight = 1.f / (1ull << kHeadroom);

typedef short s16x4_t __attribute__((ext_vector_type(4)));

// Four fp32 outputs of a row, times r, rounded.
template <typename T>
__device__ __forceinline__ void store_out(void *out, int64_t at, f32x4_t o, float r) {
  if constexpr (sizeof(T) == 2) {
    u32x2_t w;
    w[0] = pack_bf16x2(o[0] * r, o[1] * r), w[1] = pack_bf16x2(o[2] * r, o[3] * r);
    *reinterpret_cast<u32x2_t *>(static_cast<uint16_t *>(out) + at) = w;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] *= r;
    *reinterpret_cast<f32x4_t *>(static_cast<float *>(out) + at) = o;
  }
}

// Whether any of the 16 bytes' numbers is an infinity or a NaN.
template <typename T>
__device__ __forceinline__ bool not_finite(u32x4_t x) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if constexpr (sizeof(T) == 2)
      bad |= (x[i] & 0x7f800000u) == 0x7f800000u || (x[i] & 0x7f80u) == 0x7f80u;
    else
      bad |= (x[i] & 0x7f800000u) == 0x7f800000u;
  return bad;
}

// The 16 bytes' numbers with 0 in place of those that are not finite.
template <typename T>
__device__ __forceinline__ u32x4_t finite_of(u32x4_t x) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if constexpr (sizeof(T) == 2) {
      if ((x[i] & 0x7f800000u) == 0x7f800000u) x[i] &= 0xffffu;
      if ((x[i] & 0x7f80u) == 0x7f80u) x[i] &= 0xffff0000u;
    } else if ((x[i] & 0x7f800000u) == 0x7f800000u) {
      x[i] = 0;
    }
  return x;
}

// 1 KB of zeros: what a lane reads in place of a key or value that is not
// there, so that weights of zero never meet a NaN or an infinity.
static __device__ const u32x4_t kZeroRow[64] = {};

struct Seq {
  int q0, q, n;  // first row of the batch, new tokens, all tokens
};

// The batch as the device's arrays give it, held to its bounds, in LDS: read
// from memory once, because each read there is a round trip that a short call
// waits for.
struct Batch {
  int *tile_base;  // [S + 1] items before sequence i's
  int *q0, *q, *n; // [S]
  __device__ __forceinline__ Batch(void *lds, int S)
      : tile_base(static_cast<int *>(lds)), q0(tile_base + S + 1), q(q0 + S), n(q + S) {}
  __device__ __forceinline__ Seq operator[](int i) const { return {q0[i], q[i], n[i]}; }
  // the same for an i that all lanes share, in scalar registers
  __device__ __forceinline__ Seq uniform(int i) const {
    return {__builtin_amdgcn_readfirstlane(q0[i]), __builtin_amdgcn_readfirstlane(q[i]),
            __builtin_amdgcn_readfirstlane(n[i])};
  }
};
constexpr int batch_ints(int S) { return 4 * S + 1; }

// Keys [begin, end) that some row of tile r sees.
struct KeyRange {
  int begin, end;
};
__device__ __forceinline__ KeyRange keys_of(const AttnArgs &a, const Seq &s, int r, int BM) {
  KeyRange k{0, s.n};
  if (a.causal) {
    const int first = s.n - s.q + (int)fast_div((uint32_t)r * BM, a.div_group);
    const int last = s.n - s.q + min((int)fast_div((uint32_t)r * BM + BM - 1, a.div_group), s.q - 1);
    k.end = max(last + 1, 0);
    if (a.window) k.begin = (int)max((int64_t)first + 1 - a.window, (int64_t)0);
  }
  if (k.begin >= k.end) k.begin = k.end = 0;
  return k;
}
__device__ __forceinline__ int blocks_of(const KeyRange &k, int UK) {
  return k.end > k.begin ? (k.end + UK - 1) / UK - k.begin / UK : 0;
}

// Exclusive prefix sum over the workgroup of values that are not negative; `part`
// holds N / 64 values.  `stop`, if given: whether it is set in some thread, where
// the sums are not to be used.
template <int N>
__device__ __forceinline__ int scan(int v, int *part, int *total, bool *stop = nullptr) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = wave_scan(v);
  if (stop && __ballot(*stop)) x = -1;
  __syncthreads();
  if (lane == 63) part[wave] = x;
  __syncthreads();
  int before = 0, sum = 0, all = 0;
#pragma unroll
  for (int w = 0; w < N / 64; ++w) {
    const int y = part[w];
    if (w < wave) before += y;
    sum += y, all |= y;
  }
  if (stop) *stop = __builtin_amdgcn_readfirstlane(all) < 0;
  *total = __builtin_amdgcn_readfirstlane(sum);
  return before + x - v;
}

// a / b, in 32 bits where they fit (they do but for the longest calls).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}

struct PlanShared {
  int part[16];
  int item, before, most;
};

struct Plan {
  bool descends;       // cu_seqlens does somewhere: nothing is done
  int items, wg;       // items of a head; this workgroup's place in the order of spans
  int64_t per;         // length of a span
  int64_t from, to;    // this workgroup's
  int head, item;      // the (item, head) that `from` lies in
  int64_t base;        // and where that begins
};

// The sequence of item x: the last i with tile_base[i] <= x.
__device__ __forceinline__ int seq_of_item(const int *tile_base, int S, int x) {
  int lo = 0, hi = S - 1;
  while (lo < hi) {
    const int m = (lo + hi + 1) / 2;
    if (tile_base[m] <= x) lo = m;
    else hi = m - 1;
  }
  return lo;
}

// The cost of a block of an item of `rows` rows, and the least span.
struct RowCost {  // every row kernel's unit is the same bytes
  static constexpr int kLead = 1, kMost = 1, kLeast = 1;
  static __device__ __forceinline__ int of(int) { return 1; }
};

template <int N, typename Cost>
__device__ __forceinline__ Plan make_plan(const AttnArgs &a, int BM, int UK, const Batch &batch,
                                          PlanShared *sh) {
  const int tid = threadIdx.x;
  Plan p{};
  for (int i0 = 0; i0 < a.S; i0 += N) {
    const int i = i0 + tid;
    int tiles = 0, total;
    bool down = false;
    if (i < a.S) {
      const int from = a.cu[i], to = a.cu[i + 1];
      down = to < from;
      const int T = (int)a.T, q0 = min(max(from, 0), T), q = min(max(to, q0), T) - q0;
      batch.q0[i] = q0, batch.q[i] = q, batch.n[i] = min(max(a.ctx[i], 0), a.W * a.page_size);
      tiles = (int)((uint32_t)(q * a.group + BM - 1) / (uint32_t)BM);
    }
    const int before = scan<N>(tiles, sh->part, &total, &down);
    if (i < a.S) batch.tile_base[i] = p.items + before;
    p.items += total, p.descends |= down;
  }
  // Sequences that overlap could be more rows than any count here has room for.
  if (p.descends) p.items = 0;
  if (tid == 0) batch.tile_base[a.S] = p.items;
  __syncthreads();
  auto cost_of = [&](int x) {
    if (x >= p.items) return 0;
    const int i = seq_of_item(batch.tile_base, a.S, x), tile = x - batch.tile_base[i];
    const Seq s = batch[i];
    const int nb = blocks_of(keys_of(a, s, tile, BM), UK);
    return nb ? Cost::kLead + nb * Cost::of(min(BM, s.q * a.group - tile * BM)) : 0;
  };
  int sum = 0, cost = 0, before = 0;
  for (int x0 = 0; x0 < p.items; x0 += N) {
    int total;
    cost = cost_of(x0 + tid);
    before = scan<N>(cost, sh->part, &total);
    sum += total;
  }
  p.wg = xcd_contiguous_tile(blockIdx.x, gridDim.x);
  // About as many (item, head)s as workgroups, of about one length: each
  // workgroup takes a whole one, and nothing has to be joined.  What is uneven
  // about them the two workgroups of a CU share, so the second half of an
  // XCD's workgroups takes its items from the far end.  Such are chunks that fill
  // a budget of tokens (2048 of 32 heads fill the grid of 512), of one sequence or
  // of several.  Measured, whole items against equal spans, head_dim 128, us:
  //   2048 tokens behind 6144      273 / 283    2048 behind 30000       1043 / 1110
  //   2 x 1024 behind 2048         119 / 132    4 x 512 behind 2048      107 / 126
  //   8 x 256 behind 2048          101 / 116    16 x 128 behind 2048     101 / 99
  // Below 31 / 32 of the grid the workgroups without an item cost one long
  // sequence more than that (1984 tokens behind 6144, 496 items: 272 / 275; 1920:
  // 273 / 265; 1792: 271 / 249), where several short ones would gain further
  // (4 x 448 behind 2048: 105 / 117).
  const int pairs = p.items * a.KV, grid = (int)gridDim.x;
  if (p.items <= N && pairs <= grid && 32 * (int64_t)pairs >= 31 * (int64_t)grid) {
    if (tid == 0) sh->most = 0;
    __syncthreads();
    if (cost) atomicMax(&sh->most, cost);
    __syncthreads();
    if ((int64_t)sh->most * p.items <= (int64_t)sum + sum / 4) {
      const int xcd = blockIdx.x & 7, each = grid / 8, i = blockIdx.x >> 3;
      if (grid % 16 == 0 && i >= each / 2) p.wg = xcd * each + each / 2 + each - 1 - i;
      if (p.wg >= pairs) return p;
      p.head = p.wg / p.items, p.item = p.wg - p.head * p.items;
      if (p.item == tid) sh->before = before, sh->item = cost;
      __syncthreads();
      const int length = __builtin_amdgcn_readfirstlane(sh->item);
      p.base = p.from = (int64_t)p.head * sum + __builtin_amdgcn_readfirstlane(sh->before);
      p.to = p.from + length, p.per = max(length, 1);
      return p;
    }
  }
  const int64_t all = (int64_t)sum * a.KV;
  // kLeast is no shorter than a block, so that every span inside a long item
  // has the start of one
  static_assert(Cost::kLeast >= Cost::kMost, "a span may hold no block");
  p.per = max(quotient(all + gridDim.x - 1, gridDim.x), (int64_t)Cost::kLeast);
  p.from = p.per * p.wg, p.to = min(p.from + p.per, all);
  if (p.from >= p.to) {  // nothing is left: an empty span at the line's start
    p.from = p.to = 0;
    return p;
  }
  p.head = (int)quotient(p.from, sum);
  const int at = (int)(p.from - (int64_t)p.head * sum);
  if (p.items <= N) {  // the only round's values are still at hand
    if (at >= before && at < before + cost) sh->item = tid, sh->before = before;
  } else {
    int base = 0;
    for (int x0 = 0; base <= at; x0 += N) {
      int total;
      cost = cost_of(x0 + tid);
      before = base + scan<N>(cost, sh->part, &total);
      if (at >= before && at < before + cost) sh->item = x0 + tid, sh->before = before;
      base += total;
    }
  }
  __syncthreads();
  p.item = __builtin_amdgcn_readfirstlane(sh->item);
  p.base = (int64_t)p.head * sum + __builtin_amdgcn_readfirstlane(sh->before);
  return p;
}

// A workgroup's way along its span: for each (item, head) the blocks [bb, bb +
// take) of its nb.
struct Segment {
  int head, tile, seq;
  KeyRange keys;
  int b0, nb, bb, take;  // first block of the sequence, blocks, the span's
  int64_t slot;          // of its partial result
  int64_t last;          // the workgroup that has the item's last block
  bool complete;
};
template <typename Cost>
struct Walk {
  int head, item;
  int64_t base;
  __device__ __forceinline__ explicit Walk(const Plan &p) : head(p.head), item(p.item), base(p.base) {}
  __device__ __forceinline__ bool next(const AttnArgs &a, const Plan &p, const Batch &batch, int BM, int UK,
                                       Segment *g) {
    while (base < p.to) {
      if (item == p.items) ++head, item = 0;
      g->head = head;
      g->seq = __builtin_amdgcn_readfirstlane(seq_of_item(batch.tile_base, a.S, item));
      g->tile = item - __builtin_amdgcn_readfirstlane(batch.tile_base[g->seq]);
      const Seq s = batch.uniform(g->seq);
      g->keys = keys_of(a, s, g->tile, BM);
      g->nb = blocks_of(g->keys, UK), g->b0 = g->keys.begin / UK;
      ++item;
      if (g->nb == 0) continue;
      const int w = Cost::of(min(BM, s.q * a.group - g->tile * BM));
      const int64_t first = base + Cost::kLead, odd = base > p.from;
      // blocks that start in [from, to)
      const int64_t lo = max(p.from - first, (int64_t)0), hi = p.to - first;
      const int b = (int)min(quotient(lo + w - 1, w), (int64_t)g->nb);
      const int e = hi > 0 ? (int)min(quotient(hi + w - 1, w), (int64_t)g->nb) : 0;
      base = first + (int64_t)g->nb * w;
      if (b >= e) continue;
      g->bb = b, g->take = e - b;
      g->slot = 2 * (int64_t)p.wg + odd;
      g->complete = g->take == g->nb;
      g->last = quotient(first + (int64_t)(g->nb - 1) * w, p.per);
      return true;
    }
    return false;
  }
};

// Where the keys of one sequence are: a lane's lookup of its key's page, kept
// as it was loaded (a use right behind the load would wait for everything in
// flight), and the offset of its row of K or V in units of 16 bytes.
struct Pages {
  const int *table;
  int begin, end;  // keys that some row of the item sees
  __device__ __forceinline__ int lookup(const AttnArgs &a, int tok) const {
    return table[tok >= begin && tok < end ? fast_div(tok, a.div_page) : 0];
  }
  __device__ __forceinline__ bool there(const AttnArgs &a, int tok, int page) const {
    return tok >= begin && tok < end && page >= 0 && page < a.pages;
  }
};
__device__ __forceinline__ uint32_t row_offset(const AttnArgs &a, const uint32_t (&ld)[2], int tok, int page) {
  const uint32_t off = tok - fast_div(tok, a.div_page) * a.page_size;
  return (uint32_t)page * ld[0] + off * ld[1];
}

// A weight of zero times an infinity or a NaN is a NaN, so where the rows of an
// item see different keys of a block (an edge of what they see), values that are
// not finite are taken out of it.  If there were any, they are added to what the
// rows that do see them have stored, from memory, at the end of the segment, where
// that costs the kernels' loops no registers.  Whether the item's rows differ, and
// the keys they all see:
struct Shared {
  bool differ;
  int from, to;
  __device__ __forceinline__ Shared(const AttnArgs &a, const Seq &s, int tile, int BM) {
    const int a0 = (int)fast_div((uint32_t)tile * BM, a.div_group);
    const int a1 = min((int)fast_div((uint32_t)tile * BM + BM - 1, a.div_group), s.q - 1);
    differ = a.causal && a1 > a0;
    to = s.n - s.q + a0 + 1;
    from = a.window ? (int)max((int64_t)s.n - s.q + a1 + 1 - a.window, (int64_t)0) : 0;
  }
  __device__ __forceinline__ bool edge(int k0, int n) const { return differ && (k0 + n > to || k0 < from); }
};

// What a workgroup leaves about the (item, head) that it began and did not
// finish (rows = 0: none): the partial results are in slots `slot` and 2 * w for
// each workgroup w after it up to `last`.
struct Split {
  int64_t slot, last;
  int row0, rows, head;  // its rows of that cache head, from row0 of the sequence on
  int q0;                // the sequence's first row of the batch
};

// Zeros for the rows that see no key: those of items without units and those
// of no sequence.
template <int N>
__device__ __forceinline__ void zero_rows(const AttnArgs &a, const Plan &p, int BM, int UK,
                                          const Batch &batch) {
  const int esize = a.dtype == ZT_DT_F32 ? 4 : 2, chunks = a.D * esize / 16;  // of 16 bytes a head
  char *out = static_cast<char *>(a.out);
  for (int x = blockIdx.x; x < p.items; x += gridDim.x) {
    const int i = seq_of_item(batch.tile_base, a.S, x), tile = x - batch.tile_base[i];
    const Seq s = batch[i];
    if (blocks_of(keys_of(a, s, tile, BM), UK)) continue;
    // the item's rows, of every cache head
    const int r0 = tile * BM, rows = min(BM, s.q * a.group - r0);
    const int64_t n = (int64_t)rows * a.KV * chunks;
    for (int64_t e = threadIdx.x; e < n; e += N) {
      const int c = (int)(e % chunks), y = (int)(e / chunks), h = y / rows, row = r0 + y - h * rows;
      const int t = (int)fast_div(row, a.div_group);
      const int64_t at = ((int64_t)(s.q0 + t) * a.H + h * a.group + row - t * a.group) * chunks + c;
      reinterpret_cast<u32x4_t *>(out)[at] = u32x4_t{0, 0, 0, 0};
    }
  }
  const bool none = a.S == 0 || p.descends;
  const int64_t T = a.T, lo = none ? T : batch.q0[0], hi = none ? T : batch.q0[a.S - 1] + batch.q[a.S - 1];
  const int64_t row = (int64_t)a.H * chunks, n = (lo + T - hi) * row;
  for (int64_t e = (int64_t)blockIdx.x * N + threadIdx.x; e < n; e += (int64_t)gridDim.x * N)
    reinterpret_cast<u32x4_t *>(out)[e < lo * row ? e : e - lo * row + hi * row] = u32x4_t{0, 0, 0, 0};
}

// Adds the values that edges left out of the segment's keys [k0, kend), in blocks
// of n, to four numbers that one row has stored (`at` in its item).
template <typename T>
__device__ __forceinline__ void add_edges(const AttnArgs &a, const Segment &seg, const Seq &s, int BM, int at,
                                          int col, const Shared &shared, const Pages &pages, const char *vbase,
                                          int k0, int kend, int n) {
  const int row = seg.tile * BM + at, token = (int)fast_div(row, a.div_group);
  if (token >= s.q) return;
  const int pos = s.n - s.q + token, hi = a.causal ? pos + 1 : s.n;
  const int lo = a.causal && a.window ? (int)max((int64_t)pos + 1 - a.window, (int64_t)0) : 0;
  for (int k = k0; k < kend; k += n) {
    if (!shared.edge(k, n)) continue;
    for (int key = max(k, lo); key < min(k + n, hi); ++key) {
      const int page = pages.lookup(a, key);
      if (!pages.there(a, key, page)) continue;
      const T *v = reinterpret_cast<const T *>(vbase + (uint64_t)row_offset(a, a.v_row, key, page) * 16) + col;
#pragma unroll 1
      for (int e = 0; e < 4; ++e) {
        float x;
        if constexpr (sizeof(T) == 2) x = bf16_bits_to_f32(v[e]);
        else x = v[e];
        if (fabsf(x) < INFINITY) continue;
        float *part = a.part_o + (seg.slot * BM + at) * a.D + col + e;
        T *out = static_cast<T *>(a.out) +
            ((int64_t)(s.q0 + token) * a.H + seg.head * a.group + row - token * a.group) * a.D + col + e;
        if (!seg.complete) *part += x;
        else if constexpr (sizeof(T) == 2) *out = (T)f32_to_bf16_bits(bf16_bits_to_f32(*out) + x);
        else *out += x;
      }
    }
  }
}

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32); }

// The 32 rows of a wave of the tile kernels, as one lane sees them: its row is
// n = lane % 32, and of 32 scores it holds those of keys 8 (i / 4) + 4 half +
// i % 4, half = lane / 32.
struct Rows32 {
  int row, token;  // of the sequence's rows and new tokens
  bool live;
  int lo, hi;      // the keys it sees
  bool any;        // over the wave's rows; live ones come first, and their
  int hi_min, lo_min, hi_max, lo_max;  // tokens ascend with the rows

  __device__ __forceinline__ Rows32(const AttnArgs &a, const Seq &s, int row) : row(row) {
    token = (int)fast_div(row, a.div_group);
    live = token < s.q;
    const int pos = s.n - s.q + token;
    hi = !live ? INT32_MAX : a.causal ? pos + 1 : s.n;
    lo = live && a.causal && a.window ? (int)max((int64_t)pos + 1 - a.window, (int64_t)0) : 0;
    const uint32_t alive = (uint32_t)__ballot(live);
    any = alive != 0;
    const int last = 31 - __builtin_clz(alive | 1u);
    hi_min = __builtin_amdgcn_readlane(hi, 0), lo_min = __builtin_amdgcn_readlane(lo, 0);
    hi_max = __builtin_amdgcn_readlane(hi, last), lo_max = __builtin_amdgcn_readlane(lo, last);
  }
  __device__ __forceinline__ bool see(int k0, int n) const { return any && k0 < hi_max && k0 + n > lo_min; }
  __device__ __forceinline__ bool see_all(int k0, int n) const { return k0 + n <= hi_min && k0 >= lo_max; }
  // whether the row sees a key of `bad`, bit i being key k0 + i
  __device__ __forceinline__ bool sees_of(uint64_t bad, int k0) const {
    const int from = min(max(lo - k0, 0), 64), to = min(max(hi - k0, 0), 64);
    const uint64_t below = from >= 64 ? ~0ull : (1ull << from) - 1, up = to >= 64 ? ~0ull : (1ull << to) - 1;
    return live && (bad & up & ~below) != 0;
  }
  // scores of keys k0 .. k0 + 31 that the row does not see, or that are not there
  __device__ __forceinline__ void mask(f32x16_t &sc, int k0, uint32_t there) const {
    const int from = min(max(lo - k0, 0), 32), to = min(max(hi - k0, 0), 32);
    const uint64_t range = (1ull << to) - (1ull << min(from, to));
    const uint32_t seen = ((uint32_t)range & there) >> (4 * ((threadIdx.x >> 5) & 1));
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (!(seen & (1u << (8 * (e / 4) + e % 4)))) sc[e] = -INFINITY;
  }
  // Outputs, or a part of them: the lane holds columns 32 d + 8 k + 4 half .. + 3.
  template <typename T, int DT>
  __device__ __forceinline__ void store(const AttnArgs &a, const Segment &seg, const Seq &s, int BM, int at,
                                        const f32x16_t (&o)[DT], float m, float l) const {
    if (!live) return;
    const int half = (threadIdx.x >> 5) & 1;
    const int64_t pr = seg.slot * BM + at;
    const int64_t to =
        ((int64_t)(s.q0 + token) * a.H + seg.head * a.group + row - token * a.group) * a.D;
    const float r = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int col = 32 * d + 8 * k + 4 * half;
        const f32x4_t y = {o[d][4 * k], o[d][4 * k + 1], o[d][4 * k + 2], o[d][4 * k + 3]};
        if (col >= a.D) continue;
        if (seg.complete) store_out<T>(a.out, to + col, y, r);
        else *reinterpret_cast<f32x4_t *>(a.part_o + pr * a.D + col) = y;
      }
    if (!seg.complete && half == 0) a.part_ml[2 * pr] = m, a.part_ml[2 * pr + 1] = l;
  }
};

// The tile kernel (paged_attn_tile.hip): its rows per item and workgroups.
int tile_rows(const AttnArgs &a);
int tile_grid(const AttnArgs &a);
hipError_t launch_tiles(const AttnArgs &a, int grid, hipStream_t s);
hipError_t launch_split(const AttnArgs &a, int grid, hipStream_t s);  // paged_attn_split.hip
constexpr int kTileCostLead = 15, kTileCostMost = 6;  // the most of TileCost

}  // namespace zt
