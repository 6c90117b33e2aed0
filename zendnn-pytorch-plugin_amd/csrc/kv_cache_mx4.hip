// Writing and reading a key / value cache held in 4 bits, for gfx950.  The
// format is described in mx4.hpp.
//
// Both kernels move bytes: they are bound by HBM where the operands are large and
// by their launch where they are small.  Slots and positions come from the device
// and are checked before they are used as an address.
#include "mx4.hpp"

namespace zt {

namespace {

constexpr int kThreads = 256;

// A slot's page, and its place there.
__device__ __forceinline__ int64_t page_of(int64_t slot, int page_size, FastDiv d, int64_t *off) {
  const int64_t page = slot <= INT32_MAX ? (int64_t)fast_div((uint32_t)slot, d) : slot / page_size;
  *off = slot - page * page_size;
  return page;
}

// Eight consecutive elements as floats.
template <typename T, bool WIDE>
__device__ __forceinline__ void load8(const T *p, float (&f)[8]) {
  if constexpr (sizeof(T) == 2 && WIDE) {
    const u32x4_t v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(v[i] << 16), f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
  } else if constexpr (WIDE) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f32x4_t v = __builtin_nontemporal_load(reinterpret_cast<const f32x4_t *>(p) + j);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[4 * j + i] = v[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if constexpr (sizeof(T) == 2) f[i] = bf16_bits_to_f32(p[i]);
      else f[i] = p[i];
  }
}

// y in fp32, with the last bit set where that is not exact: such a number lies on
// the same side of every border between two codes (and of 1.75 times a power of
// two) as y, because those have no digits that far down.
__device__ __forceinline__ float sticky(double y) {
  const float f = (float)y;
  const double back = f;
  uint32_t b = __float_as_uint(f);
  if (back != y) b = (fabs(back) > fabs(y) ? b - 1 : b) | 1u;
  return __uint_as_float(b);
}
__device__ __forceinline__ float in_fp32(double y) { return sticky(y); }
__device__ __forceinline__ float in_fp32(float y) { return y; }

// Eight consecutive cosines or sines; ALIGNED: on 16 bytes.
template <bool ALIGNED>
__device__ __forceinline__ void factors(const float *p, bool inside, float (&f)[8]) {
  if (!inside) {  // no such position: NaN, so that it does not pass unseen
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(0x7fc00000u);
  } else if constexpr (ALIGNED) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f32x4_t v = reinterpret_cast<const f32x4_t *>(p)[j];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[4 * j + i] = v[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = p[i];
  }
}

// How a thread takes a row: eight elements at any place, one by one; eight whose
// loads are of 16 bytes and which no border of a half divides; or eight of each half,
// with their pairs' frequencies in between.
enum Mode { kAny, kWide, kPair };

// Elements e0 .. e0 + 7 of a row turned to position p: of a pair (a, b) of
// frequency i, a cos - b sin or b cos + a sin.  The pairs are (x[i], x[R / 2 + i])
// or, interleaved, (x[2 i], x[2 i + 1]); what is past R is as it was, and so is
// the row of a negative position.  A thread computes its eight elements only, and
// reads the pairs' other ones beside them, which a neighbour has read.
template <typename A, typename T, bool IL, bool WIDE>
__device__ __forceinline__ void rotated(const Mx4AppendArgs &a, const T *src, int e0, int64_t p, float (&y)[8]) {
  float x[8];
  load8<T, WIDE>(src + e0, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = x[i];
  const int R = a.R, half = R / 2;
  if (p < 0 || e0 >= R) return;
  const bool inside = p < a.length;
  const float *row = a.table + p * a.table_ld;
  const float nan = __uint_as_float(0x7fc00000u);
  if constexpr (IL) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const int f = (e0 + i) / 2;
      if (!WIDE && f >= half) continue;
      const A c = inside ? row[f] : nan, s = inside ? row[half + f] : nan;
      y[i] = in_fp32((A)x[i] * c - (A)x[i + 1] * s), y[i + 1] = in_fp32((A)x[i + 1] * c + (A)x[i] * s);
    }
  } else if constexpr (WIDE) {
    const bool second = e0 >= half;
    const int f = second ? e0 - half : e0;
    float z[8], c[8], s[8];
    load8<T, WIDE>(src + (second ? f : e0 + half), z);
    factors<false>(row + f, inside, c);
    factors<false>(row + half + f, inside, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const A other = (A)z[i] * (A)s[i];
      y[i] = in_fp32((A)x[i] * (A)c[i] + (second ? other : -other));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = e0 + i;
      if (e >= R) break;
      const bool second = e >= half;
      const int f = second ? e - half : e;
      float z;
      if constexpr (sizeof(T) == 2) z = bf16_bits_to_f32(src[second ? f : e + half]);
      else z = src[second ? f : e + half];
      const A c = inside ? row[f] : nan, s = inside ? row[half + f] : nan;
      const A other = (A)z * s;
      y[i] = in_fp32((A)x[i] * c + (second ? other : -other));
    }
  }
}

// Elements e0 .. e0 + 7 of both halves.
template <typename A, typename T>
__device__ __forceinline__ void rotated_pair(const Mx4AppendArgs &a, const T *src, int e0, int64_t p, float (&y0)[8],
                                             float (&y1)[8]) {
  const int half = a.R / 2;
  float x0[8], x1[8], c[8], s[8];
  load8<T, true>(src + e0, x0);
  load8<T, true>(src + half + e0, x1);
  const float *row = a.table + p * a.table_ld + e0;
  factors<true>(row, p >= 0 && p < a.length, c);
  factors<true>(row + half, p >= 0 && p < a.length, s);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y0[i] = p < 0 ? x0[i] : in_fp32((A)x0[i] * (A)c[i] - (A)x1[i] * (A)s[i]);
    y1[i] = p < 0 ? x1[i] : in_fp32((A)x1[i] * (A)c[i] + (A)x0[i] * (A)s[i]);
  }
}

template <typename T, bool WIDE>
__device__ __forceinline__ void store8(T *to, const float (&y)[8]) {
  if constexpr (!WIDE) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if constexpr (sizeof(T) == 2) to[i] = (T)f32_to_bf16_bits(y[i]);
      else to[i] = y[i];
  } else if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<u32x4_t *>(to) = u32x4_t{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]),
                                               pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7])};
  } else {
    *reinterpret_cast<f32x4_t *>(to) = f32x4_t{y[0], y[1], y[2], y[3]};
    *reinterpret_cast<f32x4_t *>(to + 4) = f32x4_t{y[4], y[5], y[6], y[7]};
  }
}

// Four threads' 32 elements as a block: the w-th eight of the row.
__device__ __forceinline__ void store_block(const float (&x)[8], uint8_t *codes, uint8_t *scales, int w) {
  int amax = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max(amax, (int)(__float_as_uint(x[i]) & 0x7fffffffu));
  amax = max(amax, __builtin_amdgcn_mov_dpp(amax, 0xb1, 0xf, 0xf, true));  // lanes 1 0 3 2 of four
  amax = max(amax, __builtin_amdgcn_mov_dpp(amax, 0x4e, 0xf, 0xf, true));  // lanes 2 3 0 1
  const uint32_t byte = mx_byte((uint32_t)amax);
  *reinterpret_cast<uint32_t *>(codes + 4 * w) = byte == kMxNan ? 0u : mx_codes(x, mx_scale(byte));
  if ((w & 3) == 0) scales[w / 4] = (uint8_t)byte;
}

// One thread takes eight elements of a token's row of a query, key or value head,
// or eight of each half of it, and four threads a block of 32, whose largest
// magnitude they find among themselves.  Queries are turned in fp32 and rounded
// once.  Keys are turned in 64 bits, where the products are exact and their sum has 53
// digits, so that a code next to a border does not depend on an order of roundings;
// nothing else is rounded between that and the code.
//
// Measured (bf16, 32 + 8 + 8 heads of 128): 8191 tokens 36-38 us, 4.7 TB/s; 93 with eight
// elements a thread and the table's numbers one by one (each is read by 48 rows), 51
// before the doubles were rounded one at a time (46 registers for 101).  8 tokens 4 us.
template <typename T, bool IL, Mode MODE>
__global__ __launch_bounds__(kThreads) void append_mx4_kernel(Mx4AppendArgs a) {
  constexpr bool WIDE = MODE != kAny;
  const uint32_t idx = blockIdx.x * kThreads + threadIdx.x;
  const int64_t t = fast_div(idx, a.div_units);
  if (t >= a.T) return;
  int u = (int)(idx - (uint32_t)t * a.units);
  const int k_threads = a.KV * a.k_units, v_threads = a.KV * 4 * a.NB;
  const int pairs = MODE == kPair ? a.R / 16 : 0;  // threads of a row with eight elements of each half
  if (u >= k_threads + v_threads) {
    u -= k_threads + v_threads;
    const int h = (int)fast_div(u, a.div_q), w = u - h * a.q_units;
    if (h >= a.H) return;
    const T *src = static_cast<const T *>(a.q) + t * a.q_ld[0] + h * a.q_ld[1];
    T *to = static_cast<T *>(a.q_out) + (t * a.H + h) * a.D;
    float y[8];
    if (w < pairs) {
      float z[8];
      rotated_pair<float, T>(a, src, 8 * w, a.pos[t], y, z);
      store8<T, WIDE>(to + 8 * w, y);
      store8<T, WIDE>(to + 8 * (w + pairs), z);
    } else {
      rotated<float, T, IL, WIDE>(a, src, 8 * (w + pairs), a.pos[t], y);
      store8<T, WIDE>(to + 8 * (w + pairs), y);
    }
    return;
  }
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= a.pages * a.page_size) return;  // a padding token, for the whole block
  int64_t off;
  const int64_t page = page_of(slot, a.page_size, a.div_page, &off);
  const bool value = u >= k_threads;
  if (value) u -= k_threads;
  const int h = (int)fast_div(u, value ? a.div_v : a.div_k);
  int w = u - h * (value ? 4 * a.NB : a.k_units);  // the row's w-th eight elements
  const Mx4Rows &to = value ? a.values : a.keys;
  uint8_t *codes = to.codes + page * to.ld[0] + h * to.ld[1] + off * to.ld[2];
  uint8_t *scales = to.scales + page * to.sc_ld[0] + h * to.sc_ld[1] + off * to.sc_ld[2];
  const T *k = static_cast<const T *>(a.k) + t * a.k_ld[0] + h * a.k_ld[1];
  float x[8];
  if (!value && w < pairs) {
    float z[8];
    rotated_pair<double, T>(a, k, 8 * w, a.pos[t], x, z);
    store_block(x, codes, scales, w);
    store_block(z, codes, scales, w + pairs);
    return;
  }
  if (!value) w += pairs;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 0.f;
  if (8 * w < a.D) {
    if (value) load8<T, WIDE>(static_cast<const T *>(a.v) + t * a.v_ld[0] + h * a.v_ld[1] + 8 * w, x);
    else rotated<double, T, IL, WIDE>(a, k, 8 * w, a.pos[t], x);
  }
  store_block(x, codes, scales, w);
}

// One thread gives eight elements of a token's key and of its value.  Bound by HBM,
// four times as much out as in (65536 tokens of 8 heads of 128: 54 us, 6.3 TB/s).
template <typename T>
__global__ __launch_bounds__(kThreads) void read_mx4_kernel(Mx4ReadArgs a) {
  const uint32_t idx = blockIdx.x * kThreads + threadIdx.x;
  const int64_t t = fast_div(idx, a.div_units);
  if (t >= a.n) return;
  const int u = (int)(idx - (uint32_t)t * a.units);
  const int h = (int)fast_div(u, a.div_row), w = u - h * (a.D / 8);
  const int64_t slot = a.slots[t];
  uint32_t codes[2] = {0u, 0u}, byte[2] = {0u, 0u};
  if (slot >= 0 && slot < a.pages * a.page_size) {
    int64_t off;
    const int64_t page = page_of(slot, a.page_size, a.div_page, &off);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const Mx4Rows &r = i ? a.values : a.keys;
      codes[i] = *reinterpret_cast<const uint32_t *>(r.codes + page * r.ld[0] + h * r.ld[1] + off * r.ld[2] + 4 * w);
      byte[i] = r.scales[page * r.sc_ld[0] + h * r.sc_ld[1] + off * r.sc_ld[2] + w / 4];
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x4_t y = mx_values(codes[i], mx_scale(byte[i]));
    T *to = static_cast<T *>(i ? a.v_out : a.k_out) + (t * a.KV + h) * a.D + 8 * w;
    if constexpr (sizeof(T) == 2) {
      __builtin_nontemporal_store(y, reinterpret_cast<u32x4_t *>(to));
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const u32x4_t z = {y[2 * j] << 16, y[2 * j] & 0xffff0000u, y[2 * j + 1] << 16, y[2 * j + 1] & 0xffff0000u};
        __builtin_nontemporal_store(z, reinterpret_cast<u32x4_t *>(to) + j);
      }
    }
  }
}

// Threads of a launch, at most: a thread's number is divided in 31 bits.
constexpr int64_t kMostThreads = 1 << 30;

}  // namespace

hipError_t launch_append_mx4(Mx4AppendArgs a, int dtype, bool wide, hipStream_t s) {
  // halves of whole blocks, and a table on 16 bytes
  const bool pair = wide && !a.interleaved && a.R % 64 == 0 && a.table_ld % 4 == 0 &&
                    reinterpret_cast<uintptr_t>(a.table) % 16 == 0;
  const int saved = pair ? a.R / 16 : 0;  // threads of a row that another one's second half saves
  a.q_units = a.D / 8 - saved, a.k_units = 4 * a.NB - saved;
  // whole fours of threads, which share a block
  a.units = a.KV * (a.k_units + 4 * a.NB) + (a.H * a.q_units + 3) / 4 * 4;
  a.div_units = make_div(a.units), a.div_k = make_div(a.k_units), a.div_v = make_div(4 * a.NB), a.div_q = make_div(a.q_units);
  a.div_page = make_div(a.page_size);
  const int64_t T = a.T, most = std::max<int64_t>(kMostThreads / a.units, 1), es = dtype == ZT_DT_F32 ? 4 : 2;
  const Mx4AppendArgs all = a;
  for (int64_t t0 = 0; t0 < T; t0 += most) {
    a = all;
    a.T = std::min(most, T - t0);
    a.q = static_cast<const char *>(all.q) + t0 * a.q_ld[0] * es;
    a.k = static_cast<const char *>(all.k) + t0 * a.k_ld[0] * es;
    a.v = static_cast<const char *>(all.v) + t0 * a.v_ld[0] * es;
    a.q_out = static_cast<char *>(all.q_out) + t0 * a.H * a.D * es;
    a.pos = all.pos + t0, a.slots = all.slots + t0;
    const int grid = (int)((a.T * a.units + kThreads - 1) / kThreads);
    auto go = [&](auto kernel) { kernel<<<grid, kThreads, 0, s>>>(a); };
    if (dtype == ZT_DT_BF16) {
      if (pair) go(append_mx4_kernel<uint16_t, false, kPair>);
      else if (wide) a.interleaved ? go(append_mx4_kernel<uint16_t, true, kWide>) : go(append_mx4_kernel<uint16_t, false, kWide>);
      else a.interleaved ? go(append_mx4_kernel<uint16_t, true, kAny>) : go(append_mx4_kernel<uint16_t, false, kAny>);
    } else {
      if (pair) go(append_mx4_kernel<float, false, kPair>);
      else if (wide) a.interleaved ? go(append_mx4_kernel<float, true, kWide>) : go(append_mx4_kernel<float, false, kWide>);
      else a.interleaved ? go(append_mx4_kernel<float, true, kAny>) : go(append_mx4_kernel<float, false, kAny>);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_read_mx4(Mx4ReadArgs a, int dtype, hipStream_t s) {
  a.units = a.KV * (a.D / 8);
  a.div_units = make_div(a.units), a.div_row = make_div(a.D / 8), a.div_page = make_div(a.page_size);
  const int64_t n = a.n, most = std::max<int64_t>(kMostThreads / a.units, 1), es = dtype == ZT_DT_F32 ? 4 : 2;
  const Mx4ReadArgs all = a;
  for (int64_t t0 = 0; t0 < n; t0 += most) {
    a = all;
    a.n = std::min(most, n - t0);
    a.slots = all.slots + t0;
    a.k_out = static_cast<char *>(all.k_out) + t0 * a.KV * a.D * es;
    a.v_out = static_cast<char *>(all.v_out) + t0 * a.KV * a.D * es;
    const int grid = (int)((a.n * a.units + kThreads - 1) / kThreads);
    if (dtype == ZT_DT_BF16) read_mx4_kernel<uint16_t><<<grid, kThreads, 0, s>>>(a);
    else read_mx4_kernel<float><<<grid, kThreads, 0, s>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace zt
