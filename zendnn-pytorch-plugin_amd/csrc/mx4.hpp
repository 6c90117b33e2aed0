// A key / value cache held in 4 bits (MXFP4): the format, and the launch
// interface of its kernels (kv_cache_mx4.hip, paged_attn_mx4.hip).
//
// A head row is cut into blocks of 32 elements, the last one filled with zeros.
// A block has a scale 2^E, kept as the byte E + 127, and 32 codes of 4 bits, the
// element of even index in a byte's low half: bit 3 is the sign, the others name
// one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  E is such that 3.5 <= amax / 2^E < 7 for the
// block's largest magnitude (a number is off by one scale at most: from 7 on the next
// E's codes are nearer), held to -125 .. 125: every value then is a normal bf16
// number, exactly (and the largest fp32 number, of nearly 8 scales, becomes 6).  A code is the
// nearest one, of two equally near ones the even one.  A block with an infinity or
// a NaN has the byte 255 and codes of 0.  Read, 255 stands for NaN throughout, and
// so do 253 and 254, with which some codes' values would be past bf16's largest.
//
// gfx950 has all of it in instructions: v_cvt_scalef32_pk_fp4_f32 rounds two
// numbers to codes like that, v_cvt_scalef32_pk_bf16_fp4 gives the values of two
// codes, and gives NaN for the byte 255 as an exponent.
#pragma once

#include "zt_cache.hpp"

namespace zt {

constexpr int kMxBlock = 32;   // elements that share a scale
constexpr uint32_t kMxNan = 255, kMxLast = 252;  // from kMxLast + 1 on a byte is NaN

// The scale byte of a block with this largest magnitude (fp32 bits without sign).
// A quarter added to the fraction carries into the exponent from 1.75 on.
__device__ __forceinline__ uint32_t mx_byte(uint32_t amax) {
  if (amax >= 0x7f800000u) return kMxNan;
  const int field = (int)((amax + 0x00200000u) >> 23);
  return (uint32_t)(min(max(field, 4), 254) - 2);
}
__device__ __forceinline__ float mx_scale(uint32_t byte) {
  return __uint_as_float((byte > kMxLast ? kMxNan : byte) << 23);
}

// Whether one of a word's four bytes is kMxLast or past it.
__device__ __forceinline__ bool mx_some_past(uint32_t w) {
  const uint32_t y = ~w & 0xfcfcfcfcu;  // such a byte is 0 here
  return ((y - 0x01010101u) & ~y & 0x80808080u) != 0;
}

// Eight numbers as codes, the first in the lowest bits.
__device__ __forceinline__ uint32_t mx_codes(const float (&x)[8], float scale) {
  uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
}
// Eight codes' values, as four pairs of bf16.
__device__ __forceinline__ u32x4_t mx_values(uint32_t w, float scale) {
  u32x4_t y;
  y[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
  y[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
  y[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
  y[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
  return y;
}

// The upper 16 bits of two numbers, as a pair of bf16, and of one: the first of the
// bf16 parts that an fp32 number is cut into.
__device__ __forceinline__ uint32_t tops(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
__device__ __forceinline__ float top(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

// Codes and scales of keys or values: strides of page, head and token in bytes.
struct Mx4Rows {
  uint8_t *codes, *scales;
  int64_t ld[3], sc_ld[3];
};

struct Mx4AppendArgs {
  const void *q, *k, *v;              // [T, H | KV | KV, D], unit last stride
  int64_t q_ld[2], k_ld[2], v_ld[2];  // token and head strides, elements
  void *q_out;                        // [T, H, D]
  Mx4Rows keys, values;
  const int64_t *pos, *slots;
  const float *table;  // [length, R]: cos, then sin
  int64_t length, table_ld, pages, T;
  int H, KV, D, R, NB, page_size;
  bool interleaved;
  // set by launch_append_mx4: threads of a query's and a key's row, and of a token
  int q_units, k_units, units;
  FastDiv div_units, div_k, div_v, div_q, div_page;
};
hipError_t launch_append_mx4(Mx4AppendArgs a, int dtype, bool wide, hipStream_t s);

struct Mx4ReadArgs {
  Mx4Rows keys, values;
  const int64_t *slots;
  int64_t n, pages;
  int KV, D, page_size;
  void *k_out, *v_out;  // [n, KV, D]
  int units;            // threads of a token, set by launch_read_mx4
  FastDiv div_units, div_row, div_page;
};
hipError_t launch_read_mx4(Mx4ReadArgs a, int dtype, hipStream_t s);

// k, v and their strides of AttnArgs are the codes' (k_row and v_row in 16 bytes).
struct Mx4AttnArgs : AttnArgs {
  const uint8_t *k_sc, *v_sc;
  int64_t k_sc_ld[3], v_sc_ld[3];
  int NB;  // blocks of a row
  // Set by launch_paged_attn_mx4.  Most caches are near: keys and values are laid out
  // alike (strides of page and token in bytes, of codes and of scales), within 2^32
  // bytes of the first, by strides and numbers of 24 bits, which multiply in one
  // full-rate instruction.  words: a row's scales are whole aligned words, or a half.
  bool near, words;
  uint32_t ld[2], sc_ld[2];
  int step_off;  // a tile's length less its whole pages
};
// The tile kernel (paged_attn_mx4_tile.hip): its rows per item and workgroups.
int mx4_tile_rows();
int mx4_tile_grid(const Mx4AttnArgs &a);
hipError_t launch_mx4_tiles(const Mx4AttnArgs &a, int grid, hipStream_t s);
bool paged_attn_mx4_countable(const Mx4AttnArgs &a);
size_t paged_attn_mx4_workspace(const Mx4AttnArgs &a);
hipError_t launch_paged_attn_mx4(Mx4AttnArgs a, void *workspace, hipStream_t s);

}  // namespace zt
