// Pages of a cache held in 4 bits: the format and its layout.
//
// A head's vector is held in groups of 64 values.  A group has a bf16 scale s and a bf16 minimum m, and a code c of 0 .. 15 a value, which stands for m + s c:
//   m = the largest bf16 <= min x,   s = the least bf16 >= 0 with 15 s >= max x - m,   c = the integer nearest to (x - m) / s, ties to even (0 where s = 0)
// so that no value lies outside the codes' range and a value is off by at most s / 2.  A group with a NaN, or a magnitude above 2^126, stands for NaN.
// 4.5 bits a value: groups of 32 would hold normal values 13 % closer (0.080 against 0.092 of their deviation) for 11 % more bytes, which is
// what attention over the cache is bound by.
//
// A page has 16 tokens; the record of a page and head has 18 D bytes, one bulk copy: codes of K (8 D), parameters of K (D), codes of V, parameters of V.
// Codes lie as m16n8k16 operand fragments: word j of the 16 bytes of (group, lane) is the four registers of one product, register r in the nibbles r and r + 4.
//   K: rows are tokens.  Byte [g][t][c][j][b] has token t + 8 (b & 1), dim 64 g + 16 j + 2 c + (b >> 1) in its low nibble, the dim eight behind it in its high one.
//   V: rows are dims.    Byte [g][i][c][j][b] has token 2 c + (b >> 1) + 8 (b & 1), dim 64 g + 16 j + i in its low nibble, the dim eight behind it in its high one.
// A byte has one token's codes alone, so that tokens are written without reading what is there.  K's word is V's word transposed as an 8 x 8 matrix of
// pairs of bytes (movmatrix).  Parameters: [t][half][group][s, m] for token t + 8 half.
#pragma once

#include "common.cuh"

#include <cuda_fp16.h>

namespace mfq {

constexpr float kKv4Most = 8.507059173023462e37f;  // 2^126

struct Kv4Group {
  float s, m;
};

__device__ __forceinline__ float bf16_down(float x) {  // the largest bf16 <= x
  uint32_t b = __float_as_uint(x);
  if (int(b) < 0) b += 0xffffu;
  return __uint_as_float(b & 0xffff0000u);
}
// From the least and the greatest value, both NaN if one value is.  s is the least bf16 that reaches d = max - m fifteenfold: 15 s has 12 bits and is exact, so
// it reaches d if it reaches d rounded up to 24.  The search begins at d / 15 or less and ends after two steps at most.
__device__ __forceinline__ Kv4Group kv4_group(float least, float most) {
  if (!(least >= -kKv4Most && most <= kKv4Most)) return {__uint_as_float(0x7fc00000u), __uint_as_float(0x7fc00000u)};
  const float m = bf16_down(least) + 0.f;  // no negative zeros
  const float d = __fsub_ru(most, m) + 0.f;
  uint32_t s = __float_as_uint(__fmul_rd(d, 0.06666666f)) & 0xffff0000u;  // 1 / 15 rounded down
#pragma unroll
  for (int i = 0; i < 2; ++i) s += 15.f * __uint_as_float(s) < d ? 0x10000u : 0u;
  return {__uint_as_float(s), m};
}
__device__ __forceinline__ uint32_t kv4_params(Kv4Group g) { return __float_as_uint(g.s) >> 16 | __float_as_uint(g.m); }

// Whether x - m is above (1), at (0) or below (-1) t, without rounding: h = x - m as rounded decides unless it is t itself, then what was lost does.
__device__ __forceinline__ int kv4_side(float x, float m, float t) {
  const float h = x - m;
  if (h != t) return h > t ? 1 : -1;
  const float b = h - x, lost = (x - (h - b)) + (-m - b);
  return lost > 0.f ? 1 : (lost < 0.f ? -1 : 0);
}
// The nearest code; s (c +- 1/2) has 13 bits and is exact.
static __device__ __noinline__ uint32_t kv4_code(float x, Kv4Group g) {
  if (!(g.s > 0.f)) return 0;
  int c = int(fminf(rintf((x - g.m) / g.s), 15.f));
  const int down = kv4_side(x, g.m, g.s * (float(c) - 0.5f));
  if (down < 0 || (down == 0 && (c & 1))) --c;
  const int up = kv4_side(x, g.m, g.s * (float(c) + 0.5f));
  if (up > 0 || (up == 0 && (c & 1))) ++c;
  return uint32_t(min(max(c, 0), 15));
}

// Where token t (0 .. 15) has the codes of dims 64 g + 16 j + i and the one eight behind it, in K's or V's codes of a record
__host__ __device__ __forceinline__ int kv4_k_byte(int t, int g, int j, int i) { return 512 * g + 64 * (t & 7) + 16 * (i >> 1) + 4 * j + 2 * (i & 1) + (t >> 3); }
__host__ __device__ __forceinline__ int kv4_v_byte(int t, int g, int j, int i) { return 512 * g + 64 * i + 16 * ((t & 7) >> 1) + 4 * j + 2 * (t & 1) + (t >> 3); }
// ... and, in bytes, its parameters of group 0
template <int D>
__host__ __device__ __forceinline__ int kv4_param_byte(int t) { return ((t & 7) * 2 + (t >> 3)) * (D / 16); }

}  // namespace mfq
