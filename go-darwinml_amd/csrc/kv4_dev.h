// The 4-bit form of a key-value cache's rows: E2M1 codes, two to a byte, and a power of two
// for each 32 values (the Open Compute Project's MX format of 4 bits).
//
//   value = +-{0, 1/2, 1, 3/2, 2, 3, 4, 6}[code & 7] * 2^(scale - 127),  scale 255: NaN
//
// A byte holds value 2i in its low half and 2i + 1 in its high one.  gfx950 converts both
// ways in one instruction a pair, the scale as the exponent of an fp32 operand.
#pragma once

#include "common.h"

namespace ghip {
namespace kv4 {

constexpr int kGroup = 32;  // values that share a scale

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Bytes of a row's scales: whole words.
constexpr __host__ __device__ int64_t scale_bytes(int64_t D) { return (D + 127) / 128 * 4; }

// The scale of 32 values of which `most` has the largest magnitude (its bits without the sign,
// compared as integers, so NaN is above infinity above all numbers): the least power of two
// of which they are at most 6, 2^-126 at least (2^125 at most, where the largest fp32 values
// become 6), so no value is clipped; 255 if one is not finite.
__device__ __forceinline__ uint32_t scale_of(uint32_t most) {
  const int e = static_cast<int>(most >> 23);
  if (e == 255) return 255;
  return static_cast<uint32_t>(min(max(e - 2 + ((most & 0x7fffff) > 0x400000 ? 1 : 0), 1), 252));
}

__device__ __forceinline__ float scale_f32(uint32_t byte) { return __uint_as_float(byte << 23); }

// The codes of 8 values, rounded to nearest, ties to the even code.
__device__ __forceinline__ uint32_t encode8(const float (&x)[8], uint32_t scale) {
  const float s = scale_f32(scale);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
  return w;
}

// Two values as bf16 (exact: two significant bits), of byte B of a word.
template <int B>
__device__ __forceinline__ uint32_t decode2(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, B));
}
__device__ __forceinline__ uint4 decode8(uint32_t w, float scale) {
  return make_uint4(decode2<0>(w, scale), decode2<1>(w, scale), decode2<2>(w, scale), decode2<3>(w, scale));
}

}  // namespace kv4
}  // namespace ghip
