// Rotary positions on the device: the angles of a workgroup's tokens, and the rotation.
#pragma once

#include "common.h"

namespace ghip {
namespace rope {

constexpr int kMostAxes = 4;
constexpr int kMostHalf = 128;  // pairs of a row

// Which angle turns which pair: pair i of token (b, s) by positions[axis(i)][b][s] * freqs[i].
struct Angles {
  const int32_t* positions;  // nullptr: starts[b] + s
  const int32_t* starts;
  const float* freqs;
  int64_t p_sa, p_sb, p_ss;  // element strides of axis, sequence, token
  int half;                  // pairs of a row
  int ends[kMostAxes];       // where each axis' pairs end
  int neighbours;            // pairs (2i, 2i + 1); 0: (i, i + half)
  int inverse;
};

// The position that turns pair i of token (b, s).
__device__ __forceinline__ double position(const Angles& a, int b, int s, int i) {
  if (!a.positions) return static_cast<double>(static_cast<int64_t>(a.starts[b]) + s);
  const int axis = (i >= a.ends[0]) + (i >= a.ends[1]) + (i >= a.ends[2]);
  return static_cast<double>(a.positions[axis * a.p_sa + b * a.p_sb + s * a.p_ss]);
}

// (cos, sin) of pos * freq.  The angle is a product in 64 bits, reduced by whole quarter turns in two
// steps (pi / 2 as the sum of two doubles) to |r| <= pi / 4, so positions of any size keep 2^-52
// of the angle; there the Taylor sums to r^13 and r^12 are off by less than 2^-45 and 2^-41, and each of
// the two is rounded to fp32 once.  (An fp32 angle of 10^5 is off by 2^-8.  The library's sincos,
// good to 2^-52, takes four times the instructions: a batch of prompts into 4 bits was bound by it.)
__device__ __forceinline__ float2 turn(double pos, float freq, int inverse) {
  const double a = pos * static_cast<double>(freq);
  const double k = rint(a * 0.6366197723675814);  // 2 / pi
  double r = fma(-k, 1.5707963267948966, a);
  r = fma(-k, 6.123233995736766e-17, r);
  const double z = r * r;
  double s = fma(z, 1. / 6227020800., -1. / 39916800.);
  s = fma(z, s, 1. / 362880.);
  s = fma(z, s, -1. / 5040.);
  s = fma(z, s, 1. / 120.);
  s = fma(z, s, -1. / 6.);
  s = fma(z * r, s, r);
  double c = fma(z, 1. / 479001600., -1. / 3628800.);
  c = fma(z, c, 1. / 40320.);
  c = fma(z, c, -1. / 720.);
  c = fma(z, c, 1. / 24.);
  c = fma(z, c, -0.5);
  c = fma(z, c, 1.);
  const int quarter = static_cast<int>(fma(floor(k * 0.25), -4., k));  // 0 .. 3
  const float sf = static_cast<float>(s), cf = static_cast<float>(c);
  const float sn = quarter & 1 ? cf : sf, cs = quarter & 1 ? sf : cf;
  const float si = quarter & 2 ? -sn : sn;
  return make_float2(((quarter + 1) & 2) ? -cs : cs, inverse ? -si : si);
}

// (x, y) turned.  Each product is rounded by itself: left to be fused with the sum, which of
// them is would depend on the kernel, and a key's code in a 4-bit cache with it.
__device__ __forceinline__ float2 turned(float x, float y, float2 cs) {
#pragma clang fp contract(off)
  const float xc = x * cs.x, ys = y * cs.y, xs = x * cs.y, yc = y * cs.x;
  return make_float2(xc - ys, xs + yc);
}

}  // namespace rope
}  // namespace ghip
