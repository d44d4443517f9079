// The int8 form of activation checkpoints and cached states: groups of 64
// consecutive values share one float32 scale,
//     code = rint(127 x / max|x|)  (ties to even),   scale = max|x| / 127,
//     value = code * scale.
// The code is the correctly rounded one: it does not depend on the order or
// the precision of the arithmetic that a caller compares with.  The error of a
// value is at most half a step, max|x| / 254.
//   * A group whose largest |x| is below 2^-100 is stored as zeros (its scale
//     would leave the normal range).
//   * A group that holds a NaN or an infinity gets a NaN scale, so all of it
//     reads back as NaN: one scale cannot hold an infinity next to other values,
//     and a silent 0 would hide it.
// Uniform codes rather than an 8-bit float: within a group of 64 the rounding
// error of a value is 1/254 of the largest, against 1/16 of the value itself in
// e4m3 (on normally distributed values 0.6% against 2.6% of their size, rms).
#pragma once
#include "gdn2_common.cuh"

namespace gdn2 {

constexpr int kGroup = 64;            // values that share a scale
constexpr float kInt8Tiny = 0x1p-100f;

// |x| as an ordered integer: NaN above infinity above every finite value, so
// an integer maximum keeps NaN (a float maximum would drop it).
__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

struct GroupScale {
  float top, inv, scale;   // max|x|, 127 / max|x| (0: every code is 0), max|x| / 127
};
__device__ __forceinline__ GroupScale group_scale(unsigned top_bits) {
  GroupScale s;
  s.top = __uint_as_float(top_bits);
  const bool fits = top_bits < 0x7f800000u, some = s.top >= kInt8Tiny;
  s.inv = fits && some ? __fdiv_rn(127.f, s.top) : 0.f;
  s.scale = !fits ? __uint_as_float(0x7fc00000u) : some ? __fdiv_rn(s.top, 127.f) : 0.f;
  return s;
}

// y = x * inv is off by at most 127 * 2^-23 = 1.5e-5, so only a y within 1e-4
// of a half can round the wrong way; there 254 |x| is compared with
// (2 floor + 1) * top, both exact in float64 (24 + 8 bits).  One value in 5000
// takes this path.
static __device__ __noinline__ float int8_border(float x, float y, float top) {
  const float lo = floorf(fabsf(y));
  const double l = 254.0 * (double)fabsf(x), r = (2.0 * (double)lo + 1.0) * (double)top;
  const bool up = l > r || (l == r && ((int)lo & 1));
  return copysignf(lo + (up ? 1.f : 0.f), x);
}
__device__ __forceinline__ int int8_code(float x, const GroupScale& s) {
  const float y = x * s.inv;
  float r = rintf(y);
  if (fabsf(y - r) > 0.4999f) r = int8_border(x, y, s.top);
  return __float2int_rn(r);   // NaN (inv = 0 times an infinity) gives 0
}
// The nearest code by float32 arithmetic alone, for values that carry rounding
// errors of their own: off from a half step by at most 1.5e-5 of a step.
// 1.5 * 2^23 added to |y| <= 127.01 leaves rint(y) in the low byte.
__device__ __forceinline__ unsigned int8_code_near(float x, float inv) {
  return __float_as_uint(fmaf(x, inv, 12582912.f));
}
__device__ __forceinline__ unsigned pack4(int a, int b, int c, int d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// Byte I of four codes as a float: the code moved to 0..255 becomes the low
// byte of 2^23 + code, and one exact subtraction takes both offsets off (the
// conversion instruction runs at an eighth of the rate).
template <int I>
__device__ __forceinline__ float code_f(unsigned biased) {   // biased = codes ^ 0x80808080
  return __uint_as_float(__byte_perm(biased, 0x4b000000u, 0x7440 + I)) - 8388736.f;
}

}  // namespace gdn2
