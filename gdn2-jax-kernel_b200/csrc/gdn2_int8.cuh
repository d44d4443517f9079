// The int8 form of activation checkpoints and cached states: groups of 64
// consecutive values share one float32 scale,
//     code = rint(127 x / max|x|)  (ties to even),   scale = max|x| / 127,
//     value = code * scale.
// The code is the correctly rounded one (except where the cached decode stores a
// state): it does not depend on the order or the precision of the arithmetic that
// a caller compares with.  The error of a
// value is at most half a step, max|x| / 254.
//   * A group whose largest |x| is below 2^-100 gets the scale 0 and reads back as
//     zeros (its scale would leave the normal range).
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
// 1.5 * 2^23: added to |y| < 2^22 it leaves rint(y) in the low bits
constexpr float kCodeBias = 12582912.f;

// max|x|, |y| that keeps a NaN.
__device__ __forceinline__ float max_abs(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(x)), "f"(fabsf(y)));
  return r;
}

// Two values as one operand of the packed float32 instructions.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{.reg .b64 x, y;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{.reg .b64 x, y;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// max|.| of three values; NaN stays.
__device__ __forceinline__ float max_abs3(float x, float y, float z) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

// 127 / top for the codes, to 2^-22.5 of itself (what that leaves open the border
// check decides).  Finite for every top: a group without a scale reads back as 0
// or NaN whatever its codes.  The reciprocal is that of top / 16: of a top above
// 2^126 it would lie below the normal range, with fewer bits.
__device__ __forceinline__ float group_inv(float top) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(0.0625f * fmaxf(top, kInt8Tiny)));
  return 7.9375f * r;   // 127 / 16
}
// The stored scale, rounded once.
__device__ __forceinline__ float group_scale(float top) {
  return !(top <= 3.402823466e38f) ? __uint_as_float(0x7fc00000u)
         : top >= kInt8Tiny ? __fdiv_rn(top, 127.f) : 0.f;
}

// 254 |x| against (2 floor + 1) * top, both exact in float64 (24 + 8 bits).
static __device__ __noinline__ float int8_border(float x, float y, float top) {
  const float lo = floorf(fabsf(y));
  const double l = 254.0 * (double)fabsf(x), r = (2.0 * (double)lo + 1.0) * (double)top;
  const bool up = l > r || (l == r && ((int)lo & 1));
  return copysignf(lo + (up ? 1.f : 0.f), x);
}
// The codes of N (even) values of one group, each in the low byte of a word.
// kCodeBias added to y, |y| <= 127.01, rounds it to a whole number in the low bits
// (the conversion and rounding instructions run at an eighth of the rate).
//
// float32: y = x * inv is off by at most 127 * 2^-22.5 = 2.2e-5, so only a y within
// 3e-5 of a half can round the wrong way; one value in 17000 is decided in float64.
template <int N>
__device__ __forceinline__ void int8_codes_f32(const float (&x)[N], float top, unsigned (&code)[N]) {
  const float inv = group_inv(top);
  float far = 0.f;   // the largest distance of a y from its code
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 v = make_float2(x[i], x[i + 1]), t = fma2(v, both(inv), both(kCodeBias));
    const float2 r = fma2(v, both(inv), fma2(t, both(-1.f), both(kCodeBias)));
    far = max_abs3(far, r.x, r.y);
    code[i] = __float_as_uint(t.x);
    code[i + 1] = __float_as_uint(t.y);
  }
  if (far > 0.49997f) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float y = x[i] * inv, r = __uint_as_float(code[i]) - kCodeBias;
      if (fabsf(y - r) > 0.4999f)
        code[i] = __float_as_uint(int8_border(x[i], y, top) + kCodeBias);
    }
  }
}
// bf16: exact ties are common (8-bit mantissas: one value in 500), but 127 x / top
// is either a half or at least 2^-16 away from it, and one correction makes the
// quotient exact where it is a half: with q = x * inv the remainder 127 x - q top
// has 10 bits and is exact, and q + remainder / top rounds to the quotient.
template <int N>
__device__ __forceinline__ void int8_codes_bf16(const float (&x)[N], float top, unsigned (&code)[N]) {
  const float f = top > 0x1p100f ? 0x1p-100f : 1.f;   // 127 x stays finite
  const float t1 = top * f, c1 = 127.f * f;
  float rc;
  asm("rcp.approx.f32 %0, %1;" : "=f"(rc) : "f"(fmaxf(t1, kInt8Tiny)));
  const float inv = c1 * rc;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 v = make_float2(x[i], x[i + 1]), q = mul2(v, both(inv));
    const float2 r = fma2(q, both(-t1), mul2(v, both(c1)));
    const float2 t = add2(fma2(r, both(rc), q), both(kCodeBias));
    code[i] = __float_as_uint(t.x);
    code[i + 1] = __float_as_uint(t.y);
  }
}
template <typename T, int N>
__device__ __forceinline__ void int8_codes(const float (&x)[N], float top, unsigned (&code)[N]) {
  if constexpr (sizeof(T) == 4) int8_codes_f32(x, top, code);
  else int8_codes_bf16(x, top, code);
}
__device__ __forceinline__ unsigned pack4(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// Byte I of four codes as a float: the code moved to 0..255 becomes the low
// byte of 2^23 + code, and one exact subtraction takes both offsets off (the
// conversion instruction runs at an eighth of the rate).
template <int I>
__device__ __forceinline__ float biased_f(unsigned biased) {   // biased = codes ^ 0x80808080
  return __uint_as_float(__byte_perm(biased, 0x4b000000u, 0x7440 + I));
}
template <int I>
__device__ __forceinline__ float code_f(unsigned biased) { return biased_f<I>(biased) - 8388736.f; }

}  // namespace gdn2
