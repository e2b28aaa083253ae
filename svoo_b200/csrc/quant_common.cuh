// Quantisation to e4m3 with one 32-bit scale per block of 128 values:
//   scale = max(amax / 448, 2^-126),  q = e4m3(x / scale)         both quotients rounded to 32 bits, q to nearest, ties to even
// 448 is the largest e4m3 number.  The largest magnitude is taken over bit patterns, where NaN is above infinity and both
// above every number: a block with a value that is not finite gets a scale that is not, and stands for nothing but NaN.
#pragma once

#include <cuda_fp8.h>

#include "rows_common.cuh"

namespace svoo {

constexpr int kBlock = 128;

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// max(amax / 448, 2^-126); amax not finite stays what it is.  The quotient as in BlockDivide below: 1 / 448 to nearest, twice
// corrected by the remainder, which a factor of 2^64 keeps from underflowing.
__device__ __forceinline__ float block_scale(uint32_t amax) {
  const float a = __uint_as_float(amax);
  const float up = a < 0x1p-60f ? 0x1p64f : 1.f, down = a < 0x1p-60f ? 0x1p-64f : 1.f, x = a * up, y = 1.f / 448.f;
  float q = x * y;
  q = fmaf(fmaf(q, -448.f, x), y, q);
  q = fmaf(fmaf(q, -448.f, x), y, q);
  return amax >= 0x7f800000u ? a : fmaxf(q * down, 0x1p-126f);
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// x / s, correctly rounded, for many x of one s.  With y = 1 / s rounded to nearest, q1 = x y + (x - x y s) y is within
// one unit of x / s; then x - q1 s is a 32-bit number, and q1 + (x - q1 s) y rounds to the quotient (P. Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor", 1990).  Needs a remainder that does not underflow: quotients of
// 2^-11 and more (all that e4m3 tells from zero and ties) have one when s >= 2^-90; below, x and s are multiplied by 2^64
// first, which is exact.  An infinite s gives 0 (NaN for an x that is not finite).  Five operations on pairs of values, against
// some twenty instructions for each division.
struct BlockDivide {
  float y, ns, up;
  __device__ __forceinline__ static float reciprocal(float s) {
    return s == INFINITY ? 0.f : __fdiv_rn(1.f, s * (s < 0x1p-90f ? 0x1p64f : 1.f));
  }
  __device__ __forceinline__ explicit BlockDivide(float s) : BlockDivide(s, reciprocal(s)) {}
  __device__ __forceinline__ BlockDivide(float s, float reciprocal_of_s) {
    y = reciprocal_of_s;
    up = s < 0x1p-90f ? 0x1p64f : 1.f;
    ns = s == INFINITY ? -1.f : -s * up;
  }
  // Of x that are 16-bit numbers, as is the amax that s came from, q1 is enough: it is off the rounded quotient only
  // where x / s lies within 2^-46 of the middle of two 32-bit numbers, and e4m3 tells that only beside its ties, 32-bit numbers t
  // of five bits.  x = t s (1 +- 2^-24) has no solution in x of 11 bits but t = 2^-10, x a power of two and s one step
  // below another, which no amax of 11 bits over 448 is.
  template <bool kOnce = false>
  __device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) const {
    if (__builtin_expect(up != 1.f, 0)) a *= up, b *= up, c *= up, d *= up;
    pair<kOnce>(a, b);
    pair<kOnce>(c, d);
    return e4m3x2(a, b) | e4m3x2(c, d) << 16;
  }
  // eight values, in one branch
  template <bool kOnce>
  __device__ __forceinline__ uint2 e4m3x8(float (&v)[8]) const {
    if (__builtin_expect(up != 1.f, 0)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= up;
    }
#pragma unroll
    for (int i = 0; i < 8; i += 2) pair<kOnce>(v[i], v[i + 1]);
    return make_uint2(e4m3x2(v[0], v[1]) | e4m3x2(v[2], v[3]) << 16, e4m3x2(v[4], v[5]) | e4m3x2(v[6], v[7]) << 16);
  }
  template <bool kOnce>
  __device__ __forceinline__ void pair(float& a, float& b) const {
    if constexpr (kOnce) {
      asm("{\n\t.reg .b64 x, ns, y, q, r;\n\t"
          "mov.b64 x, {%0, %1};\n\tmov.b64 ns, {%2, %2};\n\tmov.b64 y, {%3, %3};\n\t"
          "mul.rn.f32x2 q, x, y;\n\tfma.rn.f32x2 r, q, ns, x;\n\tfma.rn.f32x2 q, r, y, q;\n\t"
          "mov.b64 {%0, %1}, q;\n\t}\n" : "+f"(a), "+f"(b) : "f"(ns), "f"(y));
      return;
    }
    asm("{\n\t.reg .b64 x, ns, y, q, r;\n\t"
        "mov.b64 x, {%0, %1};\n\tmov.b64 ns, {%2, %2};\n\tmov.b64 y, {%3, %3};\n\t"
        "mul.rn.f32x2 q, x, y;\n\t"
        "fma.rn.f32x2 r, q, ns, x;\n\tfma.rn.f32x2 q, r, y, q;\n\t"
        "fma.rn.f32x2 r, q, ns, x;\n\tfma.rn.f32x2 q, r, y, q;\n\t"
        "mov.b64 {%0, %1}, q;\n\t}\n" : "+f"(a), "+f"(b) : "f"(ns), "f"(y));
  }
};

}  // namespace svoo
