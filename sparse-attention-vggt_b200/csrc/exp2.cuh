// Exponentials of column pairs on the multi-function unit and on the FMA pipe.
#pragma once

#include "common.cuh"

namespace vggt {

// (d0, d1) = (a0, a1) * b + c with one packed instruction
__device__ __forceinline__ void fma_pair(float& d0, float& d1, float a0, float a1, float b,
                                         float c) {
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\t"
      "mov.b64 rb, {%4, %4};\n\t"
      "mov.b64 rc, {%5, %5};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\t"
      "mov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b), "f"(c));
}

__device__ __forceinline__ void add_pair(float& d0, float& d1, float a0, float a1) {
  asm("{\n\t.reg .b64 ra, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\t"
      "mov.b64 rd, {%0, %1};\n\t"
      "add.rn.f32x2 rd, rd, ra;\n\t"
      "mov.b64 {%0, %1}, rd;\n\t}"
      : "+f"(d0), "+f"(d1)
      : "f"(a0), "f"(a1));
}

// 2^a, 2^b for arguments up to 126 without the multi-function unit: x = n + f
// with n = round(x) (adding 1.5 * 2^23 leaves it in the low mantissa bits), a
// polynomial of degree 4 for 2^f on [-1/2, 1/2] (fitted to the least largest
// relative error, 2.7e-6 in fp32), n added to its exponent.  Arguments below
// -126 give 2^-126 at most.
__device__ __forceinline__ void exp2_poly_pair(float& ea, float& eb, float a, float b) {
  a = fmaxf(a, -126.f);
  b = fmaxf(b, -126.f);
  float qa, qb, ta, tb;
  asm("{\n\t.reg .b64 x, m, t, n, f, q, c4, c3, c2, c1, c0;\n\t"
      "mov.b64 x, {%4, %5};\n\t"
      "mov.b64 m, {%6, %6};\n\t"
      "mov.b64 c4, {%7, %7};\n\t"
      "mov.b64 c3, {%8, %8};\n\t"
      "mov.b64 c2, {%9, %9};\n\t"
      "mov.b64 c1, {%10, %10};\n\t"
      "mov.b64 c0, {%11, %11};\n\t"
      "add.rn.f32x2 t, x, m;\n\t"
      "sub.rn.f32x2 n, t, m;\n\t"
      "sub.rn.f32x2 f, x, n;\n\t"
      "fma.rn.f32x2 q, f, c4, c3;\n\t"
      "fma.rn.f32x2 q, q, f, c2;\n\t"
      "fma.rn.f32x2 q, q, f, c1;\n\t"
      "fma.rn.f32x2 q, q, f, c0;\n\t"
      "mov.b64 {%0, %1}, q;\n\t"
      "mov.b64 {%2, %3}, t;\n\t}"
      : "=f"(qa), "=f"(qb), "=f"(ta), "=f"(tb)
      : "f"(a), "f"(b), "f"(12582912.f), "f"(0.0095701022f), "f"(0.0559178591f),
        "f"(0.2402474433f), "f"(0.6931217909f), "f"(0.9999992847f));
  ea = __int_as_float(__float_as_int(qa) + (__float_as_int(ta) << 23));
  eb = __int_as_float(__float_as_int(qb) + (__float_as_int(tb) << 23));
}

// Maximum of three that keeps a NaN.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

}  // namespace vggt
