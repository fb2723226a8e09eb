// Exponentials of column pairs on the multi-function unit and on the FMA pipe.
#pragma once

#include "common.cuh"

namespace vggt {

// Two floats in a 64-bit register, as the packed instructions take them.
// Operands that do not change are packed once: a packing inside the loop costs
// up to four moves per packed instruction, more than the instruction saves.
typedef uint64_t float_pair;

__device__ __forceinline__ float_pair pack_pair(float a, float b) {
  float_pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack_pair(float& a, float& b, float_pair v) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ float_pair fma_pair(float_pair a, float_pair b, float_pair c) {
  float_pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float_pair mul_pair(float_pair a, float_pair b) {
  float_pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float_pair add_pair(float_pair a, float_pair b) {
  float_pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float_pair sub_pair(float_pair a, float_pair b) {
  float_pair r;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// 2^x of a pair for arguments up to 126 without the multi-function unit, as
// q * scale: x = n + f with n = round(x) (adding 1.5 * 2^23 leaves it in the low
// mantissa bits), q a polynomial of degree 4 for 2^f on [-1/2, 1/2] (fitted to
// the least largest relative error, 2.7e-6 in fp32), scale = 2^n.  Where n would
// be below -126 the exponent's bits come to zero, and scale with them: -inf
// gives exactly 0, as a masked score must (2^-126 is a number of bf16, and times
// a value of 1e38 one that shows).  A NaN stays one (in q).  (The block-sparse
// attention's cubic, attn_tc05.cu, goes under the rounding of its P; here the
// exponentials are summed in fp32 for log-sum-exps and weights.)
struct Exp2Poly {
  float_pair magic, c4, c3, c2, c1, c0;
  __device__ __forceinline__ Exp2Poly()
      : magic(pack_pair(12582912.f, 12582912.f)),
        c4(pack_pair(0.0095701022f, 0.0095701022f)),
        c3(pack_pair(0.0559178591f, 0.0559178591f)),
        c2(pack_pair(0.2402474433f, 0.2402474433f)),
        c1(pack_pair(0.6931217909f, 0.6931217909f)),
        c0(pack_pair(0.9999992847f, 0.9999992847f)) {}
  __device__ __forceinline__ void operator()(float_pair& q, float_pair& scale, float_pair x) const {
    float a, b, ta, tb;
    unpack_pair(a, b, x);
    x = pack_pair(max_nan(a, -127.f), max_nan(b, -127.f));
    const float_pair t = add_pair(x, magic);
    const float_pair f = sub_pair(x, sub_pair(t, magic));
    q = fma_pair(f, c4, c3);
    q = fma_pair(q, f, c2);
    q = fma_pair(q, f, c1);
    q = fma_pair(q, f, c0);
    unpack_pair(ta, tb, t);
    // of a NaN the exponent is any
    scale = pack_pair(__int_as_float((__float_as_int(ta) << 23) + 0x3f800000),
                      __int_as_float((__float_as_int(tb) << 23) + 0x3f800000));
  }
};

// Maximum of three that keeps a NaN.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

}  // namespace vggt
