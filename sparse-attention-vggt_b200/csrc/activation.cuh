// The activations of `linear` and their derivatives, in fp32.
#pragma once

#include <type_traits>

#include "exp2.cuh"
#include "vggt_block.h"

namespace vggt {
namespace act {

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

constexpr float kLog2e = 1.4426950408889634f;

// Upper tail of the normal distribution at u = min(|z|, 64) as q = exp(-u^2 / 2) R(u), and
// e = exp(-u^2 / 2).  R is t times a polynomial of degree 5 in t = 1 / (1 + 0.3 u), fitted to
// the least largest relative error on [0, 9] (2.1e-6; with the exponential in fp32 5.7e-6):
// relative, so that an activation far on the negative side is as exact as elsewhere.  Beyond 64
// both are zero, and the cut keeps an infinity from meeting that zero.
struct Tail {
  float u, q, e;
  __device__ __forceinline__ explicit Tail(float z) {
    u = min_nan(fabsf(z), 64.f);
    const float t = rcp(fmaf(0.3f, u, 1.f));
    e = fast_exp2(u * u * (-0.5f * kLog2e));
    float r = fmaf(-0.0818372592f, t, 0.230586097f);
    r = fmaf(r, t, -0.0340376124f);
    r = fmaf(r, t, 0.153751031f);
    r = fmaf(r, t, 0.111210488f);
    r = fmaf(r, t, 0.120327726f);
    q = r * t * e;
  }
};

__device__ __forceinline__ float sigmoid(float z) { return rcp(1.f + fast_exp2(-kLog2e * z)); }

constexpr float kTanhIn = 0.7978845608028654f;  // sqrt(2 / pi)

// a(z); KIND is VGGT_ACT_*
template <int KIND>
__device__ __forceinline__ float value(float z) {
  if (KIND == VGGT_ACT_GELU) {  // z Phi(z) = max(z, 0) - |z| q(|z|)
    const Tail t(z);
    return fmaf(-t.u, t.q, max_nan(z, 0.f));
  }
  if (KIND == VGGT_ACT_GELU_TANH) {
    const float c = max_nan(min_nan(z, 64.f), -64.f);
    return max_nan(z, -64.f) * sigmoid(2.f * kTanhIn * c * fmaf(0.044715f * c, c, 1.f));
  }
  if (KIND == VGGT_ACT_SILU) return max_nan(z, -256.f) * sigmoid(z);
  if (KIND == VGGT_ACT_RELU) return max_nan(z, 0.f);
  return z;
}

// a(z) and a'(z)
template <int KIND>
__device__ __forceinline__ float value_slope(float z, float& slope) {
  if (KIND == VGGT_ACT_GELU) {  // a' = Phi(z) + z phi(z)
    const Tail t(z);
    const float c = z < 0.f ? -t.u : t.u;
    slope = fmaf(c * t.e, 0.3989422804f, z < 0.f ? t.q : 1.f - t.q);
    return fmaf(-t.u, t.q, max_nan(z, 0.f));
  }
  if (KIND == VGGT_ACT_GELU_TANH) {
    const float c = max_nan(min_nan(z, 64.f), -64.f);
    const float s = sigmoid(2.f * kTanhIn * c * fmaf(0.044715f * c, c, 1.f));
    slope = fmaf(c * s * (1.f - s), 2.f * kTanhIn * fmaf(3.f * 0.044715f * c, c, 1.f), s);
    return max_nan(z, -64.f) * s;
  }
  if (KIND == VGGT_ACT_SILU) {
    const float c = max_nan(min_nan(z, 256.f), -256.f), s = sigmoid(c);
    slope = fmaf(c * s, 1.f - s, s);
    return max_nan(z, -256.f) * s;
  }
  if (KIND == VGGT_ACT_RELU) {
    slope = z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
    return max_nan(z, 0.f);
  }
  slope = 1.f;
  return z;
}

// a(z) of a pair, in packed instructions where there are some: half of what the epilogue of a
// product issues (32 frames widened with gelu took 392 us with value(), 246 without an activation).
template <int KIND>
__device__ __forceinline__ float_pair value_pair(float_pair z) {
  float a, b;
  unpack_pair(a, b, z);
  if (KIND == VGGT_ACT_GELU) {
    const float ua = min_nan(fabsf(a), 64.f), ub = min_nan(fabsf(b), 64.f);
    const float_pair u = pack_pair(ua, ub);
    float da, db, ea, eb;
    unpack_pair(da, db, fma_pair(u, pack_pair(0.3f, 0.3f), pack_pair(1.f, 1.f)));
    const float_pair t = pack_pair(rcp(da), rcp(db));
    unpack_pair(ea, eb, mul_pair(mul_pair(u, u), pack_pair(-0.5f * kLog2e, -0.5f * kLog2e)));
    const float_pair e = pack_pair(fast_exp2(ea), fast_exp2(eb));
    // the polynomial with its sign turned: -q
    float_pair r = fma_pair(pack_pair(0.0818372592f, 0.0818372592f), t,
                            pack_pair(-0.230586097f, -0.230586097f));
    r = fma_pair(r, t, pack_pair(0.0340376124f, 0.0340376124f));
    r = fma_pair(r, t, pack_pair(-0.153751031f, -0.153751031f));
    r = fma_pair(r, t, pack_pair(-0.111210488f, -0.111210488f));
    r = fma_pair(r, t, pack_pair(-0.120327726f, -0.120327726f));
    const float_pair q = mul_pair(mul_pair(r, t), e);
    return fma_pair(q, u, pack_pair(max_nan(a, 0.f), max_nan(b, 0.f)));
  }
  return pack_pair(value<KIND>(a), value<KIND>(b));
}

// f with the activation as a compile-time constant: f(std::integral_constant<int, KIND>)
template <typename F>
__device__ __forceinline__ void dispatch(int kind, F&& f) {
  switch (kind) {
    case VGGT_ACT_GELU: f(std::integral_constant<int, VGGT_ACT_GELU>()); break;
    case VGGT_ACT_GELU_TANH: f(std::integral_constant<int, VGGT_ACT_GELU_TANH>()); break;
    case VGGT_ACT_SILU: f(std::integral_constant<int, VGGT_ACT_SILU>()); break;
    case VGGT_ACT_RELU: f(std::integral_constant<int, VGGT_ACT_RELU>()); break;
    default: f(std::integral_constant<int, VGGT_ACT_NONE>()); break;
  }
}

}  // namespace act
}  // namespace vggt
