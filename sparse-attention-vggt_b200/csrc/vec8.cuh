// Eight consecutive elements of bf16, fp16 or fp32 to and from fp32 registers.
#pragma once

#include "common.cuh"
#include "vggt_block.h"

namespace vggt {

template <typename E>
struct Elem {  // bf16 and fp16
  static __device__ __forceinline__ void load8(const E* p, float* v) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = ElemOps<E>::to_float2(u[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ void store8(E* p, const float* v) {
    uint4 w;
    w.x = ElemOps<E>::pack2(v[0], v[1]);
    w.y = ElemOps<E>::pack2(v[2], v[3]);
    w.z = ElemOps<E>::pack2(v[4], v[5]);
    w.w = ElemOps<E>::pack2(v[6], v[7]);
    *reinterpret_cast<uint4*>(p) = w;
  }
  static __device__ __forceinline__ float load(const E* p) { return (float)*p; }
  static __device__ __forceinline__ void store(E* p, float v) { *p = ElemOps<E>::from_float(v); }
};
template <>
struct Elem<float> {
  static __device__ __forceinline__ void load8(const float* p, float* v) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
  static __device__ __forceinline__ void store8(float* p, const float* v) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
};

// The first `n` of 8 elements (the rest read as zero), by one wide access where `vec`.
template <typename E>
__device__ __forceinline__ void get8(const E* p, int n, bool vec, float* v) {
  if (vec && n == 8) {
    Elem<E>::load8(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? Elem<E>::load(p + i) : 0.f;
  }
}
template <typename E>
__device__ __forceinline__ void put8(E* p, int n, bool vec, const float* v) {
  if (vec && n == 8) {
    Elem<E>::store8(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) Elem<E>::store(p + i, v[i]);
  }
}
// An element, or eight, of a vector that is of T or fp32.
template <typename T>
__device__ __forceinline__ float vector_at(const void* p, bool fp32, int64_t i) {
  return fp32 ? static_cast<const float*>(p)[i] : (float)static_cast<const T*>(p)[i];
}
template <typename T>
__device__ __forceinline__ void vector_get8(const void* p, bool fp32, int64_t at, int n, bool vec,
                                            float* v) {
  if (fp32)
    get8(static_cast<const float*>(p) + at, n, vec, v);
  else
    get8(static_cast<const T*>(p) + at, n, vec, v);
}
// Whether rows at `p` with this stride (in elements of VGGT_DTYPE_*) allow the wide accesses.
inline bool wide_rows(const void* p, int64_t stride, int type) {
  return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15u) == 0 &&
                          stride % (type == VGGT_DTYPE_FP32 ? 4 : 8) == 0);
}

}  // namespace vggt
