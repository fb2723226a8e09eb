// One row of paged attention formed key by key: the path of the few rows
// where a tensor-core product would multiply a masked zero by a value that is
// not finite.
#pragma once

#include "paged.cuh"

namespace vggt {

// Whether either 16-bit value is infinite or NaN (all exponent bits set).
template <typename T>
__device__ __forceinline__ bool has_nonfinite(uint32_t two);
template <>
__device__ __forceinline__ bool has_nonfinite<__nv_bfloat16>(uint32_t v) {
  return (v & 0x7f80u) == 0x7f80u || (v & 0x7f800000u) == 0x7f800000u;
}
template <>
__device__ __forceinline__ bool has_nonfinite<__half>(uint32_t v) {
  return (v & 0x7c00u) == 0x7c00u || (v & 0x7c000000u) == 0x7c000000u;
}

// Row r of the tile over the keys [key0, key1) that lie below `limit`: the
// unnormalised output (D floats), the maximum in units of log2, the sum.
// Called by a full warp; a lane holds D / 32 elements.
template <typename T, int D>
__device__ __noinline__ void slow_row(const PagedAttnArgs& a, const RowTile& rt, int r, int head,
                                      float scale_log2, int64_t key0, int64_t key1, int64_t limit,
                                      float* out, float* m_out, float* l_out) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int row = rt.row0 + r;
  const T* q = static_cast<const T*>(a.q) + (rt.first + row / a.group) * a.q_token +
               ((int64_t)head * a.group + row % a.group) * a.q_head;
  float qv[E], o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qv[e] = (float)q[lane * E + e];
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  if (key1 > limit) key1 = limit;
  for (int64_t j = key0; j < key1; ++j) {
    const int page = checked_page(a.t, a.pool, rt.seq, j >> a.pool.page_shift);
    const int64_t at = page * a.pool.page_stride + head * a.pool.head_stride +
                       (j & (a.pool.page - 1)) * a.pool.row_stride + lane * E;
    float s = 0.f, v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[e] = page < 0 ? 0.f : (float)static_cast<const T*>(a.v_pages)[at + e];
      s = fmaf(qv[e], page < 0 ? 0.f : (float)static_cast<const T*>(a.k_pages)[at + e], s);
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    s *= scale_log2;
    const float mx = fmaxf(m, s);
    const float base = mx == -INFINITY ? 0.f : mx;
    const float f = m == mx ? 1.f : fast_exp2(m - base), e = fast_exp2(s - base);
    l = fmaf(l, f, e);
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = fmaf(e, v[i], o[i] * f);
    m = mx;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) out[lane * E + e] = o[e];
  if (lane == 0) {
    *m_out = m;
    *l_out = l;
  }
}

}  // namespace vggt
