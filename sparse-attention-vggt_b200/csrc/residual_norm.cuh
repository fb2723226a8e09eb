// What the forward and the backward kernels of the gated residual with its norms share.
//
//   p = post(branch)             post: none, or a norm with post_weight, post_bias
//   h = x + gate * p             gate: per channel, or per channel and run of rows
//   y = norm(h) * weight + bias  norm: (h - mean) / sqrt(var + eps), or h / sqrt(mean h^2 + eps)
//
// A row is held in registers by WPR warps, 8 * J elements a lane, in chunks of 8 that are 16-byte
// loads where the layout allows (`vec`): chunk j of lane l of the row's warp w starts at column
// 8 * ((j * WPR + w) * 32 + l).  All arithmetic is in fp32; means are formed first and variances
// from what is left after them, so that a row far from zero loses nothing.
#pragma once

#include "vec8.cuh"

namespace vggt {
namespace rnorm {

constexpr int kNormLayer = VGGT_NORM_LAYER, kNormRms = VGGT_NORM_RMS;

// A vector of parameters in any of the three element types, or none.
struct Param {
  const void* p = nullptr;
  int type = VGGT_DTYPE_FP32;
};

__device__ __forceinline__ void get_param8(const Param& q, int64_t at, int n, bool vec,
                                           float* v) {
  if (q.type == VGGT_DTYPE_FP32)
    get8(static_cast<const float*>(q.p) + at, n, vec, v);
  else if (q.type == VGGT_DTYPE_BF16)
    get8(static_cast<const __nv_bfloat16*>(q.p) + at, n, vec, v);
  else
    get8(static_cast<const __half*>(q.p) + at, n, vec, v);
}

// Sums over the row's WPR warps; every thread gets them, added in the same order.  `scratch`
// holds two floats per warp of the block, twice: consecutive calls alternate (`turn`), so that
// one barrier is enough between a call's writes and the next but one's.
template <int WPR>
struct RowSum {
  float* scratch;
  int slot, warp, turn = 0;
  __device__ __forceinline__ RowSum(float* s) : scratch(s) {
    slot = (threadIdx.x >> 5) / WPR;
    warp = (threadIdx.x >> 5) % WPR;
  }
  __device__ __forceinline__ void two(float& a, float& b) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (WPR > 1) {
      float2* s = reinterpret_cast<float2*>(scratch) + (turn * (blockDim.x >> 5)) + slot * WPR;
      turn ^= 1;
      if ((threadIdx.x & 31) == 0) s[warp] = make_float2(a, b);
      asm volatile("bar.sync %0, %1;" ::"r"(1 + slot), "n"(WPR * 32) : "memory");
      a = b = 0.f;
#pragma unroll
      for (int i = 0; i < WPR; ++i) {
        const float2 t = s[i];
        a += t.x;
        b += t.y;
      }
    }
  }
  __device__ __forceinline__ float one(float a) {
    float b = 0.f;
    two(a, b);
    return a;
  }
};

// v normed in place (elements past the row's end stay zero); returns 1 / deviation.
template <int WPR, int J>
__device__ __forceinline__ float norm_row(float (*v)[8], const int* n, int kind, float inv_width,
                                          float eps, RowSum<WPR>& sum) {
  if (kind == kNormLayer) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[j][i];
    const float mean = sum.one(s) * inv_width;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = i < n[j] ? v[j][i] - mean : 0.f;
  }
  float q = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) q = fmaf(v[j][i], v[j][i], q);
  const float r = 1.f / sqrtf(sum.one(q) * inv_width + eps);
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j][i] *= r;
  return r;
}

// A call's tensors (vggt_block.h).
struct Args {
  const void* x;
  const void* branch;
  Param gate, weight, bias, post_weight, post_bias;
  int64_t rows, width, x_stride, branch_stride, rows_per_gate;
  int stream_type, type;  // of x and h, and of branch and y
  int norm, post;         // VGGT_NORM_*
  float eps;
  bool vec;
};

// residual_norm.cu: checks a call's arguments and fills `a`; 0, or the error
int check(const vggt_residual_norm_args* c, Args* a);

}  // namespace rnorm
}  // namespace vggt
