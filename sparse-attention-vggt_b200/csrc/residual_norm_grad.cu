// Gradients of the gated residual with its norms (residual_norm.cuh has the formulas).
//
// With hat the normed row, r one over its deviation, a bar for a row's mean:
//   g = dy * weight,  dh' = dh + r (g - hat mean(g hat) [- mean(g), layer norm])
//   dx = dh',  dweight = sum dy hat,  dbias = sum dy
//   dgate = sum dh' p,  dp = dh' gate,  and p's norm likewise back to the branch
// h is formed again from x and the branch, in fp32: x is read instead of h, so that the
// parameters' gradients carry no rounding of a 16-bit h.
//
// Bound by memory (x, branch, dy, dh read, dx, dbranch written, once each).  A row lies in the
// registers of WPR warps (16 elements a lane: the row's values and the parameters' sums, three
// to five fp32 numbers an element, fit together).  Each group of warps takes a run of rows; its
// parameters' sums are added over the block's groups in shared memory and written as one partial
// per block, which a second kernel adds in order.  No atomics: equal calls give equal bits.
#include <algorithm>

#include "kernels.h"
#include "residual_norm.cuh"

namespace vggt {
namespace rnorm {

enum { kWeight, kBias, kGate, kPostWeight, kPostBias, kArrays };

struct Bwd {
  Args a;
  const void* dy;
  const void* dh;
  void* dx;
  void* dbranch;
  int64_t dy_stride, dh_stride, dx_stride, dbranch_stride;
  void* out[kArrays];      // the parameters' gradients, or null
  int out_type[kArrays];
  float* part[kArrays];    // [blocks][width] partial sums; of a gate per run of rows
                           // [slots + gates][width]
  int64_t slots;           // groups of warps that have rows (one at least): group s takes
                           // [s rows / slots, (s + 1) rows / slots)
};

__device__ __forceinline__ void put_param8(void* p, int type, int64_t at, int n, bool vec,
                                           const float* v) {
  if (type == VGGT_DTYPE_FP32)
    put8(static_cast<float*>(p) + at, n, vec, v);
  else if (type == VGGT_DTYPE_BF16)
    put8(static_cast<__nv_bfloat16*>(p) + at, n, vec, v);
  else
    put8(static_cast<__half*>(p) + at, n, vec, v);
}

template <int WPR>
constexpr int bwd_threads() {
  return WPR > 8 ? WPR * 32 : 256;
}

// The gradient of what was normed to hat, from that of hat (d, in place).
template <int WPR, int J>
__device__ __forceinline__ void norm_back(float (*d)[8], const float (*hat)[8], const int* n,
                                          int kind, float r, float inv_width, RowSum<WPR>& sum) {
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s = fmaf(d[j][i], hat[j][i], s);
      t += d[j][i];
    }
  sum.two(s, t);
  s *= inv_width;
  t = kind == kNormLayer ? t * inv_width : 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) d[j][i] = i < n[j] ? r * (d[j][i] - t - hat[j][i] * s) : 0.f;
}

template <typename S, typename T, int WPR, int J, bool POST>
__global__ void __launch_bounds__(bwd_threads<WPR>()) backward_kernel(const Bwd f) {
  constexpr int kThreads = bwd_threads<WPR>(), kSlots = kThreads / 32 / WPR;
  constexpr int kAccs = POST ? 5 : 3;
  constexpr int kRow = WPR * 32 * 8 * J;  // columns that a group of warps holds
  __shared__ float scratch[2 * 2 * 32];
  __shared__ float fold[kSlots > 1 ? kSlots * kRow : 1];
  const Args& a = f.a;
  RowSum<WPR> sum(scratch);
  const int lane = threadIdx.x & 31;
  const float inv_width = 1.f / (float)a.width;
  const bool vec = a.vec;
  int n[J];
#pragma unroll
  for (int j = 0; j < J; ++j)
    n[j] = max(0, min(8, (int)a.width - 8 * ((j * WPR + sum.warp) * 32 + lane)));
  const int first = 8 * (sum.warp * 32 + lane);
  constexpr int step = 8 * WPR * 32;
  const int64_t slot = (int64_t)blockIdx.x * kSlots + sum.slot;
  const int64_t row0 = slot < f.slots ? slot * a.rows / f.slots : 0;
  const int64_t row1 = slot < f.slots ? (slot + 1) * a.rows / f.slots : 0;

  float acc[kAccs][J][8];
#pragma unroll
  for (int k = 0; k < kAccs; ++k)
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[k][j][i] = 0.f;

  const bool gates = a.gate.p != nullptr && a.rows_per_gate > 0;  // a gate per run of rows
  for (int64_t row = row0; row < row1; ++row) {
    float h[J][8], p[J][8], hat[J][8], d[J][8], gv[J][8];
    const S* x = static_cast<const S*>(a.x) + row * a.x_stride + first;
#pragma unroll
    for (int j = 0; j < J; ++j) get8(x + j * step, n[j], vec, h[j]);
    float pr = 0.f;
    const int64_t gate_row = gates ? row / a.rows_per_gate : 0;
    if (a.branch != nullptr) {
      const T* b = static_cast<const T*>(a.branch) + row * a.branch_stride + first;
#pragma unroll
      for (int j = 0; j < J; ++j) get8(b + j * step, n[j], vec, p[j]);
      if (POST) {
        pr = norm_row<WPR, J>(p, n, a.post, inv_width, a.eps, sum);
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) hat[j][i] = p[j][i];
        if (a.post_weight.p != nullptr)
#pragma unroll
          for (int j = 0; j < J; ++j) {
            float w[8];
            get_param8(a.post_weight, first + j * step, n[j], vec, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) p[j][i] *= w[i];
          }
        if (a.post_bias.p != nullptr)
#pragma unroll
          for (int j = 0; j < J; ++j) {
            float w[8];
            get_param8(a.post_bias, first + j * step, n[j], vec, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) p[j][i] += w[i];
          }
      }
      const int64_t at = gate_row * a.width;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (a.gate.p != nullptr) {
          get_param8(a.gate, at + first + j * step, n[j], vec, gv[j]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) gv[j][i] = 1.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) h[j][i] = fmaf(gv[j][i], p[j][i], h[j][i]);
      }
    }
    const float r = norm_row<WPR, J>(h, n, a.norm, inv_width, a.eps, sum);  // h is normed now
    if (f.dy != nullptr) {
      const T* dy = static_cast<const T*>(f.dy) + row * f.dy_stride + first;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        get8(dy + j * step, n[j], vec, d[j]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc[kWeight][j][i] = fmaf(d[j][i], h[j][i], acc[kWeight][j][i]);
          acc[kBias][j][i] += d[j][i];
        }
        if (a.weight.p != nullptr) {
          float w[8];
          get_param8(a.weight, first + j * step, n[j], vec, w);
#pragma unroll
          for (int i = 0; i < 8; ++i) d[j][i] *= w[i];
        }
      }
      norm_back<WPR, J>(d, h, n, a.norm, r, inv_width, sum);
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) d[j][i] = 0.f;
    }
    if (f.dh != nullptr) {
      const S* dh = static_cast<const S*>(f.dh) + row * f.dh_stride + first;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        float t[8];
        get8(dh + j * step, n[j], vec, t);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[j][i] += t[i];
      }
    }
    if (f.dx != nullptr) {
      S* dx = static_cast<S*>(f.dx) + row * f.dx_stride + first;
#pragma unroll
      for (int j = 0; j < J; ++j) put8(dx + j * step, n[j], vec, d[j]);
    }
    if (a.branch != nullptr) {
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc[kGate][j][i] = fmaf(d[j][i], p[j][i], acc[kGate][j][i]);
          d[j][i] *= gv[j][i];
        }
      if (POST) {
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            acc[kPostWeight % kAccs][j][i] = fmaf(d[j][i], hat[j][i], acc[kPostWeight % kAccs][j][i]);
            acc[kPostBias % kAccs][j][i] += d[j][i];
          }
        if (a.post_weight.p != nullptr)
#pragma unroll
          for (int j = 0; j < J; ++j) {
            float w[8];
            get_param8(a.post_weight, first + j * step, n[j], vec, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[j][i] *= w[i];
          }
        norm_back<WPR, J>(d, hat, n, a.post, pr, inv_width, sum);
      }
      if (f.dbranch != nullptr) {
        T* db = static_cast<T*>(f.dbranch) + row * f.dbranch_stride + first;
#pragma unroll
        for (int j = 0; j < J; ++j) put8(db + j * step, n[j], vec, d[j]);
      }
      // the last row here of a run of rows with one gate: its sum goes out
      if (gates && f.out[kGate] != nullptr &&
          (row + 1 == row1 || (row + 1) % a.rows_per_gate == 0)) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
          if (a.rows_per_gate == 1)
            put_param8(f.out[kGate], f.out_type[kGate], gate_row * a.width + first + j * step, n[j],
                       vec, acc[kGate][j]);
          else
            put8(f.part[kGate] + (slot + gate_row) * a.width + first + j * step, n[j], vec,
                 acc[kGate][j]);
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[kGate][j][i] = 0.f;
        }
      }
    }
  }

#pragma unroll
  for (int k = 0; k < kAccs; ++k) {
    if (f.out[k] == nullptr || (k == kGate && gates)) continue;  // the same for all threads
    float* to = f.part[k] + (int64_t)blockIdx.x * a.width;
    if (kSlots == 1) {
#pragma unroll
      for (int j = 0; j < J; ++j) put8(to + first + j * step, n[j], vec, acc[k][j]);
    } else {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < J; ++j)
        Elem<float>::store8(fold + sum.slot * kRow + first + j * step, acc[k][j]);
      __syncthreads();
      for (int c = threadIdx.x; c < (int)a.width; c += kThreads) {
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < kSlots; ++q) s += fold[q * kRow + c];
        to[c] = s;
      }
    }
  }
}

// Adds the partial sums: blockIdx.y below kArrays an array over all blocks, from kArrays on the
// gates of runs of rows.  32 columns x 8 lanes over the partials.
__global__ void __launch_bounds__(256) finish_kernel(const Bwd f, int64_t blocks, int64_t gates) {
  __shared__ float fold[8][32];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int64_t width = f.a.width, c = (int64_t)blockIdx.x * 32 + cx;
  const bool runs = blockIdx.y >= kArrays;
  const int k = runs ? kGate : (int)blockIdx.y;
  if (f.out[k] == nullptr || (!runs && k == kGate && gates > 0)) return;
  const int64_t count = runs ? gates : 1, step = runs ? gridDim.y - kArrays : 1;
  for (int64_t g = runs ? blockIdx.y - kArrays : 0; g < count; g += step) {
    int64_t lo = 0, hi = blocks;
    if (runs) {
      // the groups of warps whose rows meet the run's: group s starts at row s rows / slots
      const int64_t r0 = g * f.a.rows_per_gate, r1 = r0 + f.a.rows_per_gate - 1;
      lo = ((r0 + 1) * f.slots - 1) / f.a.rows + g;
      hi = ((r1 + 1) * f.slots - 1) / f.a.rows + g + 1;
    }
    float s = 0.f;
    if (c < width)
      for (int64_t i = lo + ry; i < hi; i += 8) s += f.part[k][i * width + c];
    fold[ry][cx] = s;
    __syncthreads();
    if (ry == 0 && c < width) {
#pragma unroll
      for (int q = 1; q < 8; ++q) s += fold[q][cx];
      put_param8(f.out[k], f.out_type[k], g * width + c, 1, false, &s);
    }
    __syncthreads();
  }
}

// Warps to a row.
int row_warps(int64_t width) {
  return width <= 512 ? 1 : width <= 1024 ? 2 : width <= 2048 ? 4 : width <= 4096 ? 8 : 16;
}

// Blocks of a call: two of 256 threads to an SM are resident; with few rows a group of warps
// takes one row each.
int64_t bwd_blocks(int64_t rows, int64_t width) {
  const int wpr = row_warps(width), slots = wpr > 8 ? 1 : 8 / wpr;
  return std::min<int64_t>((rows + slots - 1) / slots, 2 * 148);
}

template <typename S, typename T, int WPR, int J>
cudaError_t launch_back(const Bwd& f, int64_t blocks, cudaStream_t stream) {
  if (f.a.post != 0)
    backward_kernel<S, T, WPR, J, true><<<(unsigned)blocks, bwd_threads<WPR>(), 0, stream>>>(f);
  else
    backward_kernel<S, T, WPR, J, false><<<(unsigned)blocks, bwd_threads<WPR>(), 0, stream>>>(f);
  return cudaGetLastError();
}

template <typename S, typename T>
cudaError_t launch_back_types(const Bwd& f, int64_t blocks, cudaStream_t stream) {
  const int64_t w = f.a.width;
  if (w <= 256) return launch_back<S, T, 1, 1>(f, blocks, stream);
  if (w <= 512) return launch_back<S, T, 1, 2>(f, blocks, stream);
  if (w <= 1024) return launch_back<S, T, 2, 2>(f, blocks, stream);
  if (w <= 2048) return launch_back<S, T, 4, 2>(f, blocks, stream);
  if (w <= 4096) return launch_back<S, T, 8, 2>(f, blocks, stream);
  if (w <= 8192) return launch_back<S, T, 16, 2>(f, blocks, stream);
  return launch_back<S, T, 16, 4>(f, blocks, stream);
}

cudaError_t launch_residual_norm_grad(const Bwd& f, int64_t blocks, int64_t gates,
                                      cudaStream_t stream) {
  const int s = f.a.stream_type, t = f.a.type;
  cudaError_t e;
  if (s == VGGT_DTYPE_FP32 && t == VGGT_DTYPE_FP32)
    e = launch_back_types<float, float>(f, blocks, stream);
  else if (s == VGGT_DTYPE_FP32 && t == VGGT_DTYPE_BF16)
    e = launch_back_types<float, __nv_bfloat16>(f, blocks, stream);
  else if (s == VGGT_DTYPE_FP32)
    e = launch_back_types<float, __half>(f, blocks, stream);
  else if (t == VGGT_DTYPE_BF16)
    e = launch_back_types<__nv_bfloat16, __nv_bfloat16>(f, blocks, stream);
  else
    e = launch_back_types<__half, __half>(f, blocks, stream);
  if (e != cudaSuccess) return e;
  bool any = false;
  for (int k = 0; k < kArrays; ++k) any = any || f.out[k] != nullptr;
  if (!any) return cudaSuccess;
  // gates per row are written by the first kernel
  const int64_t runs = f.a.rows_per_gate > 1 && f.out[kGate] ? gates : 0;
  const dim3 grid((unsigned)((f.a.width + 31) / 32),
                  (unsigned)(kArrays + std::min<int64_t>(runs, 4096)));
  finish_kernel<<<grid, 256, 0, stream>>>(f, blocks, gates);
  return cudaGetLastError();
}

}  // namespace rnorm
}  // namespace vggt

extern "C" size_t vggt_residual_norm_grad_workspace_size(int64_t rows, int64_t width,
                                                         int64_t rows_per_gate) {
  using namespace vggt::rnorm;
  if (rows <= 0 || width <= 0 || width > VGGT_NORM_MAX_WIDTH || rows_per_gate < 0) return 0;
  const int64_t blocks = bwd_blocks(rows, width), wpr = row_warps(width);
  const int64_t slots = blocks * (wpr > 8 ? 1 : 8 / wpr);
  int64_t lines = kArrays * blocks;
  if (rows_per_gate > 1) lines += slots + rows / rows_per_gate;
  return (size_t)(lines * ((width + 3) / 4 * 4) * 4);
}

extern "C" int vggt_residual_norm_grad(const vggt_residual_norm_args* args,
                                       const vggt_residual_norm_grads* g, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  using namespace vggt;
  using namespace vggt::rnorm;
  Bwd f{};
  if (int rc = check(args, &f.a)) return rc;
  if (!g) return api_fail("grads must be non-NULL");
  const int64_t rows = args->rows, width = args->width;
  const bool both = args->branch != nullptr;
  void* const outs[kArrays] = {args->weight.data ? g->dweight : nullptr,
                               args->bias.data ? g->dbias : nullptr,
                               args->gate.data ? g->dgate : nullptr,
                               args->post_weight.data ? g->dpost_weight : nullptr,
                               args->post_bias.data ? g->dpost_bias : nullptr};
  const vggt_vector* params[kArrays] = {&args->weight, &args->bias, &args->gate, &args->post_weight,
                                        &args->post_bias};
  const int64_t gates = f.a.rows_per_gate > 0 ? rows / f.a.rows_per_gate : 0;
  if (rows == 0) {  // the sums of no rows
    for (int k = 0; k < kArrays; ++k) {
      if (!outs[k] || (k == kGate && args->rows_per_gate > 0)) continue;
      const size_t size = params[k]->dtype == VGGT_DTYPE_FP32 ? 4 : 2;
      if (int rc = api_cuda(cudaMemsetAsync(outs[k], 0, size * width,
                                            static_cast<cudaStream_t>(stream))))
        return rc;
    }
    return api_fail(nullptr);
  }
  f.dy = g->dy;
  f.dh = g->dh;
  f.dx = g->dx;
  f.dbranch = both ? g->dbranch : nullptr;
  f.dy_stride = g->dy_stride;
  f.dh_stride = g->dh_stride;
  f.dx_stride = g->dx_stride;
  f.dbranch_stride = g->dbranch_stride;
  if (rows > 1 && ((f.dx && f.dx_stride < width) || (f.dbranch && f.dbranch_stride < width)))
    return api_fail("an output's rows overlap: its stride is below the width");
  if (rows > 1 && ((f.dy && f.dy_stride < 0) || (f.dh && f.dh_stride < 0)))
    return api_fail("negative stride");
  if (workspace_bytes < vggt_residual_norm_grad_workspace_size(rows, width, f.a.rows_per_gate) ||
      !workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u))
    return api_fail("the workspace is too small or not 16-byte aligned");
  f.a.vec = f.a.vec && wide_rows(f.dy, f.dy_stride, f.a.type) && wide_rows(f.dh, f.dh_stride, f.a.stream_type) &&
            wide_rows(f.dx, f.dx_stride, f.a.stream_type) && wide_rows(f.dbranch, f.dbranch_stride, f.a.type);
  const int64_t blocks = bwd_blocks(rows, width), wpr = row_warps(width);
  f.slots = std::min(rows, blocks * (wpr > 8 ? 1 : 8 / wpr));
  float* at = static_cast<float*>(workspace);
  for (int k = 0; k < kArrays; ++k) {
    f.out[k] = outs[k];
    f.out_type[k] = params[k]->dtype;
    f.a.vec = f.a.vec && wide_rows(outs[k], 8, f.out_type[k]);
    f.part[k] = at;
    at += (k == kGate && f.a.rows_per_gate > 1 ? f.slots + gates : blocks) * width;
    at += (4 - (at - static_cast<float*>(workspace)) % 4) % 4;
  }
  return api_cuda(launch_residual_norm_grad(f, blocks, gates, static_cast<cudaStream_t>(stream)));
}
