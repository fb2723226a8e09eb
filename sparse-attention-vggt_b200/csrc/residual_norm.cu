// The gated residual with the norms around it, forward (residual_norm.cuh has the formulas).
//
// Bound by memory: x and branch are read once, h and y written once, and everything between lies
// in registers.
#include <algorithm>

#include "kernels.h"
#include "residual_norm.cuh"

namespace vggt {
namespace rnorm {

struct Fwd {
  Args a;
  void* h;
  void* y;
  int64_t h_stride, y_stride;
};

template <typename S, typename T, int WPR, int J>
__global__ void __launch_bounds__(WPR > 8 ? WPR * 32 : 256) forward_kernel(const Fwd f) {
  __shared__ float scratch[2 * 2 * 32];
  const Args& a = f.a;
  RowSum<WPR> sum(scratch);
  const int lane = threadIdx.x & 31, slots = (blockDim.x >> 5) / WPR;
  const float inv_width = 1.f / (float)a.width;
  const bool vec = a.vec;
  int n[J];
#pragma unroll
  for (int j = 0; j < J; ++j)
    n[j] = max(0, min(8, (int)a.width - 8 * ((j * WPR + sum.warp) * 32 + lane)));
  const int first = 8 * (sum.warp * 32 + lane);
  constexpr int step = 8 * WPR * 32;
  for (int64_t row = (int64_t)blockIdx.x * slots + sum.slot; row < a.rows;
       row += (int64_t)gridDim.x * slots) {
    float v[J][8];
    const S* x = static_cast<const S*>(a.x) + row * a.x_stride + first;
#pragma unroll
    for (int j = 0; j < J; ++j) get8(x + j * step, n[j], vec, v[j]);
    if (a.branch != nullptr) {
      float p[J][8];
      const T* b = static_cast<const T*>(a.branch) + row * a.branch_stride + first;
#pragma unroll
      for (int j = 0; j < J; ++j) get8(b + j * step, n[j], vec, p[j]);
      if (a.post != 0) {
        norm_row<WPR, J>(p, n, a.post, inv_width, a.eps, sum);
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
      const int64_t at = a.rows_per_gate > 0 ? row / a.rows_per_gate * a.width : 0;
      S* h = static_cast<S*>(f.h) + row * f.h_stride + first;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (a.gate.p != nullptr) {
          float g[8];
          get_param8(a.gate, at + first + j * step, n[j], vec, g);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j][i] = fmaf(g[i], p[j][i], v[j][i]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j][i] += p[j][i];
        }
        put8(h + j * step, n[j], vec, v[j]);
      }
    }
    norm_row<WPR, J>(v, n, a.norm, inv_width, a.eps, sum);
    T* y = static_cast<T*>(f.y) + row * f.y_stride + first;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (a.weight.p != nullptr) {
        float w[8];
        get_param8(a.weight, first + j * step, n[j], vec, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] *= w[i];
      }
      if (a.bias.p != nullptr) {
        float w[8];
        get_param8(a.bias, first + j * step, n[j], vec, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] += w[i];
      }
      put8(y + j * step, n[j], vec, v[j]);
    }
  }
}

template <typename S, typename T, int WPR, int J>
cudaError_t launch_shape(const Fwd& f, int sms, cudaStream_t stream) {
  const int threads = WPR > 8 ? WPR * 32 : 256, slots = threads / 32 / WPR;
  const int64_t blocks = std::min<int64_t>((f.a.rows + slots - 1) / slots, (int64_t)sms * 32);
  forward_kernel<S, T, WPR, J><<<(unsigned)blocks, threads, 0, stream>>>(f);
  return cudaGetLastError();
}

template <typename S, typename T>
cudaError_t launch_types(const Fwd& f, int sms, cudaStream_t stream) {
  const int64_t w = f.a.width;
  if (w <= 256) return launch_shape<S, T, 1, 1>(f, sms, stream);
  if (w <= 1024) return launch_shape<S, T, 1, 4>(f, sms, stream);
  if (w <= 2048) return launch_shape<S, T, 2, 4>(f, sms, stream);
  if (w <= 4096) return launch_shape<S, T, 4, 4>(f, sms, stream);
  if (w <= 8192) return launch_shape<S, T, 8, 4>(f, sms, stream);
  return launch_shape<S, T, 16, 4>(f, sms, stream);
}

}  // namespace rnorm

cudaError_t device_sms(int* sms) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  return e != cudaSuccess ? e
                          : cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
}

static cudaError_t launch_residual_norm(const rnorm::Fwd& f, int sms, cudaStream_t stream) {
  const int s = f.a.stream_type, t = f.a.type;
  if (s == VGGT_DTYPE_FP32 && t == VGGT_DTYPE_FP32)
    return rnorm::launch_types<float, float>(f, sms, stream);
  if (s == VGGT_DTYPE_FP32 && t == VGGT_DTYPE_BF16)
    return rnorm::launch_types<float, __nv_bfloat16>(f, sms, stream);
  if (s == VGGT_DTYPE_FP32) return rnorm::launch_types<float, __half>(f, sms, stream);
  if (t == VGGT_DTYPE_BF16) return rnorm::launch_types<__nv_bfloat16, __nv_bfloat16>(f, sms, stream);
  return rnorm::launch_types<__half, __half>(f, sms, stream);
}

}  // namespace vggt

namespace vggt {
namespace rnorm {

// Argument checks that both directions share; fills `a`.
int check(const vggt_residual_norm_args* c, Args* a) {
  if (c == nullptr) return api_fail("args must be non-NULL");
  const int s = c->stream_dtype, t = c->dtype;
  auto known = [](int d) {
    return d == VGGT_DTYPE_BF16 || d == VGGT_DTYPE_FP16 || d == VGGT_DTYPE_FP32;
  };
  if (!known(s) || !known(t) || (s != t && s != VGGT_DTYPE_FP32))
    return api_fail("residual_norm takes BF16, FP16 or FP32, and a stream of the same type or FP32");
  if (c->rows < 0) return api_fail("negative number of rows");
  if (c->width < 1 || c->width > VGGT_NORM_MAX_WIDTH)
    return api_fail("width %lld is not in [1, %d]", (long long)c->width, VGGT_NORM_MAX_WIDTH);
  if (c->norm != VGGT_NORM_LAYER && c->norm != VGGT_NORM_RMS)
    return api_fail("norm must be VGGT_NORM_LAYER or VGGT_NORM_RMS");
  if (c->post_norm < VGGT_NORM_NONE || c->post_norm > VGGT_NORM_RMS)
    return api_fail("unknown post_norm %d", c->post_norm);
  if (!(c->eps >= 0.f)) return api_fail("eps must not be negative");
  if (c->rows > 0 && c->branch == nullptr && (c->gate.data || c->post_norm != VGGT_NORM_NONE))
    return api_fail("gate and post_norm need a branch");
  if (c->post_norm == VGGT_NORM_NONE && (c->post_weight.data || c->post_bias.data))
    return api_fail("post_weight and post_bias need a post_norm");
  if (c->gate.data && c->rows_per_gate != 0 &&
      (c->rows_per_gate < 0 || c->rows % c->rows_per_gate != 0))
    return api_fail("rows (%lld) must be a multiple of rows_per_gate (%lld)", (long long)c->rows,
                    (long long)c->rows_per_gate);
  for (const vggt_vector* v : {&c->gate, &c->weight, &c->bias, &c->post_weight, &c->post_bias})
    if (v->data && !known(v->dtype)) return api_fail("unknown parameter type %d", v->dtype);
  if (c->rows > 0) {
    if (!c->x) return api_fail("x must be non-NULL");
    if (c->rows > 1 && (c->x_stride < 0 || (c->branch && c->branch_stride < 0)))
      return api_fail("negative stride");
  }
  auto param = [](const vggt_vector& v) { return Param{v.data, v.dtype}; };
  *a = Args{};
  a->x = c->x;
  a->branch = c->branch;
  a->gate = param(c->gate);
  a->weight = param(c->weight);
  a->bias = param(c->bias);
  a->post_weight = param(c->post_weight);
  a->post_bias = param(c->post_bias);
  a->rows = c->rows;
  a->width = c->width;
  a->x_stride = c->x_stride;
  a->branch_stride = c->branch_stride;
  a->rows_per_gate = c->gate.data ? c->rows_per_gate : 0;
  a->stream_type = s;
  a->type = t;
  a->norm = c->norm;
  a->post = c->branch ? c->post_norm : VGGT_NORM_NONE;
  a->eps = c->eps;
  a->vec = c->width % 8 == 0 && wide_rows(c->x, c->x_stride, s) && wide_rows(c->branch, c->branch_stride, t);
  for (const Param* q : {&a->gate, &a->weight, &a->bias, &a->post_weight, &a->post_bias})
    a->vec = a->vec && wide_rows(q->p, 8, q->type);
  return 0;
}

}  // namespace rnorm
}  // namespace vggt

extern "C" int vggt_residual_norm(const vggt_residual_norm_args* args, void* h, int64_t h_stride,
                                  void* y, int64_t y_stride, void* stream) {
  using namespace vggt;
  rnorm::Fwd f;
  if (int rc = rnorm::check(args, &f.a)) return rc;
  if (args->rows == 0) return api_fail(nullptr);
  const bool both = args->branch != nullptr;
  if (!y || (both && !h)) return api_fail("y, and h where there is a branch, must be non-NULL");
  if (args->rows > 1 && (y_stride < args->width || (both && h_stride < args->width)))
    return api_fail("an output's rows overlap: its stride is below the width");
  f.h = both ? h : nullptr;
  f.y = y;
  f.h_stride = h_stride;
  f.y_stride = y_stride;
  f.a.vec = f.a.vec && wide_rows(f.h, h_stride, f.a.stream_type) &&
            wide_rows(y, y_stride, f.a.type);
  int sms = 0;
  if (int rc = api_cuda(device_sms(&sms))) return rc;
  return api_cuda(launch_residual_norm(f, sms, static_cast<cudaStream_t>(stream)));
}
