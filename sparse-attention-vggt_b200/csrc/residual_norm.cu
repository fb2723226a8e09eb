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

// Threads of a block.  Rows over four or eight warps wait for one another's sums, and a third slot
// fills the gaps (8,000 rows of 4096 with two norms: 51 us with 512, 45 with 768); shorter rows are
// slower for it (44,000 of 1024: 59 and 65 us).
template <int WPR, bool DIRECT>
constexpr int block_threads() {
  return !DIRECT && (WPR == 4 || WPR == 8) ? 768 : kMaxThreads;
}

template <typename S, typename T, int WPR, int J, bool DIRECT>
__global__ void __launch_bounds__(block_threads<WPR, DIRECT>(), 1) forward_kernel(const Fwd f) {
  constexpr int kThreads = block_threads<WPR, DIRECT>();
  constexpr int kX = sizeof(S) / 2, kF = sizeof(T) / 2;  // 16-byte units of 8 elements
  constexpr int kUnits = J * (kX + kF);
  typedef Shared<kThreads, WPR, J, kUnits, DIRECT> SH;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float scratch[2 * 2 * 32];
  const Args& a = f.a;
  RowSum<WPR> sum(scratch);
  const Pipe<kThreads, kUnits> pipe(smem);
  const int lane = threadIdx.x & 31, slots = (blockDim.x >> 5) / WPR;
  const float inv_width = 1.f / (float)a.width;
  const bool vec = !DIRECT || a.vec, branch = a.branch != nullptr;
  int n[J];
#pragma unroll
  for (int j = 0; j < J; ++j)
    n[j] = max(0, min(8, (int)a.width - 8 * ((j * WPR + sum.warp) * 32 + lane)));
  const int first = 8 * (sum.warp * 32 + lane);
  constexpr int step = 8 * WPR * 32;
  // The slots go over the rows side by side, which keeps what they read and write near each other
  // in memory; with a gate for each run of rows every slot takes a run of its own instead, so that
  // gates change seldom.
  const bool gates = a.gate.p != nullptr && a.rows_per_gate > 0;
  const int64_t slot = (int64_t)blockIdx.x * slots + sum.slot, all = (int64_t)gridDim.x * slots;
  int64_t row = slot, end = a.rows;
  const int64_t step_rows = gates ? 1 : all;
  if (gates) {
    row = slot * a.rows / all;
    end = (slot + 1) * a.rows / all;
  }
  grid_wait();
  const S* x = static_cast<const S*>(a.x) + row * a.x_stride + first;
  const T* b = static_cast<const T*>(a.branch) + (branch ? row * a.branch_stride + first : 0);
  S* h = static_cast<S*>(f.h) + (branch ? row * f.h_stride + first : 0);
  T* y = static_cast<T*>(f.y) + row * f.y_stride + first;
  // x and b are a row ahead where rows are copied ahead
  auto fetch = [&](bool there, int stage) {
    if (there) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        pipe.fetch(stage, j * (kX + kF), x + j * step, n[j] > 0);
        if (branch) pipe.fetch(stage, j * (kX + kF) + kX, b + j * step, n[j] > 0);
      }
      x += step_rows * a.x_stride;
      if (branch) b += step_rows * a.branch_stride;
    }
    cp_async_commit();
  };
  // what DIRECT has of the row to come: all of it at once
  Raw8 xr[J], br[J];
  auto ahead = [&] {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      xr[j].load(x, TypeOf<S>::value, j * step, n[j]);
      if (branch) br[j].load(b, TypeOf<T>::value, j * step, n[j]);
    }
  };
  if (!DIRECT) {
    pipe.clear();
    fetch(row < end, 0);
  } else if (vec && row < end) {
    ahead();
  }
  int64_t gate_row = gates ? min(row, a.rows - 1) / a.rows_per_gate : 0;
  int64_t gate_end = gates ? (gate_row + 1) * a.rows_per_gate : a.rows;
  Params<WPR, J, SH, DIRECT> params(a, smem + SH::kAfterRows, first, n, gate_row);
  if (SH::kParams) __syncthreads();
  for (int stage = 0; row < end; row += step_rows, stage ^= 1) {
    float_pair v[J][4], p[J][4];
    if (DIRECT) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (vec) {
          xr[j].convert(v[j]);
          if (branch) br[j].convert(p[j]);
        } else {
          get_pairs(x + j * step, n[j], false, v[j]);
          if (branch) get_pairs(b + j * step, n[j], false, p[j]);
        }
      }
      x += step_rows * a.x_stride;
      if (branch) b += step_rows * a.branch_stride;
      if (vec && row + step_rows < end) ahead();
    } else {
      __syncwarp();  // all lanes are done with the stage
      fetch(row + step_rows < end, stage ^ 1);
      cp_async_wait<1>();
      __syncwarp();
#pragma unroll
      for (int j = 0; j < J; ++j) {
        pipe.template read<S>(stage, j * (kX + kF), v[j]);
        pipe.template read<T>(stage, j * (kX + kF) + kX, p[j]);
      }
    }
    if (branch) {
      if (a.post != 0) {
        norm_row<!DIRECT, WPR, J>(p, n, a.post, inv_width, a.eps, sum);
#pragma unroll
        for (int j = 0; j < J; ++j) {
          params.scale(kPostWeight, j, p[j]);
          params.shift(kPostBias, j, p[j]);
        }
      }
      if (gates && row == gate_end) {
        gate_end += a.rows_per_gate;
        params.turn_to(++gate_row);
      }
#pragma unroll
      for (int j = 0; j < J; ++j) {
        params.gated(j, p[j], v[j]);
        if (DIRECT)
          put_pairs<false>(h + j * step, n[j], vec, v[j]);
        else
          pipe.store(stage, j * (kX + kF), h + j * step, n[j] > 0, v[j]);
      }
      h += step_rows * f.h_stride;
    }
    norm_row<!DIRECT, WPR, J>(v, n, a.norm, inv_width, a.eps, sum);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      params.scale(kWeight, j, v[j]);
      params.shift(kBias, j, v[j]);
      if (DIRECT)
        put_pairs<false>(y + j * step, n[j], vec, v[j]);
      else
        pipe.store(stage, j * (kX + kF) + (sizeof(S) == 4 && sizeof(T) == 4 ? kX : 0), y + j * step,
                   n[j] > 0, v[j]);
    }
    y += step_rows * f.y_stride;
  }
}

template <typename S, typename T, int WPR, int J, bool DIRECT>
cudaError_t launch_shape(const Fwd& f, int64_t blocks, int slots, cudaStream_t stream) {
  constexpr uint32_t bytes =
      Shared<block_threads<WPR, DIRECT>(), WPR, J, J*(sizeof(S) / 2 + sizeof(T) / 2),
             DIRECT>::kBytes;
  auto k = forward_kernel<S, T, WPR, J, DIRECT>;
  static OncePerDevice allowed;
  if (cudaError_t e = allow_shared(k, (int)bytes, &allowed)) return e;
  return launch_early(k, dim3((unsigned)blocks), dim3(slots * WPR * 32), bytes, stream, f);
}

// Rows copied ahead where they are aligned, fit and are more than the slots; false where not.
template <typename S, typename T, int WPR, int J>
bool launch_ahead(const Fwd& f, int sms, cudaStream_t stream, cudaError_t* e) {
  constexpr int threads = block_threads<WPR, false>(), slots = threads / 32 / WPR;
  if constexpr (Shared<threads, WPR, J, J*(sizeof(S) / 2 + sizeof(T) / 2), false>::kFits)
    if (f.a.vec && f.a.rows > (int64_t)sms * slots) {
      *e = launch_shape<S, T, WPR, J, false>(f, sms, slots, stream);
      return true;
    }
  return false;
}

// Rows read straight into registers: few rows spread over the SMs, each with a slot of its own.
template <typename S, typename T, int WPR, int J>
cudaError_t launch_direct(const Fwd& f, int sms, cudaStream_t stream) {
  constexpr int most = kMaxThreads / 32 / WPR;
  const int slots = (int)std::min<int64_t>(most, (f.a.rows + sms - 1) / sms);
  const int64_t blocks = std::min<int64_t>(sms, (f.a.rows + slots - 1) / slots);
  return launch_shape<S, T, WPR, J, true>(f, blocks, slots, stream);
}

template <typename S, typename T>
cudaError_t launch_types(const Fwd& f, int sms, cudaStream_t stream) {
  const int64_t w = f.a.width;
  cudaError_t e = cudaSuccess;
  if (w <= 256    ? launch_ahead<S, T, 1, 1>(f, sms, stream, &e)
      : w <= 512  ? launch_ahead<S, T, 1, 2>(f, sms, stream, &e)
      : w <= 1024 ? launch_ahead<S, T, 2, 2>(f, sms, stream, &e)
      : w <= 2048 ? launch_ahead<S, T, 4, 2>(f, sms, stream, &e)
      : w <= 4096 ? launch_ahead<S, T, 8, 2>(f, sms, stream, &e)
      : w <= 8192 ? launch_ahead<S, T, 16, 2>(f, sms, stream, &e)
                  : launch_ahead<S, T, 16, 4>(f, sms, stream, &e))
    return e;
  if (w <= 256) return launch_direct<S, T, 1, 1>(f, sms, stream);
  if (w <= 512) return launch_direct<S, T, 1, 2>(f, sms, stream);
  if (w <= 1024) return launch_direct<S, T, 2, 2>(f, sms, stream);
  if (w <= 2048) return launch_direct<S, T, 4, 2>(f, sms, stream);
  if (w <= 4096) return launch_direct<S, T, 8, 2>(f, sms, stream);
  if (w <= 8192) return launch_direct<S, T, 16, 2>(f, sms, stream);
  return launch_direct<S, T, 16, 4>(f, sms, stream);
}

}  // namespace rnorm

cudaError_t device_sms(int* sms) {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  if (dev < 64 && (*sms = known[dev].load(std::memory_order_relaxed)) > 0) return cudaSuccess;
  const cudaError_t e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess && dev < 64) known[dev].store(*sms, std::memory_order_relaxed);
  return e;
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
