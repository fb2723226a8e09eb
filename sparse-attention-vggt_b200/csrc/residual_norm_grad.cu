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
// registers of WPR warps, 8 or 16 elements a lane: the row's values and the parameters' sums, three
// to five fp32 numbers an element, fit together.  Each group of warps takes rows of its own; its
// parameters' sums are added over the block's groups in shared memory and written as one partial
// per block, which a second kernel adds in order.  No atomics: equal calls give equal bits.
#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "residual_norm.cuh"

namespace vggt {
namespace rnorm {

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
  int64_t slots;           // slots that have rows; with gates of runs of rows slot s takes the rows
                           // [s rows / slots, (s + 1) rows / slots), else every slots-th row
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

// The gradient of what was normed to hat, from that of hat (d, in place).
template <bool VEC, int WPR, int J>
__device__ __forceinline__ void norm_back(float_pair (*d)[4], const float_pair (*hat)[4],
                                          const int* n, int kind, float r, float inv_width,
                                          RowSum<WPR>& sum) {
  float_pair s2 = both(0.f), t2 = both(0.f);
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s2 = fma_pair(d[j][i], hat[j][i], s2);
      t2 = add_pair(t2, d[j][i]);
    }
  float s = sum_pair(s2), t = sum_pair(t2);
  sum.two(s, t);
  const float_pair m = both(-s * inv_width), rr = both(r);
  t *= inv_width;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    if (kind == kNormLayer) subtract<VEC>(d[j], n[j], t);
#pragma unroll
    for (int i = 0; i < 4; ++i) d[j][i] = mul_pair(rr, fma_pair(hat[j][i], m, d[j][i]));
  }
}

// POST: a norm of the branch.  Its sums are three without biases (POST 1) or five (2);
// without it they are three.
template <int POST>
constexpr int acc_of(int k) {
  return POST != 1 ? k : k == kWeight ? 0 : k == kGate ? 1 : k == kPostWeight ? 2 : -1;
}

template <typename S, typename T, int WPR, int J, int POST, bool DIRECT>
__global__ void __launch_bounds__(kMaxThreads, 1) backward_kernel(const Bwd f) {
  constexpr int kAccs = POST == 2 ? 5 : 3;
  constexpr int kGateAcc = acc_of<POST>(kGate), kPostAcc = POST ? acc_of<POST>(kPostWeight) : 0;
  constexpr int kRow = WPR * 32 * 8 * J;  // columns that a slot holds
  constexpr int kX = sizeof(S) / 2, kF = sizeof(T) / 2, kUnits = 2 * (kX + kF);
  typedef Shared<kMaxThreads, WPR, J, J * kUnits, DIRECT> SH;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float scratch[2 * 2 * 32];
  float* fold = reinterpret_cast<float*>(smem);  // after the rows
  const Args& a = f.a;
  RowSum<WPR> sum(scratch);
  const Pipe<kMaxThreads, J * kUnits> pipe(smem);
  const int slots = (blockDim.x >> 5) / WPR;
  const int lane = threadIdx.x & 31;
  const float inv_width = 1.f / (float)a.width;
  const bool vec = !DIRECT || a.vec, branch = a.branch != nullptr, has_dy = f.dy != nullptr,
             has_dh = f.dh != nullptr;
  int n[J];
#pragma unroll
  for (int j = 0; j < J; ++j)
    n[j] = max(0, min(8, (int)a.width - 8 * ((j * WPR + sum.warp) * 32 + lane)));
  const int first = 8 * (sum.warp * 32 + lane);
  constexpr int step = 8 * WPR * 32;
  const int64_t slot = (int64_t)blockIdx.x * slots + sum.slot;
  // side by side over the rows, or with a gate for each run of rows a run to a slot, as forward
  const bool gates = a.gate.p != nullptr && a.rows_per_gate > 0;
  int64_t row0 = 0, row1 = 0;
  const int64_t step_rows = gates ? 1 : f.slots;
  if (slot < f.slots) {
    row0 = gates ? slot * a.rows / f.slots : slot;
    row1 = gates ? (slot + 1) * a.rows / f.slots : a.rows;
  }

  grid_wait();
  float_pair acc[kAccs][J][4];
#pragma unroll
  for (int k = 0; k < kAccs; ++k)
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[k][j][i] = both(0.f);

  // a row of a tensor (one that is not there is not read); addresses are formed where they are
  // used, which takes fewer registers than six running pointers
  auto at = [&](auto* p, int64_t row, int64_t stride) { return p + (row * stride + first); };
  auto x = [&](int64_t row) { return at(static_cast<const S*>(a.x), row, a.x_stride); };
  auto b = [&](int64_t row) { return at(static_cast<const T*>(a.branch), row, a.branch_stride); };
  auto dy = [&](int64_t row) { return at(static_cast<const T*>(f.dy), row, f.dy_stride); };
  auto dh = [&](int64_t row) { return at(static_cast<const S*>(f.dh), row, f.dh_stride); };
  auto fetch = [&](int64_t row, int stage) {
    if (row < row1) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const bool in = n[j] > 0;
        pipe.fetch(stage, j * kUnits, x(row) + j * step, in);
        if (branch) pipe.fetch(stage, j * kUnits + kX, b(row) + j * step, in);
        if (has_dy) pipe.fetch(stage, j * kUnits + kX + kF, dy(row) + j * step, in);
        if (has_dh) pipe.fetch(stage, j * kUnits + kX + 2 * kF, dh(row) + j * step, in);
      }
    }
    cp_async_commit();
  };
  // chunk j of one of the row's four tensors; DIRECT has asked for the row's before
  Raw8 raw[DIRECT ? 4 : 1][DIRECT ? J : 1];
  auto ask = [&](int64_t row) {
#pragma unroll
    for (int j = 0; j < (DIRECT ? J : 0); ++j) {
      raw[0][j].load(x(row), TypeOf<S>::value, j * step, n[j]);
      if (branch) raw[DIRECT ? 1 : 0][j].load(b(row), TypeOf<T>::value, j * step, n[j]);
      if (has_dy) raw[DIRECT ? 2 : 0][j].load(dy(row), TypeOf<T>::value, j * step, n[j]);
      if (has_dh) raw[DIRECT ? 3 : 0][j].load(dh(row), TypeOf<S>::value, j * step, n[j]);
    }
  };
  auto take = [&](auto* p, int stage, int which, int j, float_pair* v) {
    typedef std::remove_cv_t<std::remove_pointer_t<decltype(p)>> E;
    constexpr int unit[4] = {0, kX, kX + kF, kX + 2 * kF};
    if (!DIRECT)
      pipe.template read<E>(stage, j * kUnits + unit[which], v);
    else if (vec)
      raw[DIRECT ? which : 0][DIRECT ? j : 0].convert(v);
    else
      get_pairs(p + j * step, n[j], false, v);
  };

  int64_t gate_row = gates ? row0 / a.rows_per_gate : 0;
  int64_t gate_end = gates ? (gate_row + 1) * a.rows_per_gate : row1;  // the run's end
  if (!DIRECT) {
    pipe.clear();
    fetch(row0, 0);
  } else if (vec && row0 < row1) {
    ask(row0);
  }
  Params<WPR, J, SH, DIRECT> params(a, smem + SH::kAfterRows, first, n, gate_row);
  if (SH::kParams) __syncthreads();
  int stage = 0;
  for (int64_t row = row0; row < row1; row += step_rows, stage ^= 1) {
    if (!DIRECT) {
      __syncwarp();  // all lanes are done with the stage
      fetch(row + step_rows, stage ^ 1);
      cp_async_wait<1>();
      __syncwarp();
    } else if (vec && row > row0) {
      ask(row);
    }
    // the branch: as it is, or normed; what is added is formed from it again where it is needed
    float_pair h[J][4], p[J][4], d[J][4];
    auto added = [&](int j, float_pair* v) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = p[j][i];
      if (POST) {
        params.scale(kPostWeight, j, v);
        params.shift(kPostBias, j, v);
      }
    };
#pragma unroll
    for (int j = 0; j < J; ++j) take(x(row), stage, 0, j, h[j]);
    float pr = 0.f;
    if (branch) {
#pragma unroll
      for (int j = 0; j < J; ++j) take(b(row), stage, 1, j, p[j]);
      if (POST) pr = norm_row<!DIRECT, WPR, J>(p, n, a.post, inv_width, a.eps, sum);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        float_pair v[4];
        added(j, v);
        params.gated(j, v, h[j]);
      }
    }
    const float r = norm_row<!DIRECT, WPR, J>(h, n, a.norm, inv_width, a.eps, sum);  // h is normed now
    if (has_dy) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        take(dy(row), stage, 2, j, d[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float_pair& w = acc[acc_of<POST>(kWeight)][j][i];
          w = fma_pair(d[j][i], h[j][i], w);
          if (POST != 1) acc[kBias % kAccs][j][i] = add_pair(acc[kBias % kAccs][j][i], d[j][i]);
        }
        params.scale(kWeight, j, d[j]);
      }
      norm_back<!DIRECT, WPR, J>(d, h, n, a.norm, r, inv_width, sum);
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) d[j][i] = both(0.f);
    }
    if (has_dh) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        float_pair t[4];
        take(dh(row), stage, 3, j, t);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[j][i] = add_pair(d[j][i], t[i]);
      }
    }
    if (f.dx != nullptr) {
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (DIRECT)
          put_pairs<false>(at(static_cast<S*>(f.dx), row, f.dx_stride) + j * step, n[j], vec, d[j]);
        else
          pipe.store(stage, j * kUnits, at(static_cast<S*>(f.dx), row, f.dx_stride) + j * step,
                     n[j] > 0, d[j]);
    }
    if (!branch) continue;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float_pair v[4];
      added(j, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float_pair& g = acc[kGateAcc][j][i];
        g = fma_pair(d[j][i], v[i], g);
      }
      params.scale(kGate, j, d[j]);
    }
    if (POST) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float_pair& w = acc[kPostAcc][j][i];
          w = fma_pair(d[j][i], p[j][i], w);
          if (POST == 2) acc[kPostBias % kAccs][j][i] = add_pair(acc[kPostBias % kAccs][j][i], d[j][i]);
        }
        params.scale(kPostWeight, j, d[j]);
      }
      norm_back<!DIRECT, WPR, J>(d, p, n, a.post, pr, inv_width, sum);
    }
    if (f.dbranch != nullptr) {
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (DIRECT)
          put_pairs<false>(at(static_cast<T*>(f.dbranch), row, f.dbranch_stride) + j * step, n[j], vec,
                           d[j]);
        else
          pipe.store(stage, j * kUnits + kX,
                     at(static_cast<T*>(f.dbranch), row, f.dbranch_stride) + j * step, n[j] > 0, d[j]);
    }
    if (gates && (row + 1 == row1 || row + 1 == gate_end)) {
      // the last row here of a run of rows with one gate: its sum goes out
      if (f.out[kGate] != nullptr) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int64_t c = first + j * step;
          if (a.rows_per_gate == 1) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) unpack_pair(v[2 * i], v[2 * i + 1], acc[kGateAcc][j][i]);
            put_param8(f.out[kGate], f.out_type[kGate], gate_row * a.width + c, n[j], vec, v);
          } else {
            put_pairs<!DIRECT>(f.part[kGate] + (slot + gate_row) * a.width + c, n[j], vec, acc[kGateAcc][j]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[kGateAcc][j][i] = both(0.f);
        }
      }
      ++gate_row;
      gate_end += a.rows_per_gate;
      if (row + 1 < row1) params.turn_to(gate_row);
    }
  }
  cp_async_wait<0>();

#pragma unroll
  for (int k = 0; k < (POST ? kArrays : 3); ++k) {
    constexpr int kLast = kAccs - 1;
    const int q = acc_of<POST>(k);  // known at compile time
    if (q < 0 || f.out[k] == nullptr || (k == kGate && gates)) continue;  // the same for all threads
    const float_pair(&sums)[J][4] = acc[q < 0 ? kLast : q];
    float* to = f.part[k] + (int64_t)blockIdx.x * a.width;
    if (slots == 1) {
#pragma unroll
      for (int j = 0; j < J; ++j) put_pairs<!DIRECT>(to + first + j * step, n[j], vec, sums[j]);
    } else {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < J; ++j)
        put_pairs<true>(fold + sum.slot * kRow + first + j * step, 8, true, sums[j]);
      __syncthreads();
      for (int c = threadIdx.x; c < (int)a.width; c += blockDim.x) {
        float s = 0.f;
        for (int o = 0; o < slots; ++o) s += fold[o * kRow + c];
        to[c] = s;
      }
    }
  }
}

// Adds the partial sums: blockIdx.y below kArrays an array over all blocks, from kArrays on the
// gates of runs of rows.  32 columns x 8 lanes over the partials.
__global__ void __launch_bounds__(256) finish_kernel(const Bwd f, int64_t blocks, int64_t gates) {
  __shared__ float fold[8][32];
  grid_wait();
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

// Blocks of a call and slots of a block: one full block to an SM; few rows are spread over the SMs.
struct Grid {
  int64_t blocks;
  int slots;
};
Grid grid_of(int64_t rows, int64_t width, int post) {
  constexpr int sms = 148;
  const int most = kMaxThreads / 32 / row_warps(width, post == 2);
  const int slots = (int)std::min<int64_t>(most, (rows + sms - 1) / sms);
  return {std::min<int64_t>(sms, (rows + slots - 1) / slots), slots};
}

template <typename S, typename T, int WPR, int J, int POST, bool DIRECT>
cudaError_t launch_grid(const Bwd& f, const Grid& g, cudaStream_t stream) {
  constexpr uint32_t rows = Shared<kMaxThreads, WPR, J, J*(sizeof(S) + sizeof(T)), DIRECT>::kBytes;
  constexpr uint32_t fold = kMaxThreads * 8 * J * 4;
  constexpr uint32_t bytes = rows > fold ? rows : fold;
  auto k = backward_kernel<S, T, WPR, J, POST, DIRECT>;
  static OncePerDevice allowed;
  if (cudaError_t e = allow_shared(k, (int)bytes, &allowed)) return e;
  return launch_early(k, dim3((unsigned)g.blocks), dim3(g.slots * WPR * 32), bytes, stream, f);
}

template <typename S, typename T, int WPR, int J, int POST>
cudaError_t launch_back(const Bwd& f, const Grid& g, cudaStream_t stream) {
  constexpr bool fits = Shared<kMaxThreads, WPR, J, J*(sizeof(S) + sizeof(T)), false>::kFits;
  if constexpr (fits)
    if (f.a.vec && f.a.rows > g.blocks * g.slots)
      return launch_grid<S, T, WPR, J, POST, false>(f, g, stream);
  return launch_grid<S, T, WPR, J, POST, true>(f, g, stream);
}

template <typename S, typename T, int POST>
cudaError_t launch_back_wide(const Bwd& f, const Grid& g, cudaStream_t stream) {
  const int64_t w = f.a.width;
  if (w <= 256) return launch_back<S, T, 1, 1, POST>(f, g, stream);
  if (w <= 512) return launch_back<S, T, 1, 2, POST>(f, g, stream);
  if (w <= 1024) return launch_back<S, T, 2, 2, POST>(f, g, stream);
  if (w <= 2048) return launch_back<S, T, 4, 2, POST>(f, g, stream);
  if (w <= 4096) return launch_back<S, T, 8, 2, POST>(f, g, stream);
  if (w <= 8192) return launch_back<S, T, 16, 2, POST>(f, g, stream);
  return launch_back<S, T, 16, 4, POST>(f, g, stream);
}

template <typename S, typename T>
cudaError_t launch_back_types(const Bwd& f, const Grid& g, int post, cudaStream_t stream) {
  const int64_t w = f.a.width;
  if (post == 0) return launch_back_wide<S, T, 0>(f, g, stream);
  if (post == 1) return launch_back_wide<S, T, 1>(f, g, stream);
  if (w <= 256) return launch_back<S, T, 1, 1, 2>(f, g, stream);
  if (w <= 512) return launch_back<S, T, 2, 1, 2>(f, g, stream);
  if (w <= 1024) return launch_back<S, T, 4, 1, 2>(f, g, stream);
  if (w <= 2048) return launch_back<S, T, 8, 1, 2>(f, g, stream);
  if (w <= 4096) return launch_back<S, T, 16, 1, 2>(f, g, stream);
  if (w <= 8192) return launch_back<S, T, 16, 2, 2>(f, g, stream);
  return launch_back<S, T, 16, 4, 2>(f, g, stream);
}

cudaError_t launch_residual_norm_grad(const Bwd& f, const Grid& g, int post, int64_t gates,
                                      cudaStream_t stream) {
  const int s = f.a.stream_type, t = f.a.type;
  cudaError_t e;
  if (s == VGGT_DTYPE_FP32 && t == VGGT_DTYPE_FP32)
    e = launch_back_types<float, float>(f, g, post, stream);
  else if (s == VGGT_DTYPE_FP32 && t == VGGT_DTYPE_BF16)
    e = launch_back_types<float, __nv_bfloat16>(f, g, post, stream);
  else if (s == VGGT_DTYPE_FP32)
    e = launch_back_types<float, __half>(f, g, post, stream);
  else if (t == VGGT_DTYPE_BF16)
    e = launch_back_types<__nv_bfloat16, __nv_bfloat16>(f, g, post, stream);
  else
    e = launch_back_types<__half, __half>(f, g, post, stream);
  if (e != cudaSuccess) return e;
  bool any = false;
  for (int k = 0; k < kArrays; ++k) any = any || f.out[k] != nullptr;
  if (!any) return cudaSuccess;
  // gates per row are written by the first kernel
  const int64_t runs = f.a.rows_per_gate > 1 && f.out[kGate] ? gates : 0;
  const dim3 grid((unsigned)((f.a.width + 31) / 32),
                  (unsigned)(kArrays + std::min<int64_t>(runs, 4096)));
  return launch_early(finish_kernel, grid, dim3(256), 0, stream, f, g.blocks, gates);
}

}  // namespace rnorm
}  // namespace vggt

extern "C" size_t vggt_residual_norm_grad_workspace_size(int64_t rows, int64_t width,
                                                         int64_t rows_per_gate) {
  using namespace vggt::rnorm;
  if (rows <= 0 || width <= 0 || width > VGGT_NORM_MAX_WIDTH || rows_per_gate < 0) return 0;
  // the kernel that takes most
  size_t most = 0;
  for (int post = 0; post < 3; ++post) {
    const Grid g = grid_of(rows, width, post);
    int64_t lines = kArrays * g.blocks;
    if (rows_per_gate > 1) lines += g.blocks * g.slots + rows / rows_per_gate;
    most = std::max(most, (size_t)(lines * ((width + 3) / 4 * 4) * 4));
  }
  return most;
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
  // by what the call has, not by what is wanted of it: the kernels add in different orders, and a
  // gradient is the same alone and among others (where biases are there and their gradients are not
  // wanted, the kernel without their sums would be faster: 7,996 x 4096 with the forward pass 206 us
  // against 241, 30,000 x 1024 174 against 195)
  const bool biases = args->bias.data != nullptr || args->post_bias.data != nullptr;
  const int post = f.a.post == 0 ? 0 : biases ? 2 : 1;
  const Grid grid = grid_of(rows, width, post);
  f.slots = std::min(rows, grid.blocks * grid.slots);
  float* at = static_cast<float*>(workspace);
  for (int k = 0; k < kArrays; ++k) {
    f.out[k] = outs[k];
    f.out_type[k] = params[k]->dtype;
    f.a.vec = f.a.vec && wide_rows(outs[k], 8, f.out_type[k]);
    f.part[k] = at;
    at += (k == kGate && f.a.rows_per_gate > 1 ? f.slots + gates : grid.blocks) * width;
    at += (4 - (at - static_cast<float*>(workspace)) % 4) % 4;
  }
  return api_cuda(launch_residual_norm_grad(f, grid, post, gates, static_cast<cudaStream_t>(stream)));
}
