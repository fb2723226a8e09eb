// Gradients of y = residual + gate * act(x W^T + b).
//
// With an activation: dz = dy gate act'(z) and, from z, dgate = sum dy act(z); then
//   dx = dz W,  dW = dz^T x,  db = sum dz.
// Without one, z is not needed.  With G = dy^T x and s = sum dy (over the rows),
//   dW = gate G,  db = gate s,  dgate_n = <W_n, G_n> + b_n s_n,  dx = dy (gate W):
// the only pass over [rows][outer] beside the two products is the one that forms s.
//
// dW is a product over the rows.  Its epilogue scales the rows by the gate and sums their products
// with W's rows for dgate.  Where its tiles are few it is cut evenly over the SMs, and the partial
// sums lie in fp32 in the workspace until finish_weight adds them and does the same.  Nothing is
// added with atomics: equal calls give equal bits.
#include <algorithm>
#include <type_traits>

#include "activation.cuh"
#include "linear.cuh"

namespace vggt {
namespace lin {

// The pass over dy: column sums of dz (and of dy act(z)) per block of rows, and dz rounded for the
// products.  A thread takes 8 columns of every 8th row of its block.
struct Sums {
  const void* dy;
  int64_t dy_stride;
  const void* z;
  int64_t z_stride;
  const void* gate;
  bool gate_fp32;
  int act;
  void* dz;      // [rows][dz_stride], or null
  void* scaled;  // gate dy (no activation), or null
  int64_t dz_stride;
  float* bias_part;  // [row blocks][outer], or null
  float* gate_part;
  int64_t rows, outer, per_block;
  bool wide;
};

template <typename S, typename Z, typename T, int ACT, bool WIDE>
__global__ void __launch_bounds__(256, ACT == VGGT_ACT_NONE ? 4 : 2) sums_kernel(const Sums a) {
  __shared__ float fold[8][256];
  // rows whose loads are in flight (with a branch for unaligned ones in the loop none were, and
  // the sums of 22,000 x 1024 took 34 us)
  constexpr int kAhead = 4;
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int64_t c = ((int64_t)blockIdx.x * 32 + cx) * 8;
  const int n = (int)max((int64_t)0, min((int64_t)8, a.outer - c));
  const int64_t r0 = blockIdx.y * a.per_block, r1 = min(a.rows, r0 + a.per_block);
  float sb[8], sg[8], gate[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sb[i] = sg[i] = 0.f, gate[i] = 1.f;
  auto get = [&](const auto* p, float* v) {
    typedef std::remove_cv_t<std::remove_pointer_t<decltype(p)>> E;
    if (WIDE)
      Elem<E>::load8(p, v);
    else
      get8(p, n, false, v);
  };
  if (n > 0) {
    if (a.gate != nullptr) vector_get8<T>(a.gate, a.gate_fp32, c, n, WIDE, gate);
    for (int64_t rr = r0 + ry; rr < r1; rr += 8 * kAhead) {
      float d[kAhead][8], z[ACT != VGGT_ACT_NONE ? kAhead : 1][8];
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        const int64_t r = min(rr + 8 * q, r1 - 1);  // past the end the last row, unused
        get(static_cast<const S*>(a.dy) + r * a.dy_stride + c, d[q]);
        if (ACT != VGGT_ACT_NONE) get(static_cast<const Z*>(a.z) + r * a.z_stride + c, z[q]);
      }
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        const int64_t r = rr + 8 * q;
        if (r >= r1) break;
        if (ACT != VGGT_ACT_NONE) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float slope;
            const float v = act::value_slope<ACT>(z[q][i], slope);
            sg[i] = fmaf(d[q][i], v, sg[i]);
            // rounded as it stands: whether dz goes out as well must not change the sums
            d[q][i] = __fmul_rn(d[q][i], __fmul_rn(gate[i], slope));
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sb[i] += d[q][i];
        if (a.dz != nullptr) put8(static_cast<T*>(a.dz) + r * a.dz_stride + c, n, WIDE, d[q]);
        if (a.scaled != nullptr) {
#pragma unroll
          for (int i = 0; i < 8; ++i) d[q][i] *= gate[i];
          put8(static_cast<T*>(a.scaled) + r * a.dz_stride + c, n, WIDE, d[q]);
        }
      }
    }
  }
  for (int which = 0; which < 2; ++which) {
    float* out = which == 0 ? a.bias_part : a.gate_part;
    if (out == nullptr) continue;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) fold[ry][cx * 8 + i] = which == 0 ? sb[i] : sg[i];
    __syncthreads();
    const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (col < a.outer) {
      float s = 0.f;
#pragma unroll
      for (int q = 0; q < 8; ++q) s += fold[q][threadIdx.x];
      out[blockIdx.y * a.outer + col] = s;
    }
  }
}

template <typename S, typename Z, typename T, bool WIDE>
static void launch_sums(const Sums& a, dim3 grid, cudaStream_t stream) {
  switch (a.act) {
    case VGGT_ACT_GELU: sums_kernel<S, Z, T, VGGT_ACT_GELU, WIDE><<<grid, 256, 0, stream>>>(a); break;
    case VGGT_ACT_GELU_TANH:
      sums_kernel<S, Z, T, VGGT_ACT_GELU_TANH, WIDE><<<grid, 256, 0, stream>>>(a);
      break;
    case VGGT_ACT_SILU: sums_kernel<S, Z, T, VGGT_ACT_SILU, WIDE><<<grid, 256, 0, stream>>>(a); break;
    case VGGT_ACT_RELU: sums_kernel<S, Z, T, VGGT_ACT_RELU, WIDE><<<grid, 256, 0, stream>>>(a); break;
    default: sums_kernel<S, T, T, VGGT_ACT_NONE, WIDE><<<grid, 256, 0, stream>>>(a);
  }
}

template <typename S, typename T>
static void launch_sums(const Sums& a, bool z_fp32, dim3 grid, cudaStream_t stream) {
  if (z_fp32)
    a.wide ? launch_sums<S, float, T, true>(a, grid, stream)
           : launch_sums<S, float, T, false>(a, grid, stream);
  else
    a.wide ? launch_sums<S, T, T, true>(a, grid, stream)
           : launch_sums<S, T, T, false>(a, grid, stream);
}

// gate W, rounded once more to W's type (bf16): one rounding of dx's factors, as dy gate would be.
__global__ void __launch_bounds__(256)
    scale_weight_kernel(const __nv_bfloat16* w, int64_t stride, const void* gate, bool gate_fp32,
                        __nv_bfloat16* to, int64_t pad, int64_t outer, int64_t inner) {
  const int64_t groups = (inner + 7) / 8, all = outer * groups;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < all;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / groups, c = (i - r * groups) * 8;
    float v[8];
    const int n = (int)min((int64_t)8, inner - c);
    get8(w + r * stride + c, n, true, v);
    const float g = vector_at<__nv_bfloat16>(gate, gate_fp32, r);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= g;
    put8(to + r * pad + c, n, true, v);
  }
}

// A block per row of W: adds the partial sums of dW's row, and what the row's bias and gate get.
struct Weights {
  const void* weight;
  int64_t weight_stride;
  const void* bias;
  const void* gate;
  bool gate_fp32;
  bool act;       // with an activation dz has the gate already, and gate_part the gate's sums
  void* dweight;  // or null
  int64_t dweight_stride;
  void* dbias;
  void* dgate;
  const float* bias_part;
  const float* gate_part;
  int64_t row_blocks, outer, inner;
  bool product;  // whether there are partial sums of a product
  const float* dots;  // or its rows' products with W's, [dot_groups][outer]
  int64_t dot_groups;
  bool wide;
};

__device__ __forceinline__ float block_sum(float v, float* fold) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) fold[threadIdx.x >> 5] = v;
  __syncthreads();
  return fold[0] + fold[1] + fold[2] + fold[3];
}

template <typename T>
__global__ void __launch_bounds__(128) finish_weight_kernel(const Slots s, const Weights a) {
  __shared__ float fold[4];
  const int64_t r = blockIdx.x;
  const float gate = a.gate != nullptr && !a.act ? vector_at<T>(a.gate, a.gate_fp32, r) : 1.f;
  const bool want_dot = a.dgate != nullptr && !a.act;
  float dot = 0.f;
  if (a.product)
    for (int64_t c = threadIdx.x * 8; c < a.inner; c += 128 * 8) {
      const int n = (int)min((int64_t)8, a.inner - c);
      float v[8];
      s.get8(r, c, v);
      if (want_dot) {
        float w[8];
        get8(static_cast<const T*>(a.weight) + r * a.weight_stride + c, n, true, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) dot = fmaf(v[i], w[i], dot);
      }
      if (a.dweight != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= gate;
        put8(static_cast<T*>(a.dweight) + r * a.dweight_stride + c, n, a.wide, v);
      }
    }
  float sum = 0.f;
  if (a.bias_part != nullptr) {
    for (int64_t i = threadIdx.x; i < a.row_blocks; i += 128) sum += a.bias_part[i * a.outer + r];
    sum = block_sum(sum, fold);
  }
  if (a.dbias != nullptr && threadIdx.x == 0)
    static_cast<T*>(a.dbias)[r] = ElemOps<T>::from_float(gate * sum);
  if (a.dgate == nullptr) return;
  float g = 0.f;
  if (a.act) {
    for (int64_t i = threadIdx.x; i < a.row_blocks; i += 128) g += a.gate_part[i * a.outer + r];
  } else if (a.dots != nullptr) {
    for (int64_t i = threadIdx.x; i < a.dot_groups; i += 128) g += a.dots[i * a.outer + r];
  } else {
    g = dot;
  }
  g = block_sum(g, fold);
  if (threadIdx.x == 0) {
    if (!a.act && a.bias != nullptr) g = fmaf((float)static_cast<const T*>(a.bias)[r], sum, g);
    if (a.gate_fp32)
      static_cast<float*>(a.dgate)[r] = g;
    else
      static_cast<T*>(a.dgate)[r] = ElemOps<T>::from_float(g);
  }
}

// What a backward call does, and where its workspace lies (offsets in bytes).
struct Back {
  bool act, dx, product, dot, sums, copy_dy, scale_dy, scale_w;
  int64_t row_blocks, per_block, pad;  // pad: row stride of dz
  Laid laid;
  Plan px, pw;
  size_t dz, scaled, weight, bias_part, gate_part, dots, slots, bytes;
};

static bool tma_rows(const void* p, int64_t stride, int64_t width, int64_t rows) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 &&
         (rows <= 1 || (stride % 8 == 0 && stride >= width));
}

static Back plan_back(const vggt_linear_args* a, const vggt_linear_grads* g) {
  Back b{};
  b.act = a->activation != VGGT_ACT_NONE;
  const bool dgate = g->dgate && a->gate;
  b.dx = g->dx != nullptr;
  b.product = g->dweight != nullptr || (dgate && !b.act);
  // dy as it lies, where it is of the products' type and TMA can read it
  b.copy_dy = (b.dx || b.product) &&
              (b.act || a->stream_dtype == VGGT_DTYPE_FP32 ||
               !tma_rows(g->dy, g->dy_stride, a->outer, a->rows));
  if (b.dx && a->gate && !b.act) {
    // the gate goes to the smaller factor of dx, or to dy where that is rounded anyway: one
    // rounding of a factor in either case.  In fp16 always to dy: gate W would fall among the
    // subnormal numbers for a gate of 1e-4 (dx off by 1 %; by 10 % for 1e-5) and, unlike gate dy,
    // not come out of them with a scaled loss (22,000 rows of 4096 -> 1024, forward and gradient:
    // 444 to 464 us with the gate on W, 439 to 494 on dy)
    b.scale_dy = b.copy_dy || a->dtype == VGGT_DTYPE_FP16 || a->rows < a->inner;
    b.scale_w = !b.scale_dy;
  }
  b.sums = b.copy_dy || b.scale_dy || (g->dbias && a->bias) || dgate;
  b.laid = plan_operands(a, b.product, b.dx || (dgate && !b.act));
  b.bytes = b.laid.bytes;
  const int64_t cols = (a->outer + 255) / 256;
  b.row_blocks = std::max<int64_t>(1, std::min<int64_t>((a->rows + 31) / 32, 148 * 8 / cols));
  b.per_block = (a->rows + b.row_blocks - 1) / b.row_blocks;
  b.row_blocks = (a->rows + b.per_block - 1) / b.per_block;
  b.pad = (a->outer + 7) / 8 * 8;
  auto take = [&](bool need, size_t bytes) {
    const size_t at = b.bytes;
    if (need) b.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  b.dz = take(b.copy_dy, (size_t)a->rows * b.pad * 2);
  b.scaled = take(b.scale_dy, (size_t)a->rows * b.pad * 2);
  b.weight = take(b.scale_w, (size_t)a->outer * b.laid.pad * 2);
  b.bias_part = take(b.sums, (size_t)b.row_blocks * a->outer * 4);
  b.gate_part = take(b.sums && b.act, (size_t)b.row_blocks * a->outer * 4);
  if (b.dx) b.px = plan_product(a->rows, a->inner, a->outer);
  if (b.product) b.pw = plan_product(a->outer, a->inner, a->rows);
  b.dot = b.product && !b.pw.split && dgate && !b.act;
  b.dots = take(b.dot, b.dot ? (size_t)dot_groups(b.pw, a->inner) * a->outer * 4 : 0);
  // the products run one after the other
  b.slots = take(true, std::max(b.dx ? b.px.slot_bytes() : 0, b.product ? b.pw.slot_bytes() : 0));
  return b;
}

template <typename T>
static cudaError_t run_back(const vggt_linear_args* a, const vggt_linear_grads* g, const Back& b,
                            int32_t* status, unsigned char* ws, cudaStream_t stream) {
  const int64_t rows = a->rows, inner = a->inner, outer = a->outer;
  float* bias_part = reinterpret_cast<float*>(ws + b.bias_part);
  float* gate_part = reinterpret_cast<float*>(ws + b.gate_part);
  float* slots = reinterpret_cast<float*>(ws + b.slots);
  T* scaled = reinterpret_cast<T*>(ws + b.scaled);
  const bool gate_fp32 = a->gate_fp32 != 0;
  if (b.sums) {
    Sums s{};
    s.dy = g->dy;
    s.dy_stride = g->dy_stride;
    s.z = g->z;
    s.z_stride = g->z_stride;
    s.gate = a->gate;
    s.gate_fp32 = gate_fp32;
    s.act = a->activation;
    s.dz = b.copy_dy ? ws + b.dz : nullptr;
    s.scaled = b.scale_dy ? scaled : nullptr;
    s.dz_stride = b.pad;
    s.bias_part = bias_part;
    s.gate_part = b.act ? gate_part : nullptr;
    s.rows = rows;
    s.outer = outer;
    s.per_block = b.per_block;
    s.wide = outer % 8 == 0 && wide_rows(g->dy, g->dy_stride, a->stream_dtype) &&
             (!b.act || wide_rows(g->z, g->z_stride, a->z_dtype)) &&
             wide_rows(a->gate, 8, gate_fp32 ? VGGT_DTYPE_FP32 : a->dtype);
    const dim3 grid((unsigned)((outer + 255) / 256), (unsigned)b.row_blocks);
    const bool z_fp32 = a->z_dtype == VGGT_DTYPE_FP32;
    if (a->stream_dtype == VGGT_DTYPE_FP32)
      launch_sums<float, T>(s, z_fp32, grid, stream);
    else
      launch_sums<T, T>(s, z_fp32, grid, stream);
    if (cudaError_t e = cudaGetLastError()) return e;
  }
  if (cudaError_t e = copy_operands(a, b.laid, ws, stream)) return e;
  const Operand weight = w_operand(a, b.laid, ws, true);
  const void* dz = b.copy_dy ? ws + b.dz : g->dy;
  const int64_t dz_stride = b.copy_dy ? b.pad : g->dy_stride;
  if (b.dx) {
    Operand w = weight;
    if (b.scale_w) {
      typedef __nv_bfloat16 B;
      B* to = reinterpret_cast<B*>(ws + b.weight);
      const int64_t all = outer * ((inner + 7) / 8);
      scale_weight_kernel<<<(unsigned)std::min<int64_t>((all + 255) / 256, 148 * 16), 256, 0,
                            stream>>>(static_cast<const B*>(w.p), w.stride, a->gate, gate_fp32, to,
                                      b.laid.pad, outer, inner);
      if (cudaError_t e = cudaGetLastError()) return e;
      w.p = to;
      w.stride = b.laid.pad;
    }
    Epilogue e;
    e.y = g->dx;
    e.y_stride = g->dx_stride;
    e.y_head_stride = g->dx_head_stride;
    e.y_heads = a->heads > 1 && g->dx_head_stride > 0 ? a->heads : 1;
    e.y_dim = inner / e.y_heads;
    e.y_type = a->dtype;
    const Operand d = b.scale_dy ? matrix(scaled, outer, b.pad, false)
                                 : matrix(dz, outer, dz_stride, false);
    if (cudaError_t rc =
            launch_product(b.px, a->dtype, rows, inner, outer, d, w, e, slots, status, stream))
      return rc;
    if (b.px.split)
      if (cudaError_t rc = finish_product(b.px, a->dtype, rows, inner, e, slots, stream)) return rc;
  }
  if (b.product) {
    Epilogue e;  // of a product that is not split
    e.y = g->dweight;
    e.y_stride = g->dweight_stride;
    e.y_dim = inner;
    e.y_type = a->dtype;
    if (a->gate && !b.act) e.row_gate = a->gate;
    e.gate_fp32 = gate_fp32;
    if (b.dot) {
      e.residual = weight.p;
      e.residual_stride = weight.stride;
      e.row_dot = reinterpret_cast<float*>(ws + b.dots);
    }
    if (cudaError_t rc = launch_product(b.pw, a->dtype, outer, inner, rows,
                                        matrix(dz, outer, dz_stride, true),
                                        x_operand(a, b.laid, ws, true), e, slots, status, stream))
      return rc;
  }
  Weights f{};
  f.weight = weight.p;
  f.weight_stride = weight.stride;
  f.bias = a->bias;
  f.gate = a->gate;
  f.gate_fp32 = gate_fp32;
  f.act = b.act;
  f.dweight = g->dweight;
  f.dweight_stride = g->dweight_stride;
  f.dbias = a->bias ? g->dbias : nullptr;
  f.dgate = a->gate ? g->dgate : nullptr;
  const bool partial = b.product && b.pw.split;
  if (!partial && !f.dbias && !f.dgate) return cudaSuccess;
  f.bias_part = b.sums ? bias_part : nullptr;
  f.gate_part = gate_part;
  f.row_blocks = b.row_blocks;
  f.outer = outer;
  f.inner = inner;
  f.product = partial;
  f.dots = b.dot ? reinterpret_cast<float*>(ws + b.dots) : nullptr;
  f.dot_groups = b.dot ? dot_groups(b.pw, inner) : 0;
  f.wide = wide_rows(g->dweight, g->dweight_stride, a->dtype);
  const Slots s = partial ? slots_of(b.pw, slots) : Slots{};
  finish_weight_kernel<T><<<(unsigned)outer, 128, 0, stream>>>(s, f);
  return cudaGetLastError();
}

}  // namespace lin
}  // namespace vggt

extern "C" size_t vggt_linear_grad_workspace_size(const vggt_linear_args* a,
                                                  const vggt_linear_grads* g) {
  if (!a || !g || a->rows <= 0 || a->inner < 1 || a->outer < 1) return 0;
  return vggt::lin::plan_back(a, g).bytes;
}

extern "C" int vggt_linear_grad(const vggt_linear_args* a, const vggt_linear_grads* g,
                                int32_t* status, void* workspace, size_t workspace_bytes,
                                void* stream) {
  using namespace vggt;
  using namespace vggt::lin;
  if (int rc = check(a)) return rc;
  if (!g) return api_fail("grads must be non-NULL");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (g->dweight && a->outer > 1 && g->dweight_stride < a->inner)
    return api_fail("dweight's stride is below inner");
  if (a->rows == 0) {  // the sums of no rows
    if (g->dweight)
      if (int rc = api_cuda(cudaMemset2DAsync(g->dweight, (size_t)g->dweight_stride * 2, 0,
                                              (size_t)a->inner * 2, (size_t)a->outer, st)))
        return rc;
    void* const sums[2] = {a->bias ? g->dbias : nullptr, a->gate ? g->dgate : nullptr};
    for (int k = 0; k < 2; ++k) {
      const size_t size = k == 1 && a->gate_fp32 ? 4 : 2;
      if (sums[k])
        if (int rc = api_cuda(cudaMemsetAsync(sums[k], 0, (size_t)a->outer * size, st))) return rc;
    }
    return api_fail(nullptr);
  }
  if (!g->dy) return api_fail("dy must be non-NULL");
  if (a->activation != VGGT_ACT_NONE && !g->z)
    return api_fail("with an activation the gradient needs z");
  if (a->rows > 1 && (g->dy_stride < 0 || (g->z && g->z_stride < 0)))
    return api_fail("negative stride");
  const bool split_dx = a->heads > 1 && g->dx_head_stride > 0;
  const int64_t dim = split_dx ? a->inner / a->heads : a->inner;
  if (g->dx && split_dx && dim % 64)
    return api_fail("a head-major dx needs heads of a multiple of 64 elements");
  if (g->dx && ((a->rows > 1 && g->dx_stride < dim) || (split_dx && g->dx_head_stride < dim)))
    return api_fail("a stride of dx is below the row's width");
  const Back b = plan_back(a, g);
  if (b.bytes > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) ||
                      workspace_bytes < b.bytes))
    return api_fail("the workspace is too small or not 256-byte aligned");
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  return api_cuda(a->dtype == VGGT_DTYPE_BF16
                      ? run_back<__nv_bfloat16>(a, g, b, status, ws, st)
                      : run_back<__half>(a, g, b, status, ws, st));
}
