// The matrix products of `linear` and its gradients: what host and kernels share.
#pragma once

#include <cuda.h>

#include "kernels.h"
#include "vec8.cuh"

namespace vggt {
namespace lin {

// One product C [m][n] = A B over `red` reduced elements, fp32 accumulators, with an epilogue:
//   z = C + bias, y = residual + gate * act(z)
// or, with split, only partial sums, which a launch of its own adds up.
//
// An operand is K-major (rows of reduced elements, as x and weight in y = x weight^T) or
// MN-major (rows of m or n, one per reduced element).  Its rows may lie in several heads:
// element c of a row at head c / dim, element c % dim, dim a multiple of 64.
struct Operand {
  const void* p = nullptr;
  int64_t stride = 0, head_stride = 0;
  int64_t heads = 1, dim = 0;  // dim: elements of a row in one head
  bool mn_major = false;
};

struct Epilogue {
  const void* bias = nullptr;  // [n]
  const void* gate = nullptr;  // [n]
  bool gate_fp32 = false;      // of gate and row_gate: fp32, or the operands' type
  int act = VGGT_ACT_NONE;
  const void* residual = nullptr;
  int64_t residual_stride = 0;
  void* y = nullptr;
  int64_t y_stride = 0, y_head_stride = 0, y_heads = 1, y_dim = 0;
  int y_type = 0;  // of y and the residual
  void* z = nullptr;
  int64_t z_stride = 0;
  int z_type = 0;
  // of a weight's gradient C [outer][inner] that is not split: rows scaled by row_gate, and where
  // row_dot is given their products (unscaled) with the rows of `residual`, which is then not
  // added: one sum for each row and each of dot_groups pieces of columns, [dot_groups][m].  y may
  // be null then.
  const void* row_gate = nullptr;
  float* row_dot = nullptr;
};

// How a product is cut: tiles of 128 cta x bnc cta (cta CTAs work on one), dealt out whole to
// `workers` groups of CTAs (split 0), or as equal runs of the tiles' reduction blocks (split 1).
struct Plan {
  int cta = 1, bnc = 128, split = 0, workers = 1;
  int64_t tiles_m = 0, tiles_n = 0, blocks = 0;  // blocks: of 64 reduced elements
  int64_t units() const { return tiles_m * tiles_n * (split ? blocks : 1); }
  size_t slot_bytes() const;                     // partial sums of a split product
};

Plan plan_product(int64_t m, int64_t n, int64_t red);
// pieces of columns in which a row's product with another is summed (Epilogue::row_dot)
int64_t dot_groups(const Plan& plan, int64_t n);

// A split product's partial sums.  All tiles' reduction blocks, one tile after the other, are dealt
// out in runs: the first `rest` workers take per + 1 of them, the others per.  Worker w's part of
// tile t is slot w + t: per CTA 32-column pieces of 128 rows, in the epilogue buffers' layout.
struct Slots {
  const float* p;
  uint32_t tiles_n, blocks, per, rest;
  int cta, bn;
  __device__ __forceinline__ uint32_t worker_of(uint32_t unit) const {
    const uint32_t border = rest * (per + 1);
    return unit < border ? unit / (per + 1) : rest + (unit - border) / per;
  }
  // the sums at row r, columns c .. c + 8, c a multiple of 8
  __device__ __forceinline__ void get8(int64_t r, int64_t c, float* v) const {
    const uint32_t bm = 128 * cta;
    const uint32_t tm = (uint32_t)r / bm, tn = (uint32_t)c / bn, tile = tm * tiles_n + tn;
    const uint32_t rank = ((uint32_t)r - tm * bm) / 128, row = (uint32_t)r & 127, in = (uint32_t)c - tn * bn;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
    const uint32_t j = (in & 31) / 4;
    for (uint32_t w = worker_of(tile * blocks), e = worker_of((tile + 1) * blocks - 1); w <= e; ++w) {
      const float* q = p + (((int64_t)(w + tile) * cta + rank) * (bn / 32) + in / 32) * (128 * 32) + row * 32;
      const float4 a = *reinterpret_cast<const float4*>(q + ((j ^ (row & 7)) << 2));
      const float4 b = *reinterpret_cast<const float4*>(q + (((j + 1) ^ (row & 7)) << 2));
      v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w;
      v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
    }
  }
};
Slots slots_of(const Plan& plan, const float* p);

// Launches the product; with plan.split the partial sums go to `slots` and finish_product or
// finish_weight (linear_grad.cu) adds them up.
cudaError_t launch_product(const Plan& plan, int dtype, int64_t m, int64_t n, int64_t red,
                           const Operand& a, const Operand& b, const Epilogue& e, float* slots,
                           int32_t* status, cudaStream_t stream);
cudaError_t finish_product(const Plan& plan, int dtype, int64_t m, int64_t n, const Epilogue& e,
                           const float* slots, cudaStream_t stream);

// linear_rows.cu: the product for few rows of x, all epilogues, no workspace.
bool few_rows(int64_t m, int64_t n, int64_t k);
cudaError_t launch_rows(int dtype, int64_t m, int64_t n, int64_t k, const Operand& x,
                        const Operand& w, const Epilogue& e, cudaStream_t stream);

// Argument checks (0, or the error) and operands of a call.
int check(const vggt_linear_args* a);
Operand matrix(const void* p, int64_t width, int64_t stride, bool mn_major);

// x and weight as the kernels read them: in place, or copied into rows that start on 16 bytes.
struct Laid {
  bool copy_x, copy_w;
  int64_t pad;  // row stride of the copies
  size_t x_at, w_at, bytes;
};
Laid plan_operands(const vggt_linear_args* a, bool need_x, bool need_w);
cudaError_t copy_operands(const vggt_linear_args* a, const Laid& l, unsigned char* workspace,
                          cudaStream_t stream);
Operand x_operand(const vggt_linear_args* a, const Laid& l, const unsigned char* workspace,
                  bool mn_major);
Operand w_operand(const vggt_linear_args* a, const Laid& l, const unsigned char* workspace,
                  bool mn_major);

}  // namespace lin
}  // namespace vggt
