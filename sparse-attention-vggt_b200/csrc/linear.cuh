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
  int act = VGGT_ACT_NONE;
  const void* residual = nullptr;
  int64_t residual_stride = 0;
  void* y = nullptr;
  int64_t y_stride = 0, y_head_stride = 0, y_heads = 1, y_dim = 0;
  int y_type = 0;  // of y and the residual
  void* z = nullptr;
  int64_t z_stride = 0;
};

// How a product is cut: tiles of 128 cta x 128 cta, worked on by `workers` groups of cta CTAs,
// whole (split 0), or as equal runs of the tiles' reduction blocks (split 1).
struct Plan {
  int cta = 1, split = 0, workers = 1;
  int64_t tiles_m = 0, tiles_n = 0, blocks = 0;  // blocks: of 64 reduced elements
  size_t slot_bytes() const;                     // partial sums of a split product
};

Plan plan_product(int64_t m, int64_t n, int64_t red, bool must_split);

// A split product's partial sums.  Tile t's reduction blocks [t blocks, (t + 1) blocks) of all lie with the workers that begin at
// or before them; worker w's part is slot w + t.
struct Slots {
  const float* p;
  int64_t units;
  int64_t tiles_n;
  int cta, blocks, workers;
  __device__ __forceinline__ int first(int64_t tile) const {
    return (int)(((tile * blocks + 1) * workers - 1) / units);
  }
  __device__ __forceinline__ int last(int64_t tile) const {
    return (int)(((tile + 1) * blocks * workers - 1) / units);
  }
  // the sums at row r, columns c .. c + 8, c a multiple of 8
  __device__ __forceinline__ void get8(int64_t r, int64_t c, float* v) const {
    const int bn = 128 * cta;
    const int64_t tm = r / bn, tn = c / bn, tile = tm * tiles_n + tn;
    const int rank = (int)(r - tm * bn) / 128, row = (int)(r & 127), in = (int)(c - tn * bn);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
    const int j = (in & 31) / 4;
    for (int w = first(tile), e = last(tile); w <= e; ++w) {
      const float* q = p + (((w + tile) * cta + rank) * (bn / 32) + in / 32) * (128 * 32) + row * 32;
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

// Argument checks (0, or the error) and operands of a call.
int check(const vggt_linear_args* a);
Operand x_operand(const vggt_linear_args* a, bool mn_major);
Operand matrix(const void* p, int64_t width, int64_t stride, bool mn_major);

}  // namespace lin
}  // namespace vggt
