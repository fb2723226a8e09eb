// The matrix product of `linear` for few rows (single tokens, a decode batch).
//
// Bound by reading the weight once.  A block takes COLS = 8, 16 or 32 columns of y, i.e. as many rows
// of the weight; its warps deal out the reduced length in pieces of 64 elements.  A lane reads 16
// bytes of a weight row and of x's rows straight into the registers of mma.sync m16n8k16 (x the
// 16 rows, the weight the 8 columns): the instruction sums over the reduced index, so that which
// lane holds which elements does not matter as long as both operands agree, and nothing goes
// through shared memory.  All of a warp's loads of a piece are in flight at once; the warps' sums
// are added in shared memory in a fixed order.  The tensor core's tcgen05 form would need 128 rows.
#include <algorithm>

#include "activation.cuh"
#include "linear.cuh"

namespace vggt {
namespace lin {

struct RowsArgs {
  const void* x;
  int64_t x_stride, x_head_stride;
  int dim;  // elements of x's row in one head, a multiple of 64 where there are several
  const void* weight;
  int64_t weight_stride;
  int m, n, k;
  Epilogue e;
};

template <typename T>
__device__ __forceinline__ void mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                    uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 load16(const void* p, bool there) {
  return there ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
}

// Warps of a block at most: their sums share 48 KB.
template <int MT, int COLS>
constexpr int most_warps() {
  return MT * COLS >= 64 ? 8 : 16;
}

// MT blocks of 16 rows of x, COLS columns of y.
template <typename T, int MT, int COLS>
__global__ void __launch_bounds__(most_warps<MT, COLS>() * 32) rows_kernel(const RowsArgs a) {
  constexpr int NT = COLS / 8, DEPTH = 4 / NT;
  __shared__ float part[most_warps<MT, COLS>()][MT * 16 * COLS];  // of each warp
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int g = lane >> 2, t = lane & 3, n0 = blockIdx.x * COLS;
  grid_wait();
  float c[MT][NT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) c[i][j][q] = 0.f;
  const T* x = static_cast<const T*>(a.x);
  const T* w = static_cast<const T*>(a.weight) + (int64_t)(n0 + g) * a.weight_stride;
  for (int kk = warp * 64; kk < a.k; kk += warps * 64 * DEPTH) {
    // the weight's pieces, which come from memory, all at once
    uint4 b[DEPTH][NT][2];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = kk + d * warps * 64 + h * 32 + t * 8;
          b[d][j][h] = load16(w + (int64_t)(8 * j) * a.weight_stride + k,
                              n0 + g + 8 * j < a.n && k < a.k);
        }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int k0 = kk + d * warps * 64;
      if (d > 0 && k0 >= a.k) break;
      // a piece lies within one head
      const int head = k0 / a.dim;
      const T* xk = x + head * a.x_head_stride + (k0 - head * a.dim);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        uint4 lo[2], hi[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = h * 32 + t * 8, r = i * 16 + g;
          const bool in = k0 + k < a.k;
          lo[h] = load16(xk + r * a.x_stride + k, in && r < a.m);
          hi[h] = load16(xk + (r + 8) * a.x_stride + k, in && r + 8 < a.m);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            mma<T>(c[i][j], lo[h].x, hi[h].x, lo[h].y, hi[h].y, b[d][j][h].x, b[d][j][h].y);
            mma<T>(c[i][j], lo[h].z, hi[h].z, lo[h].w, hi[h].w, b[d][j][h].z, b[d][j][h].w);
          }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float* p = part[warp] + (i * 16 + g) * COLS + j * 8 + t * 2;
      *reinterpret_cast<float2*>(p) = make_float2(c[i][j][0], c[i][j][1]);
      *reinterpret_cast<float2*>(p + 8 * COLS) = make_float2(c[i][j][2], c[i][j][3]);
    }
  __syncthreads();
  const Epilogue& e = a.e;
  for (int i = threadIdx.x; i < MT * 16 * COLS; i += blockDim.x) {
    const int r = i / COLS, n = n0 + i % COLS;
    if (r >= a.m || n >= a.n) continue;
    float v = 0.f;
    for (int q = 0; q < warps; ++q) v += part[q][i];
    if (e.bias != nullptr) v += (float)static_cast<const T*>(e.bias)[n];
    if (e.z != nullptr && e.z_type == VGGT_DTYPE_FP32)
      static_cast<float*>(e.z)[r * e.z_stride + n] = v;
    else if (e.z != nullptr)
      static_cast<T*>(e.z)[r * e.z_stride + n] = ElemOps<T>::from_float(v);
    act::dispatch(e.act, [&](auto k) { v = act::value<decltype(k)::value>(v); });
    if (e.gate != nullptr) v *= vector_at<T>(e.gate, e.gate_fp32, n);
    if (e.y_type == VGGT_DTYPE_FP32) {
      if (e.residual != nullptr)
        v += static_cast<const float*>(e.residual)[r * e.residual_stride + n];
      static_cast<float*>(e.y)[r * e.y_stride + n] = v;
    } else {
      if (e.residual != nullptr)
        v += (float)static_cast<const T*>(e.residual)[r * e.residual_stride + n];
      static_cast<T*>(e.y)[r * e.y_stride + n] = ElemOps<T>::from_float(v);
    }
  }
}

// 64 rows of a narrow product at most, 32 of another: there the tiles of linear.cu catch up (64
// rows, 1024 -> 1024: 5.7 against 6.7 us; 4096 -> 1024: 10.5 against 12.2; 1024 -> 4096: 11.6 against
// 7.5; 32 rows, 8192 -> 8192: 32 against 33).
bool few_rows(int64_t m, int64_t n, int64_t k) {
  return k % 8 == 0 && (m <= 32 || (m <= 64 && n < 2048));
}

template <typename T, int MT, int COLS>
static cudaError_t launch(const RowsArgs& a, cudaStream_t stream) {
  // two pieces of 64 to a warp at least
  const int warps = std::max(1, std::min(most_warps<MT, COLS>(), a.k / 128));
  return launch_early(rows_kernel<T, MT, COLS>, dim3((unsigned)((a.n + COLS - 1) / COLS)),
                      dim3(warps * 32), 0, stream, a);
}

template <typename T>
static cudaError_t launch_rows(const RowsArgs& a, cudaStream_t stream) {
  // As many columns to a block as still leave every SM one: more columns read x less often
  // (us, one B200, weights from memory; rows: 8 / 16 / 32 columns.  1024 -> 4096, 1 row: 6.1 / 4.8 /
  // 5.7; 4096 -> 1024, 1 row: 5.4 / 7.4 / 9.1; 4096 -> 4096, 32 rows: 23.4 / 18.9 / 15.0;
  // 4096 -> 1024, 32 rows: 7.0 / 9.8 / 13.3)
  if (a.m <= 16) return a.n >= 2048 ? launch<T, 1, 16>(a, stream) : launch<T, 1, 8>(a, stream);
  if (a.m <= 32) return a.n >= 4096 ? launch<T, 2, 32>(a, stream) : launch<T, 2, 8>(a, stream);
  return launch<T, 4, 8>(a, stream);
}

cudaError_t launch_rows(int dtype, int64_t m, int64_t n, int64_t k, const Operand& x,
                        const Operand& w, const Epilogue& e, cudaStream_t stream) {
  RowsArgs a;
  a.x = x.p;
  a.x_stride = x.stride;
  a.x_head_stride = x.head_stride;
  a.dim = x.heads > 1 ? (int)x.dim : (int)((k + 63) / 64 * 64);
  a.weight = w.p;
  a.weight_stride = w.stride;
  a.m = (int)m;
  a.n = (int)n;
  a.k = (int)k;
  a.e = e;
  return dtype == VGGT_DTYPE_BF16 ? launch_rows<__nv_bfloat16>(a, stream)
                                  : launch_rows<__half>(a, stream);
}

}  // namespace lin
}  // namespace vggt
