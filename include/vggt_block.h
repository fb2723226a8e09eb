/*
 * vggt_block.h — C ABI of the dense operators around a block's attention: a
 * matrix product whose epilogue adds the bias, applies the activation, scales
 * by a gate and adds the residual, a gated residual with the norms around it,
 * and the gradients of both.
 *
 * As in vggt_sparse.h every entry point takes plain device pointers, sizes
 * and a cudaStream_t (as void*), enqueues on that stream, never synchronises
 * and never allocates.  0: enqueued; negative: argument error (message from
 * vggt_sparse_last_error()); positive: CUDA error code of the launch.
 *
 * Element types are VGGT_DTYPE_BF16, _FP16 and _FP32.  Strides are in elements
 * and lie between rows; rows are contiguous.  Pointers that are "or NULL" may
 * be; outputs that are NULL are not computed.  All sums, statistics and
 * activations are formed in fp32 and rounded once, to the output's type.
 */
#ifndef VGGT_BLOCK_H
#define VGGT_BLOCK_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#ifndef VGGT_DTYPE_FP32
#define VGGT_DTYPE_FP32 2
#endif

/* activations */
#define VGGT_ACT_NONE 0
#define VGGT_ACT_GELU 1      /* z Phi(z), Phi the normal distribution */
#define VGGT_ACT_GELU_TANH 2 /* z sigmoid(2 sqrt(2 / pi) (z + 0.044715 z^3)) */
#define VGGT_ACT_SILU 3      /* z sigmoid(z) */
#define VGGT_ACT_RELU 4      /* max(z, 0) */

/* norms */
#define VGGT_NORM_NONE 0  /* post_norm only: the branch as it is */
#define VGGT_NORM_LAYER 1 /* (v - mean v) / sqrt(var v + eps) */
#define VGGT_NORM_RMS 2   /* v / sqrt(mean v^2 + eps) */

/* widest row of vggt_residual_norm */
#define VGGT_NORM_MAX_WIDTH 16384

/* a parameter vector, of any of the element types, or none (data NULL) */
typedef struct vggt_vector {
  const void* data;
  int dtype;
} vggt_vector;

/*
 * z = x weight^T + bias
 * y = residual + gate * activation(z)
 *
 * x [rows][inner], or with heads > 1 head-major: [heads][rows][inner / heads]
 * with x_head_stride between heads, read as [rows][inner].  weight
 * [outer][inner], bias [outer], x of dtype (BF16 or FP16); gate [outer] of
 * dtype, or with gate_fp32 FP32; residual and y [rows][outer] of stream_dtype,
 * which is dtype or FP32.  z [rows][outer] of z_dtype (dtype or FP32), where
 * non-NULL, gets the activation's argument for the backward pass.  residual and
 * y may be the same; otherwise the outputs lie apart from the inputs.
 *
 * x and weight are read in place where their rows (and heads, then of a multiple
 * of 64 elements) start on 16 bytes, else copied into the workspace first.
 *
 * The workspace needs vggt_linear_workspace_size bytes (none: it may be NULL),
 * 256-byte aligned, and no clearing.
 * status, where non-NULL, gets VGGT_STATUS_TIMEOUT if a wait ran out.
 */
typedef struct vggt_linear_args {
  int64_t rows, inner, outer;
  int dtype, stream_dtype;
  const void* x;
  int64_t x_stride, x_head_stride;
  int64_t heads; /* 0 or 1: x is [rows][inner] */
  const void* weight;
  int64_t weight_stride;
  const void* bias;     /* or NULL */
  const void* gate;     /* or NULL */
  const void* residual; /* or NULL */
  int64_t residual_stride;
  int activation;
  int z_dtype;          /* of z, here and in the backward pass */
  int gate_fp32;        /* nonzero: gate and its gradient are FP32, not of dtype */
} vggt_linear_args;

size_t vggt_linear_workspace_size(const vggt_linear_args* args);
int vggt_linear(const vggt_linear_args* args, void* y, int64_t y_stride, void* z, int64_t z_stride,
                int32_t* status, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Gradients of the above from that of y (dy, of stream_dtype): dx [rows][inner]
 * or, with dx_head_stride > 0, head-major like x (heads of a multiple of 64
 * elements), dweight [outer][inner], dbias [outer], all of dtype, and dgate
 * [outer] of the gate's type; that of residual is dy.  z is what vggt_linear wrote;
 * without an activation it is not needed.  Sums are formed in a fixed order.
 */
typedef struct vggt_linear_grads {
  const void* dy;
  int64_t dy_stride;
  const void* z;
  int64_t z_stride;
  void* dx;
  int64_t dx_stride, dx_head_stride;
  void* dweight;
  int64_t dweight_stride;
  void *dbias, *dgate;
} vggt_linear_grads;

size_t vggt_linear_grad_workspace_size(const vggt_linear_args* args,
                                       const vggt_linear_grads* grads);
int vggt_linear_grad(const vggt_linear_args* args, const vggt_linear_grads* grads, int32_t* status,
                     void* workspace, size_t workspace_bytes, void* stream);

/*
 * p = post_norm(branch) * post_weight + post_bias
 * h = x + gate * p
 * y = norm(h) * weight + bias
 *
 * x, h [rows][width] of stream_dtype; branch, y of dtype, which is stream_dtype
 * or, where that is fp32, any.  gate is one row, or with rows_per_gate > 0 one
 * row for each rows_per_gate rows (rows is then a multiple of it).  Without a
 * branch h is x: neither gate, post_norm nor h is used.  h may be x.
 */
typedef struct vggt_residual_norm_args {
  int64_t rows, width;
  int stream_dtype, dtype;
  const void* x;
  int64_t x_stride;
  const void* branch; /* or NULL */
  int64_t branch_stride;
  vggt_vector gate, weight, bias, post_weight, post_bias;
  int64_t rows_per_gate;
  int norm, post_norm;
  float eps;
} vggt_residual_norm_args;

int vggt_residual_norm(const vggt_residual_norm_args* args, void* h, int64_t h_stride, void* y,
                       int64_t y_stride, void* stream);

/*
 * Gradients of the above from those of y (dy, of dtype) and h (dh, of
 * stream_dtype), either of which may be NULL (zero): dx of stream_dtype,
 * dbranch of dtype, and the parameters' gradients in the parameters' own types
 * and shapes, contiguous.  Every output may be NULL.  The workspace needs
 * vggt_residual_norm_grad_workspace_size bytes, 16-byte aligned, and no
 * clearing.  Sums over rows are formed in a fixed order: equal calls give equal
 * results.
 */
typedef struct vggt_residual_norm_grads {
  const void* dy; /* or NULL */
  int64_t dy_stride;
  const void* dh; /* or NULL */
  int64_t dh_stride;
  void* dx;
  int64_t dx_stride;
  void* dbranch;
  int64_t dbranch_stride;
  void *dgate, *dweight, *dbias, *dpost_weight, *dpost_bias;
} vggt_residual_norm_grads;

size_t vggt_residual_norm_grad_workspace_size(int64_t rows, int64_t width, int64_t rows_per_gate);
int vggt_residual_norm_grad(const vggt_residual_norm_args* args,
                            const vggt_residual_norm_grads* grads, void* workspace,
                            size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* VGGT_BLOCK_H */
