// Python binding of the dense operators around a block's attention (include/vggt_block.h).
//
// As cache_binding.cpp: a call's checks, allocations and the launch, in a few microseconds.  The
// graph of a call that needs a gradient is made here too, with the backward pass as C++ (through
// Python a small call with its gradient took 200 us on the host).  vggt_sparse/block_ops.py
// documents the arguments, which come by position.
#include "vggt_block.h"

#include "binding.h"

#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>
#include <optional>
#include <tuple>
#include <utility>
#include <vector>

namespace {

int dtype_of(const char* name, at::ScalarType t, bool fp32) {
  if (t == at::kBFloat16) return VGGT_DTYPE_BF16;
  if (t == at::kHalf) return VGGT_DTYPE_FP16;
  if (fp32 && t == at::kFloat) return VGGT_DTYPE_FP32;
  refuse("%s must be BF16%s", name, fp32 ? ", FP16 or FP32" : " or FP16");
}

bool is(PyObject* o, const char* text) {
  return PyUnicode_Check(o) && PyUnicode_CompareWithASCIIString(o, text) == 0;
}

int norm_of(PyObject* o, const char* name, bool none) {
  if (none && o == Py_None) return VGGT_NORM_NONE;
  if (is(o, "layer")) return VGGT_NORM_LAYER;
  if (is(o, "rms")) return VGGT_NORM_RMS;
  refuse("%s must be 'layer'%s 'rms'%s", name, none ? "," : " or", none ? " or None" : "");
}

int activation_of(PyObject* o) {
  if (o == Py_None) return VGGT_ACT_NONE;
  if (is(o, "gelu")) return VGGT_ACT_GELU;
  if (is(o, "gelu_tanh")) return VGGT_ACT_GELU_TANH;
  if (is(o, "silu")) return VGGT_ACT_SILU;
  if (is(o, "relu")) return VGGT_ACT_RELU;
  refuse("activation must be None, 'gelu', 'gelu_tanh', 'silu' or 'relu'");
}

// A tensor [..., width] as rows with one stride between them, or a contiguous copy.
struct Rows {
  at::Tensor t;
  int64_t rows = 0, width = 0, stride = 0;
  Rows() = default;
  explicit Rows(const at::Tensor& x) : t(x) {
    width = x.size(-1);
    rows = width > 0 ? x.numel() / width : 0;
    stride = width;
    if (x.is_contiguous() || rows <= 1) {
      if (rows == 1 && width > 1 && x.stride(-1) != 1) t = x.contiguous();
      return;
    }
    if (x.dim() == 2 && (x.stride(1) == 1 || width == 1)) {
      stride = x.stride(0);
      return;
    }
    t = x.contiguous();
  }
  void* data() const { return t.data_ptr(); }
};

void check_rows(const char* name, const at::Tensor& t) {
  if (t.dim() < 1 || t.size(-1) < 1) refuse("%s must be [..., width]", name);
}

// A tensor of the caller's that is written in place: graphs that hold it find out.
void written(const at::Tensor& t) {
  if (t.defined()) t.unsafeGetTensorImpl()->bump_version();
}

// An output that the caller gives.
void check_given(const char* name, const at::Tensor& t, at::IntArrayRef sizes, at::ScalarType type) {
  if (t.sizes() != sizes || t.scalar_type() != type || !t.is_contiguous())
    refuse("%s must be contiguous, of the result's shape and dtype", name);
}

// Whether an element of a strided tensor at byte `at` lies in [lo, hi).  The dimension of the largest
// stride is taken first: of its steps only those whose elements can lie there are looked into, and
// all but the outer two of those lie there whole.
bool meets(at::IntArrayRef sizes, at::IntArrayRef strides, int64_t item, uint32_t taken, int64_t at,
           int64_t lo, int64_t hi) {
  int64_t span = item;
  int most = -1;
  for (int k = 0; k < (int)sizes.size(); ++k) {
    if ((taken >> k & 1) || sizes[k] == 1 || strides[k] == 0) continue;
    span += (sizes[k] - 1) * strides[k] * item;
    if (most < 0 || strides[k] > strides[most]) most = k;
  }
  if (at >= hi || at + span <= lo) return false;
  if (most < 0 || at >= lo) return true;
  const int64_t step = strides[most] * item, inner = span - (sizes[most] - 1) * step;
  int64_t i = std::max<int64_t>(0, (lo - at - inner) / step);
  for (; i < sizes[most] && at + i * step < hi; ++i)
    if (meets(sizes, strides, item, taken | 1u << most, at + i * step, lo, hi)) return true;
  return false;
}

// An output that the caller gives lies apart from an input, or, where `same` allows that, in its
// very elements.
void check_apart(const char* name, const at::Tensor& out, const char* input, const at::Tensor& t,
                 bool same) {
  if (!out.defined() || !t.defined() || out.numel() == 0 || t.numel() == 0) return;
  if (same && t.data_ptr() == out.data_ptr() && t.is_contiguous() &&
      t.scalar_type() == out.scalar_type())
    return;
  const int64_t lo = (int64_t)out.data_ptr();
  if (t.dim() <= 32 && !meets(t.sizes(), t.strides(), t.element_size(), 0, (int64_t)t.data_ptr(), lo,
                              lo + (int64_t)out.nbytes()))
    return;
  refuse("%s must not lie in %s%s", name, input, same ? " (unless it is that very tensor)" : "");
}

at::Tensor workspace(size_t bytes, c10::Device device) {
  return at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(device));
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

at::Tensor given_or_none(PyObject* o, const char* name) {
  const at::Tensor* t = tensor_or_none(o, name);
  return t ? *t : at::Tensor();
}
const at::Tensor* there(const at::Tensor& t) { return t.defined() ? &t : nullptr; }

// An argument of a function of the graph: an undefined tensor is none.
typedef std::optional<at::Tensor> Maybe;
Maybe maybe(const at::Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
at::Tensor value(const Maybe& t) { return t.has_value() ? *t : at::Tensor(); }

template <typename... Ts>
bool needs_graph(const Ts&... t) {
  return c10::GradMode::is_enabled() && ((t.defined() && t.requires_grad()) || ...);
}

// Tensors with a tangent (dual tensors need no backward graph) are refused: the kernels form none,
// and a result without one reads as zero.
template <typename... Ts>
void no_tangents(const Ts&... t) {
  if (((t.defined() && t._fw_grad(0).defined()) || ...))
    refuse("there is no forward-mode derivative of this operator");
}

// Gradients that a second differentiation must not go through raise there.
variable_list once(variable_list grads) {
  if (!c10::GradMode::is_enabled()) return grads;
  for (at::Tensor& g : grads)
    if (g.defined()) {
      g = g.detach();
      g.set_requires_grad(true);
    }
  auto raise = std::make_shared<torch::autograd::DelayedError>(
      "this operator is differentiable once", (int)grads.size());
  return (*raise)(std::move(grads));
}

// ---- residual_norm ----------------------------------------------------------------------------
enum { kX, kBranch, kWeight, kBias, kGate, kPostWeight, kPostBias, kNormTensors };

// A call's arguments.
struct NormIn {
  at::Tensor t[kNormTensors];
  int norm = 0, post = 0;
  double eps = 0;
  at::ScalarType type;  // of y

  // a: x, branch, weight, bias, gate, post_weight, post_bias, norm, post_norm, eps, dtype
  explicit NormIn(PyObject* const* o) {
    static const char* names[kNormTensors] = {"x",    "branch",      "weight",   "bias",
                                              "gate", "post_weight", "post_bias"};
    t[kX] = tensor(o[0], "x");
    for (int k = kBranch; k < kNormTensors; ++k) t[k] = given_or_none(o[k], names[k]);
    type = t[kBranch].defined() ? t[kBranch].scalar_type() : t[kX].scalar_type();
    if (o[10] != Py_None) {
      if (!THPDtype_Check(o[10])) refuse("dtype must be a torch.dtype");
      const at::ScalarType asked = reinterpret_cast<THPDtype*>(o[10])->scalar_type;
      if (t[kBranch].defined() && asked != type) refuse("dtype is the branch's where there is one");
      type = asked;
    }
    norm = norm_of(o[7], "norm", false);
    post = norm_of(o[8], "post_norm", true);
    eps = number(o[9], "eps");
  }
  NormIn(const variable_list& tensors, int n, int p, double e, at::ScalarType y)
      : norm(n), post(p), eps(e), type(y) {
    for (int k = 0; k < kNormTensors; ++k) t[k] = tensors[k];
  }
};

// Checked, and as the C ABI takes it.
struct NormCall {
  vggt_residual_norm_args a{};
  Rows x, branch;
  at::ScalarType stream;
  at::Tensor held[kNormTensors];

  explicit NormCall(const NormIn& in) {
    const at::Tensor &xt = in.t[kX], &bt = in.t[kBranch];
    check_rows("x", xt);
    stream = xt.scalar_type();
    a.stream_dtype = dtype_of("x", stream, true);
    a.dtype = dtype_of(bt.defined() ? "branch" : "dtype", in.type, true);
    if (in.type != stream && stream != at::kFloat)
      refuse("x must be of the branch's dtype, or FP32");
    x = Rows(xt);
    a.rows = x.rows;
    a.width = x.width;
    if (bt.defined()) {
      if (bt.sizes() != xt.sizes()) refuse("branch must have x's shape");
      branch = Rows(bt);
      a.branch = branch.data();
      a.branch_stride = branch.stride;
    }
    a.x = x.data();
    a.x_stride = x.stride;
    vggt_vector* to[kNormTensors] = {nullptr,        nullptr, &a.weight, &a.bias, &a.gate,
                                     &a.post_weight, &a.post_bias};
    static const char* names[kNormTensors] = {"", "", "weight", "bias", "gate", "post_weight",
                                              "post_bias"};
    for (int k = kWeight; k < kNormTensors; ++k) {
      const at::Tensor& t = in.t[k];
      if (!t.defined()) continue;
      if (k == kGate) {
        if ((t.dim() != 1 && t.dim() != 2) || t.size(-1) != x.width)
          refuse("gate must be [width] or [groups, width]");
        if (t.dim() == 2) {
          const int64_t groups = t.size(0);
          if (groups < 1 ? a.rows > 0 : a.rows % groups != 0)
            refuse("x's rows (%lld) must be a multiple of gate's (%lld)", (long long)a.rows,
                   (long long)groups);
          // one row for all is a gate per channel
          a.rows_per_gate = groups > 1 ? a.rows / groups : 0;
        }
      } else if (t.dim() != 1 || t.size(0) != x.width) {
        refuse("%s must be [width]", names[k]);
      }
      to[k]->dtype = dtype_of(names[k], t.scalar_type(), true);
      held[k] = t.is_contiguous() ? t : t.contiguous();
      to[k]->data = held[k].data_ptr();
    }
    if (!bt.defined() && (in.t[kGate].defined() || in.post != VGGT_NORM_NONE))
      refuse("gate and post_norm need a branch");
    if (in.post == VGGT_NORM_NONE && (in.t[kPostWeight].defined() || in.t[kPostBias].defined()))
      refuse("post_weight and post_bias need a post_norm");
    a.norm = in.norm;
    a.post_norm = in.post;
    a.eps = (float)in.eps;
  }
};

c10::Device device_of(const NormIn& in, const at::Tensor& a, const at::Tensor& b) {
  return one_device(in.t[kX], there(in.t[kBranch]), there(in.t[kWeight]), there(in.t[kBias]),
                    there(in.t[kGate]), there(in.t[kPostWeight]), there(in.t[kPostBias]), there(a),
                    there(b));
}

// (y, h); h undefined without a branch
std::pair<at::Tensor, at::Tensor> norm_forward(const NormIn& in, const at::Tensor& out,
                                               const at::Tensor& hout) {
  NormCall c(in);
  const at::Tensor& xt = in.t[kX];
  const bool both = in.t[kBranch].defined();
  if (out.defined()) check_given("out", out, xt.sizes(), in.type);
  if (hout.defined()) {
    if (!both) refuse("stream_out needs a branch: without one the stream is x");
    check_given("stream_out", hout, xt.sizes(), c.stream);
  }
  static const char* inputs[kNormTensors] = {"x",    "branch",      "weight",   "bias",
                                             "gate", "post_weight", "post_bias"};
  // a row is read whole before it is written
  for (int k = 0; k < kNormTensors; ++k) {
    check_apart("out", out, inputs[k], in.t[k], k <= kBranch);
    check_apart("stream_out", hout, inputs[k], in.t[k], k <= kBranch);
  }
  check_apart("out", out, "stream_out", hout, false);
  const c10::cuda::CUDAGuard guard(device_of(in, out, hout));
  at::Tensor y = out.defined() ? out : at::empty(xt.sizes(), xt.options().dtype(in.type));
  at::Tensor h = !both ? at::Tensor() : hout.defined() ? hout : at::empty(xt.sizes(), xt.options());
  written(out);
  written(hout);
  check(vggt_residual_norm(&c.a, both ? h.data_ptr() : nullptr, c.a.width, y.data_ptr(), c.a.width,
                           c10::cuda::getCurrentCUDAStream().stream()));
  return {y, h};
}

// The gradients of the call's tensors, in their order, where `wanted`.
variable_list norm_backward(const NormIn& in, const at::Tensor& dy, const at::Tensor& dh,
                            const bool* wanted) {
  NormCall c(in);
  const at::Tensor& xt = in.t[kX];
  if ((dy.defined() && (dy.sizes() != xt.sizes() || dy.scalar_type() != in.type)) ||
      (dh.defined() && (dh.sizes() != xt.sizes() || dh.scalar_type() != c.stream)))
    refuse("the gradients must have the outputs' shapes and dtypes");
  const c10::Device device = device_of(in, dy, dh);
  const c10::cuda::CUDAGuard guard(device);
  vggt_residual_norm_grads g{};
  Rows ry, rh;
  if (dy.defined()) {
    ry = Rows(dy);
    g.dy = ry.data();
    g.dy_stride = ry.stride;
  }
  if (dh.defined()) {
    rh = Rows(dh);
    g.dh = rh.data();
    g.dh_stride = rh.stride;
  }
  variable_list d(kNormTensors);
  void** to[kNormTensors] = {&g.dx,    &g.dbranch,      &g.dweight,   &g.dbias,
                             &g.dgate, &g.dpost_weight, &g.dpost_bias};
  for (int k = 0; k < kNormTensors; ++k) {
    const at::Tensor& t = in.t[k];
    if (!wanted[k] || !t.defined()) continue;
    // the sums of no rows are zeros
    d[k] = c.a.rows > 0 ? at::empty(t.sizes(), t.options()) : at::zeros(t.sizes(), t.options());
    *to[k] = d[k].data_ptr();
  }
  g.dx_stride = g.dbranch_stride = c.a.width;
  if (c.a.rows == 0) return d;
  const size_t bytes =
      vggt_residual_norm_grad_workspace_size(c.a.rows, c.a.width, c.a.rows_per_gate);
  const at::Tensor ws = workspace(bytes, device);
  check(vggt_residual_norm_grad(&c.a, &g, ws.data_ptr(), bytes,
                                c10::cuda::getCurrentCUDAStream().stream()));
  return d;
}

struct NormFunction : public torch::autograd::Function<NormFunction> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const Maybe& branch,
                               const Maybe& weight, const Maybe& bias, const Maybe& gate,
                               const Maybe& post_weight, const Maybe& post_bias, int64_t norm,
                               int64_t post, double eps, int64_t type) {
    const variable_list t = {x,           value(branch),      value(weight),   value(bias),
                             value(gate), value(post_weight), value(post_bias)};
    const NormIn in(t, (int)norm, (int)post, eps, (at::ScalarType)type);
    auto both = norm_forward(in, {}, {});
    ctx->save_for_backward(t);
    ctx->saved_data["norm"] = norm;
    ctx->saved_data["post"] = post;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["type"] = type;
    ctx->set_materialize_grads(false);
    if (!branch.has_value()) return {both.first};
    return {both.first, both.second};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const at::Tensor dy = grads[0], dh = grads.size() > 1 ? grads[1] : at::Tensor();
    variable_list out(kNormTensors + 4);
    if (!dy.defined() && !dh.defined()) return out;
    const NormIn in(ctx->get_saved_variables(), (int)ctx->saved_data["norm"].toInt(),
                    (int)ctx->saved_data["post"].toInt(), ctx->saved_data["eps"].toDouble(),
                    (at::ScalarType)ctx->saved_data["type"].toInt());
    bool wanted[kNormTensors];
    for (int k = 0, edge = 0; k < kNormTensors; ++k)  // only what was given has an edge
      wanted[k] = in.t[k].defined() && ctx->needs_input_grad(edge++);
    variable_list d;
    {
      c10::AutoGradMode off(false);
      d = norm_backward(in, dy, dh, wanted);
    }
    d = once(std::move(d));
    std::copy(d.begin(), d.end(), out.begin());
    return out;
  }
};

// a: x, branch, weight, bias, gate, post_weight, post_bias, norm, post_norm, eps, dtype, out,
// stream_out -> (y, h)
PyObject* residual_norm(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded(n, 13, [&]() -> PyObject* {
    const NormIn in(o);
    const at::Tensor out = given_or_none(o[11], "out"), hout = given_or_none(o[12], "stream_out");
    const at::Tensor* t = in.t;
    no_tangents(t[0], t[1], t[2], t[3], t[4], t[5], t[6], out, hout);
    at::Tensor y, h;
    if (needs_graph(t[0], t[1], t[2], t[3], t[4], t[5], t[6], out, hout)) {
      if (out.defined() || hout.defined())
        refuse("out and stream_out are for calls without a gradient");
      variable_list both = NormFunction::apply(
          t[0], maybe(t[1]), maybe(t[2]), maybe(t[3]), maybe(t[4]), maybe(t[5]), maybe(t[6]),
          (int64_t)in.norm, (int64_t)in.post, in.eps, (int64_t)in.type);
      y = both[0];
      if (both.size() > 1) h = both[1];
    } else {
      std::tie(y, h) = norm_forward(in, out, hout);
    }
    PyObject *py = returned(o[11], y), *ph;
    if (h.defined()) {
      ph = returned(o[12], h);
    } else {
      ph = o[0];
      Py_INCREF(ph);
    }
    PyObject* both = py && ph ? PyTuple_Pack(2, py, ph) : nullptr;
    Py_XDECREF(py);
    Py_XDECREF(ph);
    return both;
  });
}

// ---- linear -----------------------------------------------------------------------------------
struct LinearIn {
  at::Tensor x, weight, bias, gate, residual, status;
  int activation = 0;
  bool head_major = false;
};

struct LinearCall {
  vggt_linear_args a{};
  const LinearIn& in;
  at::Tensor x, weight, held[2];
  Rows residual;
  at::ScalarType type, stream, z_type;

  // Checks; nothing is copied before lay_out.
  explicit LinearCall(const LinearIn& call) : in(call) {
    const at::Tensor &xt = in.x, &wt = in.weight;
    a.activation = in.activation;
    type = xt.scalar_type();
    a.dtype = dtype_of("x", type, false);
    if (wt.dim() != 2 || wt.scalar_type() != type || wt.size(0) < 1 || wt.size(1) < 1)
      refuse("weight must be [outer, inner], of x's dtype");
    a.outer = wt.size(0);
    a.inner = wt.size(1);
    if (in.head_major) {
      if (xt.dim() != 3 || xt.size(0) * xt.size(2) != a.inner)
        refuse("a head-major x must be [heads, rows, dim] with heads * dim the weight's inner size");
      a.rows = xt.size(1);
    } else {
      if (xt.dim() < 1 || xt.size(-1) != a.inner)
        refuse("x must be [..., inner] with the weight's inner size");
      a.rows = xt.numel() / a.inner;
    }
    const at::Tensor &bt = in.bias, &gt = in.gate;
    if (bt.defined() && (bt.dim() != 1 || bt.size(0) != a.outer || bt.scalar_type() != type))
      refuse("bias must be [outer], of x's dtype");
    if (gt.defined()) {
      if (gt.dim() != 1 || gt.size(0) != a.outer ||
          (gt.scalar_type() != type && gt.scalar_type() != at::kFloat))
        refuse("gate must be [outer], of x's dtype or FP32");
      a.gate_fp32 = gt.scalar_type() != type;
    }
    stream = type;
    if (in.residual.defined()) {
      stream = in.residual.scalar_type();
      if (stream != type && stream != at::kFloat) refuse("residual must be of x's dtype, or FP32");
      if (in.residual.sizes() != at::IntArrayRef(y_shape()))
        refuse("residual must have the result's shape");
    }
    a.stream_dtype = dtype_of("residual", stream, true);
    // the gate's gradient is a sum of what is formed from z: in fp32, so that it rounds but once
    z_type = in.gate.defined() ? at::kFloat : type;
    a.z_dtype = dtype_of("z", z_type, true);
  }

  std::vector<int64_t> y_shape() const {
    if (in.head_major) return {a.rows, a.outer};
    std::vector<int64_t> s(in.x.sizes().begin(), in.x.sizes().end());
    s.back() = a.outer;
    return s;
  }

  // The tensors as the C ABI takes them (on the device that the caller has made current).
  void lay_out() {
    const Rows w(in.weight);
    weight = w.t;
    a.weight = w.data();
    a.weight_stride = w.stride;
    if (in.head_major && in.x.size(0) > 1) {
      x = in.x.size(2) > 1 && in.x.stride(2) != 1 ? in.x.contiguous() : in.x;
      a.heads = x.size(0);
      a.x_head_stride = x.stride(0);
      a.x_stride = a.rows > 1 ? x.stride(1) : x.size(2);
    } else {
      const Rows rows(in.head_major ? in.x.squeeze(0) : in.x);
      x = rows.t;
      a.x_stride = rows.stride;
    }
    a.x = x.data_ptr();
    const at::Tensor* vectors[2] = {&in.bias, &in.gate};
    const void** to[2] = {&a.bias, &a.gate};
    for (int k = 0; k < 2; ++k)
      if (vectors[k]->defined()) {
        held[k] = vectors[k]->is_contiguous() ? *vectors[k] : vectors[k]->contiguous();
        *to[k] = held[k].data_ptr();
      }
  }
};

// (y, z); z, the activation's argument, only where `keep`
std::pair<at::Tensor, at::Tensor> linear_forward(const LinearIn& in, const at::Tensor& out,
                                                 bool keep) {
  LinearCall c(in);
  const std::vector<int64_t> shape = c.y_shape();
  if (out.defined()) check_given("out", out, shape, c.stream);
  int32_t* word = status_of(there(in.status));
  // tiles are read while others are written
  check_apart("out", out, "x", in.x, false);
  check_apart("out", out, "weight", in.weight, false);
  check_apart("out", out, "bias", in.bias, false);
  check_apart("out", out, "gate", in.gate, false);
  check_apart("out", out, "residual", in.residual, true);
  check_apart("out", out, "status", in.status, false);
  const c10::Device device = one_device(in.x, there(in.weight), there(in.bias), there(in.gate),
                                        there(in.residual), there(out), there(in.status));
  const c10::cuda::CUDAGuard guard(device);
  c.lay_out();
  if (in.residual.defined()) {
    c.residual = Rows(in.residual);
    c.a.residual = c.residual.data();
    c.a.residual_stride = c.residual.stride;
  }
  at::Tensor y = out.defined() ? out : at::empty(shape, in.x.options().dtype(c.stream)), z;
  if (keep) z = at::empty(shape, in.x.options().dtype(c.z_type));
  const size_t bytes = vggt_linear_workspace_size(&c.a);
  at::Tensor ws;
  if (bytes) ws = workspace(bytes, device);
  written(out);
  check(vggt_linear(&c.a, y.data_ptr(), c.a.outer, keep ? z.data_ptr() : nullptr, c.a.outer, word,
                    bytes ? ws.data_ptr() : nullptr, bytes,
                    c10::cuda::getCurrentCUDAStream().stream()));
  return {y, z};
}

// The gradients of x, weight, bias and gate, where `wanted`.
variable_list linear_backward(const LinearIn& in, const at::Tensor& dy, const at::Tensor& z,
                              const bool* wanted) {
  LinearCall c(in);
  if (dy.sizes() != at::IntArrayRef(c.y_shape())) refuse("the gradient must have the result's shape");
  c.a.stream_dtype = dtype_of("the gradient", dy.scalar_type(), true);
  int32_t* word = status_of(there(in.status));
  const c10::Device device = one_device(in.x, there(in.weight), there(in.bias), there(in.gate), &dy,
                                        there(z), there(in.status));
  const c10::cuda::CUDAGuard guard(device);
  c.lay_out();
  vggt_linear_grads g{};
  const Rows rdy(dy);
  Rows rz;
  g.dy = rdy.data();
  g.dy_stride = rdy.stride;
  if (z.defined()) {
    rz = Rows(z);
    g.z = rz.data();
    g.z_stride = rz.stride;
  }
  variable_list d(4);
  // a head-major dx whose heads do not end on 64 elements is turned round afterwards
  const bool heads = c.a.heads > 1, turn = heads && in.x.size(2) % 64 != 0;
  if (wanted[0]) {
    d[0] = turn ? at::empty({c.a.rows, c.a.inner}, in.x.options())
                : at::empty(in.x.sizes(), in.x.options());
    g.dx_stride = heads && !turn ? in.x.size(2) : c.a.inner;
    g.dx_head_stride = heads && !turn ? c.a.rows * in.x.size(2) : 0;
    g.dx = d[0].data_ptr();
  }
  if (wanted[1]) {
    d[1] = at::empty({c.a.outer, c.a.inner}, in.weight.options());
    g.dweight = d[1].data_ptr();
    g.dweight_stride = c.a.inner;
  }
  if (wanted[2] && in.bias.defined()) {
    d[2] = at::empty({c.a.outer}, in.x.options());
    g.dbias = d[2].data_ptr();
  }
  if (wanted[3] && in.gate.defined()) {
    d[3] = at::empty({c.a.outer}, in.gate.options());
    g.dgate = d[3].data_ptr();
  }
  const size_t bytes = vggt_linear_grad_workspace_size(&c.a, &g);
  at::Tensor ws;
  if (bytes) ws = workspace(bytes, device);
  check(vggt_linear_grad(&c.a, &g, word, bytes ? ws.data_ptr() : nullptr, bytes,
                         c10::cuda::getCurrentCUDAStream().stream()));
  if (d[0].defined() && turn)
    d[0] = d[0].view({c.a.rows, in.x.size(0), in.x.size(2)}).transpose(0, 1).contiguous();
  return d;
}

struct LinearFunction : public torch::autograd::Function<LinearFunction> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight,
                            const Maybe& bias, const Maybe& gate, const Maybe& residual,
                            int64_t activation, bool head_major, const Maybe& status) {
    LinearIn in{x, weight, value(bias), value(gate), value(residual), value(status),
                (int)activation, head_major};
    auto both = linear_forward(in, {}, activation != VGGT_ACT_NONE);
    ctx->save_for_backward({x, weight, in.bias, in.gate, both.second});
    ctx->saved_data["residual"] = in.residual.defined();
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["head_major"] = head_major;
    if (in.status.defined()) ctx->saved_data["status"] = in.status;
    ctx->set_materialize_grads(false);
    return both.first;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const at::Tensor dy = grads[0];
    variable_list out(8);
    if (!dy.defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    LinearIn in{saved[0], saved[1], saved[2], saved[3], at::Tensor(), at::Tensor(),
                (int)ctx->saved_data["activation"].toInt(), ctx->saved_data["head_major"].toBool()};
    const auto status = ctx->saved_data.find("status");
    if (status != ctx->saved_data.end()) in.status = status->second.toTensor();
    bool wanted[4], any = false;
    int edge = 0;  // only what was given has one
    for (int k = 0; k < 4; ++k) {
      wanted[k] = saved[k].defined() && ctx->needs_input_grad(edge++);
      any = any || wanted[k];
    }
    if (any) {
      variable_list d;
      {
        c10::AutoGradMode off(false);
        d = linear_backward(in, dy, saved[4], wanted);
      }
      d = once(std::move(d));
      std::copy(d.begin(), d.end(), out.begin());
    }
    if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(edge)) out[4] = dy;
    return out;
  }
};

// a: x, weight, bias, activation, gate, residual, head_major, out, status -> y
PyObject* linear(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    LinearIn in;
    in.x = tensor(o[0], "x");
    in.weight = tensor(o[1], "weight");
    in.bias = given_or_none(o[2], "bias");
    in.activation = activation_of(o[3]);
    in.gate = given_or_none(o[4], "gate");
    in.residual = given_or_none(o[5], "residual");
    in.head_major = truth(o[6], "head_major");
    in.status = given_or_none(o[8], "status");
    const at::Tensor out = given_or_none(o[7], "out");
    no_tangents(in.x, in.weight, in.bias, in.gate, in.residual, out);
    if (needs_graph(in.x, in.weight, in.bias, in.gate, in.residual, out)) {
      if (out.defined()) refuse("out is for calls without a gradient");
      return THPVariable_Wrap(LinearFunction::apply(
          in.x, in.weight, maybe(in.bias), maybe(in.gate), maybe(in.residual), (int64_t)in.activation,
          in.head_major, maybe(in.status)));
    }
    return returned(o[7], linear_forward(in, out, false).first);
  });
}

#define VGGT_METHOD(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {VGGT_METHOD(residual_norm), VGGT_METHOD(linear),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_block_binding", nullptr, -1, methods,
                      nullptr,               nullptr,          nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__block_binding() { return PyModule_Create(&module); }
