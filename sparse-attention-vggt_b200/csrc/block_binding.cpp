// Python binding of the dense operators around a block's attention (include/vggt_block.h).
//
// As cache_binding.cpp: a call's checks, allocations and the launch, in a few microseconds.
// vggt_sparse/block_ops.py documents the arguments, which come by position.
#include "vggt_block.h"

#include "binding.h"

#include <torch/csrc/Dtype.h>

#include <initializer_list>
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

// An output that the caller gives.
void check_given(const char* name, const at::Tensor& t, at::IntArrayRef sizes, at::ScalarType type) {
  if (t.sizes() != sizes || t.scalar_type() != type || !t.is_contiguous())
    refuse("%s must be contiguous, of the result's shape and dtype", name);
}

at::Tensor workspace(size_t bytes, c10::Device device) {
  return at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(device));
}

PyObject* tuple_of(std::initializer_list<const at::Tensor*> items) {
  PyObject* out = PyTuple_New((Py_ssize_t)items.size());
  if (!out) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor* t : items) {
    PyObject* o;
    if (t && t->defined()) {
      o = THPVariable_Wrap(*t);
      if (!o) {
        Py_DECREF(out);
        return nullptr;
      }
    } else {
      o = Py_None;
      Py_INCREF(o);
    }
    PyTuple_SET_ITEM(out, i++, o);
  }
  return out;
}

// ---- residual_norm ----------------------------------------------------------------------------
struct NormCall {
  vggt_residual_norm_args a{};
  Rows x, branch;
  at::ScalarType type, stream;
  const at::Tensor* params[5];  // weight, bias, gate, post_weight, post_bias
  at::Tensor held[5];

  // a: x, branch, weight, bias, gate, post_weight, post_bias, norm, post_norm, eps
  NormCall(PyObject* const* o, const at::Tensor* dtype_from, PyObject* dtype) {
    const at::Tensor& xt = tensor(o[0], "x");
    const at::Tensor* bt = tensor_or_none(o[1], "branch");
    check_rows("x", xt);
    stream = xt.scalar_type();
    a.stream_dtype = dtype_of("x", stream, true);
    type = dtype_from ? dtype_from->scalar_type() : bt ? bt->scalar_type() : stream;
    if (dtype != Py_None) {
      if (!THPDtype_Check(dtype)) refuse("dtype must be a torch.dtype");
      const at::ScalarType asked = reinterpret_cast<THPDtype*>(dtype)->scalar_type;
      if (bt && asked != type) refuse("dtype is the branch's where there is one");
      type = asked;
    }
    a.dtype = dtype_of(bt ? "branch" : "dtype", type, true);
    if (type != stream && stream != at::kFloat)
      refuse("x must be of the branch's dtype, or FP32");
    x = Rows(xt);
    a.rows = x.rows;
    a.width = x.width;
    if (bt) {
      if (bt->sizes() != xt.sizes()) refuse("branch must have x's shape");
      branch = Rows(*bt);
      a.branch = branch.data();
      a.branch_stride = branch.stride;
    }
    a.x = x.data();
    a.x_stride = x.stride;
    static const char* names[5] = {"weight", "bias", "gate", "post_weight", "post_bias"};
    vggt_vector* to[5] = {&a.weight, &a.bias, &a.gate, &a.post_weight, &a.post_bias};
    for (int k = 0; k < 5; ++k) {
      params[k] = tensor_or_none(o[2 + k], names[k]);
      if (!params[k]) continue;
      const at::Tensor& t = *params[k];
      if (k == 2) {
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
    if (!bt && (params[2] || o[8] != Py_None)) refuse("gate and post_norm need a branch");
    if (o[8] == Py_None && (params[3] || params[4]))
      refuse("post_weight and post_bias need a post_norm");
    a.norm = norm_of(o[7], "norm", false);
    a.post_norm = norm_of(o[8], "post_norm", true);
    a.eps = (float)number(o[9], "eps");
  }
};

PyObject* residual_norm(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded(n, 13, [&]() -> PyObject* {
    NormCall c(o, nullptr, o[10]);
    const at::Tensor &xt = tensor(o[0], "x");
    const at::Tensor *bt = tensor_or_none(o[1], "branch"), *out = tensor_or_none(o[11], "out"),
                     *hout = tensor_or_none(o[12], "stream_out");
    if (out) check_given("out", *out, xt.sizes(), c.type);
    if (hout) {
      if (!bt) refuse("stream_out needs a branch: without one the stream is x");
      check_given("stream_out", *hout, xt.sizes(), c.stream);
    }
    const c10::Device device = one_device(xt, bt, c.params[0], c.params[1], c.params[2],
                                          c.params[3], c.params[4], out, hout);
    const c10::cuda::CUDAGuard guard(device);
    const at::Tensor y = out ? *out : at::empty(xt.sizes(), xt.options().dtype(c.type));
    const at::Tensor h = !bt ? xt : hout ? *hout : at::empty(xt.sizes(), xt.options());
    check(vggt_residual_norm(&c.a, bt ? h.data_ptr() : nullptr, c.a.width, y.data_ptr(), c.a.width,
                             c10::cuda::getCurrentCUDAStream().stream()));
    PyObject *py = returned(o[11], y), *ph;
    if (bt) {
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

// (dx, dbranch, dweight, dbias, dgate, dpost_weight, dpost_bias); `wanted` has a bit for each.
PyObject* residual_norm_grad(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded(n, 14, [&]() -> PyObject* {
    const at::Tensor *dy = tensor_or_none(o[11], "dy"), *dh = tensor_or_none(o[12], "dh");
    NormCall c(o, nullptr, o[10]);
    const int64_t wanted = integer(o[13], "wanted");
    const at::Tensor& xt = tensor(o[0], "x");
    const at::Tensor* bt = tensor_or_none(o[1], "branch");
    if ((dy && (dy->sizes() != xt.sizes() || dy->scalar_type() != c.type)) ||
        (dh && (dh->sizes() != xt.sizes() || dh->scalar_type() != c.stream)))
      refuse("the gradients must have the outputs' shapes and dtypes");
    const c10::Device device = one_device(xt, bt, c.params[0], c.params[1], c.params[2],
                                          c.params[3], c.params[4], dy, dh);
    const c10::cuda::CUDAGuard guard(device);
    vggt_residual_norm_grads g{};
    Rows ry, rh;
    if (dy) {
      ry = Rows(*dy);
      g.dy = ry.data();
      g.dy_stride = ry.stride;
    }
    if (dh) {
      rh = Rows(*dh);
      g.dh = rh.data();
      g.dh_stride = rh.stride;
    }
    at::Tensor dx, db, dp[5];
    if (wanted & 1) {
      dx = at::empty(xt.sizes(), xt.options());
      g.dx = dx.data_ptr();
      g.dx_stride = c.a.width;
    }
    if ((wanted & 2) && bt) {
      db = at::empty(bt->sizes(), bt->options());
      g.dbranch = db.data_ptr();
      g.dbranch_stride = c.a.width;
    }
    void** to[5] = {&g.dweight, &g.dbias, &g.dgate, &g.dpost_weight, &g.dpost_bias};
    for (int k = 0; k < 5; ++k)
      if ((wanted & (4 << k)) && c.params[k]) {
        // the sums of no rows are zeros
        dp[k] = c.a.rows > 0 ? at::empty(c.params[k]->sizes(), c.params[k]->options())
                             : at::zeros(c.params[k]->sizes(), c.params[k]->options());
        *to[k] = dp[k].data_ptr();
      }
    if (c.a.rows == 0) return tuple_of({&dx, &db, &dp[0], &dp[1], &dp[2], &dp[3], &dp[4]});
    const size_t bytes =
        vggt_residual_norm_grad_workspace_size(c.a.rows, c.a.width, c.a.rows_per_gate);
    const at::Tensor ws = workspace(bytes, device);
    check(vggt_residual_norm_grad(&c.a, &g, bytes ? ws.data_ptr() : nullptr, bytes,
                                  c10::cuda::getCurrentCUDAStream().stream()));
    return tuple_of({&dx, &db, &dp[0], &dp[1], &dp[2], &dp[3], &dp[4]});
  });
}

// ---- linear -----------------------------------------------------------------------------------
struct LinearCall {
  vggt_linear_args a{};
  at::Tensor x, weight, held[2];
  Rows residual;
  const at::Tensor *xt, *wt, *params[2], *rt;
  int64_t inner = 0;
  bool head_major = false;
  at::ScalarType type, stream;

  // o: x, weight, bias, activation, gate, residual, head_major
  explicit LinearCall(PyObject* const* o) {
    xt = &tensor(o[0], "x");
    wt = &tensor(o[1], "weight");
    params[0] = tensor_or_none(o[2], "bias");
    params[1] = tensor_or_none(o[4], "gate");
    rt = tensor_or_none(o[5], "residual");
    a.activation = activation_of(o[3]);
    head_major = truth(o[6]);
    type = xt->scalar_type();
    a.dtype = dtype_of("x", type, false);
    if (wt->dim() != 2 || wt->scalar_type() != type || wt->size(0) < 1 || wt->size(1) < 1)
      refuse("weight must be [outer, inner], of x's dtype");
    a.outer = wt->size(0);
    inner = wt->size(1);
    if (head_major) {
      if (xt->dim() != 3 || xt->size(0) * xt->size(2) != inner)
        refuse("a head-major x must be [heads, rows, dim] with heads * dim the weight's inner size");
      a.rows = xt->size(1);
    } else {
      if (xt->dim() < 1 || xt->size(-1) != inner)
        refuse("x must be [..., inner] with the weight's inner size");
      a.rows = xt->numel() / inner;
    }
    for (int k = 0; k < 2; ++k) {
      if (!params[k]) continue;
      const at::Tensor& t = *params[k];
      if (t.dim() != 1 || t.size(0) != a.outer || t.scalar_type() != type)
        refuse("%s must be [outer], of x's dtype", k == 0 ? "bias" : "gate");
    }
    stream = type;
    if (rt) {
      stream = rt->scalar_type();
      if (stream != type && stream != at::kFloat) refuse("residual must be of x's dtype, or FP32");
      if (rt->sizes() != at::IntArrayRef(y_shape())) refuse("residual must have the result's shape");
    }
    a.stream_dtype = dtype_of("residual", stream, true);
  }

  std::vector<int64_t> y_shape() const {
    if (head_major) return {a.rows, a.outer};
    std::vector<int64_t> s(xt->sizes().begin(), xt->sizes().end());
    s.back() = a.outer;
    return s;
  }

  // The tensors as the kernels take them (on the device that the caller has made current).
  void lay_out() {
    a.inner = inner;
    const Rows w(*wt);
    weight = w.t;
    a.weight = w.data();
    a.weight_stride = w.stride;
    if (head_major && xt->size(0) > 1) {
      x = xt->size(2) > 1 && xt->stride(2) != 1 ? xt->contiguous() : *xt;
      a.heads = x.size(0);
      a.x_head_stride = x.stride(0);
      a.x_stride = a.rows > 1 ? x.stride(1) : x.size(2);
    } else {
      const Rows rows(head_major ? xt->squeeze(0) : *xt);
      x = rows.t;
      a.x_stride = rows.stride;
    }
    a.x = x.data_ptr();
    const void** to[2] = {&a.bias, &a.gate};
    for (int k = 0; k < 2; ++k)
      if (params[k]) {
        held[k] = params[k]->is_contiguous() ? *params[k] : params[k]->contiguous();
        *to[k] = held[k].data_ptr();
      }
    if (rt) {
      residual = Rows(*rt);
      a.residual = residual.data();
      a.residual_stride = residual.stride;
    }
  }
};

// y, or (y, z) with keep_z
PyObject* linear(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded(n, 10, [&]() -> PyObject* {
    LinearCall c(o);
    const at::Tensor *out = tensor_or_none(o[7], "out"), *status = tensor_or_none(o[9], "status");
    const bool keep_z = truth(o[8]);
    const std::vector<int64_t> shape = c.y_shape();
    if (out) check_given("out", *out, shape, c.stream);
    int32_t* word = status_of(status);
    const c10::Device device =
        one_device(*c.xt, c.wt, c.params[0], c.params[1], c.rt, out, status);
    const c10::cuda::CUDAGuard guard(device);
    c.lay_out();
    const at::Tensor y = out ? *out : at::empty(shape, c.xt->options().dtype(c.stream));
    at::Tensor z;
    if (keep_z) z = at::empty(shape, c.xt->options());
    const size_t bytes = vggt_linear_workspace_size(&c.a);
    at::Tensor ws;
    if (bytes) ws = workspace(bytes, device);
    check(vggt_linear(&c.a, y.data_ptr(), c.a.outer, keep_z ? z.data_ptr() : nullptr, c.a.outer,
                      word, bytes ? ws.data_ptr() : nullptr, bytes,
                      c10::cuda::getCurrentCUDAStream().stream()));
    if (!keep_z) return returned(o[7], y);
    return tuple_of({&y, &z});
  });
}

// (dx, dweight, dbias, dgate); `wanted` has a bit for each.
PyObject* linear_grad(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject* {
    LinearCall c(o);
    const at::Tensor& dy = tensor(o[7], "dy");
    const at::Tensor *z = tensor_or_none(o[8], "z"), *status = tensor_or_none(o[10], "status");
    const int64_t wanted = integer(o[9], "wanted");
    const std::vector<int64_t> shape = c.y_shape();
    if (dy.sizes() != at::IntArrayRef(shape)) refuse("the gradient must have the result's shape");
    // without the residual its type tells the result's
    c.a.stream_dtype = dtype_of("dy", dy.scalar_type(), true);
    int32_t* word = status_of(status);
    const c10::Device device =
        one_device(*c.xt, c.wt, c.params[0], c.params[1], c.rt, &dy, z, status);
    const c10::cuda::CUDAGuard guard(device);
    c.lay_out();
    c.a.residual = nullptr;
    vggt_linear_grads g{};
    const Rows rdy(dy);
    Rows rz;
    g.dy = rdy.data();
    g.dy_stride = rdy.stride;
    if (z) {
      rz = Rows(*z);
      g.z = rz.data();
      g.z_stride = rz.stride;
    }
    at::Tensor dx, dw, db, dg;
    // a head-major dx whose heads do not end on 64 elements is turned round afterwards
    const bool turn = c.a.heads > 1 && c.xt->size(2) % 64 != 0;
    if (wanted & 1) {
      if (turn)
        dx = at::empty({c.a.rows, c.inner}, c.xt->options());
      else
        dx = at::empty(c.xt->sizes(), c.xt->options());
      g.dx_stride = c.inner;
      if (c.a.heads > 1 && !turn) {
        g.dx_head_stride = c.a.rows * c.xt->size(2);
        g.dx_stride = c.xt->size(2);
      }
      g.dx = dx.data_ptr();
    }
    if (wanted & 2) {
      dw = at::empty({c.a.outer, c.inner}, c.wt->options());
      g.dweight = dw.data_ptr();
      g.dweight_stride = c.inner;
    }
    if ((wanted & 4) && c.params[0]) {
      db = at::empty({c.a.outer}, c.xt->options());
      g.dbias = db.data_ptr();
    }
    if ((wanted & 8) && c.params[1]) {
      dg = at::empty({c.a.outer}, c.xt->options());
      g.dgate = dg.data_ptr();
    }
    const size_t bytes = vggt_linear_grad_workspace_size(&c.a, &g);
    at::Tensor ws;
    if (bytes) ws = workspace(bytes, device);
    check(vggt_linear_grad(&c.a, &g, word, bytes ? ws.data_ptr() : nullptr, bytes,
                           c10::cuda::getCurrentCUDAStream().stream()));
    if (dx.defined() && turn)
      dx = dx.view({c.a.rows, c.xt->size(0), c.xt->size(2)}).transpose(0, 1).contiguous();
    return tuple_of({&dx, &dw, &db, &dg});
  });
}

#define VGGT_METHOD(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {VGGT_METHOD(residual_norm), VGGT_METHOD(residual_norm_grad),
                         VGGT_METHOD(linear),        VGGT_METHOD(linear_grad),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_block_binding", nullptr, -1, methods,
                      nullptr,               nullptr,          nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__block_binding() { return PyModule_Create(&module); }
