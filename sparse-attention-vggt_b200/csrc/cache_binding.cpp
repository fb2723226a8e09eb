// Python binding of the streaming cache's entry points (include/vggt_cache.h).
//
// These calls are short, single tokens above all, so that what a call costs on
// the host counts: checked in Python and passed through ctypes a call took 15
// to 25 us, here it takes a third of that.  A function takes its arguments by position from
// vggt_sparse/kv_cache.py (which documents them), checks them, allocates what
// is not given and enqueues on the current stream of the tensors' device.
#include "binding.h"

#include <c10/cuda/CUDAGraphsC10Utils.h>

#include <map>
#include <utility>

#include "vggt_cache.h"

namespace {

int layout_of(PyObject* o) {
  if (PyUnicode_Check(o)) {
    if (PyUnicode_CompareWithASCIIString(o, "half") == 0) return VGGT_ROTARY_HALF;
    if (PyUnicode_CompareWithASCIIString(o, "interleaved") == 0) return VGGT_ROTARY_INTERLEAVED;
  }
  refuse("layout must be 'half' or 'interleaved'");
}

int half_dtype(const at::Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return VGGT_DTYPE_BF16;
  if (t.scalar_type() == at::kHalf) return VGGT_DTYPE_FP16;
  refuse("the paged cache requires BF16 or FP16");
}

void need(const char* name, const at::Tensor& t, at::ScalarType type, at::IntArrayRef sizes) {
  if (t.scalar_type() == type && t.sizes() == sizes && t.is_contiguous()) return;
  std::string shape;
  for (int64_t s : sizes) shape += (shape.empty() ? "" : ", ") + std::to_string(s);
  refuse("%s must be a contiguous %s tensor of shape (%s)", name,
         type == at::kInt ? "int32" : "float32", shape.c_str());
}

struct Pools {
  int dtype;
  int64_t pages, heads, page, dim, page_stride, head_stride, row_stride, width, seqs;
  const int32_t* table;
  int64_t slots() const { return width * page; }
};

Pools pools_of(const at::Tensor& k, const at::Tensor* v, const at::Tensor& table) {
  Pools p;
  p.dtype = half_dtype(k);
  if (k.dim() != 4 || k.stride(3) != 1)
    refuse("pools must be [pages, kv_heads, page, dim], last dimension contiguous");
  if (v && (v->sizes() != k.sizes() || v->strides() != k.strides() ||
            v->scalar_type() != k.scalar_type()))
    refuse("k_pages and v_pages must have the same shape, strides and dtype");
  if (table.dim() != 2 || table.scalar_type() != at::kInt || !table.is_contiguous())
    refuse("table must be contiguous int32 [seqs, width]");
  p.pages = k.size(0);
  p.heads = k.size(1);
  p.page = k.size(2);
  p.dim = k.size(3);
  p.page_stride = k.stride(0);
  p.head_stride = k.stride(1);
  p.row_stride = k.stride(2);
  p.width = table.size(1);
  p.seqs = table.size(0);
  p.table = static_cast<const int32_t*>(table.data_ptr());
  if (p.heads > 65535 || p.page > 1024 || p.dim > 1024) refuse("unsupported pool shape");
  return p;
}

// Strides of a dimension of size one are never used: any will do.
void plain_strides(Pools& p) {
  if (p.heads == 1) p.head_stride = p.page * p.row_stride;
  if (p.pages == 1) p.page_stride = p.heads * p.head_stride;
}

// Packed rows [tokens, heads, dim] and their strides.
struct Rows {
  at::Tensor t;
  int64_t token, head;
  explicit Rows(const at::Tensor& x) : t(x) {
    // those of a dimension of size one are never used, and may be anything
    head = t.size(1) == 1 ? t.size(2) : t.stride(1);
    token = t.size(0) == 1 ? t.size(1) * head : t.stride(0);
  }
  // whether the attention kernels take them as they are
  bool fit() const {
    return t.stride(2) == 1 && token % 8 == 0 && head % 8 == 0 &&
           reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  }
};

// A tensor argument with strides and an address that the kernels take, else a
// copy.  (A contiguous one at any address will do for append.)
Rows rows_of(const char* name, const at::Tensor& t, const at::Tensor& pages, int64_t heads,
             bool aligned) {
  if (t.dim() != 3 || t.size(2) != pages.size(3) || t.scalar_type() != pages.scalar_type() ||
      (heads > 0 && t.size(1) != heads))
    refuse("%s must be [tokens, heads, dim] with the pools' dim, dtype%s", name,
           heads > 0 ? " and heads" : "");
  const Rows rows(t);
  if (rows.fit()) return rows;
  return Rows(aligned ? t.clone(at::MemoryFormat::Contiguous) : t.contiguous());
}

struct Turn {
  const int32_t* positions = nullptr;
  const double* freq = nullptr;
  int axes = 0, pairs = 0, layout = 0;
};

Turn turn_of(const at::Tensor* positions, const at::Tensor* freq, PyObject* layout,
             int64_t tokens) {
  Turn t;
  if (!positions) return t;
  if (positions->dim() < 1 || positions->dim() > 2 || positions->size(0) != tokens ||
      positions->scalar_type() != at::kInt || !positions->is_contiguous())
    refuse("positions must be contiguous int32 [tokens] or [tokens, axes]");
  if (!freq || freq->scalar_type() != at::kDouble || freq->dim() != 1 || !freq->is_contiguous())
    refuse("frequencies must be a contiguous float64 vector (rotary_frequencies)");
  const int64_t axes = positions->dim() == 1 ? 1 : positions->size(1);
  if (axes > 4 || freq->size(0) > 65536) refuse("too many axes or frequencies");
  t.positions = static_cast<const int32_t*>(positions->data_ptr());
  t.freq = static_cast<const double*>(freq->data_ptr());
  t.axes = (int)axes;
  t.pairs = (int)freq->size(0);
  t.layout = layout_of(layout);
  return t;
}

// One workspace per stream, its front zeroed once: the stream's calls run one
// after another and each leaves the front at zero.  A call under graph capture
// gets a workspace of its own, since the graph may be replayed on any stream.
// Never freed: the allocator may be gone by the time statics are destroyed.
at::Tensor workspace_of(size_t bytes, c10::Device device, cudaStream_t stream) {
  constexpr int64_t kFront = VGGT_PAGED_WORKSPACE_ZERO_BYTES;
  const int64_t size = (int64_t)bytes < kFront ? kFront : (int64_t)bytes;
  auto make = [&](int64_t n) {
    at::Tensor t = at::empty({n}, at::TensorOptions().dtype(at::kByte).device(device));
    t.narrow(0, 0, kFront).zero_();
    return t;
  };
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None)
    return make(size);
  static auto* spaces = new std::map<std::pair<int, cudaStream_t>, at::Tensor>();
  at::Tensor& t = (*spaces)[{device.index(), stream}];
  if (!t.defined() || t.numel() < size) t = make(size < (1 << 20) ? 1 << 20 : size);
  return t;
}

PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    const at::Tensor &x = tensor(a[0], "x"), &pos = tensor(a[1], "positions"),
                     &freq = tensor(a[2], "frequencies");
    const at::Tensor* given = tensor_or_none(a[6], "out");
    int dtype;
    switch (x.scalar_type()) {
      case at::kBFloat16: dtype = VGGT_DTYPE_BF16; break;
      case at::kHalf: dtype = VGGT_DTYPE_FP16; break;
      case at::kFloat: dtype = VGGT_DTYPE_FP32; break;
      default: refuse("x must be BF16, FP16 or FP32");
    }
    if (x.dim() != 3 || x.stride(2) != 1)
      refuse("x must be [tokens, heads, dim], last dimension contiguous");
    if (x.size(1) > 65535 || x.size(2) > 65536) refuse("too many heads, or too wide ones");
    const Turn t = turn_of(&pos, &freq, a[3], x.size(0));
    if (given && (given->sizes() != x.sizes() || given->scalar_type() != x.scalar_type() ||
                  given->stride(2) != 1))
      refuse("out must have x's shape and dtype, last dimension contiguous");
    const c10::Device device = one_device(x, &pos, &freq, given);
    const c10::cuda::CUDAGuard guard(device);
    const at::Tensor out = given ? *given : at::empty(x.sizes(), x.options());
    check(vggt_rotary(x.data_ptr(), dtype, x.size(0), (int)x.size(1), (int)x.size(2), x.stride(0),
                      x.stride(1), t.positions, t.axes, t.freq, t.pairs, t.layout,
                      (float)number(a[4], "lengthen"), truth(a[5], "inverse"), out.data_ptr(), out.stride(0),
                      out.stride(1), c10::cuda::getCurrentCUDAStream().stream()));
    return returned(a[6], out);
  });
}

PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 17, [&]() -> PyObject* {
    const at::Tensor &kp = tensor(a[2], "k_pages"), &vp = tensor(a[3], "v_pages"),
                     &table = tensor(a[4], "table"), &before = tensor(a[5], "before"),
                     &starts = tensor(a[6], "starts");
    const at::Tensor *pos = tensor_or_none(a[7], "positions"),
                     *freq = tensor_or_none(a[8], "frequencies"),
                     *ids = tensor_or_none(a[11], "ids"),
                     *new_ids = tensor_or_none(a[12], "new_ids"),
                     *weights = tensor_or_none(a[13], "weights"),
                     *new_weights = tensor_or_none(a[14], "new_weights"),
                     *given = tensor_or_none(a[15], "after"),
                     *status = tensor_or_none(a[16], "status");
    Pools p = pools_of(kp, &vp, table);
    plain_strides(p);
    const Rows kr = rows_of("k", tensor(a[0], "k"), kp, p.heads, false);
    const Rows vr = rows_of("v", tensor(a[1], "v"), kp, p.heads, false);
    const at::Tensor &k = kr.t, &v = vr.t;
    const int64_t total = k.size(0);
    if (v.size(0) != total) refuse("k and v must have the same shape");
    const Turn t = turn_of(pos, freq, a[9], total);
    need("before", before, at::kInt, {p.seqs});
    need("starts", starts, at::kInt, {p.seqs + 1});
    if (ids) {
      need("ids", *ids, at::kInt, {p.seqs, p.heads, p.slots()});
      if (!new_ids) refuse("ids needs new_ids");
      need("new_ids", *new_ids, at::kInt, {total});
    }
    if (weights) {
      need("weights", *weights, at::kFloat, {p.seqs, p.heads, p.slots()});
      if (new_weights) need("new_weights", *new_weights, at::kFloat, {total});
    }
    if (given) {
      need("after", *given, at::kInt, {p.seqs});
      if (given->data_ptr() == before.data_ptr() && p.seqs > 0) refuse("after must not be before");
    }
    int32_t* word = status_of(status);
    const c10::Device device = one_device(k, &v, &kp, &vp, &table, &before, &starts, pos, freq,
                                          ids, new_ids, weights, new_weights, given, status);
    const c10::cuda::CUDAGuard guard(device);
    const at::Tensor after = given ? *given : at::empty({p.seqs}, before.options());
    check(vggt_paged_append(
        k.data_ptr(), v.data_ptr(), p.dtype, total, kr.token, kr.head, vr.token,
        vr.head, kp.data_ptr(), vp.data_ptr(), p.pages, (int)p.heads, (int)p.page, (int)p.dim,
        p.page_stride, p.head_stride, p.row_stride, p.table, p.width, p.seqs,
        static_cast<const int32_t*>(before.data_ptr()),
        static_cast<const int32_t*>(starts.data_ptr()), t.positions, t.axes, t.freq, t.pairs,
        t.layout, (float)number(a[10], "lengthen"), static_cast<int32_t*>(ptr(ids)),
        static_cast<const int32_t*>(ptr(new_ids)), static_cast<float*>(ptr(weights)),
        static_cast<const float*>(ptr(new_weights)), static_cast<int32_t*>(after.data_ptr()), word,
        c10::cuda::getCurrentCUDAStream().stream()));
    return returned(a[15], after);
  });
}

// q's heads over the pools': the group.
int64_t group_of(const at::Tensor& q, const Pools& p) {
  if (p.heads < 1 || q.size(1) < 1 || q.size(1) % p.heads)
    refuse("q's heads (%lld) must be a multiple of the pools' (%lld)", (long long)q.size(1),
           (long long)p.heads);
  return q.size(1) / p.heads;
}

PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 14, [&]() -> PyObject* {
    const at::Tensor &kp = tensor(a[1], "k_pages"), &vp = tensor(a[2], "v_pages"),
                     &table = tensor(a[3], "table"), &lengths = tensor(a[4], "lengths"),
                     &starts = tensor(a[5], "starts");
    const at::Tensor *given = tensor_or_none(a[10], "out"), *given_lse = tensor_or_none(a[11], "lse"),
                     *space = tensor_or_none(a[12], "workspace"),
                     *status = tensor_or_none(a[13], "status");
    Pools p = pools_of(kp, &vp, table);
    plain_strides(p);
    const Rows qr = rows_of("q", tensor(a[0], "q"), kp, 0, true);
    const at::Tensor& q = qr.t;
    const int64_t total = q.size(0), heads = q.size(1), group = group_of(q, p);
    if (group > 65535) refuse("too many heads");
    need("lengths", lengths, at::kInt, {p.seqs});
    need("starts", starts, at::kInt, {p.seqs + 1});
    const int64_t max_new = integer(a[6], "max_new");
    const int64_t max_len = a[7] == Py_None ? p.slots() : integer(a[7], "max_len");
    const float scale =
        a[9] == Py_None ? 1.f / std::sqrt((float)p.dim) : (float)number(a[9], "scale");
    if (given && (given->sizes() != q.sizes() || given->scalar_type() != q.scalar_type() ||
                  !Rows(*given).fit()))
      refuse("out must have q's shape and dtype and 16-byte aligned rows");
    if (given_lse) need("lse", *given_lse, at::kFloat, {total, heads});
    // its elements are taken as bytes that lie one behind the other
    if (space && !space->is_contiguous()) refuse("workspace must be contiguous");
    int32_t* word = status_of(status);
    const c10::Device device = one_device(q, &kp, &vp, &table, &lengths, &starts, given, given_lse,
                                          space, status);
    const c10::cuda::CUDAGuard guard(device);
    const at::Tensor out = given ? *given : at::empty(q.sizes(), q.options());
    const Rows to(out);
    const at::Tensor lse =
        given_lse ? *given_lse : at::empty({total, heads}, q.options().dtype(at::kFloat));
    if (p.seqs == 0) {  // the rows belong to no sequence; no kernel will run
      out.zero_();
      lse.fill_(-INFINITY);
      if (status && total > 0) status->as_strided({1}, {1}).bitwise_or_(VGGT_STATUS_BAD_LENGTH);
    }
    const size_t bytes = vggt_paged_attention_workspace_size(
        total, p.seqs, (int)p.heads, (int)group, (int)p.dim, max_new, max_len);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream().stream();
    const at::Tensor ws = space ? *space : workspace_of(bytes, device, stream);
    check(vggt_paged_attention(
        q.data_ptr(), p.dtype, total, qr.token, qr.head, kp.data_ptr(), vp.data_ptr(),
        p.pages, (int)p.heads, (int)p.page, (int)p.dim, p.page_stride, p.head_stride, p.row_stride,
        p.table, p.width, p.seqs, static_cast<const int32_t*>(lengths.data_ptr()),
        static_cast<const int32_t*>(starts.data_ptr()), (int)group, truth(a[8], "causal"), scale, max_new,
        max_len, out.data_ptr(), to.token, to.head, static_cast<float*>(lse.data_ptr()),
        word, ws.data_ptr(), ws.numel() * ws.element_size(), stream));
    PyObject *o = returned(a[10], out), *l = returned(a[11], lse);
    PyObject* both = o && l ? PyTuple_Pack(2, o, l) : nullptr;
    Py_XDECREF(o);
    Py_XDECREF(l);
    return both;
  });
}

PyObject* weigh(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 13, [&]() -> PyObject* {
    const at::Tensor &lse = tensor(a[1], "lse"), &kp = tensor(a[2], "k_pages"),
                     &table = tensor(a[3], "table"), &lengths = tensor(a[4], "lengths"),
                     &starts = tensor(a[5], "starts"), &weights = tensor(a[6], "weights");
    const at::Tensor* status = tensor_or_none(a[12], "status");
    Pools p = pools_of(kp, nullptr, table);
    plain_strides(p);
    const Rows qr = rows_of("q", tensor(a[0], "q"), kp, 0, true);
    const at::Tensor& q = qr.t;
    const int64_t total = q.size(0), heads = q.size(1), group = group_of(q, p);
    if (group > 65535) refuse("too many heads");
    need("lse", lse, at::kFloat, {total, heads});
    need("weights", weights, at::kFloat, {p.seqs, p.heads, p.slots()});
    need("lengths", lengths, at::kInt, {p.seqs});
    need("starts", starts, at::kInt, {p.seqs + 1});
    const int64_t max_len = a[8] == Py_None ? p.slots() : integer(a[8], "max_len");
    const float scale =
        a[10] == Py_None ? 1.f / std::sqrt((float)p.dim) : (float)number(a[10], "scale");
    int32_t* word = status_of(status);
    const c10::cuda::CUDAGuard guard(
        one_device(q, &lse, &kp, &table, &lengths, &starts, &weights, status));
    check(vggt_paged_weights(
        q.data_ptr(), p.dtype, total, qr.token, qr.head,
        static_cast<const float*>(lse.data_ptr()), kp.data_ptr(), p.pages, (int)p.heads,
        (int)p.page, (int)p.dim, p.page_stride, p.head_stride, p.row_stride, p.table, p.width,
        p.seqs, static_cast<const int32_t*>(lengths.data_ptr()),
        static_cast<const int32_t*>(starts.data_ptr()), (int)group, truth(a[9], "causal"), scale,
        (float)number(a[11], "decay"), integer(a[7], "max_new"), max_len,
        static_cast<float*>(weights.data_ptr()), word,
        c10::cuda::getCurrentCUDAStream().stream()));
    return returned(a[6], weights);
  });
}

PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 13, [&]() -> PyObject* {
    const at::Tensor &weights = tensor(a[0], "weights"), &ids = tensor(a[1], "ids"),
                     &kp = tensor(a[2], "k_pages"), &vp = tensor(a[3], "v_pages"),
                     &table = tensor(a[4], "table"), &lengths = tensor(a[5], "lengths");
    const at::Tensor *recent = tensor_or_none(a[8], "recent_from"),
                     *new_w = tensor_or_none(a[9], "out[0]"), *new_i = tensor_or_none(a[10], "out[1]"),
                     *new_n = tensor_or_none(a[11], "out[2]"),
                     *status = tensor_or_none(a[12], "status");
    Pools p = pools_of(kp, &vp, table);
    plain_strides(p);
    const int64_t shape[3] = {p.seqs, p.heads, p.slots()};
    need("weights", weights, at::kFloat, shape);
    need("ids", ids, at::kInt, shape);
    need("lengths", lengths, at::kInt, {p.seqs});
    if (new_w) need("out[0]", *new_w, at::kFloat, shape);
    if (new_i) need("out[1]", *new_i, at::kInt, shape);
    if (new_n) need("out[2]", *new_n, at::kInt, {p.seqs});
    if (recent) need("recent_from", *recent, at::kInt, {p.seqs});
    const int64_t budget = integer(a[6], "budget");
    const int64_t max_len = a[7] == Py_None ? p.slots() : integer(a[7], "max_len");
    int32_t* word = status_of(status);
    const c10::Device device = one_device(weights, &ids, &kp, &vp, &table, &lengths, recent, new_w,
                                          new_i, new_n, status);
    const c10::cuda::CUDAGuard guard(device);
    const at::Tensor w2 = new_w ? *new_w : at::empty(shape, weights.options());
    const at::Tensor i2 = new_i ? *new_i : at::empty(shape, ids.options());
    const at::Tensor n2 = new_n ? *new_n : at::empty({p.seqs}, lengths.options());
    const size_t bytes =
        vggt_paged_evict_workspace_size(p.seqs, (int)p.heads, p.slots(), budget);
    const at::Tensor ws =
        at::empty({(int64_t)bytes + 1}, at::TensorOptions().dtype(at::kByte).device(device));
    check(vggt_paged_evict(
        static_cast<const float*>(weights.data_ptr()), static_cast<const int32_t*>(ids.data_ptr()),
        p.dtype, kp.data_ptr(), vp.data_ptr(), p.pages, (int)p.heads, (int)p.page, (int)p.dim,
        p.page_stride, p.head_stride, p.row_stride, p.table, p.width, p.seqs,
        static_cast<const int32_t*>(lengths.data_ptr()), budget,
        static_cast<const int32_t*>(ptr(recent)), max_len, static_cast<float*>(w2.data_ptr()),
        static_cast<int32_t*>(i2.data_ptr()), static_cast<int32_t*>(n2.data_ptr()), word,
        ws.data_ptr(), bytes, c10::cuda::getCurrentCUDAStream().stream()));
    PyObject *w = returned(a[9], w2), *i = returned(a[10], i2), *l = returned(a[11], n2);
    PyObject* all = w && i && l ? PyTuple_Pack(3, w, i, l) : nullptr;
    Py_XDECREF(w);
    Py_XDECREF(i);
    Py_XDECREF(l);
    return all;
  });
}

#define VGGT_METHOD(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {VGGT_METHOD(rotary), VGGT_METHOD(append), VGGT_METHOD(attention),
                         VGGT_METHOD(weigh),  VGGT_METHOD(evict),  {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_cache_binding", nullptr, -1, methods,
                      nullptr,               nullptr,          nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__cache_binding() { return PyModule_Create(&module); }
