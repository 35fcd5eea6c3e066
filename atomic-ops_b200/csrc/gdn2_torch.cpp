// The short way from a Python call of an operator to its launch, with the backward of those that have one, and the
// optimizer's step, as a CPython extension.
//
// A decode step's kernels take a few microseconds, less than the interpreter needs to look at the
// tensors, allocate the outputs and pass the pointers on.  These functions do that for calls that need
// nothing else: tensors of the expected types and layouts on the current device, no gradients.  For
// any other call they return None, and the Python path of the operator copies, converts or raises.
// The checks here are a subset of that path's, so nothing is accepted that it would refuse.
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros_like.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include "gdn2_b200.h"

namespace {

// A plain tensor argument that needs no gradient of either mode, or null.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != at::kStrided || (t.requires_grad() && c10::GradMode::is_enabled())) return nullptr;
  if (t._fw_grad(0).defined()) return nullptr;
  return &t;
}
bool on16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
at::Tensor fresh(c10::IntArrayRef size, at::ScalarType type, c10::Device dev) {
  return at::Tensor(at::detail::empty_cuda(size, type, dev, std::nullopt));
}
PyObject* pair(at::Tensor a, at::Tensor b) {
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(a)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(b)));
  return r;
}
float* floats(const at::Tensor& t) { return static_cast<float*>(t.data_ptr()); }
gdn2_dtype dtype_of(at::ScalarType t) { return t == at::kBFloat16 ? GDN2_BF16 : GDN2_F32; }
// Whether `dev` is the current device: the launch and its workspace go there.
bool current(c10::Device dev) { return dev.index() == c10::cuda::current_device(); }

// A status other than OK leaves the call to the Python path, whose own call reports it.  torch's exceptions
// (out of memory) become their Python ones.

// recurrent(q, k, v, w, b, g, h0, lengths, h_index, h_out, scale, clip, flags)
PyObject* recurrent(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 13) Py_RETURN_NONE;
  gdn2_rec_desc d{};
  const at::Tensor* x[6];
  for (int i = 0; i < 6; ++i)
    if (!(x[i] = plain(a[i]))) Py_RETURN_NONE;
  const at::Tensor& q = *x[0];
  const auto type = q.scalar_type();
  const auto dev = q.device();
  if (q.dim() != 4 || (type != at::kFloat && type != at::kBFloat16) || !current(dev)) Py_RETURN_NONE;
  const int64_t B = q.size(0), H = q.size(1), L = q.size(2), D = q.size(3);
  if (B < 1 || H < 1 || L < 1 || D != 128 || B >= (1 << 26) || H >= (1 << 26) || L >= (1 << 30)) Py_RETURN_NONE;
  const int64_t per = 16 / q.element_size();
  for (int i = 0; i < 6; ++i) {
    const at::Tensor& t = *x[i];
    if (t.scalar_type() != type || t.device() != dev || t.sizes() != q.sizes() || t.stride(3) != 1 || !on16(t))
      Py_RETURN_NONE;
    for (int j = 0; j < 3; ++j) {
      d.stride[i][j] = q.size(j) == 1 ? 0 : t.stride(j);  // of a dimension of one: never used
      if (d.stride[i][j] % per) Py_RETURN_NONE;
    }
    if (d.stride[i][2] >= 1 << 27) Py_RETURN_NONE;
  }
  const int64_t state[4] = {B, H, D, D};
  const float* h0 = nullptr;
  if (a[6] != Py_None) {
    const at::Tensor* h = plain(a[6]);
    if (!h || h->device() != dev || h->scalar_type() != at::kFloat || h->dim() != 4 || !h->is_contiguous() || !on16(*h) ||
        h->size(1) != H || h->size(2) != D || h->size(3) != D || h->size(0) < 1 || h->size(0) >= (1 << 30) ||
        (a[8] == Py_None && h->size(0) != B))
      Py_RETURN_NONE;
    h0 = static_cast<const float*>(h->data_ptr());
    d.n_states = (int32_t)h->size(0);
  }
  const int32_t* ints[2] = {nullptr, nullptr};  // lengths, h_index
  for (int i = 0; i < 2; ++i) {
    if (a[7 + i] == Py_None) continue;
    const at::Tensor* t = plain(a[7 + i]);
    if (!t || t->device() != dev || t->scalar_type() != at::kInt || t->dim() != 1 || t->size(0) != B || !t->is_contiguous())
      Py_RETURN_NONE;
    ints[i] = static_cast<const int32_t*>(t->data_ptr());
  }
  if (ints[1] && !h0) Py_RETURN_NONE;
  at::Tensor h;
  if (a[9] != Py_None) {
    const at::Tensor* t = plain(a[9]);
    if (!t || t->device() != dev || t->scalar_type() != at::kFloat || t->sizes() != c10::IntArrayRef(state) ||
        !t->is_contiguous() || !on16(*t))
      Py_RETURN_NONE;
    // h0 itself without an index, or no overlap
    const float *lo = static_cast<const float*>(t->data_ptr()), *hi = lo + t->numel();
    if (h0 && lo < h0 + (int64_t)d.n_states * H * D * D && h0 < hi && (ints[1] || lo != h0)) Py_RETURN_NONE;
    h = *t;
  } else {
    h = fresh(state, at::kFloat, dev);
  }
  at::Tensor o;
  if (q.stride(1) < q.stride(2)) {  // token-major: so is o
    const int64_t size[4] = {B, H, L, D}, st[4] = {L * H * D, D, H * D, 1};
    o = at::Tensor(at::detail::empty_strided_cuda(size, st, at::kFloat, dev));
  } else {
    const int64_t size[4] = {B, H, L, D};
    o = fresh(size, at::kFloat, dev);
  }
  d.B = (int32_t)B; d.H = (int32_t)H; d.L = (int32_t)L; d.D = (int32_t)D;
  for (int j = 0; j < 3; ++j) d.o_stride[j] = o.stride(j);
  d.in_dtype = dtype_of(type);
  d.scale = (float)PyFloat_AsDouble(a[10]);
  d.clip = (float)PyFloat_AsDouble(a[11]);
  void* flags = PyLong_AsVoidPtr(a[12]);
  if (PyErr_Occurred()) return nullptr;
  at::Tensor ws;
  if (const size_t bytes = gdn2_recurrent_workspace_bytes(&d)) {
    const int64_t size[1] = {(int64_t)bytes};
    ws = fresh(size, at::kByte, dev);
  }
  const gdn2_status s = gdn2_recurrent(
      &d, x[0]->data_ptr(), x[1]->data_ptr(), x[2]->data_ptr(), x[3]->data_ptr(), x[4]->data_ptr(), x[5]->data_ptr(), h0,
      ints[1], ints[0], static_cast<float*>(o.data_ptr()), static_cast<float*>(h.data_ptr()),
      ws.defined() ? ws.data_ptr() : nullptr, static_cast<uint32_t*>(flags),
      c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  if (s != GDN2_OK) Py_RETURN_NONE;
  if (a[9] != Py_None && !h.is_inference()) h.unsafeGetTensorImpl()->bump_version();  // autograd may have saved it
  return pair(std::move(o), std::move(h));
  END_HANDLE_TH_ERRORS
}

// w4_linear(x, packed, scales, bias, residual, din, dout, group, act)
PyObject* w4_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9) Py_RETURN_NONE;
  const at::Tensor *x = plain(a[0]), *w = plain(a[1]), *sc = plain(a[2]);
  if (!x || !w || !sc) Py_RETURN_NONE;
  const auto type = x->scalar_type();
  const auto dev = x->device();
  const int64_t din = PyLong_AsLongLong(a[5]), dout = PyLong_AsLongLong(a[6]), group = PyLong_AsLongLong(a[7]);
  const int64_t act = PyLong_AsLongLong(a[8]);
  if (PyErr_Occurred()) return nullptr;
  if ((type != at::kFloat && type != at::kBFloat16) || !current(dev) || w->device() != dev || sc->device() != dev)
    Py_RETURN_NONE;
  if (din < 1 || dout < 1 || (group != 32 && group != 64 && group != 128)) Py_RETURN_NONE;
  const int64_t blocks = (dout + 31) / 32 * ((din + 127) / 128);  // the kernel trusts the buffers' sizes
  if (w->scalar_type() != at::kInt || w->numel() != blocks * 512 || !w->is_contiguous() ||
      sc->scalar_type() != at::kBFloat16 || sc->numel() != blocks * 32 * (128 / group) || !sc->is_contiguous())
    Py_RETURN_NONE;
  if (x->dim() != 2 || x->size(1) != din || x->size(0) < 1 || x->size(0) >= (1 << 30) || x->stride(1) != 1 || !on16(*x))
    Py_RETURN_NONE;
  gdn2_w4_desc d{};
  d.M = (int32_t)x->size(0); d.K = (int32_t)din; d.N = (int32_t)dout; d.group = (int32_t)group;
  d.dtype = dtype_of(type);
  d.act = (int32_t)act;
  d.x_stride = d.M == 1 ? 0 : x->stride(0);
  d.y_stride = dout;
  const float* bias = nullptr;
  if (a[3] != Py_None) {
    const at::Tensor* t = plain(a[3]);
    if (!t || t->device() != dev || t->scalar_type() != at::kFloat || t->dim() != 1 || t->size(0) != dout || !t->is_contiguous())
      Py_RETURN_NONE;
    bias = static_cast<const float*>(t->data_ptr());
  }
  const void* res = nullptr;
  if (a[4] != Py_None) {
    const at::Tensor* t = plain(a[4]);
    if (!t || t->device() != dev || t->scalar_type() != type || t->dim() != 2 || t->size(0) != d.M || t->size(1) != dout ||
        t->stride(1) != 1)
      Py_RETURN_NONE;
    res = t->data_ptr();
    d.res_stride = t->stride(0);
  }
  const int64_t size[2] = {d.M, dout};
  at::Tensor y = fresh(size, type, dev), ws;
  if (const size_t bytes = gdn2_w4_workspace_bytes(&d)) {
    const int64_t ws_size[1] = {(int64_t)bytes};
    ws = fresh(ws_size, at::kByte, dev);
  }
  const gdn2_status s = gdn2_w4_linear(&d, x->data_ptr(), w->data_ptr(), sc->data_ptr(), bias, res, y.data_ptr(),
                                       ws.defined() ? ws.data_ptr() : nullptr,
                                       c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  if (s != GDN2_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// beam_select(logits, scores, finished, eos)
PyObject* beam_select(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) Py_RETURN_NONE;
  const at::Tensor *x = plain(a[0]), *sc = plain(a[1]);
  if (!x || !sc || x->dim() != 3 || sc->dim() != 2) Py_RETURN_NONE;
  const auto type = x->scalar_type();
  const auto dev = x->device();
  const int64_t B = x->size(0), K = x->size(1), V = x->size(2);
  if ((type != at::kFloat && type != at::kBFloat16) || !current(dev) || B < 1 || K < 1 || K > 32 || V < 1 ||
      B >= (1 << 24) || V >= (1 << 30) || x->stride(2) != 1)
    Py_RETURN_NONE;
  if (sc->device() != dev || sc->scalar_type() != at::kFloat || sc->size(0) != B || sc->size(1) != K || !sc->is_contiguous())
    Py_RETURN_NONE;
  gdn2_beam_desc d{};
  d.B = (int32_t)B; d.K = (int32_t)K; d.V = (int32_t)V;
  d.dtype = dtype_of(type);
  d.stride_b = x->stride(0);
  d.stride_k = x->stride(1);
  d.eos = -1;
  if (a[3] != Py_None) {
    if (!PyLong_CheckExact(a[3])) Py_RETURN_NONE;
    const long long eos = PyLong_AsLongLong(a[3]);
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    if (eos < 0 || eos >= V) Py_RETURN_NONE;
    d.eos = (int32_t)eos;
  }
  const uint8_t* finished = nullptr;
  if (a[2] != Py_None) {
    const at::Tensor* t = plain(a[2]);
    if (!t || d.eos < 0 || t->device() != dev || t->scalar_type() != at::kBool || t->dim() != 2 || t->size(0) != B ||
        t->size(1) != K || !t->is_contiguous())
      Py_RETURN_NONE;
    finished = static_cast<const uint8_t*>(t->data_ptr());
  }
  const int64_t size[2] = {B, K};
  at::Tensor out = fresh(size, at::kFloat, dev), rows = fresh(size, at::kInt, dev), tokens = fresh(size, at::kInt, dev),
             done = fresh(size, at::kBool, dev), ws;
  if (const size_t bytes = gdn2_beam_workspace_bytes(&d)) {
    const int64_t ws_size[1] = {(int64_t)bytes};
    ws = fresh(ws_size, at::kByte, dev);
  }
  const gdn2_status s = gdn2_beam_select(
      &d, x->data_ptr(), static_cast<const float*>(sc->data_ptr()), finished, static_cast<float*>(out.data_ptr()),
      static_cast<int32_t*>(rows.data_ptr()), static_cast<int32_t*>(tokens.data_ptr()),
      static_cast<uint8_t*>(done.data_ptr()), ws.defined() ? ws.data_ptr() : nullptr,
      c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  if (s != GDN2_OK) Py_RETURN_NONE;
  PyObject* r = PyTuple_New(4);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(out)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(rows)));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(tokens)));
  PyTuple_SET_ITEM(r, 3, THPVariable_Wrap(std::move(done)));
  return r;
  END_HANDLE_TH_ERRORS
}

// ---- differentiable operators -----------------------------------------------------------------------
// The common call of linear and gated_scan, their backward with it.  What the Python path does besides (other types,
// copies, checks at once) it does; the results are the same.

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Like plain(), for a tensor that may need a gradient; `grad` becomes true where it does.
const at::Tensor* input(PyObject* o, bool& grad) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != at::kStrided || t.is_neg() || t._fw_grad(0).defined()) return nullptr;
  grad = grad || (t.requires_grad() && c10::GradMode::is_enabled());
  return &t;
}
at::Tensor workspace(size_t bytes, c10::Device dev) {
  if (!bytes) return {};
  const int64_t size[1] = {(int64_t)bytes};
  return fresh(size, at::kByte, dev);
}
const void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
cudaStream_t stream_of(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }
// Gradients of a backward under create_graph: a second derivative raises.
variable_list once(variable_list grads, const char* what) {
  if (!c10::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(
      std::string("trying to differentiate twice through ") + what + ", which has no second derivative", (int64_t)grads.size());
  return (*node)(std::move(grads));
}

// What a backward gets of saved tensors is what their hooks gave back (one that keeps them on the host returns copies in an
// order of its own): their strides are read there, and layouts that the kernels cannot read are copied.
// A view whose values are its memory's negated (the imaginary part of a conjugate is one) is copied too.
at::Tensor dense(const at::Tensor& t) {
  return t.is_contiguous() && on16(t) && !t.is_neg() ? t : t.clone(at::MemoryFormat::Contiguous);
}
// n rows of `width` elements that do not overlap and are not further apart than the products take.
bool near_rows(int64_t n, int64_t width, int64_t ld) { return ld >= width && ld <= (1 << 28) && n * ld <= (int64_t{1} << 36); }
at::Tensor matrix(const at::Tensor& t) {
  if (t.dim() != 2) return dense(t);
  const bool rows = (t.size(1) == 1 || t.stride(1) == 1) && (t.size(0) == 1 || near_rows(t.size(0), t.size(1), t.stride(0))) && on16(t) && !t.is_neg();
  return rows ? t : t.clone(at::MemoryFormat::Contiguous);
}

struct LinearCall {
  gdn2_linear_desc d;
  std::vector<int64_t> out;            // y's shape
};
at::Tensor linear_forward(const LinearCall& c, const at::Tensor& x, const at::Tensor& w, const at::Tensor& bias,
                          const at::Tensor& res, at::Tensor* z, uint32_t* flags, gdn2_status& s) {
  at::Tensor y = fresh(c.out, x.scalar_type(), x.device());
  if (z) *z = fresh(c.out, x.scalar_type(), x.device());
  at::Tensor ws = workspace(gdn2_linear_fwd_workspace_bytes(&c.d), x.device());
  s = gdn2_linear_fwd(&c.d, x.data_ptr(), w.data_ptr(), ptr(bias), ptr(res), y.data_ptr(), z ? z->data_ptr() : nullptr, ptr(ws),
                      flags, stream_of(x.device()));
  return y;
}
struct LinearFn : torch::autograd::Function<LinearFn> {
  // Of the inputs that may be missing only those that are there have an edge.
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias,
                            const std::optional<at::Tensor>& res, const LinearCall* c, uint32_t* flags) {
    at::Tensor z;
    gdn2_status s;
    at::Tensor y = linear_forward(*c, x, w, bias.value_or(at::Tensor()), res.value_or(at::Tensor()), c->d.act ? &z : nullptr,
                                  flags, s);
    TORCH_CHECK(s == GDN2_OK, "gdn2_linear_fwd: ", gdn2_status_string(s));
    ctx->save_for_backward({x, w, z});
    auto& data = ctx->saved_data;
    const gdn2_linear_desc& d = c->d;
    data["desc"] = std::vector<int64_t>{d.M, d.K, d.N, d.dtype, d.bias_dtype, d.act, bias.has_value(), res.has_value()};
    data["flags"] = (int64_t) reinterpret_cast<intptr_t>(flags);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto v = ctx->saved_data["desc"].toIntVector();
    gdn2_linear_desc d{(int32_t)v[0], (int32_t)v[1], (int32_t)v[2], (int32_t)v[3], (int32_t)v[4], (int32_t)v[5], 0, 0, 0};
    const auto dev = grads[0].device();
    const c10::cuda::CUDAGuard guard(dev);
    for (int i = 0; i < (d.act ? 3 : 2); ++i)
      TORCH_CHECK(saved[i].device() == dev && saved[i].scalar_type() == grads[0].scalar_type() && saved[i].dim() > 1 &&
                      saved[i].size(-1) == (i ? d.N : d.K) && saved[i].numel() == (int64_t)(i == 1 ? d.K : d.M) * (i ? d.N : d.K),
                  "linear: a saved tensor came back on another device, or with another type or size");
    const at::Tensor x = matrix(saved[0]), w = matrix(saved[1]), z = d.act ? dense(saved[2]) : at::Tensor();
    d.x_stride = x.dim() == 2 && d.M > 1 ? x.stride(0) : d.K;
    d.w_stride = d.K > 1 ? w.stride(0) : d.N;
    at::Tensor dy = dense(grads[0]), dx, dw, db;
    if (ctx->needs_input_grad(0)) dx = fresh(x.sizes(), x.scalar_type(), dev);
    if (ctx->needs_input_grad(1)) dw = fresh(w.sizes(), w.scalar_type(), dev);
    const int64_t n[1] = {d.N};
    const bool has_b = v[6], has_r = v[7];
    if (has_b && ctx->needs_input_grad(2)) db = fresh(n, d.bias_dtype == GDN2_BF16 ? at::kBFloat16 : at::kFloat, dev);
    const int32_t want = (dx.defined() ? 1 : 0) + (dw.defined() ? 2 : 0) + (db.defined() ? 4 : 0);
    if (want) {
      at::Tensor ws = workspace(gdn2_linear_bwd_workspace_bytes(&d, want), dev);
      const gdn2_status s = gdn2_linear_bwd(&d, x.data_ptr(), w.data_ptr(), ptr(z), dy.data_ptr(), ptr(dx), ptr(dw), ptr(db),
                                            ptr(ws), reinterpret_cast<uint32_t*>((intptr_t)ctx->saved_data["flags"].toInt()),
                                            stream_of(dev));
      TORCH_CHECK(s == GDN2_OK, "gdn2_linear_bwd: ", gdn2_status_string(s));
    }
    variable_list r{dx, dw, db, has_r && ctx->needs_input_grad(2 + has_b) ? grads[0] : at::Tensor(), at::Tensor(), at::Tensor()};
    return once(std::move(r), "linear");
  }
};

// linear(x, weight, bias, residual, act, flags)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) Py_RETURN_NONE;
  bool grad = false;
  const at::Tensor *x = input(a[0], grad), *w = input(a[1], grad);
  if (!x || !w || w->dim() != 2 || x->dim() < 2) Py_RETURN_NONE;
  const auto type = x->scalar_type();
  const auto dev = x->device();
  if ((type != at::kFloat && type != at::kBFloat16) || w->scalar_type() != type || !current(dev) || w->device() != dev ||
      !on16(*x) || !on16(*w) || !(x->dim() == 2 || x->is_contiguous()))
    Py_RETURN_NONE;
  const int64_t K = w->size(0), N = w->size(1), last = x->dim() - 1;
  if (x->size(last) != K || K < 1 || N < 1 || x->numel() < 1 || w->stride(1) != 1 || x->stride(last) != 1) Py_RETURN_NONE;
  const int64_t M = x->numel() / K;
  if (M >= (1 << 28) || K >= (1 << 28) || N >= (1 << 28)) Py_RETURN_NONE;
  LinearCall c{};
  c.d.M = (int32_t)M; c.d.K = (int32_t)K; c.d.N = (int32_t)N;
  c.d.dtype = dtype_of(type);
  c.d.act = (int32_t)PyLong_AsLong(a[4]);
  c.d.x_stride = M > 1 && x->dim() == 2 ? x->stride(0) : K;
  c.d.w_stride = K > 1 ? w->stride(0) : N;
  if (!near_rows(M, K, c.d.x_stride) || !near_rows(K, N, c.d.w_stride) || M * N > (int64_t{1} << 36)) Py_RETURN_NONE;
  c.out = x->sizes().vec();
  c.out[last] = N;
  std::optional<at::Tensor> bias, res;
  if (a[2] != Py_None) {
    const at::Tensor* t = input(a[2], grad);
    if (!t || t->device() != dev || t->dim() != 1 || t->size(0) != N || !t->is_contiguous() ||
        (t->scalar_type() != at::kFloat && t->scalar_type() != at::kBFloat16))
      Py_RETURN_NONE;
    bias = *t;
    c.d.bias_dtype = dtype_of(t->scalar_type());
  }
  if (a[3] != Py_None) {
    const at::Tensor* t = input(a[3], grad);
    if (!t || t->device() != dev || t->scalar_type() != type || t->sizes() != c10::IntArrayRef(c.out) || !t->is_contiguous())
      Py_RETURN_NONE;
    res = *t;
    c.d.res_stride = N;
  }
  uint32_t* flags = static_cast<uint32_t*>(PyLong_AsVoidPtr(a[5]));
  if (PyErr_Occurred()) return nullptr;
  if (grad) return THPVariable_Wrap(LinearFn::apply(*x, *w, bias, res, &c, flags));
  gdn2_status s;
  at::Tensor y = linear_forward(c, *x, *w, bias.value_or(at::Tensor()), res.value_or(at::Tensor()), nullptr, flags, s);
  if (s != GDN2_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

gdn2_gated_desc gated_desc(const at::Tensor& x, const at::Tensor& g) {
  gdn2_gated_desc d{};
  d.B = (int32_t)x.size(0); d.L = (int32_t)x.size(1); d.C = (int32_t)x.size(2);
  d.dtype = dtype_of(x.scalar_type());
  for (int i = 0; i < 2; ++i) {
    d.x_stride[i] = x.size(i) > 1 ? x.stride(i) : 0;
    d.g_stride[i] = g.size(i) > 1 ? g.stride(i) : 0;
  }
  return d;
}
struct GatedMasks {
  at::Tensor lengths, reset;
};
// Unit stride along C, on 4 bytes.
at::Tensor rows(const at::Tensor& t) {
  const bool as_is = (t.size(2) == 1 || t.stride(2) == 1) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 4 == 0 && !t.is_neg();
  return as_is ? t : t.clone(at::MemoryFormat::Contiguous);
}
struct GatedFn : torch::autograd::Function<GatedFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& g, const std::optional<at::Tensor>& first,
                               const GatedMasks* masks, uint32_t* flags) {
    const auto dev = x.device();
    const at::Tensor h0 = first.value_or(at::Tensor()), &lengths = masks->lengths, &reset = masks->reset;
    gdn2_gated_desc d = gated_desc(x, g);
    d.n_states = h0.defined() ? d.B : 0;
    const int64_t state[2] = {d.B, d.C};
    at::Tensor h = fresh(x.sizes(), x.scalar_type(), dev), last = fresh(state, at::kFloat, dev),
               marks = workspace(gdn2_gated_marks_bytes(&d), dev);
    const gdn2_status s = gdn2_gated_fwd(&d, x.data_ptr(), g.data_ptr(), static_cast<const float*>(ptr(h0)), nullptr,
                                         static_cast<const int32_t*>(ptr(lengths)), static_cast<const uint8_t*>(ptr(reset)),
                                         h.data_ptr(), floats(last), floats(marks), flags, stream_of(dev));
    TORCH_CHECK(s == GDN2_OK, "gdn2_gated_fwd: ", gdn2_status_string(s));
    ctx->save_for_backward({x, g, marks, lengths, reset});
    ctx->set_materialize_grads(false);
    ctx->saved_data["h0"] = h0.defined();
    ctx->saved_data["flags"] = (int64_t) reinterpret_cast<intptr_t>(flags);
    return {h, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto dev = saved[0].device();
    TORCH_CHECK(dev.is_cuda(), "gated_scan: a saved tensor came back on another device");
    const c10::cuda::CUDAGuard guard(dev);
    for (const auto& t : saved)
      TORCH_CHECK(!t.defined() || t.device() == dev, "gated_scan: a saved tensor came back on another device");
    for (const auto& t : grads)
      TORCH_CHECK(!t.defined() || t.device() == dev, "gated_scan: a saved tensor came back on another device");
    const auto size = saved[0].sizes();
    const auto type = saved[0].scalar_type();
    TORCH_CHECK(size.size() == 3 && saved[1].sizes() == size && saved[1].scalar_type() == type &&
                    saved[2].scalar_type() == at::kByte &&
                    (!saved[3].defined() || (saved[3].numel() == size[0] && saved[3].scalar_type() == at::kInt)) &&
                    (!saved[4].defined() || (saved[4].numel() == size[0] * size[1] && saved[4].scalar_type() == at::kBool)) &&
                    (!grads[0].defined() || (grads[0].sizes() == size && grads[0].scalar_type() == type)) &&
                    (!grads[1].defined() || (grads[1].size(0) == size[0] && grads[1].size(1) == size[2])),
                "gated_scan: a saved tensor came back with another type or size");
    const at::Tensor x = rows(saved[0]), g = rows(saved[1]), marks = dense(saved[2]), lengths = saved[3].defined() ? dense(saved[3]) : saved[3],
                     reset = saved[4].defined() ? dense(saved[4]) : saved[4];
    gdn2_gated_desc d = gated_desc(x, g);
    TORCH_CHECK((int64_t)gdn2_gated_marks_bytes(&d) == marks.numel(), "gated_scan: a saved tensor came back with another type or size");
    at::Tensor dh = grads[0], dlast = grads[1], dx = fresh(x.sizes(), x.scalar_type(), dev), dg = fresh(x.sizes(), x.scalar_type(), dev), d0;
    if (dh.defined()) {
      dh = dh.resolve_neg().contiguous();
      if (reinterpret_cast<uintptr_t>(dh.data_ptr()) % 4) dh = dh.clone();
    } else {
      dh = at::zeros_like(dx);
    }
    if (dlast.defined()) dlast = dlast.resolve_neg().contiguous();
    const int64_t state[2] = {d.B, d.C};
    if (ctx->saved_data["h0"].toBool() && ctx->needs_input_grad(2)) d0 = fresh(state, at::kFloat, dev);
    const gdn2_status s = gdn2_gated_bwd(&d, x.data_ptr(), g.data_ptr(), static_cast<const int32_t*>(ptr(lengths)),
                                         static_cast<const uint8_t*>(ptr(reset)), static_cast<const float*>(marks.data_ptr()),
                                         dh.data_ptr(), static_cast<const float*>(ptr(dlast)), dx.data_ptr(), dg.data_ptr(),
                                         static_cast<float*>(ptr(d0)),
                                         reinterpret_cast<uint32_t*>((intptr_t)ctx->saved_data["flags"].toInt()), stream_of(dev));
    TORCH_CHECK(s == GDN2_OK, "gdn2_gated_bwd: ", gdn2_status_string(s));
    variable_list r{dx, dg, d0, at::Tensor(), at::Tensor()};
    return once(std::move(r), "gated_scan");
  }
};

// gated_scan(x, g, h0, lengths, reset, h_index, h_out, flags)
PyObject* gated_scan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) Py_RETURN_NONE;
  bool grad = false;
  const at::Tensor *x = input(a[0], grad), *g = input(a[1], grad);
  if (!x || !g || x->dim() != 3 || g->sizes() != x->sizes()) Py_RETURN_NONE;
  const auto type = x->scalar_type();
  const auto dev = x->device();
  const int64_t B = x->size(0), L = x->size(1), C = x->size(2);
  if ((type != at::kFloat && type != at::kBFloat16) || g->scalar_type() != type || g->device() != dev || !current(dev) || B < 1 ||
      L < 1 || C < 1 || B >= (1 << 28) || L >= (1 << 30) || C >= (1 << 30))
    Py_RETURN_NONE;
  for (const at::Tensor* t : {x, g})
    if ((C > 1 && t->stride(2) != 1) || reinterpret_cast<uintptr_t>(t->data_ptr()) % 4) Py_RETURN_NONE;
  at::Tensor h0, ints[2], reset;       // ints: lengths, h_index
  if (a[2] != Py_None) {
    const at::Tensor* t = input(a[2], grad);
    if (!t || t->device() != dev || t->scalar_type() != at::kFloat || t->dim() != 2 || !t->is_contiguous() || t->size(1) != C ||
        t->size(0) < 1 || t->size(0) >= (1 << 30) || (a[5] == Py_None && t->size(0) != B))
      Py_RETURN_NONE;
    h0 = *t;
  }
  for (int i = 0; i < 2; ++i) {
    PyObject* o = a[i ? 5 : 3];
    if (o == Py_None) continue;
    const at::Tensor* t = plain(o);
    if (!t || t->device() != dev || t->scalar_type() != at::kInt || t->dim() != 1 || t->size(0) != B || !t->is_contiguous())
      Py_RETURN_NONE;
    ints[i] = *t;
  }
  if (a[4] != Py_None) {
    const at::Tensor* t = plain(a[4]);
    if (!t || t->device() != dev || t->scalar_type() != at::kBool || t->dim() != 2 || t->size(0) != B || t->size(1) != L ||
        !t->is_contiguous())
      Py_RETURN_NONE;
    reset = *t;
  }
  uint32_t* flags = static_cast<uint32_t*>(PyLong_AsVoidPtr(a[7]));
  if (PyErr_Occurred()) return nullptr;
  if (a[6] != Py_None || (ints[1].defined() && (grad || !h0.defined()))) Py_RETURN_NONE;
  if (grad) {
    const GatedMasks masks{ints[0], reset};
    auto r = GatedFn::apply(*x, *g, h0.defined() ? std::optional<at::Tensor>(h0) : std::nullopt, &masks, flags);
    return pair(std::move(r[0]), std::move(r[1]));
  }
  gdn2_gated_desc d = gated_desc(*x, *g);
  d.n_states = h0.defined() ? (int32_t)h0.size(0) : 0;
  const int64_t state[2] = {B, C};
  at::Tensor h = fresh(x->sizes(), type, dev), last = fresh(state, at::kFloat, dev);
  const gdn2_status s =
      gdn2_gated_fwd(&d, x->data_ptr(), g->data_ptr(), static_cast<const float*>(ptr(h0)), static_cast<const int32_t*>(ptr(ints[1])),
                     static_cast<const int32_t*>(ptr(ints[0])), static_cast<const uint8_t*>(ptr(reset)), h.data_ptr(), floats(last),
                     nullptr, flags, stream_of(dev));
  if (s != GDN2_OK) Py_RETURN_NONE;
  return pair(std::move(h), std::move(last));
  END_HANDLE_TH_ERRORS
}

// ---- the optimizer ----------------------------------------------------------------------------------
// Its step is one call over lists of tensors, so these are the whole host path, with errors of their own.

std::vector<at::Tensor> tensors(PyObject* list, const char* what) {
  TORCH_CHECK_TYPE(PyList_CheckExact(list), what, " must be a list");
  std::vector<at::Tensor> r;
  r.reserve(PyList_GET_SIZE(list));
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) {
    PyObject* o = PyList_GET_ITEM(list, i);
    TORCH_CHECK_TYPE(THPVariable_Check(o), what, " must hold tensors");
    r.push_back(THPVariable_Unpack(o));
  }
  return r;
}
void changed(const at::Tensor& t) {  // in place: autograd may have saved it
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// The codes or values of a moment: p's shape and order.
void check_moment(const at::Tensor& t, const at::Tensor& p, at::ScalarType type, const char* what) {
  TORCH_CHECK_VALUE(t.device() == p.device() && t.scalar_type() == type && t.sizes() == p.sizes() &&
                        (t.strides() == p.strides() || (t.is_contiguous() && p.is_contiguous())),
                    "AdamW: ", what, " of a ", p.sizes(), " parameter must be ", type, " of its shape and order on ",
                    p.device(), "; got ", t.sizes(), " ", t.scalar_type(), " on ", t.device());
}
void check_scale(const at::Tensor& t, const at::Tensor& p, const char* what) {
  TORCH_CHECK_VALUE(t.device() == p.device() && t.scalar_type() == at::kFloat && t.is_contiguous() &&
                        t.numel() == (p.numel() + 255) / 256,
                    "AdamW: ", what, " of a ", p.sizes(), " parameter must be ", (p.numel() + 255) / 256,
                    " contiguous float32 on ", p.device());
}

// A new reference's value in a dict, borrowed, or null without an error.
PyObject* item(PyObject* dict, PyObject* key) { return PyDict_GetItemWithError(dict, key); }
// The dict's tensor: it lives as long as the dict, whose lock (the interpreter's) the call holds.
const at::Tensor& tensor_of(PyObject* dict, PyObject* key, const char* what) {
  PyObject* o = item(dict, key);
  if (!o && PyErr_Occurred()) throw python_error();
  TORCH_CHECK_VALUE(o && THPVariable_Check(o), "AdamW: the state of a parameter has no tensor ", what);
  return THPVariable_Unpack(o);
}
struct Names {
  PyObject *params = PyUnicode_InternFromString("params"), *lr = PyUnicode_InternFromString("lr"),
           *wd = PyUnicode_InternFromString("weight_decay"), *step = PyUnicode_InternFromString("step"),
           *m = PyUnicode_InternFromString("exp_avg"), *v = PyUnicode_InternFromString("exp_avg_sq"),
           *ms = PyUnicode_InternFromString("exp_avg_scale"), *vs = PyUnicode_InternFromString("exp_avg_sq_scale");
};

// adamw_step(param_groups, state, beta1, beta2, eps, clip, spike, bits, loss, control) -> status, or None where a
// parameter with a gradient has no state yet (or control is None).
PyObject* adamw_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  static const Names names;
  TORCH_CHECK_TYPE(n == 10 && PyList_Check(a[0]) && PyDict_Check(a[1]), "adamw_step takes a list, a dict and 8 values");
  gdn2_adamw_desc d{};
  d.beta1 = PyFloat_AsDouble(a[2]);
  d.beta2 = PyFloat_AsDouble(a[3]);
  d.eps = PyFloat_AsDouble(a[4]);
  d.clip = PyFloat_AsDouble(a[5]);
  d.spike = PyFloat_AsDouble(a[6]);
  d.state_bits = (int32_t)PyLong_AsLong(a[7]);
  if (PyErr_Occurred()) return nullptr;
  const bool eight = d.state_bits == 8;
  const auto moment_type = eight ? at::kByte : at::kFloat;
  std::vector<at::Tensor> kept;          // gradients
  std::vector<const at::Tensor*> written;
  std::vector<gdn2_adamw_tensor> table;
  for (Py_ssize_t gi = 0, k = 0; gi < PyList_GET_SIZE(a[0]); ++gi) {
    PyObject* params = PyDict_Check(PyList_GET_ITEM(a[0], gi)) ? item(PyList_GET_ITEM(a[0], gi), names.params) : nullptr;
    if (params && PyList_Check(params)) k += PyList_GET_SIZE(params);
    kept.reserve(k);
    table.reserve(k);
    written.reserve(6 * k);
  }
  c10::Device dev(c10::kCPU);
  for (Py_ssize_t gi = 0; gi < PyList_GET_SIZE(a[0]); ++gi) {
    PyObject* group = PyList_GET_ITEM(a[0], gi);
    TORCH_CHECK_TYPE(PyDict_Check(group), "AdamW: a parameter group must be a dict");
    PyObject *params = item(group, names.params), *lr = item(group, names.lr), *wd = item(group, names.wd);
    TORCH_CHECK_VALUE(params && PyList_Check(params) && lr && wd, "AdamW: a parameter group needs params, lr and weight_decay");
    double rate = 0.0;
    at::Tensor rate_at;
    if (THPVariable_Check(lr)) rate_at = THPVariable_Unpack(lr);
    else rate = PyFloat_AsDouble(lr);
    const double decay = PyFloat_AsDouble(wd);
    if (PyErr_Occurred()) return nullptr;
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(params); ++i) {
      PyObject* key = PyList_GET_ITEM(params, i);
      TORCH_CHECK_TYPE(THPVariable_Check(key), "AdamW: params must hold tensors");
      const at::Tensor& q = THPVariable_Unpack(key);
      at::Tensor g = q.grad();
      if (!g.defined()) continue;
      PyObject* st = item(a[1], key);
      if (!st) {
        if (PyErr_Occurred()) return nullptr;
        Py_RETURN_NONE;
      }
      TORCH_CHECK_TYPE(PyDict_Check(st), "AdamW: the state of a parameter must be a dict");
      if (!PyDict_GET_SIZE(st) || a[9] == Py_None) Py_RETURN_NONE;
      gdn2_adamw_tensor t{};
      const auto type = q.scalar_type();
      if (table.empty()) dev = q.device();
      TORCH_CHECK(q.is_cuda(), "AdamW: the parameters must be on a CUDA device (the step runs only on the B200 kernels)");
      TORCH_CHECK_VALUE(q.device() == dev, "AdamW: parameters on ", q.device(), " and on ", dev, ": one optimizer steps one device's");
      TORCH_CHECK_VALUE(type == at::kFloat || type == at::kBFloat16, "AdamW: parameters must be float32 or bfloat16, not ", type);
      TORCH_CHECK_VALUE(q.layout() == at::kStrided && q.is_non_overlapping_and_dense() && !q.is_neg(),
                        "AdamW: a parameter's values must fill their memory, each at one place");
      TORCH_CHECK_VALUE(g.layout() == at::kStrided && g.device() == dev && g.sizes() == q.sizes() && !g.is_complex(),
                        "AdamW: a gradient must be dense, of its parameter's shape and device");
      if (g.scalar_type() != type || g.is_neg() || (g.strides() != q.strides() && !(g.is_contiguous() && q.is_contiguous()))) {
        const c10::cuda::CUDAGuard guard(dev);
        const at::NoGradGuard no_grad;
        at::Tensor c = at::empty_like(q);
        c.copy_(g);
        g = std::move(c);
      }
      const at::Tensor &m = tensor_of(st, names.m, "exp_avg"), &v = tensor_of(st, names.v, "exp_avg_sq"),
                       &step = tensor_of(st, names.step, "step");
      check_moment(m, q, moment_type, "exp_avg");
      check_moment(v, q, moment_type, "exp_avg_sq");
      TORCH_CHECK_VALUE(step.device() == dev && step.scalar_type() == at::kFloat && step.numel() == 1,
                        "AdamW: step must be one float32 value on ", dev);
      t.p = q.data_ptr(); t.g = g.data_ptr(); t.m = m.data_ptr(); t.v = v.data_ptr();
      t.step = floats(step);
      if (eight) {
        const at::Tensor &ms = tensor_of(st, names.ms, "exp_avg_scale"), &vs = tensor_of(st, names.vs, "exp_avg_sq_scale");
        check_scale(ms, q, "exp_avg_scale");
        check_scale(vs, q, "exp_avg_sq_scale");
        t.m_scale = floats(ms);
        t.v_scale = floats(vs);
        written.push_back(&ms);
        written.push_back(&vs);
      }
      if (rate_at.defined()) {
        TORCH_CHECK_VALUE(rate_at.device() == dev && rate_at.scalar_type() == at::kFloat && rate_at.numel() == 1,
                          "AdamW: a tensor for lr must be one float32 value on ", dev);
        t.lr_at = floats(rate_at);
      }
      t.lr = rate;
      t.weight_decay = decay;
      t.n = q.numel();
      t.dtype = dtype_of(type);
      table.push_back(t);
      for (const at::Tensor* t : {&q, &m, &v, &step}) written.push_back(t);
      kept.push_back(std::move(g));
    }
  }
  if (table.empty()) return PyLong_FromLong(GDN2_OK);
  const int32_t k = (int32_t)table.size();
  const c10::cuda::CUDAGuard guard(dev);
  const float* loss = nullptr;
  at::Tensor loss32;
  if (a[8] != Py_None) {
    TORCH_CHECK_TYPE(THPVariable_Check(a[8]), "AdamW: loss must be a tensor");
    loss32 = THPVariable_Unpack(a[8]);
    TORCH_CHECK_VALUE(loss32.device() == dev && loss32.numel() == 1, "AdamW: loss must be one value on ", dev);
    const at::NoGradGuard no_grad;
    loss32 = loss32.to(at::kFloat);
    loss = floats(loss32);
  }
  TORCH_CHECK_TYPE(THPVariable_Check(a[9]), "AdamW: control must be a tensor");
  const at::Tensor& control = THPVariable_Unpack(a[9]);
  TORCH_CHECK_VALUE(control.device() == dev && control.scalar_type() == at::kFloat && control.numel() == 5 && control.is_contiguous(),
                    "AdamW: control must be five float32 words on ", dev);
  const int64_t size[1] = {(int64_t)gdn2_adamw_workspace_bytes(&d, table.data(), k)};
  at::Tensor ws = fresh(size, at::kByte, dev);
  const gdn2_status s = gdn2_adamw_step(&d, table.data(), k, loss, control.data_ptr(), ws.data_ptr(),
                                        c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  if (s == GDN2_OK)
    for (const at::Tensor* t : written) changed(*t);
  return PyLong_FromLong(s);
  END_HANDLE_TH_ERRORS
}

// adamw_moments(m, v, m_scales, v_scales, out_m, out_v)
PyObject* adamw_moments(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 6, "adamw_moments takes 6 arguments");
  auto m = tensors(a[0], "exp_avg"), v = tensors(a[1], "exp_avg_sq"), ms = tensors(a[2], "scales"), vs = tensors(a[3], "scales");
  auto om = tensors(a[4], "out"), ov = tensors(a[5], "out");
  const size_t k = m.size();
  TORCH_CHECK_VALUE(v.size() == k && ms.size() == k && vs.size() == k && om.size() == k && ov.size() == k,
                    "AdamW: lists of different lengths");
  if (!k) return PyLong_FromLong(GDN2_OK);
  const auto dev = m[0].device();
  TORCH_CHECK(dev.is_cuda(), "AdamW: the moments must be on a CUDA device");
  const c10::cuda::CUDAGuard guard(dev);
  std::vector<gdn2_adamw_tensor> table(k);
  for (size_t i = 0; i < k; ++i) {
    gdn2_adamw_tensor& t = table[i];
    TORCH_CHECK_VALUE(m[i].device() == dev && m[i].is_non_overlapping_and_dense(), "AdamW: moments on several devices");
    check_moment(m[i], m[i], at::kByte, "exp_avg");
    check_moment(v[i], m[i], at::kByte, "exp_avg_sq");
    check_scale(ms[i], m[i], "exp_avg_scale");
    check_scale(vs[i], m[i], "exp_avg_sq_scale");
    check_moment(om[i], m[i], at::kFloat, "out");
    check_moment(ov[i], m[i], at::kFloat, "out");
    t.m = m[i].data_ptr(); t.v = v[i].data_ptr(); t.m_scale = floats(ms[i]); t.v_scale = floats(vs[i]);
    t.p = om[i].data_ptr(); t.g = ov[i].data_ptr();
    t.n = m[i].numel();
    t.dtype = GDN2_F32;
  }
  const gdn2_status s = gdn2_adamw_moments(table.data(), (int32_t)k, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  for (size_t i = 0; i < k; ++i) { changed(om[i]); changed(ov[i]); }
  return PyLong_FromLong(s);
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"recurrent", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(recurrent)), METH_FASTCALL, nullptr},
    {"w4_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(w4_linear)), METH_FASTCALL, nullptr},
    {"beam_select", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(beam_select)), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(linear)), METH_FASTCALL, nullptr},
    {"gated_scan", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(gated_scan)), METH_FASTCALL, nullptr},
    {"adamw_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(adamw_step)), METH_FASTCALL, nullptr},
    {"adamw_moments", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(adamw_moments)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "gdn2_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_gdn2_torch() { return PyModule_Create(&module); }
