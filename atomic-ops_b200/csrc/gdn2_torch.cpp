// The short way from a Python call of a serving operator to its launch, as a CPython extension.
//
// A decode step's kernels take a few microseconds, less than the interpreter needs to look at the
// tensors, allocate the outputs and pass the pointers on.  These functions do that for calls that need
// nothing else: tensors of the expected types and layouts on the current device, no gradients.  For
// any other call they return None, and the Python path of the operator copies, converts or raises.
// The checks here are a subset of that path's, so nothing is accepted that it would refuse.
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/core/Tensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
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

PyMethodDef methods[] = {
    {"recurrent", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(recurrent)), METH_FASTCALL, nullptr},
    {"w4_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(w4_linear)), METH_FASTCALL, nullptr},
    {"beam_select", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(beam_select)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "gdn2_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_gdn2_torch() { return PyModule_Create(&module); }
