// Native form of the operator front-end for the calls a program makes every step: contiguous tensors of one
// type on the current device.  ops.py's Python form costs 25 to 30 us per call (attribute look-ups,
// torch functions and a ctypes call with 17 arguments), several times what the decode kernels take; this
// one 4 to 7 us.  Anything out of the ordinary - a cast, a copy, a broadcast, an error to report - makes a
// function here return None, and the caller goes through the Python form, which handles all of it.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "../../include/b200q.h"

namespace {

using at::Tensor;

// ---- scratch buffers: owned and grown by ops._workspaces, known here by address
struct Scratch {
  int dev, op;
  void* stream;
  void* ptr;
  size_t bytes;
};
std::vector<Scratch> g_scratch;   // a handful of (device, stream, operator) triples; guarded by the GIL

const Scratch* find_scratch(int dev, void* stream, int op, size_t need) {
  for (const Scratch& s : g_scratch)
    if (s.dev == dev && s.stream == stream && s.op == op) return s.bytes >= need ? &s : nullptr;
  return nullptr;
}

// B200Q_CHECK_STATUS=1 (read on every call, as the Python form does): status checks live there.
bool checked() {
  const char* e = getenv("B200Q_CHECK_STATUS");
  return e && e[0] == '1' && e[1] == 0;
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return B200Q_F32;
    case at::kHalf: return B200Q_F16;
    case at::kBFloat16: return B200Q_BF16;
    default: return -1;
  }
}

// A plain torch.Tensor (or Parameter) argument; nullptr for anything else.
const Tensor* tensor(PyObject* o) {
  return THPVariable_CheckTypeExact(Py_TYPE(o)) ? &THPVariable_Unpack(o) : nullptr;
}
bool integer(PyObject* o, int dflt, int* out) {
  if (o == Py_None) { *out = dflt; return true; }
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  const long v = PyLong_AsLongAndOverflow(o, &overflow);
  if (overflow != 0 || v < INT_MIN || v > INT_MAX) return false;   // the Python form says what is wrong with it
  *out = (int)v;
  return true;
}
bool affine(PyObject* o) { return PyUnicode_Check(o) && PyUnicode_CompareWithASCIIString(o, "affine") == 0; }

// Quantized matrix operands that need no cast and no copy: w uint32, scales and biases of type `t` and of one
// shape, all contiguous on `dev`.
bool plain_weights(const Tensor& w, const Tensor& s, const Tensor& b, at::ScalarType t, at::Device dev, int group, int bits) {
  if (w.scalar_type() != at::kUInt32 || s.scalar_type() != t || b.scalar_type() != t) return false;
  if (w.device() != dev || s.device() != dev || b.device() != dev) return false;
  const int64_t nd = w.dim();
  if (nd < 2 || s.dim() != nd || b.dim() != nd) return false;
  for (int64_t i = 0; i < nd - 1; ++i)
    if (s.size(i) != w.size(i) || b.size(i) != w.size(i)) return false;
  if (s.size(nd - 1) != b.size(nd - 1) || w.size(nd - 1) * 32 % bits != 0 || w.size(nd - 1) * 32 / bits != s.size(nd - 1) * group) return false;
  return w.is_contiguous() && s.is_contiguous() && b.is_contiguous();
}
bool current(at::Device dev) { return dev.is_cuda() && dev.index() == c10::cuda::current_device(); }
bool params_ok(int group, int bits) { return (group == 32 || group == 64 || group == 128) && bits >= 2 && bits <= 8 && bits != 7; }

PyObject* none() { Py_RETURN_NONE; }

// ---- quantized_matmul.  False: not an ordinary call (or the library refused it): take the Python form.
bool qmm_run(const Tensor& x, const Tensor& w, const Tensor& s, const Tensor& b, bool transpose, int group, int bits, Tensor* y) {
  const at::ScalarType t = x.scalar_type();
  const int dt = dtype_code(t);
  const at::Device dev = x.device();
  if (dt < 0 || !params_ok(group, bits) || !current(dev) || x.dim() < 2 || w.dim() != 2 || !x.is_contiguous() ||
      !plain_weights(w, s, b, t, dev, group, bits) || checked())
    return false;
  const int64_t inner = w.size(1) * 32 / bits;
  const int64_t K = x.size(-1), M = K ? x.numel() / K : 0, N = transpose ? w.size(0) : inner;
  if (M == 0 || N == 0 || K != (transpose ? inner : w.size(0))) return false;
  void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  const size_t need = b200q_qmm_workspace_bytes(dt, 1, M, N, K, group, bits, transpose);
  const Scratch* ws = find_scratch(dev.index(), stream, 0, need);
  if (!ws) return false;
  c10::SmallVector<int64_t, 6> size(x.sizes().begin(), x.sizes().end());
  size.back() = N;
  *y = at::detail::empty_cuda(size, t, dev, std::nullopt);
  return b200q_qmm(x.data_ptr(), static_cast<const uint32_t*>(w.data_ptr()), s.data_ptr(), b.data_ptr(), y->data_ptr(), dt, 1,
                   M, N, K, group, bits, transpose, 0, ws->ptr, ws->bytes, stream) == B200Q_OK;
}

// (x, w, scales, biases, transpose, group_size, bits, mode)
bool qmm_args(PyObject* const* a, Py_ssize_t n, const Tensor* (&t)[4], bool* transpose, int* group, int* bits) {
  if (n != 8) return false;
  for (int i = 0; i < 4; ++i)
    if (!(t[i] = tensor(a[i]))) return false;
  if (!PyBool_Check(a[4]) || !integer(a[5], 64, group) || !integer(a[6], 4, bits) || !affine(a[7])) return false;
  *transpose = a[4] == Py_True;
  return true;
}

PyObject* py_qmm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor* t[4];
  bool transpose;
  int group, bits;
  Tensor y;
  if (!qmm_args(a, n, t, &transpose, &group, &bits)) return none();
  if (!qmm_run(*t[0], *t[1], *t[2], *t[3], transpose, group, bits, &y)) return none();
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// ---- quantize, dequantize
PyObject* py_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {   // (w, group_size, bits, mode)
  HANDLE_TH_ERRORS
  int group, bits;
  const Tensor* w;
  if (n != 4 || !(w = tensor(a[0])) || !integer(a[1], 64, &group) || !integer(a[2], 4, &bits) || !affine(a[3])) return none();
  const at::ScalarType t = w->scalar_type();
  const int dt = dtype_code(t);
  const at::Device dev = w->device();
  if (dt < 0 || !params_ok(group, bits) || !current(dev) || w->dim() < 2 || !w->is_contiguous() || w->numel() == 0) return none();
  const int64_t K = w->size(-1);
  if (K % group != 0) return none();
  c10::SmallVector<int64_t, 6> size(w->sizes().begin(), w->sizes().end());
  size.back() = K * bits / 32;
  Tensor wq = at::detail::empty_cuda(size, at::kUInt32, dev, std::nullopt);
  size.back() = K / group;
  Tensor s = at::detail::empty_cuda(size, t, dev, std::nullopt), b = at::detail::empty_cuda(size, t, dev, std::nullopt);
  void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  if (b200q_quantize(w->data_ptr(), dt, w->numel() / K, K, group, bits, static_cast<uint32_t*>(wq.data_ptr()), s.data_ptr(),
                     b.data_ptr(), stream) != B200Q_OK)
    return none();
  PyObject* out = PyTuple_New(3);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(wq)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(s)));
  PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(std::move(b)));
  return out;
  END_HANDLE_TH_ERRORS
}

PyObject* py_dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {   // (w, scales, biases, group_size, bits, mode)
  HANDLE_TH_ERRORS
  int group, bits;
  const Tensor *w, *s, *b;
  if (n != 6 || !(w = tensor(a[0])) || !(s = tensor(a[1])) || !(b = tensor(a[2])) || !integer(a[3], 64, &group) ||
      !integer(a[4], 4, &bits) || !affine(a[5]))
    return none();
  const at::ScalarType t = s->scalar_type();
  const int dt = dtype_code(t);
  const at::Device dev = w->device();
  if (dt < 0 || !params_ok(group, bits) || !current(dev) || !plain_weights(*w, *s, *b, t, dev, group, bits) || w->numel() == 0)
    return none();
  const int64_t words = w->size(-1), K = words * 32 / bits;
  c10::SmallVector<int64_t, 6> size(w->sizes().begin(), w->sizes().end());
  size.back() = K;
  Tensor out = at::detail::empty_cuda(size, t, dev, std::nullopt);
  void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  if (b200q_dequantize(static_cast<const uint32_t*>(w->data_ptr()), s->data_ptr(), b->data_ptr(), dt, w->numel() / words, K, group,
                       bits, out.data_ptr(), stream) != B200Q_OK)
    return none();
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---- quantized_matmul with a gradient for x alone (frozen scales and biases)
struct QmmFn : public torch::autograd::Function<QmmFn> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& s, const Tensor& b,
                        bool transpose, int64_t group, int64_t bits, Tensor* y) {
    ctx->save_for_backward({w, s, b});
    ctx->saved_data["transpose"] = transpose;
    ctx->saved_data["group"] = group;
    ctx->saved_data["bits"] = bits;
    return *y;   // by address: a result passed as a tensor would come back as a view of itself
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool transpose = ctx->saved_data["transpose"].toBool();
    const int64_t group = ctx->saved_data["group"].toInt(), bits = ctx->saved_data["bits"].toInt();
    Tensor dx;
    pybind11::gil_scoped_acquire gil;   // the scratch table, and the Python forms
    auto python = [&](const char* module, const Tensor& dy) {
      auto wrap = [](const Tensor& t) { return pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(t)); };
      pybind11::object r = pybind11::module_::import(module).attr("quantized_matmul")(wrap(dy), wrap(saved[0]), wrap(saved[1]), wrap(saved[2]),
                                                                                      !transpose, group, bits);
      return Tensor(THPVariable_Unpack(r.ptr()));
    };
    if (at::GradMode::is_enabled()) {   // a graph of the gradient is asked for
      dx = python("mlx_b200.grad", grads[0].contiguous());
    } else {
      const Tensor dy = grads[0].contiguous();
      if (!qmm_run(dy, saved[0], saved[1], saved[2], !transpose, (int)group, (int)bits, &dx)) dx = python("mlx_b200.ops", dy);
    }
    return {dx, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

PyObject* py_qmm_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor* t[4];
  bool transpose;
  int group, bits;
  Tensor y;
  if (!qmm_args(a, n, t, &transpose, &group, &bits)) return none();
  if (t[2]->requires_grad() || t[3]->requires_grad()) return none();
  for (const Tensor* u : t)   // forward-mode differentiation: the Python form's autograd.Function says that it has none
    if (u->_fw_grad(0).defined()) return none();
  {
    at::AutoDispatchBelowAutograd below;
    if (!qmm_run(*t[0], *t[1], *t[2], *t[3], transpose, group, bits, &y)) return none();
  }
  if (t[0]->requires_grad() && at::GradMode::is_enabled())
    y = QmmFn::apply(*t[0], *t[1], *t[2], *t[3], transpose, (int64_t)group, (int64_t)bits, &y);
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// ---- gather_qmm and the gated expert layer
// An index operand as a view over the pairs: right-aligned to four dimensions.  `t` null: the default index, which is
// the offset into `lead` (the batch dimensions of the operand it selects from).
struct View {
  b200q_index v;
  int64_t shape[4];
};
bool make_view(const Tensor* t, at::IntArrayRef lead, at::Device dev, View* out) {
  for (int d = 0; d < 4; ++d) { out->shape[d] = 1; out->v.stride[d] = 0; }
  out->v.data = nullptr;
  out->v.elem_bytes = 4;
  const int64_t nd = t ? t->dim() : (int64_t)lead.size();
  if (nd > 4) return false;
  if (t) {
    const at::ScalarType k = t->scalar_type();
    if (t->device() != dev || (k != at::kLong && k != at::kInt && k != at::kUInt32)) return false;
    if (t->numel() == 0) return false;
    out->v.data = t->data_ptr();
    out->v.elem_bytes = k == at::kLong ? 8 : 4;
    for (int64_t d = 0; d < nd; ++d) {
      out->shape[4 - nd + d] = t->size(d);
      out->v.stride[4 - nd + d] = t->size(d) == 1 ? 0 : t->stride(d);
    }
  } else {
    int64_t st = 1;
    for (int64_t d = nd - 1; d >= 0; --d) {
      out->shape[4 - nd + d] = lead[d];
      out->v.stride[4 - nd + d] = lead[d] == 1 ? 0 : st;
      st *= lead[d];
    }
  }
  return true;
}
// The pairs' shape (and the output's leading dimensions); false where the views do not broadcast.
bool broadcast(View* a, View* b, int64_t nd_a, int64_t nd_b, int64_t shape[4], int64_t* n, c10::SmallVector<int64_t, 6>* lead) {
  *n = 1;
  for (int d = 0; d < 4; ++d) {
    if (a->shape[d] != b->shape[d] && a->shape[d] != 1 && b->shape[d] != 1) return false;
    shape[d] = a->shape[d] == 1 ? b->shape[d] : a->shape[d];
    *n *= shape[d];
  }
  lead->clear();
  for (int d = 4 - (int)std::max(nd_a, nd_b); d < 4; ++d) lead->push_back(shape[d]);
  return true;
}
int64_t product(at::IntArrayRef v) {
  int64_t n = 1;
  for (int64_t x : v) n *= x;
  return n;
}
// Index argument: None, or a plain tensor.
bool index_arg(PyObject* o, const Tensor** t) {
  if (o == Py_None) { *t = nullptr; return true; }
  return (*t = tensor(o)) != nullptr;
}

// (x, w, scales, biases, lhs_indices, rhs_indices, transpose, group_size, bits, mode)
PyObject* py_gather(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *x, *w, *s, *b, *li, *ri;
  int group, bits;
  if (n != 10 || !(x = tensor(a[0])) || !(w = tensor(a[1])) || !(s = tensor(a[2])) || !(b = tensor(a[3])) || !index_arg(a[4], &li) ||
      !index_arg(a[5], &ri) || (!li && !ri) || a[6] != Py_True || !integer(a[7], 64, &group) || !integer(a[8], 4, &bits) ||
      !affine(a[9]))
    return none();
  const at::Device dev = x->device();
  if (x->scalar_type() != at::kBFloat16 || !params_ok(group, bits) || !current(dev) || x->dim() < 2 || w->dim() < 3 ||
      !x->is_contiguous() || !plain_weights(*w, *s, *b, at::kBFloat16, dev, group, bits) || checked())
    return none();
  const int64_t M = x->size(-2), K = x->size(-1), N = w->size(-2), x_batch = product(x->sizes().slice(0, x->dim() - 2)),
                E = product(w->sizes().slice(0, w->dim() - 2));
  if (w->size(-1) * 32 / bits != K || M == 0 || N == 0 || K == 0 || x_batch == 0 || E == 0) return none();
  View l, r;
  int64_t shape[4], n_idx;
  c10::SmallVector<int64_t, 6> size;
  const auto xl = x->sizes().slice(0, x->dim() - 2), wl = w->sizes().slice(0, w->dim() - 2);
  if (!make_view(li, xl, dev, &l) || !make_view(ri, wl, dev, &r) ||
      !broadcast(&l, &r, li ? li->dim() : (int64_t)xl.size(), ri ? ri->dim() : (int64_t)wl.size(), shape, &n_idx, &size))
    return none();
  void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  const Scratch* ws = find_scratch(dev.index(), stream, 1, b200q_gather_qmm_workspace_bytes(B200Q_BF16, n_idx, x_batch, E, M, N, K, group, bits, 1));
  if (!ws) return none();
  size.push_back(M);
  size.push_back(N);
  Tensor y = at::detail::empty_cuda(size, at::kBFloat16, dev, std::nullopt);
  if (b200q_gather_qmm_indexed(x->data_ptr(), static_cast<const uint32_t*>(w->data_ptr()), s->data_ptr(), b->data_ptr(), &l.v, &r.v,
                               shape, y.data_ptr(), B200Q_BF16, x_batch, E, M, N, K, group, bits, ws->ptr, ws->bytes, stream) != B200Q_OK)
    return none();
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// A (w, scales, biases) triple of plain tensors.
bool triple(PyObject* o, const Tensor* (&t)[3]) {
  if (!(PyTuple_CheckExact(o) || PyList_CheckExact(o)) || PySequence_Fast_GET_SIZE(o) != 3) return false;
  for (int i = 0; i < 3; ++i)
    if (!(t[i] = tensor(PySequence_Fast_GET_ITEM(o, i)))) return false;
  return true;
}

// (x, gate, up, down, rhs_indices, lhs_indices, group_size, bits)
PyObject* py_swiglu(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *x, *g[3], *u[3], *d[3], *li, *ri;
  int group, bits;
  if (n != 8 || !(x = tensor(a[0])) || !triple(a[1], g) || !triple(a[2], u) || !triple(a[3], d) || !index_arg(a[4], &ri) || !ri ||
      !index_arg(a[5], &li) || !integer(a[6], 64, &group) || !integer(a[7], 4, &bits))
    return none();
  const at::Device dev = x->device();
  if (x->scalar_type() != at::kBFloat16 || !params_ok(group, bits) || !current(dev) || x->dim() < 2 || g[0]->dim() < 3 ||
      !x->is_contiguous() || checked())
    return none();
  for (const auto& t : {g, u, d})
    if (!plain_weights(*t[0], *t[1], *t[2], at::kBFloat16, dev, group, bits)) return none();
  const int64_t M = x->size(-2), K1 = x->size(-1), H = g[0]->size(-2), N2 = d[0]->size(-2),
                x_batch = product(x->sizes().slice(0, x->dim() - 2)), E = product(g[0]->sizes().slice(0, g[0]->dim() - 2));
  if (g[0]->sizes() != u[0]->sizes() || g[0]->size(-1) * 32 / bits != K1 || d[0]->size(-1) * 32 / bits != H ||
      g[0]->dim() != d[0]->dim() || g[0]->sizes().slice(0, g[0]->dim() - 2) != d[0]->sizes().slice(0, d[0]->dim() - 2) || M == 0 ||
      K1 == 0 || H == 0 || N2 == 0 || x_batch == 0 || E == 0)
    return none();
  View l, r;
  int64_t shape[4], n_idx;
  c10::SmallVector<int64_t, 6> size;
  const auto xl = x->sizes().slice(0, x->dim() - 2);
  if (!make_view(li, xl, dev, &l) || !make_view(ri, xl, dev, &r) ||
      !broadcast(&l, &r, li ? li->dim() : (int64_t)xl.size(), ri->dim(), shape, &n_idx, &size))
    return none();
  void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  const Scratch* ws = find_scratch(dev.index(), stream, 1, b200q_gather_qmm_swiglu_workspace_bytes(n_idx, E, M, H, K1));
  if (!ws) return none();
  size.push_back(M);
  size.push_back(N2);
  Tensor y = at::detail::empty_cuda(size, at::kBFloat16, dev, std::nullopt);
  auto w = [](const Tensor* t) { return static_cast<const uint32_t*>(t->data_ptr()); };
  if (b200q_gather_qmm_swiglu_indexed(x->data_ptr(), w(g[0]), g[1]->data_ptr(), g[2]->data_ptr(), w(u[0]), u[1]->data_ptr(),
                                      u[2]->data_ptr(), w(d[0]), d[1]->data_ptr(), d[2]->data_ptr(), &l.v, &r.v, shape, y.data_ptr(),
                                      B200Q_BF16, x_batch, E, M, H, K1, N2, group, bits, ws->ptr, ws->bytes, stream) != B200Q_OK)
    return none();
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// ---- microscaled 4-bit modes
// Mode argument: its code and group size; group_size and bits, where given, have to be the mode's.
bool fp4_mode(PyObject* mode, PyObject* group_size, PyObject* bits, int* code, int* group) {
  if (!PyUnicode_Check(mode)) return false;
  if (PyUnicode_CompareWithASCIIString(mode, "mxfp4") == 0) { *code = B200Q_MXFP4; *group = 32; }
  else if (PyUnicode_CompareWithASCIIString(mode, "nvfp4") == 0) { *code = B200Q_NVFP4; *group = 16; }
  else return false;
  int g, b;
  return integer(group_size, *group, &g) && integer(bits, 4, &b) && g == *group && b == 4;
}
// A global scale: None, or a contiguous float32 tensor of one element or of `each`.
bool global_arg(PyObject* o, int mode, int64_t each, at::Device dev, const float** out, bool* per_matrix) {
  *out = nullptr;
  *per_matrix = false;
  if (o == Py_None) return true;
  const Tensor* t = tensor(o);
  if (!t || mode != B200Q_NVFP4 || t->scalar_type() != at::kFloat || t->device() != dev || !t->is_contiguous()) return false;
  if (t->numel() != 1 && (t->numel() != each || each < 1)) return false;
  *per_matrix = t->numel() != 1;
  *out = static_cast<const float*>(t->data_ptr());
  return true;
}
bool on16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
bool fp4_weights(const Tensor& w, const Tensor& s, int group, at::Device dev) {
  if (w.scalar_type() != at::kUInt32 || s.scalar_type() != at::kByte || w.device() != dev || s.device() != dev) return false;
  const int64_t nd = w.dim();
  if (nd < 2 || s.dim() != nd || w.size(nd - 1) * 8 != s.size(nd - 1) * group) return false;
  for (int64_t i = 0; i < nd - 1; ++i)
    if (s.size(i) != w.size(i)) return false;
  return w.is_contiguous() && s.is_contiguous() && on16(w);
}
int64_t matrices(const Tensor& w) { return product(w.sizes().slice(0, w.dim() - 2)); }

PyObject* py_fp4_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {   // (w, group_size, bits, mode, global_scale)
  HANDLE_TH_ERRORS
  const Tensor* w;
  int mode, group;
  if (n != 5 || !(w = tensor(a[0])) || !fp4_mode(a[3], a[1], a[2], &mode, &group)) return none();
  const int dt = dtype_code(w->scalar_type());
  const at::Device dev = w->device();
  if (dt < 0 || !current(dev) || w->dim() < 2 || !w->is_contiguous() || w->numel() == 0) return none();
  const int64_t K = w->size(-1), rows = w->numel() / K;
  const float* g;
  bool each;
  if (K % group != 0 || !global_arg(a[4], mode, matrices(*w), dev, &g, &each)) return none();
  c10::SmallVector<int64_t, 6> size(w->sizes().begin(), w->sizes().end());
  size.back() = K / 8;
  Tensor wq = at::detail::empty_cuda(size, at::kUInt32, dev, std::nullopt);
  size.back() = K / group;
  Tensor s = at::detail::empty_cuda(size, at::kByte, dev, std::nullopt);
  void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  if (b200q_fp4_quantize(w->data_ptr(), dt, rows, K, mode, g, each ? w->size(-2) : rows, static_cast<uint32_t*>(wq.data_ptr()),
                         static_cast<uint8_t*>(s.data_ptr()), stream) != B200Q_OK)
    return none();
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(wq)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(s)));
  return out;
  END_HANDLE_TH_ERRORS
}

PyObject* py_fp4_dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {   // (w, scales, group_size, bits, mode, dtype code, global_scale)
  HANDLE_TH_ERRORS
  const Tensor *w, *s;
  int mode, group, dt;
  if (n != 7 || !(w = tensor(a[0])) || !(s = tensor(a[1])) || !fp4_mode(a[4], a[2], a[3], &mode, &group) || !integer(a[5], -1, &dt))
    return none();
  const at::Device dev = w->device();
  const float* g;
  bool each;
  if (dt < 0 || dt > B200Q_BF16 || !current(dev) || !fp4_weights(*w, *s, group, dev) || w->numel() == 0 ||
      !global_arg(a[6], mode, matrices(*w), dev, &g, &each))
    return none();
  const int64_t K = w->size(-1) * 8, rows = w->numel() / w->size(-1);
  c10::SmallVector<int64_t, 6> size(w->sizes().begin(), w->sizes().end());
  size.back() = K;
  Tensor out = at::detail::empty_cuda(size, dt == B200Q_F32 ? at::kFloat : (dt == B200Q_F16 ? at::kHalf : at::kBFloat16), dev, std::nullopt);
  void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  if (b200q_fp4_dequantize(static_cast<const uint32_t*>(w->data_ptr()), static_cast<const uint8_t*>(s->data_ptr()), mode, g,
                           each ? w->size(-2) : rows, dt, rows, K, out.data_ptr(), stream) != B200Q_OK)
    return none();
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---- products grouped by expert
bool sizes_ok(const Tensor& t, int64_t E, at::Device dev) {
  return (t.scalar_type() == at::kLong || t.scalar_type() == at::kInt) && t.dim() == 1 && t.size(0) == E && t.device() == dev && t.is_contiguous();
}

// (x, w, scales, sizes or None, group_size, bits, mode, global_scale_x, global_scale_w)
PyObject* py_qqmm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *x, *w, *s, *sizes;
  int mode, group;
  if (n != 9 || !(x = tensor(a[0])) || !(w = tensor(a[1])) || !(s = tensor(a[2])) || !index_arg(a[3], &sizes) ||
      !fp4_mode(a[6], a[4], a[5], &mode, &group))
    return none();
  const at::ScalarType t = x->scalar_type();
  const int dt = dtype_code(t);
  const at::Device dev = x->device();
  if (dt < 0 || !current(dev) || !x->is_contiguous() || !fp4_weights(*w, *s, group, dev) || checked()) return none();
  if (sizes ? x->dim() != 2 || w->dim() != 3 : x->dim() < 1 || w->dim() != 2) return none();
  const int64_t E = sizes ? w->size(0) : 1, N = w->size(-2), K = w->size(-1) * 8;
  const float *gx, *gw;
  bool each_x, each_w;
  if (x->size(-1) != K || x->numel() == 0 || N == 0 || E == 0 || (sizes && !sizes_ok(*sizes, E, dev)) ||
      !global_arg(a[7], mode, 1, dev, &gx, &each_x) || !global_arg(a[8], mode, E, dev, &gw, &each_w))
    return none();
  const int64_t T = x->numel() / K;
  void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  const Scratch* ws = find_scratch(dev.index(), stream, 2, b200q_grouped_qqmm_workspace_bytes(T, E, N, K, mode));
  if (!ws) return none();
  c10::SmallVector<int64_t, 6> size(x->sizes().begin(), x->sizes().end());
  size.back() = N;
  Tensor y = at::detail::empty_cuda(size, t, dev, std::nullopt);
  if (b200q_grouped_qqmm(x->data_ptr(), static_cast<const uint32_t*>(w->data_ptr()), static_cast<const uint8_t*>(s->data_ptr()),
                         sizes ? sizes->data_ptr() : nullptr, sizes && sizes->scalar_type() == at::kLong ? 8 : 4, y.data_ptr(), dt, T, E,
                         N, K, mode, gx, gw, each_w, ws->ptr, ws->bytes, stream) != B200Q_OK)
    return none();
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

bool grouped_run(const Tensor& x, const Tensor& w, const Tensor& sizes, bool transpose, Tensor* y) {
  const at::ScalarType t = x.scalar_type();
  const at::Device dev = x.device();
  if ((t != at::kHalf && t != at::kBFloat16) || w.scalar_type() != t || w.device() != dev || !current(dev) || x.dim() != 2 || w.dim() != 3 ||
      !x.is_contiguous() || !w.is_contiguous() || !on16(x) || !on16(w) || checked())
    return false;
  const int64_t E = w.size(0), N = w.size(transpose ? 1 : 2), K = w.size(transpose ? 2 : 1), T = x.size(0);
  if (x.size(1) != K || T == 0 || N == 0 || K == 0 || E == 0 || !sizes_ok(sizes, E, dev)) return false;
  void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  const Scratch* ws = find_scratch(dev.index(), stream, 2, b200q_grouped_mm_workspace_bytes(T, E, N, K, transpose));
  if (!ws) return false;
  *y = at::detail::empty_cuda({T, N}, t, dev, std::nullopt);
  return b200q_grouped_mm(x.data_ptr(), w.data_ptr(), sizes.data_ptr(), sizes.scalar_type() == at::kLong ? 8 : 4, y->data_ptr(),
                          dtype_code(t), T, E, N, K, transpose, ws->ptr, ws->bytes, stream) == B200Q_OK;
}
bool grouped_dw_run(const Tensor& dy, const Tensor& x, const Tensor& sizes, bool transpose, Tensor* dw) {
  const at::ScalarType t = x.scalar_type();
  const at::Device dev = x.device();
  if ((t != at::kHalf && t != at::kBFloat16) || dy.scalar_type() != t || dy.device() != dev || !current(dev) || x.dim() != 2 ||
      dy.dim() != 2 || sizes.dim() != 1 || !x.is_contiguous() || !dy.is_contiguous() || !on16(x) || !on16(dy) || checked())
    return false;
  const Tensor &a = transpose ? dy : x, &b = transpose ? x : dy;
  const int64_t E = sizes.size(0), N = a.size(1), K = b.size(1), T = x.size(0);
  if (dy.size(0) != T || T == 0 || N == 0 || K == 0 || E == 0 || !sizes_ok(sizes, E, dev)) return false;
  void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  const Scratch* ws = find_scratch(dev.index(), stream, 2, b200q_grouped_mm_dw_workspace_bytes(T, N, K));
  if (!ws) return false;
  *dw = at::detail::empty_cuda({E, N, K}, t, dev, std::nullopt);
  return b200q_grouped_mm_dw(a.data_ptr(), b.data_ptr(), sizes.data_ptr(), sizes.scalar_type() == at::kLong ? 8 : 4, dw->data_ptr(),
                             dtype_code(t), T, E, N, K, ws->ptr, ws->bytes, stream) == B200Q_OK;
}
bool boolean(PyObject* o, bool* out) {
  *out = o == Py_True;
  return PyBool_Check(o);
}

PyObject* py_grouped_mm(PyObject*, PyObject* const* a, Py_ssize_t n) {   // (x, w, sizes, transpose)
  HANDLE_TH_ERRORS
  const Tensor *x, *w, *sizes;
  bool transpose;
  Tensor y;
  if (n != 4 || !(x = tensor(a[0])) || !(w = tensor(a[1])) || !(sizes = tensor(a[2])) || !boolean(a[3], &transpose)) return none();
  if (!grouped_run(*x, *w, *sizes, transpose, &y)) return none();
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}
PyObject* py_grouped_mm_dw(PyObject*, PyObject* const* a, Py_ssize_t n) {   // (dy, x, sizes, transpose)
  HANDLE_TH_ERRORS
  const Tensor *dy, *x, *sizes;
  bool transpose;
  Tensor dw;
  if (n != 4 || !(dy = tensor(a[0])) || !(x = tensor(a[1])) || !(sizes = tensor(a[2])) || !boolean(a[3], &transpose)) return none();
  if (!grouped_dw_run(*dy, *x, *sizes, transpose, &dw)) return none();
  return THPVariable_Wrap(std::move(dw));
  END_HANDLE_TH_ERRORS
}

// grouped_mm with gradients for x and w
struct GroupedFn : public torch::autograd::Function<GroupedFn> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& sizes, bool transpose, Tensor* y) {
    ctx->save_for_backward({x, w, sizes});
    ctx->saved_data["transpose"] = transpose;
    return *y;   // by address: a result passed as a tensor would come back as a view of itself
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &sizes = saved[2];
    const bool transpose = ctx->saved_data["transpose"].toBool();
    Tensor dx, dw;
    if (!grads[0].defined()) return {dx, dw, Tensor(), Tensor(), Tensor()};
    const bool for_x = ctx->needs_input_grad(0), for_w = ctx->needs_input_grad(1);   // of this pass, which may want one of the two only
    pybind11::gil_scoped_acquire gil;   // the scratch table, and the Python forms
    auto wrap = [](const Tensor& v) { return pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(v)); };
    if (at::GradMode::is_enabled()) {   // a graph of the gradients is asked for: the Python form makes one
      const pybind11::tuple r = pybind11::module_::import("mlx_b200.grad").attr("_grouped_mm_vjp")(
          wrap(grads[0]), wrap(x), wrap(w), wrap(sizes), transpose, for_x, for_w);
      if (for_x) dx = THPVariable_Unpack(r[0].ptr());
      if (for_w) dw = THPVariable_Unpack(r[1].ptr());
      return {dx, dw, Tensor(), Tensor(), Tensor()};
    }
    const Tensor dy = grads[0].contiguous();
    at::AutoDispatchBelowAutograd below;
    auto python = [&](const char* name, const Tensor& p, const Tensor& q, bool t) {
      pybind11::object r = pybind11::module_::import("mlx_b200.ops").attr(name)(wrap(p), wrap(q), wrap(sizes), t);
      return Tensor(THPVariable_Unpack(r.ptr()));
    };
    if (for_x && !grouped_run(dy, w, sizes, !transpose, &dx)) dx = python("grouped_mm", dy, w, !transpose);
    if (for_w && !grouped_dw_run(dy, x, sizes, transpose, &dw)) dw = python("grouped_mm_dw", dy, x, transpose);
    return {dx, dw, Tensor(), Tensor(), Tensor()};
  }
};
PyObject* py_grouped_mm_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {   // (x, w, sizes, transpose)
  HANDLE_TH_ERRORS
  const Tensor *x, *w, *sizes;
  bool transpose;
  Tensor y;
  if (n != 4 || !(x = tensor(a[0])) || !(w = tensor(a[1])) || !(sizes = tensor(a[2])) || !boolean(a[3], &transpose)) return none();
  if (x->_fw_grad(0).defined() || w->_fw_grad(0).defined()) return none();   // the Python form says that it has no forward mode
  {
    at::AutoDispatchBelowAutograd below;
    if (!grouped_run(*x, *w, *sizes, transpose, &y)) return none();
  }
  if ((x->requires_grad() || w->requires_grad()) && at::GradMode::is_enabled()) y = GroupedFn::apply(*x, *w, *sizes, transpose, &y);
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// ---- routing, rows between tokens and experts, adapters.  None of them uses the scratch table: what scratch they need is allocated per call.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void* stream_of(at::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }
Tensor fresh(at::IntArrayRef size, at::ScalarType t, at::Device dev) { return at::detail::empty_cuda(size, t, dev, std::nullopt); }
// A tensor of int32 at `offset` of a one-dimensional one: of what a call makes, the tables share one allocation.
Tensor part(const Tensor& of, int64_t offset, at::IntArrayRef size) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(of.storage()), of.key_set(), of.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(offset);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(size);
  return t;
}
int64_t up4(int64_t n) { return (n + 3) / 4 * 4; }
bool plain(const Tensor& t, at::ScalarType type, at::Device dev) { return t.scalar_type() == type && t.device() == dev && t.is_contiguous(); }
int64_t lead_of(const Tensor& t) { return product(t.sizes().slice(0, t.dim() - 1)); }
bool tangent(const Tensor& t) { return t._fw_grad(0).defined(); }   // forward mode: the Python form says that there is none
bool number(PyObject* o, float* out) {
  if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
  const double v = PyFloat_AsDouble(o);
  if (PyErr_Occurred()) { PyErr_Clear(); return false; }
  *out = (float)v;
  return true;
}
// The tensors of a tuple (a NamedTuple, too).
template <int N>
bool members(PyObject* o, const Tensor* (&t)[N]) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != N) return false;
  for (int i = 0; i < N; ++i) t[i] = tensor(PyTuple_GET_ITEM(o, i));
  return true;
}
// As a NamedTuple of ops.py.
PyObject* pack(variable_list&& ts, const char* name, PyTypeObject** type) {
  if (!*type) {
    pybind11::object t = pybind11::module_::import("mlx_b200.ops").attr(name);
    *type = reinterpret_cast<PyTypeObject*>(t.release().ptr());
  }
  PyObject* out = (*type)->tp_alloc(*type, (Py_ssize_t)ts.size());
  if (!out) return nullptr;
  for (size_t i = 0; i < ts.size(); ++i) PyTuple_SET_ITEM(out, (Py_ssize_t)i, THPVariable_Wrap(std::move(ts[i])));
  return out;
}
PyTypeObject *g_routing = nullptr, *g_row_groups = nullptr;   // (guarded by the GIL)
pybind11::object wrapped(const Tensor& t) { return pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(t)); }
pybind11::object python(const char* module, const char* name) { return pybind11::module_::import(module).attr(name); }
Tensor unwrapped(const pybind11::handle& o) { return o.is_none() ? Tensor() : Tensor(THPVariable_Unpack(o.ptr())); }
// Gradients of first order: where a graph of them is asked for, one whose backward pass says so.
void first_order(std::initializer_list<Tensor*> grads) {
  if (!at::GradMode::is_enabled()) return;
  pybind11::gil_scoped_acquire gil;
  for (Tensor* g : grads)
    if (g->defined()) *g = unwrapped(python("mlx_b200.grad", "_first_order")(wrapped(*g)));
}

struct Route {
  int top, groups, top_groups, best, scoring;
  bool renormalize;
  float scale;
  const Tensor* bias;
};
// (logits, top, scoring, bias, groups, top_groups, group_best, renormalize, scale)
bool route_args(PyObject* const* a, Py_ssize_t n, const Tensor** logits, Route* r) {
  if (n != 9 || !(*logits = tensor(a[0])) || !PyLong_CheckExact(a[1]) || !integer(a[1], 0, &r->top) || !index_arg(a[3], &r->bias) || !PyLong_CheckExact(a[4]) ||
      !integer(a[4], 1, &r->groups) || !integer(a[5], r->groups, &r->top_groups) || !PyLong_CheckExact(a[6]) || !integer(a[6], 1, &r->best) ||
      !PyBool_Check(a[7]) || !number(a[8], &r->scale) || !PyUnicode_Check(a[2]))
    return false;
  r->renormalize = a[7] == Py_True;
  if (PyUnicode_CompareWithASCIIString(a[2], "softmax") == 0) r->scoring = B200Q_SOFTMAX;
  else if (PyUnicode_CompareWithASCIIString(a[2], "sigmoid") == 0) r->scoring = B200Q_SIGMOID;
  else return false;
  return true;
}
bool route_run(const Tensor& l, const Route& r, variable_list* out) {
  const int dt = dtype_code(l.scalar_type());
  const at::Device dev = l.device();
  if (dt < 0 || !current(dev) || l.dim() < 1 || !l.is_contiguous() || l.numel() == 0) return false;
  const int64_t E = l.size(-1), T = lead_of(l);
  if (r.top < 1 || r.top > E || (r.bias && (!plain(*r.bias, at::kFloat, dev) || r.bias->dim() != 1 || r.bias->size(0) != E))) return false;
  c10::SmallVector<int64_t, 6> size(l.sizes().begin(), l.sizes().end());
  size.back() = r.top;
  const int64_t P = T * r.top, P4 = up4(P);
  const Tensor all = fresh({3 * P4 + E}, at::kInt, dev);
  Tensor w = fresh(size, at::kFloat, dev), e = part(all, 0, size), p = part(all, P4, size), o = part(all, 2 * P4, {P}), s = part(all, 3 * P4, {E}), ws;
  const size_t need = b200q_route_workspace_bytes(T, E, r.top);
  if (need) ws = fresh({(int64_t)need}, at::kByte, dev);
  auto at = [](const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); };
  if (b200q_route(l.data_ptr(), dt, T, E, r.top, r.scoring, r.bias ? static_cast<const float*>(r.bias->data_ptr()) : nullptr, r.groups, r.top_groups, r.best,
                  r.renormalize, r.scale, static_cast<float*>(w.data_ptr()), at(e), at(s), at(p), at(o), need ? ws.data_ptr() : nullptr, need,
                  stream_of(dev)) != B200Q_OK)
    return false;
  *out = {w, e, s, p, o};
  return true;
}
PyObject* py_route(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor* l;
  Route r;
  variable_list out;
  if (!route_args(a, n, &l, &r) || !route_run(*l, r, &out)) return none();
  return pack(std::move(out), "Routing", &g_routing);
  END_HANDLE_TH_ERRORS
}
struct RouteFn : public torch::autograd::Function<RouteFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Route* r, variable_list* out) {
    ctx->save_for_backward({logits, (*out)[1]});
    ctx->saved_data["scoring"] = (int64_t)r->scoring;
    ctx->saved_data["renormalize"] = r->renormalize;
    ctx->saved_data["scale"] = (double)r->scale;
    ctx->mark_non_differentiable({(*out)[1], (*out)[2], (*out)[3], (*out)[4]});
    ctx->set_materialize_grads(false);   // (no zeros for the four that have none)
    return *out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &l = saved[0], &e = saved[1];
    Tensor dl;
    if (!grads[0].defined()) return {dl, Tensor(), Tensor()};
    const int scoring = (int)ctx->saved_data["scoring"].toInt();
    const bool renormalize = ctx->saved_data["renormalize"].toBool();
    const double scale = ctx->saved_data["scale"].toDouble();
    const at::Device dev = l.device();
    {
      at::AutoDispatchBelowAutograd below;
      const Tensor dw = grads[0].contiguous();
      if (current(dev) && l.is_contiguous() && e.is_contiguous() && e.device() == dev && plain(dw, at::kFloat, dev)) {
        dl = fresh(l.sizes(), l.scalar_type(), dev);
        if (b200q_route_dlogits(static_cast<const float*>(dw.data_ptr()), l.data_ptr(), dtype_code(l.scalar_type()), static_cast<const int32_t*>(e.data_ptr()),
                                lead_of(l), l.size(-1), e.size(-1), scoring, renormalize, (float)scale, dl.data_ptr(), stream_of(dev)) != B200Q_OK)
          dl = Tensor();
      }
      if (!dl.defined()) {
        pybind11::gil_scoped_acquire gil;
        dl = unwrapped(python("mlx_b200.ops", "route_dlogits")(wrapped(dw), wrapped(l.detach()), wrapped(e), scoring == B200Q_SOFTMAX ? "softmax" : "sigmoid",
                                                               renormalize, scale));
      }
    }
    first_order({&dl});
    return {dl, Tensor(), Tensor()};
  }
};
PyObject* py_route_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor* l;
  Route r;
  variable_list out;
  if (!route_args(a, n, &l, &r) || tangent(*l) || (r.bias && tangent(*r.bias)) || !route_run(*l, r, &out)) return none();
  if (l->requires_grad() && at::GradMode::is_enabled()) out = RouteFn::apply(*l, &r, &out);
  return pack(std::move(out), "Routing", &g_routing);
  END_HANDLE_TH_ERRORS
}

// The tables of a routing (weights, experts, sizes, places, order) that fit T = the tokens of `places`.
bool plan_ok(const Tensor* places, const Tensor* order, at::Device dev) {
  return places && order && plain(*places, at::kInt, dev) && plain(*order, at::kInt, dev) && places->dim() >= 1 && order->dim() == 1 &&
         order->size(0) == places->numel() && places->numel() > 0;
}
const int32_t* ints(const Tensor& t) { return static_cast<const int32_t*>(t.data_ptr()); }
bool dispatch_run(const Tensor& x, const Tensor* places, const Tensor* order, Tensor* xs) {
  const int dt = dtype_code(x.scalar_type());
  const at::Device dev = x.device();
  if (dt < 0 || !current(dev) || !x.is_contiguous() || x.numel() == 0 || !plan_ok(places, order, dev) || x.dim() != places->dim()) return false;
  for (int64_t i = 0; i < x.dim() - 1; ++i)
    if (x.size(i) != places->size(i)) return false;
  *xs = fresh({order->size(0), x.size(-1)}, x.scalar_type(), dev);
  return b200q_dispatch_rows(x.data_ptr(), dt, lead_of(x), places->size(-1), x.size(-1), ints(*places), ints(*order), xs->data_ptr(), stream_of(dev)) == B200Q_OK;
}
bool rows_ok(const Tensor& y, const Tensor* places, const Tensor* order, const Tensor* weights, at::Device dev) {
  return dtype_code(y.scalar_type()) >= 0 && current(dev) && y.is_contiguous() && y.dim() == 2 && y.numel() > 0 && plan_ok(places, order, dev) &&
         y.size(0) == order->size(0) && (!weights || (plain(*weights, at::kFloat, dev) && weights->sizes() == places->sizes()));
}
bool combine_run(const Tensor& y, const Tensor* places, const Tensor* order, const Tensor* weights, Tensor* out) {
  const at::Device dev = y.device();
  if (!rows_ok(y, places, order, weights, dev)) return false;
  c10::SmallVector<int64_t, 6> size(places->sizes().begin(), places->sizes().end());
  size.back() = y.size(1);
  *out = fresh(size, y.scalar_type(), dev);
  return b200q_combine_rows(y.data_ptr(), dtype_code(y.scalar_type()), lead_of(*places), places->size(-1), y.size(1), ints(*places),
                            weights ? static_cast<const float*>(weights->data_ptr()) : nullptr, out->data_ptr(), stream_of(dev)) == B200Q_OK;
}
pybind11::object routing_of(const Tensor* weights, const Tensor& places, const Tensor& order) {
  const pybind11::object no = pybind11::none();
  return python("mlx_b200.ops", "Routing")(weights ? wrapped(*weights) : no, no, no, wrapped(places), wrapped(order));
}

PyObject* py_dispatch(PyObject*, PyObject* const* a, Py_ssize_t n) {   // (x, routing)
  HANDLE_TH_ERRORS
  const Tensor *x, *r[5];
  Tensor xs;
  if (n != 2 || !(x = tensor(a[0])) || !members(a[1], r) || !dispatch_run(*x, r[3], r[4], &xs)) return none();
  return THPVariable_Wrap(std::move(xs));
  END_HANDLE_TH_ERRORS
}
struct DispatchFn : public torch::autograd::Function<DispatchFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor* places, const Tensor* order, Tensor* xs) {
    ctx->save_for_backward({*places, *order});
    return *xs;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    Tensor dx;
    if (grads[0].defined()) {
      {
        at::AutoDispatchBelowAutograd below;
        const Tensor g = grads[0].contiguous();
        if (!combine_run(g, &saved[0], &saved[1], nullptr, &dx)) {
          pybind11::gil_scoped_acquire gil;
          dx = unwrapped(python("mlx_b200.ops", "combine_rows")(wrapped(g), routing_of(nullptr, saved[0], saved[1]), false));
        }
      }
      first_order({&dx});
    }
    return {dx, Tensor(), Tensor(), Tensor()};
  }
};
PyObject* py_dispatch_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {   // (x, routing)
  HANDLE_TH_ERRORS
  const Tensor *x, *r[5];
  Tensor xs;
  if (n != 2 || !(x = tensor(a[0])) || !members(a[1], r) || tangent(*x) || !dispatch_run(*x, r[3], r[4], &xs)) return none();
  if (x->requires_grad() && at::GradMode::is_enabled()) xs = DispatchFn::apply(*x, r[3], r[4], &xs);
  return THPVariable_Wrap(std::move(xs));
  END_HANDLE_TH_ERRORS
}

PyObject* py_combine(PyObject*, PyObject* const* a, Py_ssize_t n) {   // (y, routing, weighted)
  HANDLE_TH_ERRORS
  const Tensor *y, *r[5];
  Tensor out;
  bool weighted;
  if (n != 3 || !(y = tensor(a[0])) || !members(a[1], r) || !boolean(a[2], &weighted) || (weighted && !r[0]) ||
      !combine_run(*y, r[3], r[4], weighted ? r[0] : nullptr, &out))
    return none();
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}
struct CombineFn : public torch::autograd::Function<CombineFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& weights, const Tensor* places, const Tensor* order, Tensor* out) {
    ctx->save_for_backward({y, weights, *places, *order});
    return *out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &y = saved[0], &w = saved[1], &places = saved[2], &order = saved[3];
    Tensor dys, dw;
    const bool for_y = ctx->needs_input_grad(0), for_w = ctx->needs_input_grad(1);
    if (grads[0].defined()) {
      {
        at::AutoDispatchBelowAutograd below;
        const Tensor dy = grads[0].contiguous();
        const at::Device dev = y.device();
        bool done = rows_ok(y, &places, &order, &w, dev) && plain(dy, y.scalar_type(), dev);
        if (done) {
          if (for_y) dys = fresh(y.sizes(), y.scalar_type(), dev);
          if (for_w) dw = fresh(w.sizes(), at::kFloat, dev);
          done = b200q_combine_rows_grad(dy.data_ptr(), y.data_ptr(), dtype_code(y.scalar_type()), lead_of(places), places.size(-1), y.size(1), ints(places),
                                         ints(order), static_cast<const float*>(w.data_ptr()), for_y ? dys.data_ptr() : nullptr,
                                         for_w ? static_cast<float*>(dw.data_ptr()) : nullptr, stream_of(dev)) == B200Q_OK;
        }
        if (!done) {
          pybind11::gil_scoped_acquire gil;
          const Tensor wd = w.detach();
          const pybind11::tuple r = python("mlx_b200.ops", "combine_rows_grad")(wrapped(dy), wrapped(y.detach()), routing_of(&wd, places, order), for_y, for_w);
          dys = unwrapped(r[0]);
          dw = unwrapped(r[1]);
        }
      }
      first_order({&dys, &dw});
    }
    return {dys, dw, Tensor(), Tensor(), Tensor()};
  }
};
PyObject* py_combine_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {   // (y, routing)
  HANDLE_TH_ERRORS
  const Tensor *y, *r[5];
  Tensor out;
  if (n != 2 || !(y = tensor(a[0])) || !members(a[1], r) || !r[0] || tangent(*y) || tangent(*r[0]) || !combine_run(*y, r[3], r[4], r[0], &out)) return none();
  if ((y->requires_grad() || r[0]->requires_grad()) && at::GradMode::is_enabled()) out = CombineFn::apply(*y, *r[0], r[3], r[4], &out);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyObject* py_group_rows(PyObject*, PyObject* const* a, Py_ssize_t nargs) {   // (ids, n)
  HANDLE_TH_ERRORS
  const Tensor* ids;
  int n;
  if (nargs != 2 || !(ids = tensor(a[0])) || !PyLong_CheckExact(a[1]) || !integer(a[1], 0, &n) || n < 0) return none();
  const at::Device dev = ids->device();
  const at::ScalarType t = ids->scalar_type();
  if ((t != at::kInt && t != at::kLong) || !current(dev) || !ids->is_contiguous() || ids->numel() == 0) return none();
  const int64_t T = ids->numel();
  const size_t need = b200q_group_rows_workspace_bytes(T, n);
  const int64_t t4 = b200q_group_rows_tiles(T, n);
  const Tensor all = fresh({4 * t4 + up4(T) + up4(n) + n + 1}, at::kInt, dev);   // (tiles first: on 16 bytes)
  Tensor tiles = part(all, 0, {t4, 4}), order = part(all, 4 * t4, {T}), sizes = part(all, 4 * t4 + up4(T), {n}), starts = part(all, 4 * t4 + up4(T) + up4(n), {n + 1}), ws;
  if (need) ws = fresh({(int64_t)need}, at::kByte, dev);
  auto at = [](const Tensor& v) { return static_cast<int32_t*>(v.data_ptr()); };
  if (b200q_group_rows(ids->data_ptr(), t == at::kLong ? 8 : 4, T, n, at(sizes), at(starts), at(order), at(tiles), need ? ws.data_ptr() : nullptr, need, stream_of(dev)) != B200Q_OK)
    return none();
  return pack({sizes, starts, order, tiles}, "RowGroups", &g_row_groups);
  END_HANDLE_TH_ERRORS
}

struct Adapters {
  const Tensor *y, *x, *a, *b, *g[4], *scales;   // g: sizes, starts, order, tiles
  int64_t T, L, N, K, r;
};
bool adapters_ok(Adapters* p, const Tensor& y) {   // y: what is added to, or the result's gradient
  const at::ScalarType t = p->x->scalar_type();
  const at::Device dev = p->x->device();
  if ((t != at::kHalf && t != at::kBFloat16) || !current(dev)) return false;
  for (const Tensor* v : {&y, p->x, p->a, p->b})
    if (!plain(*v, t, dev) || v->numel() == 0) return false;
  if (p->a->dim() != 3 || p->b->dim() != 3 || p->x->dim() < 1 || y.dim() != p->x->dim()) return false;
  for (int64_t i = 0; i < y.dim() - 1; ++i)
    if (y.size(i) != p->x->size(i)) return false;
  p->T = lead_of(y); p->L = p->a->size(0); p->r = p->a->size(1); p->K = p->a->size(2); p->N = p->b->size(1);
  if (p->b->size(0) != p->L || p->b->size(2) != p->r || p->x->size(-1) != p->K || y.size(-1) != p->N) return false;
  for (const Tensor* v : p->g)
    if (!v || !plain(*v, at::kInt, dev)) return false;
  if (p->g[0]->dim() != 1 || p->g[0]->size(0) != p->L || p->g[1]->dim() != 1 || p->g[1]->size(0) != p->L + 1 || p->g[2]->dim() != 1 || p->g[2]->size(0) != p->T ||
      p->g[3]->dim() != 2 || p->g[3]->size(0) != b200q_group_rows_tiles(p->T, p->L) || p->g[3]->size(1) != 4)
    return false;
  return !p->scales || (plain(*p->scales, at::kFloat, dev) && p->scales->dim() == 1 && p->scales->size(0) == p->L);
}
const float* floats(const Tensor* t) { return t ? static_cast<const float*>(t->data_ptr()) : nullptr; }
bool adapters_run(Adapters* p, Tensor* out, Tensor* h) {
  if (!adapters_ok(p, *p->y)) return false;
  const at::Device dev = p->x->device();
  if (!out->defined()) *out = fresh(p->y->sizes(), p->y->scalar_type(), dev);
  *h = fresh({p->T, 3, (p->r + 15) / 16 * 16}, at::kBFloat16, dev);
  return b200q_add_adapters(p->y->data_ptr(), p->x->data_ptr(), p->a->data_ptr(), p->b->data_ptr(), dtype_code(p->x->scalar_type()), p->T, p->L, p->N, p->K, p->r,
                            ints(*p->g[2]), ints(*p->g[3]), floats(p->scales), h->data_ptr(), out->data_ptr(), stream_of(dev)) == B200Q_OK;
}
bool overlap(const Tensor& a, const Tensor& b) {
  const char *p = static_cast<const char*>(a.data_ptr()), *q = static_cast<const char*>(b.data_ptr());
  return p < q + b.nbytes() && q < p + a.nbytes();
}
bool adapters_args(PyObject* const* a, Adapters* p) {   // (y, x, a, b, groups, scales)
  return (p->y = tensor(a[0])) && (p->x = tensor(a[1])) && (p->a = tensor(a[2])) && (p->b = tensor(a[3])) && members(a[4], p->g) && index_arg(a[5], &p->scales);
}
PyObject* py_add_adapters(PyObject*, PyObject* const* a, Py_ssize_t n) {   // (..., out): out is None or y itself
  HANDLE_TH_ERRORS
  Adapters p;
  Tensor out, h;
  if (n != 7 || !adapters_args(a, &p) || (a[6] != Py_None && a[6] != a[0])) return none();
  if (a[6] != Py_None) {
    out = *p.y;
    if (out.requires_grad() && at::GradMode::is_enabled()) return none();
    for (const Tensor* v : {p.x, p.a, p.b})
      if (overlap(out, *v)) return none();
  }
  if (!adapters_run(&p, &out, &h)) return none();
  if (a[6] != Py_None && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();   // whoever has kept it for a gradient hears of it
  PyObject* pair = PyTuple_New(2);
  if (!pair) return nullptr;
  if (a[6] != Py_None) { Py_INCREF(a[6]); PyTuple_SET_ITEM(pair, 0, a[6]); }
  else PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(out)));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(h)));
  return pair;
  END_HANDLE_TH_ERRORS
}
struct AdaptersFn : public torch::autograd::Function<AdaptersFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& x, const Tensor& a, const Tensor& b, const Adapters* p, const Tensor* h, Tensor* out) {
    variable_list saved{x, a, b, *h, *p->g[0], *p->g[1], *p->g[2], *p->g[3]};
    if (p->scales) saved.push_back(*p->scales);
    ctx->save_for_backward(std::move(saved));
    return *out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    Tensor d_y, dx, da, db;
    if (grads[0].defined()) {
      const bool for_y = ctx->needs_input_grad(0), for_x = ctx->needs_input_grad(1), for_a = ctx->needs_input_grad(2), for_b = ctx->needs_input_grad(3);
      if (for_x || for_a || for_b) {
        {
          at::AutoDispatchBelowAutograd below;
          const Tensor dy = grads[0].contiguous();
          Adapters p{nullptr, &saved[0], &saved[1], &saved[2], {&saved[4], &saved[5], &saved[6], &saved[7]}, saved.size() > 8 ? &saved[8] : nullptr};
          const Tensor& h = saved[3];
          const at::Device dev = saved[0].device();
          bool done = adapters_ok(&p, dy) && plain(h, at::kBFloat16, dev) && on16(h);
          if (done) {
            Tensor g;
            if (for_x) dx = fresh(p.x->sizes(), p.x->scalar_type(), dev);
            if (for_a) da = fresh(p.a->sizes(), p.x->scalar_type(), dev);
            if (for_b) db = fresh(p.b->sizes(), p.x->scalar_type(), dev);
            if (for_x || for_a) g = fresh(h.sizes(), at::kBFloat16, dev);
            auto at = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
            done = b200q_add_adapters_grad(dy.data_ptr(), p.x->data_ptr(), p.a->data_ptr(), p.b->data_ptr(), dtype_code(p.x->scalar_type()), p.T, p.L, p.N, p.K, p.r,
                                           ints(*p.g[2]), ints(*p.g[1]), ints(*p.g[3]), floats(p.scales), h.data_ptr(), at(g), at(dx), at(da),
                                           at(db), stream_of(dev)) == B200Q_OK;
          }
          if (!done) {
            pybind11::gil_scoped_acquire gil;
            const pybind11::object groups = python("mlx_b200.ops", "RowGroups")(wrapped(saved[4]), wrapped(saved[5]), wrapped(saved[6]), wrapped(saved[7]));
            const pybind11::object scales = p.scales ? wrapped(*p.scales) : pybind11::object(pybind11::none());
            const pybind11::tuple r = python("mlx_b200.ops", "add_adapters_grad")(wrapped(dy), wrapped(saved[0].detach()), wrapped(saved[1].detach()),
                                                                                 wrapped(saved[2].detach()), groups, wrapped(h), scales, for_x, for_a, for_b);
            dx = unwrapped(r[0]);
            da = unwrapped(r[1]);
            db = unwrapped(r[2]);
          }
        }
        first_order({&dx, &da, &db});
      }
      if (for_y) d_y = grads[0];
    }
    return {d_y, dx, da, db, Tensor(), Tensor(), Tensor()};
  }
};
PyObject* py_add_adapters_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {   // (y, x, a, b, groups, scales)
  HANDLE_TH_ERRORS
  Adapters p;
  Tensor out, h;
  if (n != 6 || !adapters_args(a, &p)) return none();
  bool graph = false;
  for (const Tensor* v : {p.y, p.x, p.a, p.b}) {
    if (tangent(*v)) return none();
    graph = graph || v->requires_grad();
  }
  if (p.scales && tangent(*p.scales)) return none();
  if (!adapters_run(&p, &out, &h)) return none();
  if (graph && at::GradMode::is_enabled()) out = AdaptersFn::apply(*p.y, *p.x, *p.a, *p.b, &p, &h, &out);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (device index, stream, operator, address, bytes): ops._workspaces has a new buffer
PyObject* py_scratch(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5) { PyErr_SetString(PyExc_TypeError, "scratch takes five arguments"); return nullptr; }
  const Scratch s{(int)PyLong_AsLong(a[0]), (int)PyLong_AsLong(a[2]), PyLong_AsVoidPtr(a[1]), PyLong_AsVoidPtr(a[3]), PyLong_AsSize_t(a[4])};
  if (PyErr_Occurred()) return nullptr;
  for (Scratch& g : g_scratch)
    if (g.dev == s.dev && g.stream == s.stream && g.op == s.op) { g = s; Py_RETURN_NONE; }
  g_scratch.push_back(s);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"qmm", (PyCFunction)(void (*)(void))py_qmm, METH_FASTCALL, nullptr},
    {"qmm_grad", (PyCFunction)(void (*)(void))py_qmm_grad, METH_FASTCALL, nullptr},
    {"quantize", (PyCFunction)(void (*)(void))py_quantize, METH_FASTCALL, nullptr},
    {"dequantize", (PyCFunction)(void (*)(void))py_dequantize, METH_FASTCALL, nullptr},
    {"gather", (PyCFunction)(void (*)(void))py_gather, METH_FASTCALL, nullptr},
    {"swiglu", (PyCFunction)(void (*)(void))py_swiglu, METH_FASTCALL, nullptr},
    {"fp4_quantize", (PyCFunction)(void (*)(void))py_fp4_quantize, METH_FASTCALL, nullptr},
    {"fp4_dequantize", (PyCFunction)(void (*)(void))py_fp4_dequantize, METH_FASTCALL, nullptr},
    {"qqmm", (PyCFunction)(void (*)(void))py_qqmm, METH_FASTCALL, nullptr},
    {"grouped_mm", (PyCFunction)(void (*)(void))py_grouped_mm, METH_FASTCALL, nullptr},
    {"grouped_mm_dw", (PyCFunction)(void (*)(void))py_grouped_mm_dw, METH_FASTCALL, nullptr},
    {"grouped_mm_grad", (PyCFunction)(void (*)(void))py_grouped_mm_grad, METH_FASTCALL, nullptr},
    {"route", (PyCFunction)(void (*)(void))py_route, METH_FASTCALL, nullptr},
    {"route_grad", (PyCFunction)(void (*)(void))py_route_grad, METH_FASTCALL, nullptr},
    {"dispatch", (PyCFunction)(void (*)(void))py_dispatch, METH_FASTCALL, nullptr},
    {"dispatch_grad", (PyCFunction)(void (*)(void))py_dispatch_grad, METH_FASTCALL, nullptr},
    {"combine", (PyCFunction)(void (*)(void))py_combine, METH_FASTCALL, nullptr},
    {"combine_grad", (PyCFunction)(void (*)(void))py_combine_grad, METH_FASTCALL, nullptr},
    {"group_rows", (PyCFunction)(void (*)(void))py_group_rows, METH_FASTCALL, nullptr},
    {"add_adapters", (PyCFunction)(void (*)(void))py_add_adapters, METH_FASTCALL, nullptr},
    {"add_adapters_grad", (PyCFunction)(void (*)(void))py_add_adapters_grad, METH_FASTCALL, nullptr},
    {"scratch", (PyCFunction)(void (*)(void))py_scratch, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_front", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__front() { return PyModule_Create(&module); }
