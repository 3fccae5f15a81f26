// h24_torch.cpp -- the short way from a torch tensor to libh24 for the calls of
// a decoding step, where a few microseconds of Python for each call would cost
// more than the kernel.  Each function takes the Python call's arguments; are
// they contiguous CUDA tensors of the current device in types that the kernel
// reads, it allocates the outputs, launches on the current stream and returns
// them.  For anything else, errors included, it returns None and the caller
// (int8.py, sampling.py) takes the general path, which checks, copies and
// raises.
//
// The module is not linked against libh24: bind() receives the entry points'
// addresses from the library that Python has loaded.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <limits>

#include "../../include/h24.h"

namespace {

struct {
  decltype(&h24_add_rms_norm_int8) norm;
  decltype(&h24_rows_int8_quantize) quantize;
  decltype(&h24_rows_int8_dequant) dequant;
  decltype(&h24_int8_linear) linear;
  decltype(&h24_sample_tokens) sample;
} g_h24;

// The tensor behind `o` if it is a contiguous CUDA tensor of device `dev` of
// which no gradient is asked.
const at::Tensor *plain(PyObject *o, int dev) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor &t = THPVariable_Unpack(o);
  return t.is_cuda() && t.get_device() == dev && t.layout() == at::kStrided && t.is_contiguous() &&
                 !(t.requires_grad() && c10::GradMode::is_enabled())
             ? &t
             : nullptr;
}

// Whether `t` has a value for each row of `x`, in their order: x's leading
// dimensions up to ones, or one of the two a flat list.  (As _holds_rows in
// int8.py, which answers for what is refused here.)
bool holds_rows(const at::Tensor &t, const at::Tensor &x) {
  const at::IntArrayRef own = t.sizes(), want = x.sizes().slice(0, x.dim() - 1);
  int64_t n = 1;
  for (const int64_t d : want) n *= d;
  if (t.numel() != n) return false;
  if (own.equals(want)) return true;
  size_t i = 0, j = 0, n_own = 0, n_want = 0;
  for (const int64_t d : own) n_own += d != 1;
  for (const int64_t d : want) n_want += d != 1;
  if (n_own <= 1 || n_want <= 1) return true;
  if (n_own != n_want) return false;
  for (;; ++i, ++j) {
    while (i < own.size() && own[i] == 1) ++i;
    while (j < want.size() && want[j] == 1) ++j;
    if (i == own.size()) return true;
    if (own[i] != want[j]) return false;
  }
}

int code_of(at::ScalarType t) {
  return t == at::kFloat ? H24_DTYPE_F32 : t == at::kHalf ? H24_DTYPE_F16 : t == at::kBFloat16 ? H24_DTYPE_BF16 : -1;
}

at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, int dev) {
  return at::detail::empty_cuda(sizes, type, at::Device(at::kCUDA, static_cast<at::DeviceIndex>(dev)), std::nullopt);
}

void *stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream(); }

bool number(PyObject *o, double *v) {
  if (PyFloat_CheckExact(o)) {
    *v = PyFloat_AS_DOUBLE(o);
    return true;
  }
  if (!PyLong_CheckExact(o)) return false;
  *v = PyLong_AsDouble(o);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

PyObject *wrap(std::initializer_list<const at::Tensor *> ts) {
  PyObject *r = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (!r) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor *t : ts) {
    PyObject *o = t ? THPVariable_Wrap(*t) : Py_NewRef(Py_None);
    if (!o) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

// A C++ exception (an allocation that fails, say) leaves the call to the general path.
template <typename F>
PyObject *guarded(F f) {
  try {
    return f();
  } catch (const std::exception &) {
  }
  Py_RETURN_NONE;
}

// (x, weight, residual or None, eps) -> (q, scale, summed or None)
PyObject *add_rms_norm_int8(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    const int dev = c10::cuda::current_device();
    const at::Tensor *x = n == 4 ? plain(a[0], dev) : nullptr;
    const at::Tensor *w = x ? plain(a[1], dev) : nullptr;
    const bool has_residual = n == 4 && a[2] != Py_None;
    const at::Tensor *r = has_residual && w ? plain(a[2], dev) : nullptr;
    double eps;
    if (!w || (has_residual && !r) || x->dim() < 1 || x->numel() == 0 || !number(a[3], &eps)) Py_RETURN_NONE;
    const int64_t cols = x->size(-1), rows = x->numel() / cols;
    const int code = code_of(x->scalar_type());
    if (code < 0 || w->numel() != cols || (w->scalar_type() != x->scalar_type() && w->scalar_type() != at::kFloat) ||
        (r && (r->scalar_type() != x->scalar_type() || !r->sizes().equals(x->sizes()))))
      Py_RETURN_NONE;
    const at::Tensor q = fresh(x->sizes(), at::kChar, dev);
    const at::Tensor scale = fresh(x->sizes().slice(0, x->dim() - 1), at::kFloat, dev);
    const at::Tensor sum = r ? fresh(x->sizes(), x->scalar_type(), dev) : at::Tensor();
    if (g_h24.norm(x->const_data_ptr(), r ? r->const_data_ptr() : nullptr, w->const_data_ptr(),
                   code_of(w->scalar_type()), rows, cols, cols, r ? cols : 0, code, static_cast<float>(eps),
                   static_cast<int8_t *>(q.data_ptr()), static_cast<float *>(scale.data_ptr()),
                   r ? sum.data_ptr() : nullptr, stream_of(dev)) != H24_OK)
      Py_RETURN_NONE;
    return wrap({&q, &scale, r ? &sum : nullptr});
  });
}

// (x) -> (q, scale)
PyObject *quantize_rows_int8(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    const int dev = c10::cuda::current_device();
    const at::Tensor *x = n == 1 ? plain(a[0], dev) : nullptr;
    if (!x || x->dim() < 1 || x->numel() == 0 || code_of(x->scalar_type()) < 0) Py_RETURN_NONE;
    const int64_t cols = x->size(-1);
    const at::Tensor q = fresh(x->sizes(), at::kChar, dev);
    const at::Tensor scale = fresh(x->sizes().slice(0, x->dim() - 1), at::kFloat, dev);
    if (g_h24.quantize(x->const_data_ptr(), x->numel() / cols, cols, cols, code_of(x->scalar_type()),
                       static_cast<int8_t *>(q.data_ptr()), static_cast<float *>(scale.data_ptr()),
                       stream_of(dev)) != H24_OK)
      Py_RETURN_NONE;
    return wrap({&q, &scale});
  });
}

bool dtype_of(PyObject *o, at::ScalarType *t) {
  if (!THPDtype_Check(o)) return false;
  *t = reinterpret_cast<THPDtype *>(o)->scalar_type;
  return code_of(*t) >= 0;
}

// (q, scale, dtype) -> tensor
PyObject *dequantize_rows_int8(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    const int dev = c10::cuda::current_device();
    const at::Tensor *q = n == 3 ? plain(a[0], dev) : nullptr;
    const at::Tensor *s = q ? plain(a[1], dev) : nullptr;
    at::ScalarType type;
    if (!s || q->dim() < 1 || q->numel() == 0 || q->scalar_type() != at::kChar || s->scalar_type() != at::kFloat ||
        !holds_rows(*s, *q) || !dtype_of(a[2], &type))
      Py_RETURN_NONE;
    const at::Tensor out = fresh(q->sizes(), type, dev);
    if (g_h24.dequant(static_cast<const int8_t *>(q->const_data_ptr()), static_cast<const float *>(s->const_data_ptr()),
                      s->numel(), q->size(-1), code_of(type), out.data_ptr(), stream_of(dev)) != H24_OK)
      Py_RETURN_NONE;
    return THPVariable_Wrap(out);
  });
}

// (q, scale, weight_int8, mu_rows, bias or None, out_dtype) -> tensor
PyObject *int8_linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    const int dev = c10::cuda::current_device();
    const at::Tensor *q = n == 6 ? plain(a[0], dev) : nullptr;
    const at::Tensor *s = q ? plain(a[1], dev) : nullptr;
    const at::Tensor *w = s ? plain(a[2], dev) : nullptr;
    const at::Tensor *mu = w ? plain(a[3], dev) : nullptr;
    const bool has_bias = n == 6 && a[4] != Py_None;
    const at::Tensor *b = has_bias && mu ? plain(a[4], dev) : nullptr;
    at::ScalarType type;
    if (!mu || (has_bias && !b) || q->dim() < 1 || q->numel() == 0 || q->scalar_type() != at::kChar ||
        s->scalar_type() != at::kFloat || w->scalar_type() != at::kChar || w->dim() != 2 || w->numel() == 0 ||
        mu->scalar_type() != at::kHalf || !dtype_of(a[5], &type))
      Py_RETURN_NONE;
    const int64_t in = w->size(1), out = w->size(0), tokens = s->numel();
    if (q->size(-1) != in || !holds_rows(*s, *q) || mu->numel() != out ||
        (b && (b->scalar_type() != at::kFloat || b->numel() != out)))
      Py_RETURN_NONE;
    at::DimVector sizes(q->sizes());
    sizes.back() = out;
    const at::Tensor y = fresh(sizes, type, dev);
    if (g_h24.linear(static_cast<const int8_t *>(q->const_data_ptr()), static_cast<const float *>(s->const_data_ptr()),
                     tokens, in, static_cast<const int8_t *>(w->const_data_ptr()),
                     static_cast<const uint16_t *>(mu->const_data_ptr()), out, in,
                     b ? static_cast<const float *>(b->const_data_ptr()) : nullptr, code_of(type), y.data_ptr(),
                     stream_of(dev)) != H24_OK)
      Py_RETURN_NONE;
    return THPVariable_Wrap(y);
  });
}

// A sampling setting: a number in [0, most] or one value a row.
bool setting(PyObject *o, int dev, const at::Tensor &logits, at::ScalarType type, double most, const void **p, double *v) {
  *p = nullptr;
  *v = 0;
  if (number(o, v)) return *v >= 0 && *v <= most;
  const at::Tensor *t = plain(o, dev);
  if (!t || t->scalar_type() != type || !holds_rows(*t, logits)) return false;
  *p = t->const_data_ptr();
  return true;
}

// (logits, u, temperature, top_k, top_p, min_p, return_logprob) -> tokens or (tokens, logprob)
PyObject *sample_tokens(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    const int dev = c10::cuda::current_device();
    const at::Tensor *l = n == 7 ? plain(a[0], dev) : nullptr;
    const at::Tensor *u = l ? plain(a[1], dev) : nullptr;
    if (!u || l->dim() < 1 || l->numel() == 0 || code_of(l->scalar_type()) < 0 || u->scalar_type() != at::kFloat)
      Py_RETURN_NONE;
    const int64_t vocab = l->size(-1), rows = l->numel() / vocab;
    const double inf = std::numeric_limits<double>::infinity();
    const void *tp, *kp, *pp, *mp;
    double t, k, p, m;
    if (!holds_rows(*u, *l) || !setting(a[2], dev, *l, at::kFloat, inf, &tp, &t) ||
        !setting(a[3], dev, *l, at::kInt, inf, &kp, &k) || !setting(a[4], dev, *l, at::kFloat, 1.0, &pp, &p) ||
        !setting(a[5], dev, *l, at::kFloat, 1.0, &mp, &m))
      Py_RETURN_NONE;
    const int want = PyObject_IsTrue(a[6]);
    const at::Tensor tokens = fresh(l->sizes().slice(0, l->dim() - 1), at::kLong, dev);
    const at::Tensor logprob = want == 1 ? fresh(tokens.sizes(), at::kFloat, dev) : at::Tensor();
    if (want < 0 ||
        g_h24.sample(l->const_data_ptr(), code_of(l->scalar_type()), rows, vocab, vocab,
                     static_cast<const float *>(u->const_data_ptr()), static_cast<const float *>(tp),
                     static_cast<float>(t), static_cast<const int32_t *>(kp),
                     static_cast<int32_t>(k < static_cast<double>(vocab) ? k : static_cast<double>(vocab)),
                     static_cast<const float *>(pp), static_cast<float>(p), static_cast<const float *>(mp),
                     static_cast<float>(m), static_cast<int64_t *>(tokens.data_ptr()),
                     want ? static_cast<float *>(logprob.data_ptr()) : nullptr, stream_of(dev)) != H24_OK) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    return want ? wrap({&tokens, &logprob}) : THPVariable_Wrap(tokens);
  });
}

PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
  void *p[5];
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "bind takes the addresses of five entry points");
    return nullptr;
  }
  for (int i = 0; i < 5; ++i) p[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  g_h24.norm = reinterpret_cast<decltype(g_h24.norm)>(p[0]);
  g_h24.quantize = reinterpret_cast<decltype(g_h24.quantize)>(p[1]);
  g_h24.dequant = reinterpret_cast<decltype(g_h24.dequant)>(p[2]);
  g_h24.linear = reinterpret_cast<decltype(g_h24.linear)>(p[3]);
  g_h24.sample = reinterpret_cast<decltype(g_h24.sample)>(p[4]);
  Py_RETURN_NONE;
}

#define H24_METHOD(name) \
  { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr }
PyMethodDef g_methods[] = {H24_METHOD(bind),        H24_METHOD(add_rms_norm_int8),
                           H24_METHOD(quantize_rows_int8), H24_METHOD(dequantize_rows_int8),
                           H24_METHOD(int8_linear), H24_METHOD(sample_tokens),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_h24_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__h24_torch() { return PyModule_Create(&g_module); }
