// h24_torch.cpp -- the short way from a torch tensor to libh24 for the calls of
// a decoding step and of a training step's norms and loss, where the
// microseconds of Python for each call would cost more than the kernel.  Each function takes the Python call's arguments; are
// they contiguous CUDA tensors of the current device in types that the kernel
// reads, it allocates the outputs, launches on the current stream and returns
// them.  For anything else, errors included, it returns None and the caller
// (int8.py, sampling.py, norm.py, loss.py) takes the general path, which checks,
// copies and raises.  The nodes of the autograd graph that norms and loss leave
// are here too.
//
// The module is not linked against libh24: bind() receives the entry points'
// addresses from the library that Python has loaded.
#include <Python.h>

#include <ATen/autocast_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <limits>
#include <memory>
#include <mutex>

#include "../../include/h24.h"

namespace {

struct {
  decltype(&h24_add_rms_norm_int8) norm;
  decltype(&h24_rows_int8_quantize) quantize;
  decltype(&h24_rows_int8_dequant) dequant;
  decltype(&h24_int8_linear) linear;
  decltype(&h24_sample_tokens) sample;
  decltype(&h24_add_norm) add_norm;
  decltype(&h24_add_norm_backward) add_norm_backward;
  decltype(&h24_linear_ce_forward) ce_forward;
  decltype(&h24_linear_ce_backward) ce_backward;
  decltype(&h24_last_error) last_error;
} g_h24;

// The tensor (or parameter, but no other subclass) behind `o` if it is a
// contiguous CUDA tensor of device `dev` without a tangent of forward-mode
// derivatives (which nothing here has: the general path says so).
const at::Tensor *dense(PyObject *o, int dev) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor &t = THPVariable_Unpack(o);
  const bool ok = t.is_cuda() && t.get_device() == dev && t.layout() == at::kStrided && t.is_contiguous() &&
                  !t._fw_grad(0).defined();
  return ok ? &t : nullptr;
}
bool tracked(const at::Tensor *t) { return t && t->requires_grad() && c10::GradMode::is_enabled(); }

// The same, and no gradient is asked of it.
const at::Tensor *plain(PyObject *o, int dev) {
  const at::Tensor *t = dense(o, dev);
  return tracked(t) ? nullptr : t;
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

// A C++ exception (an allocation that fails, say) leaves the call to the general
// path.  What Python code raised goes on to the caller: a hook on saved tensors may
// end the call that way (a checkpoint's recomputation does, once it has all it needs).
template <typename F>
PyObject *guarded(F f) {
  try {
    return f();
  } catch (python_error &e) {
    e.restore();
  } catch (const std::exception &) {
  }
  if (PyErr_Occurred()) return nullptr;
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

// ---------------------------------------------------------------------------
// Norms and loss, with their nodes in the autograd graph
// ---------------------------------------------------------------------------
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

void check(int rc, const char *what) {
  if (rc != H24_OK) throw std::runtime_error(std::string(what) + ": " + g_h24.last_error());
}

// Gradients that are themselves tracked (create_graph) say so when they are
// differentiated, as torch's once_differentiable does.
variable_list once(variable_list grads, const char *what) {
  if (!c10::GradMode::is_enabled()) return grads;
  for (at::Tensor &g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string("trying to differentiate twice: ") + what + " has one derivative", static_cast<int64_t>(grads.size()));
  return (*error)(std::move(grads));
}

// A saved tensor, as the kernels read it.  Hooks may give back another than they
// were given: its strides are put right, anything else is refused.
struct Saved {
  SavedVariable variable;
  at::ScalarType type = at::kFloat;
  at::DimVector sizes;
  at::Device device{at::kCPU};

  void keep(const at::Tensor &t, bool is_output) {
    variable = SavedVariable(t, is_output);
    type = t.scalar_type();
    sizes = t.sizes();
    device = t.device();
  }
  at::Tensor unpack(std::shared_ptr<torch::autograd::Node> owner = nullptr) const {
    const at::Tensor t = variable.unpack(std::move(owner));
    if (t.scalar_type() != type || !t.sizes().equals(sizes) || t.device() != device || t.layout() != at::kStrided)
      throw std::runtime_error("a hook on saved tensors gave back another type, shape or device than it was given");
    const at::NoGradGuard none;
    return t.contiguous();
  }
};

struct NormNode : torch::autograd::Node {
  Saved s, weight;
  at::Tensor stats;
  bool layer = false, saved_output = false;

  std::string name() const override { return layer ? "AddLayerNormBackward" : "AddRmsNormBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    s.variable.reset_data();
    weight.variable.reset_data();
    stats.reset();
  }

  // (dy, dsummed) -> (x, residual, weight, bias)
  variable_list apply(variable_list &&grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    const at::Tensor sum = s.unpack(saved_output ? shared_from_this() : nullptr), w = weight.unpack();
    const int dev = static_cast<int>(sum.get_device());
    const c10::cuda::OptionalCUDAGuard guard(sum.device());
    const bool need_x = should_compute_output(0), need_r = should_compute_output(1);
    const bool need_w = should_compute_output(2), need_b = should_compute_output(3);
    variable_list out(4);
    if (!grads[0].defined()) {  // nothing reached y
      if (need_x) out[0] = grads[1];
      if (need_r) out[1] = grads[1];
      if (need_w) out[2] = at::zeros_like(w);
      if (need_b) out[3] = at::zeros_like(w);
      return once(std::move(out), "the norm");
    }
    const at::Tensor dy = grads[0].contiguous();
    const at::Tensor dsum = grads.size() > 1 && grads[1].defined() ? grads[1].contiguous() : at::Tensor();
    const int64_t cols = sum.size(-1), rows = sum.numel() / cols;
    const at::Tensor dx = need_x || need_r ? fresh(sum.sizes(), sum.scalar_type(), dev) : at::Tensor();
    const at::Tensor dw = need_w ? fresh(w.sizes(), w.scalar_type(), dev) : at::Tensor();
    const at::Tensor db = need_b ? fresh(w.sizes(), w.scalar_type(), dev) : at::Tensor();
    check(g_h24.add_norm_backward(sum.const_data_ptr(), w.const_data_ptr(), code_of(w.scalar_type()), layer, rows, cols,
                                  cols, code_of(sum.scalar_type()), static_cast<const float *>(stats.const_data_ptr()),
                                  dy.const_data_ptr(), cols, dsum.defined() ? dsum.const_data_ptr() : nullptr, cols,
                                  dx.defined() ? dx.data_ptr() : nullptr, dw.defined() ? dw.data_ptr() : nullptr,
                                  db.defined() ? db.data_ptr() : nullptr, stream_of(dev)),
          "h24_add_norm_backward");
    if (need_x) out[0] = dx;
    if (need_r) out[1] = dx;
    out[2] = dw;
    out[3] = db;
    return once(std::move(out), "the norm");
  }
};

// (x, weight, bias or None, residual or None, eps, layer) -> (y, summed or None)
PyObject *add_norm(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    const int dev = c10::cuda::current_device();
    const at::Tensor *x = n == 6 ? dense(a[0], dev) : nullptr;
    const at::Tensor *w = x ? dense(a[1], dev) : nullptr;
    const bool has_bias = w && a[2] != Py_None, has_residual = w && a[3] != Py_None;
    const at::Tensor *b = has_bias ? dense(a[2], dev) : nullptr, *r = has_residual ? dense(a[3], dev) : nullptr;
    double eps;
    if (!w || (has_bias && !b) || (has_residual && !r) || x->dim() < 1 || x->numel() == 0 || !number(a[4], &eps) ||
        !(eps >= 0))
      Py_RETURN_NONE;
    const int64_t cols = x->size(-1), rows = x->numel() / cols;
    const int code = code_of(x->scalar_type());
    const auto param = [&](const at::Tensor *p) {
      return p->dim() == 1 && p->numel() == cols && p->scalar_type() == w->scalar_type();
    };
    if (code < 0 || !param(w) || (w->scalar_type() != x->scalar_type() && w->scalar_type() != at::kFloat) ||
        (b && !param(b)) || (r && (r->scalar_type() != x->scalar_type() || !r->sizes().equals(x->sizes()))))
      Py_RETURN_NONE;
    const bool layer = a[5] == Py_True;
    const at::Tensor y = fresh(x->sizes(), x->scalar_type(), dev);
    const at::Tensor sum = r ? fresh(x->sizes(), x->scalar_type(), dev) : at::Tensor();
    const at::Tensor stats = fresh({2 * rows}, at::kFloat, dev);
    if (g_h24.add_norm(x->const_data_ptr(), r ? r->const_data_ptr() : nullptr, w->const_data_ptr(),
                       b ? b->const_data_ptr() : nullptr, code_of(w->scalar_type()), layer, rows, cols, cols, cols, code,
                       static_cast<float>(eps), y.data_ptr(), r ? sum.data_ptr() : nullptr,
                       static_cast<float *>(stats.data_ptr()), stream_of(dev)) != H24_OK)
      Py_RETURN_NONE;
    if (tracked(x) || tracked(w) || tracked(b) || tracked(r)) {
      const at::Tensor none;
      const std::shared_ptr<NormNode> node(new NormNode(), torch::autograd::deleteNode);
      node->set_next_edges(torch::autograd::collect_next_edges(*x, r ? *r : none, *w, b ? *b : none));
      torch::autograd::set_history(y, node);
      if (r) torch::autograd::set_history(sum, node);
      node->s.keep(r ? sum : *x, r != nullptr);
      node->weight.keep(*w, false);
      node->stats = stats;
      node->layer = layer;
      node->saved_output = r != nullptr;
    }
    return wrap({&y, r ? &sum : nullptr});
  });
}

struct LossNode : torch::autograd::Node {
  Saved x, weight;
  at::Tensor state;
  int reduction = 0;

  std::string name() const override { return "LinearCrossEntropyBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    x.variable.reset_data();
    weight.variable.reset_data();
    state.reset();
  }

  variable_list apply(variable_list &&grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    const at::Tensor rows = x.unpack(), w = weight.unpack();
    variable_list out(2);
    if (!grads[0].defined()) return out;
    const int dev = static_cast<int>(rows.get_device());
    const c10::cuda::OptionalCUDAGuard guard(rows.device());
    const at::Tensor g = grads[0].dim() <= 1 ? grads[0] : grads[0].contiguous();
    const int64_t step = g.dim() == 1 ? g.stride(0) : g.dim() ? 1 : 0, in = w.size(1);
    if (should_compute_output(0)) out[0] = fresh(rows.sizes(), rows.scalar_type(), dev);
    if (should_compute_output(1)) out[1] = fresh(w.sizes(), w.scalar_type(), dev);
    check(g_h24.ce_backward(rows.const_data_ptr(), rows.numel() / in, in, w.const_data_ptr(), w.size(0), in, in,
                            code_of(w.scalar_type()), reduction, static_cast<const float *>(g.const_data_ptr()), step,
                            static_cast<const int32_t *>(state.const_data_ptr()),
                            out[0].defined() ? out[0].data_ptr() : nullptr,
                            out[1].defined() ? out[1].data_ptr() : nullptr, stream_of(dev)),
          "h24_linear_ce_backward");
    return once(std::move(out), "linear_cross_entropy");
  }
};

// (x, weight, target, ignore_index, reduction) -> loss
PyObject *linear_ce(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    const int dev = c10::cuda::current_device();
    const at::Tensor *x = n == 5 ? dense(a[0], dev) : nullptr;
    const at::Tensor *w = x ? dense(a[1], dev) : nullptr;
    const at::Tensor *t = w ? dense(a[2], dev) : nullptr;
    if (!t || x->dim() < 1 || x->numel() == 0 || w->dim() != 2 || w->numel() == 0 || x->size(-1) != w->size(1) ||
        (x->scalar_type() != at::kHalf && x->scalar_type() != at::kBFloat16) || w->scalar_type() != x->scalar_type() ||
        t->scalar_type() != at::kLong || !holds_rows(*t, *x) || at::autocast::is_autocast_enabled(at::kCUDA) ||
        !PyLong_CheckExact(a[3]) || !PyLong_CheckExact(a[4]))
      Py_RETURN_NONE;
    int overflow = 0;
    const long long ignore = PyLong_AsLongLongAndOverflow(a[3], &overflow);
    const long reduction = PyLong_AsLong(a[4]);
    if (overflow) Py_RETURN_NONE;
    const int64_t in = w->size(1), tokens = x->numel() / in;
    const at::Tensor loss = reduction == H24_REDUCE_NONE ? fresh(x->sizes().slice(0, x->dim() - 1), at::kFloat, dev)
                                                         : fresh({}, at::kFloat, dev);
    const at::Tensor state = fresh({3 * tokens + 1}, at::kInt, dev);
    if (g_h24.ce_forward(x->const_data_ptr(), tokens, in, w->const_data_ptr(), w->size(0), in, in,
                         code_of(x->scalar_type()), static_cast<const int64_t *>(t->const_data_ptr()), ignore,
                         static_cast<int>(reduction), static_cast<float *>(loss.data_ptr()),
                         static_cast<int32_t *>(state.data_ptr()), stream_of(dev)) != H24_OK)
      Py_RETURN_NONE;
    if (tracked(x) || tracked(w)) {
      const std::shared_ptr<LossNode> node(new LossNode(), torch::autograd::deleteNode);
      node->set_next_edges(torch::autograd::collect_next_edges(*x, *w));
      torch::autograd::set_history(loss, node);
      node->x.keep(*x, false);
      node->weight.keep(*w, false);
      node->state = state;
      node->reduction = static_cast<int>(reduction);
    }
    return THPVariable_Wrap(loss);
  });
}

PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
  constexpr int kEntries = 10;
  void *p[kEntries];
  if (n != kEntries) {
    PyErr_SetString(PyExc_TypeError, "bind takes the addresses of ten entry points");
    return nullptr;
  }
  for (int i = 0; i < kEntries; ++i) p[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  g_h24.norm = reinterpret_cast<decltype(g_h24.norm)>(p[0]);
  g_h24.quantize = reinterpret_cast<decltype(g_h24.quantize)>(p[1]);
  g_h24.dequant = reinterpret_cast<decltype(g_h24.dequant)>(p[2]);
  g_h24.linear = reinterpret_cast<decltype(g_h24.linear)>(p[3]);
  g_h24.sample = reinterpret_cast<decltype(g_h24.sample)>(p[4]);
  g_h24.add_norm = reinterpret_cast<decltype(g_h24.add_norm)>(p[5]);
  g_h24.add_norm_backward = reinterpret_cast<decltype(g_h24.add_norm_backward)>(p[6]);
  g_h24.ce_forward = reinterpret_cast<decltype(g_h24.ce_forward)>(p[7]);
  g_h24.ce_backward = reinterpret_cast<decltype(g_h24.ce_backward)>(p[8]);
  g_h24.last_error = reinterpret_cast<decltype(g_h24.last_error)>(p[9]);
  Py_RETURN_NONE;
}

#define H24_METHOD(name) \
  { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr }
PyMethodDef g_methods[] = {H24_METHOD(bind),        H24_METHOD(add_rms_norm_int8),
                           H24_METHOD(quantize_rows_int8), H24_METHOD(dequantize_rows_int8),
                           H24_METHOD(int8_linear), H24_METHOD(sample_tokens),
                           H24_METHOD(add_norm), H24_METHOD(linear_ce),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_h24_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__h24_torch() { return PyModule_Create(&g_module); }
