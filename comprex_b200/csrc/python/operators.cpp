// The operators of cx_ops.h on torch tensors, with their gradients: checks, outputs and workspaces from torch's
// allocators, native calls on the current stream.  In C++ because the smallest products take 5 us on the GPU: the same
// checks, descriptors and autograd functions took 22 us a call in Python, 160 us for a loss with its gradients.
//
// Errors: what a caller got wrong is a ValueError or the package's ComprexError; no other exception leaves.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/autocast_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <string>

#include "../cx_ops.h"
#include "operators.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

struct Native {
  decltype(&cx_linear_workspace_bytes) linear_bytes;
  decltype(&cx_linear_forward) linear_forward;
  decltype(&cx_linear_backward) linear_backward;
  decltype(&cx_vocab_loss_workspace_bytes) loss_bytes;
  decltype(&cx_vocab_loss_forward) loss_forward;
  decltype(&cx_vocab_loss_backward) loss_backward;
  decltype(&cx_last_error) last_error;
  PyObject* error;             // ComprexError
} native = {};

struct Refused {               // ends as ComprexError, or ValueError
  std::string why;
  bool value = false;
};
std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
// (No streams: a number put into one ended the process, with torch's and this library's C++ runtimes in it side by side.)
std::string text(const char* s) { return s; }
std::string text(const std::string& s) { return s; }
std::string text(int64_t n) { return std::to_string(n); }
std::string text(int n) { return std::to_string(n); }
std::string text(at::ScalarType t) { return c10::toString(t); }
std::string text(const c10::Device& d) { return d.str(); }
template <typename... A>
[[noreturn]] void refuse(const A&... parts) {
  throw Refused{(std::string() + ... + text(parts))};
}
void done(int rc, const char* what) {
  if (rc) refuse(what, " failed: ", native.last_error(), " (rc=", rc, ")");
}

int code_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CX_F32;
    case at::kBFloat16: return CX_BF16;
    case at::kHalf: return CX_F16;
    default: refuse("unsupported dtype ", t.scalar_type(), "; use float32, bfloat16 or float16");
  }
}
int dev_of(const Tensor& t) { return t.is_cuda() ? CX_DEV_CUDA : CX_DEV_HOST; }
void* stream_of(const Tensor& t) {
  if (!t.is_cuda()) return nullptr;
  return c10::impl::VirtualGuardImpl(c10::DeviceType::CUDA).getStream(t.device()).native_handle();
}

// `t` as a matrix of rows of `cols` consecutive elements that do not overlap, with their signs in memory: a view where that can be
Tensor rows_of(const Tensor& t, int64_t cols) {
  Tensor m = (t.dim() == 2 ? t : t.reshape({-1, cols})).resolve_neg();
  if ((m.size(0) > 1 && m.stride(0) < cols) || (cols > 1 && m.stride(1) != 1)) m = m.contiguous();
  return m;
}
int64_t ld_of(const Tensor& m) { return m.size(0) > 1 ? m.stride(0) : m.size(1); }

// scratch of one call, of the current stream, in the descriptor; the caller keeps it until the launches are out
template <typename D>
Tensor workspace(D& d, const Tensor& like, int64_t bytes) {
  d.ws_bytes = bytes;
  if (!bytes) return {};
  Tensor ws = at::empty({bytes}, like.options().dtype(at::kByte));
  d.workspace = ws.data_ptr();
  return ws;
}

// A trace sees the outputs being allocated and not the kernels that fill them: what it plays back would be memory that nobody
// wrote.  (torch.compile leaves a call to these functions out of its graphs.)  Under a mode of fake tensors the outputs would have
// no memory at all.  Asked once a call.
void for_real() {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  if (torch::jit::tracer::isTracing()) refuse("this operator cannot be put into a trace");
  if (!TorchDispatchModeTLS::any_modes_set()) return;
  if (TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY)) refuse("this operator cannot be put into a trace");
  if (TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FAKE) || TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FUNCTIONAL))
    refuse("what this operator makes would have no memory of its own under this mode");
}

// Fake tensors, those that a transform (vmap, grad) has wrapped and subclasses that dispatch in Python have no memory that the
// kernels could read.
void has_memory(const Tensor& t, const char* name) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet without({DispatchKey::Python, DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper,
                                         DispatchKey::Functionalize, DispatchKey::ZeroTensor});
  if (t.key_set().has_any(without) || !t.has_storage()) refuse(name, " has no memory of its own (a fake or wrapped tensor)");
}

// There is no forward-mode derivative: a tangent would be lost in silence.
void no_tangent(const Tensor& t, const char* name) {
  if (t._fw_grad(0).defined()) refuse(name, " has a forward-mode tangent, and this operator no forward-mode derivative");
}

// a gradient of zeros that autograd has not written down, written down
Tensor written(const Tensor& t) {
  return t.defined() && t._is_zerotensor() ? at::zeros(t.sizes(), t.options()) : t;
}

// Gradients that are computed here cannot be differentiated again: asking for it is an error of that second pass.
variable_list once(variable_list&& grads) {
  if (!at::GradMode::is_enabled()) return std::move(grads);
  for (Tensor& g : grads)
    if (g.defined()) {
      g = g.detach();
      g.set_requires_grad(true);
    }
  auto stop = std::make_shared<torch::autograd::DelayedError>("this operator's gradients cannot be differentiated again", (int64_t)grads.size());
  return (*stop)(std::move(grads));
}

// A saved tensor as it was saved, in rows without gaps: hooks may have kept it somewhere else, and must bring it back.
Tensor kept(const Tensor& t, const char* name, const Tensor& like, at::ScalarType type, at::IntArrayRef sizes) {
  if (!t.defined() || t.layout() != at::kStrided || t.device() != like.device() || t.scalar_type() != type || t.sizes() != sizes)
    refuse("the saved ", name, " has come back as another tensor");
  has_memory(t, name);
  return t.resolve_neg().contiguous();
}
// ... and a saved operand, whose rows may lie apart
void came_back(const Tensor& t, const char* name, const Tensor& like, at::ScalarType type, bool fits) {
  if (!fits || t.layout() != at::kStrided || t.device() != like.device() || t.scalar_type() != type) refuse("the saved ", name, " has come back as another tensor");
  has_memory(t, name);
}

template <typename F>
variable_list in_backward(const F& f) {
  try {
    for_real();
    return once(f());
  } catch (const Refused& r) {          // the engine may have called from a thread of its own
    const PyGILState_STATE gil = PyGILState_Ensure();
    PyErr_SetString(native.error, r.why.c_str());
    python_error e;
    e.persist();
    PyGILState_Release(gil);
    throw e;
  }
}

// ---- linear ---------------------------------------------------------------------------------------------------------
CxLinear describe(const Tensor& xm, const Tensor& wm, int act) {
  CxLinear d = {};
  d.rows = xm.size(0);
  d.inner = wm.size(1);
  d.outer = wm.size(0);
  d.x = xm.data_ptr();
  d.ldx = ld_of(xm);
  d.w = wm.data_ptr();
  d.ldw = ld_of(wm);
  d.dtype = code_of(xm);
  d.act = act;
  return d;
}

int64_t pre_columns(int64_t outer) { return (outer + 15) / 16 * 16; }

Tensor linear_forward(const Tensor& x, const Tensor& w, const Maybe& bias, int act, const Maybe& residual, Tensor* pre) {
  const int64_t outer = w.size(0), inner = w.size(1);
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = outer;
  Tensor y = at::empty(shape, x.options());
  if (!y.numel()) {
    if (pre) *pre = at::empty({0}, x.options());
    return y;
  }
  const c10::OptionalDeviceGuard guard(x.is_cuda() ? std::make_optional(x.device()) : std::nullopt);
  const Tensor xm = rows_of(x, inner), wm = rows_of(w, inner), b = bias ? bias->resolve_neg().contiguous() : Tensor(), r = residual ? rows_of(*residual, outer) : Tensor();
  CxLinear d = describe(xm, wm, act);
  if (bias) d.bias = b.data_ptr();
  if (residual) {
    d.residual = r.data_ptr();
    d.ldr = ld_of(r);
  }
  d.y = y.data_ptr();
  if (pre) {                                  // kept for the backward call, in aligned rows
    d.ldpre = pre_columns(outer);
    *pre = at::empty({d.rows, d.ldpre}, x.options());
    d.pre = pre->data_ptr();
  }
  const Tensor ws = workspace(d, x, native.linear_bytes(dev_of(x), &d, 0));
  done(native.linear_forward(dev_of(x), &d, stream_of(x)), "cx_linear_forward");
  return y;
}

struct LinearFn : torch::autograd::Function<LinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Maybe& bias, int64_t act, const Maybe& residual) {
    Tensor pre;
    Tensor y = linear_forward(x, w, bias, (int)act, residual, act != CX_ACT_NONE ? &pre : nullptr);
    ctx->saved_data["call"] = std::vector<int64_t>{act, (bias ? 1 : 0) | (residual ? 2 : 0)};
    ctx->save_for_backward({x, w, pre});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return in_backward([&]() -> variable_list {
      const variable_list saved = ctx->get_saved_variables();
      const Tensor &x = saved[0], &w = saved[1], grad = written(grads[0]);
      const auto call = ctx->saved_data["call"].toIntVector();
      const int64_t act = call[0], inputs = call[1];
      variable_list out(5);
      if (!grad.defined()) return out;
      has_memory(grad, "the gradient");
      no_tangent(grad, "the gradient");
      came_back(w, "weight", grad, grad.scalar_type(), w.dim() == 2 && w.size(0) == grad.size(-1));
      came_back(x, "x", grad, grad.scalar_type(), x.dim() == grad.dim() && x.size(-1) == w.size(1) && x.sizes().slice(0, x.dim() - 1) == grad.sizes().slice(0, x.dim() - 1));
      const bool bias = inputs & 1, residual = inputs & 2;
      const bool need_b = bias && ctx->needs_input_grad(2), need_r = residual && ctx->needs_input_grad(bias ? 3 : 2);
      const int64_t outer = w.size(0), inner = w.size(1);
      const at::AutoDispatchBelowADInplaceOrView below;
      if (ctx->needs_input_grad(0)) out[0] = at::empty(x.sizes(), x.options());
      if (ctx->needs_input_grad(1)) out[1] = at::empty(w.sizes(), x.options());
      if (need_b) out[2] = at::empty({outer}, x.options());
      if (need_r) out[4] = grad;
      if (!grad.numel()) {
        for (int i = 1; i < 3; ++i)
          if (out[i].defined()) out[i].zero_();
        return out;
      }
      if (!out[0].defined() && !out[1].defined() && !out[2].defined()) return out;
      const c10::OptionalDeviceGuard guard(x.is_cuda() ? std::make_optional(x.device()) : std::nullopt);
      const Tensor xm = rows_of(x, inner), wm = rows_of(w, inner), gm = rows_of(grad, outer);
      CxLinear d = describe(xm, wm, (int)act);
      d.grad = gm.data_ptr();
      d.ldg = ld_of(gm);
      Tensor pre;
      if (act != CX_ACT_NONE) {
        d.ldpre = pre_columns(outer);
        pre = kept(saved[2], "u", grad, grad.scalar_type(), {d.rows, d.ldpre});
        d.pre = pre.data_ptr();
      }
      if (out[0].defined()) d.dx = out[0].data_ptr();
      if (out[1].defined()) d.dw = out[1].data_ptr();
      if (out[2].defined()) d.dbias = out[2].data_ptr();
      const Tensor ws = workspace(d, x, native.linear_bytes(dev_of(x), &d, 1));
      done(native.linear_backward(dev_of(x), &d, stream_of(x)), "cx_linear_backward");
      return out;
    });
  }
};

// ---- loss over a vocabulary -------------------------------------------------------------------------------------------
CxVocabLoss describe(const Tensor& hm, const Tensor& wm, const Tensor& tm, int64_t ignore, int reduction, const Tensor& lse, const Tensor& count) {
  CxVocabLoss d = {};
  d.rows = hm.size(0);
  d.vocab = wm.size(0);
  d.dim = wm.size(1);
  d.h = hm.data_ptr();
  d.ldh = ld_of(hm);
  d.w = wm.data_ptr();
  d.ldw = ld_of(wm);
  d.targets = tm.data_ptr<int64_t>();
  d.ignore_index = ignore;
  d.lse = lse.data_ptr<float>();
  d.count = count.data_ptr<float>();
  d.dtype = code_of(hm);
  d.reduction = reduction;
  return d;
}

Tensor loss_forward(const Tensor& h, const Tensor& w, const Tensor& targets, int64_t ignore, int reduction, Tensor& tm, Tensor& lse, Tensor& count) {
  const c10::OptionalDeviceGuard guard(h.is_cuda() ? std::make_optional(h.device()) : std::nullopt);
  tm = targets.reshape({-1}).resolve_neg().contiguous();
  const auto f32 = h.options().dtype(at::kFloat);
  Tensor loss = reduction == CX_REDUCE_NONE ? at::empty(targets.sizes(), f32) : at::empty({}, f32);
  lse = at::empty({tm.numel()}, f32);
  count = at::empty({1}, f32);
  if (!tm.numel()) return reduction == CX_REDUCE_NONE ? loss : loss.fill_(reduction == CX_REDUCE_SUM ? 0.0 : NAN);
  const Tensor hm = rows_of(h, w.size(1)), wm = rows_of(w, w.size(1));
  CxVocabLoss d = describe(hm, wm, tm, ignore, reduction, lse, count);
  d.loss = loss.data_ptr<float>();
  const Tensor ws = workspace(d, h, native.loss_bytes(dev_of(h), &d, 0));
  done(native.loss_forward(dev_of(h), &d, stream_of(h)), "cx_vocab_loss_forward");
  return loss;
}

struct LossFn : torch::autograd::Function<LossFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& h, const Tensor& w, const Tensor& targets, int64_t ignore, int64_t reduction) {
    Tensor tm, lse, count;
    Tensor loss = loss_forward(h, w, targets, ignore, (int)reduction, tm, lse, count);
    ctx->saved_data["call"] = std::vector<int64_t>{ignore, reduction, tm.numel(), static_cast<int64_t>(h.scalar_type())};
    ctx->save_for_backward({h, w, tm, lse, count});
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return in_backward([&]() -> variable_list {
      const variable_list saved = ctx->get_saved_variables();
      const Tensor &h = saved[0], &w = saved[1];
      grads[0] = written(grads[0]);
      variable_list out(5);
      if (!grads[0].defined()) return out;
      has_memory(grads[0], "the gradient");
      no_tangent(grads[0], "the gradient");
      const auto call = ctx->saved_data["call"].toIntVector();
      const int64_t ignore = call[0], rows = call[2];
      const int reduction = (int)call[1];
      const auto type = static_cast<at::ScalarType>(call[3]);
      came_back(w, "weight", grads[0], type, w.dim() == 2 && w.numel());
      came_back(h, "hidden", grads[0], type, h.dim() >= 1 && h.size(-1) == w.size(1) && h.numel() == rows * w.size(1));
      const Tensor tm = kept(saved[2], "targets", grads[0], at::kLong, {rows}), lse = kept(saved[3], "sums", grads[0], at::kFloat, {rows}),
                   count = kept(saved[4], "count", grads[0], at::kFloat, {1});
      const at::AutoDispatchBelowADInplaceOrView below;
      if (ctx->needs_input_grad(0)) out[0] = at::empty(h.sizes(), h.options());
      if (ctx->needs_input_grad(1)) out[1] = at::empty(w.sizes(), w.options());
      if (!tm.numel()) {
        if (out[1].defined()) out[1].zero_();
        return out;
      }
      const c10::OptionalDeviceGuard guard(h.is_cuda() ? std::make_optional(h.device()) : std::nullopt);
      const Tensor hm = rows_of(h, w.size(1)), wm = rows_of(w, w.size(1));
      CxVocabLoss d = describe(hm, wm, tm, ignore, reduction, lse, count);
      Tensor g = grads[0].to(at::kFloat).resolve_neg();
      if (g.dim() > 1) g = g.reshape({-1});
      d.grad = g.data_ptr<float>();
      d.grad_stride = g.dim() ? g.stride(0) : 0;
      if (out[0].defined()) d.dh = out[0].data_ptr();
      if (out[1].defined()) d.dw = out[1].data_ptr();
      const Tensor ws = workspace(d, h, native.loss_bytes(dev_of(h), &d, 1));
      done(native.loss_backward(dev_of(h), &d, stream_of(h)), "cx_vocab_loss_backward");
      return out;
    });
  }
};

// ---- calls from Python --------------------------------------------------------------------------------------------------
// a strided tensor on the device of `like` (itself where that is NULL)
const Tensor& tensor(PyObject* o, const char* name, const Tensor* like) {
  if (!THPVariable_Check(o)) refuse(name, " must be a strided tensor");
  const Tensor& t = THPVariable_Unpack(o);
  if (t.layout() != at::kStrided) refuse(name, " must be a strided tensor");
  if (!like) for_real();
  if (!like && !t.is_cuda() && !t.is_cpu()) refuse("tensors on ", t.device(), " are not supported");
  if (like && t.device() != like->device()) refuse(name, " is on ", t.device(), ", not on ", like->device());
  has_memory(t, name);
  no_tangent(t, name);
  return t;
}
const Tensor& same_type(const Tensor& t, const char* name, const Tensor& like) {
  if (t.scalar_type() != like.scalar_type()) refuse(name, " is ", t.scalar_type(), ", not ", like.scalar_type(), ": one type is needed");
  return t;
}

// The type that torch's own product would be in: autocast's, where that is on and casts such a tensor; else the tensor's.
struct Cast {
  bool on;
  at::ScalarType type;
  explicit Cast(const Tensor& x) : on(at::autocast::is_autocast_enabled(x.device().type())), type(x.scalar_type()) {
    if (on && x.is_floating_point() && type != at::kDouble) type = at::autocast::get_autocast_dtype(x.device().type());
  }
  // an operand in it, by autocast's rules and through its cache of weights
  Tensor of(const Tensor& t) const { return on ? at::autocast::cached_cast(type, t, t.device().type()) : t; }
};

void out_of_memory(const c10::OutOfMemoryError& e) {
  PyObject* torch = PyImport_ImportModule("torch");
  PyObject* kind = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
  PyErr_Clear();
  PyErr_SetString(kind ? kind : PyExc_MemoryError, e.what_without_backtrace());
  Py_XDECREF(kind);
  Py_XDECREF(torch);
}

template <typename F>
PyObject* guarded(const F& f) {
  try {
    Tensor out;
    {
      struct Without {                   // other threads may run: the native calls need no Python
        PyThreadState* state = PyEval_SaveThread();
        ~Without() { PyEval_RestoreThread(state); }
      } without;
      out = f();
    }
    return THPVariable_Wrap(std::move(out));
  } catch (const Refused& r) {
    PyErr_SetString(r.value ? PyExc_ValueError : native.error, r.why.c_str());
  } catch (python_error& e) {
    e.restore();
  } catch (const c10::OutOfMemoryError& e) {
    out_of_memory(e);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

}  // namespace

// linear(x, weight, bias or None, activation, residual or None); activation: CX_ACT_*
PyObject* cx_py_linear(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  if (nargs != 5) {
    PyErr_SetString(PyExc_TypeError, "linear: five arguments");
    return nullptr;
  }
  const long act = PyLong_AsLong(a[3]);
  if (PyErr_Occurred()) return nullptr;
  Tensor x, w;
  Maybe bias, residual;
  bool apart = false;          // the residual is added to the result, in the type that torch adds the two in
  try {
    const Tensor& given = tensor(a[0], "x", nullptr);
    const Cast cast(given);
    x = cast.of(given);
    code_of(x);
    w = same_type(cast.of(tensor(a[1], "weight", &x)), "weight", x);
    if (a[2] != Py_None) bias = same_type(cast.of(tensor(a[2], "bias", &x)), "bias", x);
    if (a[4] != Py_None) {
      residual = tensor(a[4], "residual", &x);
      if (cast.on && residual->scalar_type() != cast.type) apart = true;       // (autocast leaves sums as they are)
      else residual = same_type(*residual, "residual", x);
    }
    if (w.dim() != 2 || x.dim() < 1 || x.size(-1) != w.size(1) || !w.numel()) refuse("x ", shape_of(x), " does not fit weight ", shape_of(w));
    if (bias && (bias->dim() != 1 || bias->size(0) != w.size(0))) refuse("bias ", shape_of(*bias), " does not fit weight ", shape_of(w));
    if (residual) {
      bool fits = residual->dim() == x.dim() && residual->size(-1) == w.size(0);
      for (int64_t i = 0; fits && i + 1 < x.dim(); ++i) fits = residual->size(i) == x.size(i);
      if (!fits) refuse("residual ", shape_of(*residual), " does not have the result's shape");
    }
  } catch (const Refused& r) {
    PyErr_SetString(native.error, r.why.c_str());
    return nullptr;
  } catch (const c10::OutOfMemoryError& e) {
    out_of_memory(e);
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(native.error, e.what());
    return nullptr;
  }
  Tensor more;
  if (apart) {
    more = *residual;
    residual.reset();
  }
  const bool train = at::GradMode::is_enabled() &&
                     (x.requires_grad() || w.requires_grad() || (bias && bias->requires_grad()) || (residual && residual->requires_grad()));
  return guarded([&] {
    const Tensor y = train ? LinearFn::apply(x, w, bias, (int64_t)act, residual) : linear_forward(x, w, bias, (int)act, residual, nullptr);
    return apart ? y + more : y;
  });
}

// vocab_loss(hidden, weight, targets, ignore_index, reduction); reduction: CX_REDUCE_*
PyObject* cx_py_vocab_loss(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  if (nargs != 5) {
    PyErr_SetString(PyExc_TypeError, "vocab_loss: five arguments");
    return nullptr;
  }
  const long long ignore = PyLong_AsLongLong(a[3]);
  const long reduction = PyLong_AsLong(a[4]);
  if (PyErr_Occurred()) return nullptr;
  Tensor h, w, targets;
  try {
    const Tensor& given = tensor(a[0], "hidden", nullptr);
    const Cast cast(given);
    h = cast.of(given);
    code_of(h);
    w = same_type(cast.of(tensor(a[1], "weight", &h)), "weight", h);
    targets = tensor(a[2], "targets", &h);
    if (targets.scalar_type() != at::kLong) refuse("targets must be int64, not ", targets.scalar_type());
    if (w.dim() != 2 || !w.numel() || h.dim() < 1 || h.size(-1) != w.size(1)) refuse("hidden ", shape_of(h), " does not fit weight ", shape_of(w));
    if (targets.sizes() != h.sizes().slice(0, h.dim() - 1)) refuse("targets ", shape_of(targets), " do not fit hidden ", shape_of(h));
  } catch (const Refused& r) {
    PyErr_SetString(native.error, r.why.c_str());
    return nullptr;
  } catch (const c10::OutOfMemoryError& e) {
    out_of_memory(e);
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(native.error, e.what());
    return nullptr;
  }
  const bool train = at::GradMode::is_enabled() && (h.requires_grad() || w.requires_grad());
  return guarded([&]() -> Tensor {
    if (train) return LossFn::apply(h, w, targets, (int64_t)ignore, (int64_t)reduction);
    Tensor tm, lse, count;
    return loss_forward(h, w, targets, ignore, (int)reduction, tm, lse, count);
  });
}

// bind_operators(error class, addresses of the seven native functions in the order of Native)
PyObject* cx_py_bind_operators(PyObject*, PyObject* args) {
  unsigned long long f[7];
  PyObject* error;
  if (!PyArg_ParseTuple(args, "OKKKKKKK", &error, f, f + 1, f + 2, f + 3, f + 4, f + 5, f + 6)) return nullptr;
  native.linear_bytes = reinterpret_cast<decltype(native.linear_bytes)>(f[0]);
  native.linear_forward = reinterpret_cast<decltype(native.linear_forward)>(f[1]);
  native.linear_backward = reinterpret_cast<decltype(native.linear_backward)>(f[2]);
  native.loss_bytes = reinterpret_cast<decltype(native.loss_bytes)>(f[3]);
  native.loss_forward = reinterpret_cast<decltype(native.loss_forward)>(f[4]);
  native.loss_backward = reinterpret_cast<decltype(native.loss_backward)>(f[5]);
  native.last_error = reinterpret_cast<decltype(native.last_error)>(f[6]);
  Py_INCREF(error);
  Py_XDECREF(native.error);
  native.error = error;
  Py_RETURN_NONE;
}
