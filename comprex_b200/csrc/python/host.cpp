// Host work on torch tensors for the Python side, where attribute look-ups in Python would cost as
// much as the GPU's work:
//  * collect: the addresses of an optimizer's gradients (161 parameters: 60 us in Python, 3 us here,
//    next to 110 us of GPU work for the step),
//  * layout, addresses: those of the tensors themselves, as long as the tensors are what they were,
//  * graded: which tensors have a gradient; stepped: tells autograd which have been written,
//  * run_vector: the launches of one message of a prepared connection.  Checks of the vector,
//    descriptors and native calls took 20 us per exchange in Python, the kernels of a 64 k-element
//    exchange take 15 us,
//  * linear, vocab_loss: the operators of operators.cpp.
// Tensors of unusual kinds (nested, sparse, wrapped by a transform) throw at the questions asked here.  No
// exception may leave these functions: such a tensor is not the plain case, and the caller's general path
// says what is wrong with it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "../cx_common.h"
#include "operators.h"

namespace {

// the same memory order: strides of dimensions of size 1 say nothing
bool same_layout(const at::Tensor& a, const at::Tensor& b) {
  const auto n = b.sizes();
  if (a.sizes() != n) return false;
  const auto x = a.strides(), y = b.strides();
  for (size_t d = 0; d < n.size(); ++d)
    if (n[d] != 1 && x[d] != y[d]) return false;
  return true;
}

// Whether the elements lie in memory as strides say.  (Fake tensors, wrapped ones, zeros that are not written down and signs that
// are only noted do not.)
bool plain(const at::Tensor& t) {
  const c10::DispatchKeySet keys = t.key_set();
  return t.layout() == at::kStrided && t.has_storage() && !t.is_neg() && !keys.has(c10::DispatchKey::Python) &&
         !keys.has(c10::DispatchKey::ZeroTensor) && !keys.has(c10::DispatchKey::Functionalize);
}

// collect(params, scalar_type, zeros, out) -> 0: the table at address `out` (one int64 per parameter)
// already held these addresses, 1: it has changed, 2: some gradient has another element type, device
// or memory order than its parameter, or no plain memory (the table is incomplete).  `zeros` stands in for a missing one.
PyObject* collect(PyObject*, PyObject* args) {
  PyObject* params;
  int scalar_type;
  unsigned long long zeros, out;
  if (!PyArg_ParseTuple(args, "O!iKK", &PyList_Type, &params, &scalar_type, &zeros, &out)) return nullptr;
  int64_t* table = reinterpret_cast<int64_t*>(out);
  long changed = 0;
  const Py_ssize_t n = PyList_GET_SIZE(params);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PyList_GET_ITEM(params, i);
    if (!THPVariable_Check(o)) {
      PyErr_SetString(PyExc_TypeError, "collect: not a tensor");
      return nullptr;
    }
    int64_t a = static_cast<int64_t>(zeros);
    try {
      const at::Tensor& p = THPVariable_Unpack(o);
      const at::Tensor& g = p.grad();
      if (g.defined()) {
        if (static_cast<int>(g.scalar_type()) != scalar_type || !plain(g) || g.device() != p.device() || !same_layout(g, p))
          return PyLong_FromLong(2);
        a = reinterpret_cast<int64_t>(g.data_ptr());
      }
    } catch (const std::exception&) {
      return PyLong_FromLong(2);
    }
    changed |= table[i] != a;
    table[i] = a;
  }
  return PyLong_FromLong(changed);
}

// What the flat states of an optimizer go by: element type, device, sizes and strides of each of its tensors.
void describe(const at::Tensor& t, std::vector<int64_t>& out) {
  out.push_back(static_cast<int64_t>(t.scalar_type()));
  out.push_back(static_cast<int64_t>(t.device().type()));
  out.push_back(t.device().index());
  out.push_back(t.dim());
  for (int64_t d = 0; d < t.dim(); ++d) {
    out.push_back(t.size(d));
    out.push_back(t.size(d) == 1 ? 0 : t.stride(d));
  }
}
// the end of the description at `d` if it is that of `t`, else NULL; nothing is read from `end` on
const int64_t* as_described(const at::Tensor& t, const int64_t* d, const int64_t* end) {
  if (end - d < 4 || !plain(t) || d[0] != static_cast<int64_t>(t.scalar_type()) || d[1] != static_cast<int64_t>(t.device().type()) ||
      d[2] != t.device().index() || d[3] != t.dim())
    return nullptr;
  d += 4;
  if (end - d < 2 * t.dim()) return nullptr;
  const auto size = t.sizes(), stride = t.strides();
  for (size_t i = 0; i < size.size(); ++i, d += 2)
    if (d[0] != size[i] || (size[i] != 1 && d[1] != stride[i])) return nullptr;
  return d;
}

// layout(tensors) -> bytes for `addresses`; None where one has no plain memory, or what is made now would not have any
PyObject* layout(PyObject*, PyObject* tensors) {
  if (!PyList_Check(tensors)) {
    PyErr_SetString(PyExc_TypeError, "layout: a list of tensors");
    return nullptr;
  }
  try {
    std::vector<int64_t> all;
    if (c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::FAKE)) Py_RETURN_NONE;
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(tensors); ++i) {
      PyObject* o = PyList_GET_ITEM(tensors, i);
      if (!THPVariable_Check(o)) {
        PyErr_SetString(PyExc_TypeError, "layout: not a tensor");
        return nullptr;
      }
      if (!plain(THPVariable_Unpack(o))) Py_RETURN_NONE;
      describe(THPVariable_Unpack(o), all);
    }
    return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(all.data()), static_cast<Py_ssize_t>(all.size() * sizeof(int64_t)));
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// addresses(tensors, layout, out) -> 0: the table at address `out` (one int64 per tensor) already held these addresses, 1: it
// has changed, -1 - i: tensor i is not what `layout` says of it (the table is as it was)
PyObject* addresses(PyObject*, PyObject* args) {
  PyObject *tensors, *bytes;
  unsigned long long out;
  if (!PyArg_ParseTuple(args, "O!SK", &PyList_Type, &tensors, &bytes, &out)) return nullptr;
  int64_t* table = reinterpret_cast<int64_t*>(out);
  const int64_t* d = reinterpret_cast<const int64_t*>(PyBytes_AS_STRING(bytes));
  const int64_t* end = d + PyBytes_GET_SIZE(bytes) / static_cast<Py_ssize_t>(sizeof(int64_t));
  bool changed = false;
  const Py_ssize_t n = PyList_GET_SIZE(tensors);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PyList_GET_ITEM(tensors, i);
    if (!THPVariable_Check(o)) {
      PyErr_SetString(PyExc_TypeError, "addresses: not a tensor");
      return nullptr;
    }
    try {
      const at::Tensor& t = THPVariable_Unpack(o);
      d = as_described(t, d, end);
      if (!d) return PyLong_FromLong(-1 - static_cast<long>(i));
      changed |= table[i] != reinterpret_cast<int64_t>(t.data_ptr());
    } catch (const std::exception&) {
      return PyLong_FromLong(-1 - static_cast<long>(i));
    }
  }
  if (!changed) return PyLong_FromLong(0);
  for (Py_ssize_t i = 0; i < n; ++i) table[i] = reinterpret_cast<int64_t>(THPVariable_Unpack(PyList_GET_ITEM(tensors, i)).data_ptr());
  return PyLong_FromLong(1);
}

// graded(tensors) -> a list of those that have a gradient
PyObject* graded(PyObject*, PyObject* tensors) {
  if (!PyList_Check(tensors)) {
    PyErr_SetString(PyExc_TypeError, "graded: a list of tensors");
    return nullptr;
  }
  PyObject* found = PyList_New(0);
  for (Py_ssize_t i = 0; found && i < PyList_GET_SIZE(tensors); ++i) {
    PyObject* o = PyList_GET_ITEM(tensors, i);
    bool has = false;
    try {
      has = THPVariable_Check(o) && THPVariable_Unpack(o).grad().defined();
    } catch (const std::exception& e) {
      PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    if (PyErr_Occurred() || (has && PyList_Append(found, o) != 0)) Py_CLEAR(found);
  }
  return found;
}

// stepped(tensors, table): those with an address at `table` (one int64 per tensor, 0: none) have been written in place
PyObject* stepped(PyObject*, PyObject* args) {
  PyObject* tensors;
  unsigned long long at;
  if (!PyArg_ParseTuple(args, "O!K", &PyList_Type, &tensors, &at)) return nullptr;
  const int64_t* table = reinterpret_cast<const int64_t*>(at);
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(tensors); ++i) {
    PyObject* o = PyList_GET_ITEM(tensors, i);
    if (!THPVariable_Check(o)) {
      PyErr_SetString(PyExc_TypeError, "stepped: not a tensor");
      return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (table[i] && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
  Py_RETURN_NONE;
}

int element_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CX_F32;
    case at::kBFloat16: return CX_BF16;
    case at::kHalf: return CX_F16;
    default: return -1;
  }
}

typedef int (*RunOps)(CxOp*, int, uint64_t, void*);
enum Role { kSend = 0, kApply = 1, kDenseSend = 2, kDenseRead = 3, kDenseAdd = 4, kRleRead = 5 };

// run_vector(role, run_ops, ops, count, seq, stream, vector, device, n) -> what cx_run_ops returns, or
// None when the vector is not the plain case (a contiguous CUDA tensor of the right size and type on
// `device`): nothing has happened then, the caller takes its general path.
//   kSend: input of a threshold + compress (or run-length send) list, n elements.  kApply: destination of an
//   apply op, n elements.  kDense*: a dense message of the vector's length, at most n, of the op's element type.
//   kRleRead: destination of a run-length receive, n fp32 elements.
PyObject* run_vector(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  if (nargs != 9) {
    PyErr_SetString(PyExc_TypeError, "run_vector: nine arguments");
    return nullptr;
  }
  const long role = PyLong_AsLong(a[0]);
  RunOps run = reinterpret_cast<RunOps>(PyLong_AsUnsignedLongLong(a[1]));
  CxOp* ops = reinterpret_cast<CxOp*>(PyLong_AsUnsignedLongLong(a[2]));
  const long count = PyLong_AsLong(a[3]);
  const uint64_t seq = PyLong_AsUnsignedLongLong(a[4]);
  void* stream = reinterpret_cast<void*>(PyLong_AsUnsignedLongLong(a[5]));
  const long device = PyLong_AsLong(a[7]);
  const int64_t n = PyLong_AsLongLong(a[8]);
  if (PyErr_Occurred()) return nullptr;
  if (!THPVariable_CheckExact(a[6])) Py_RETURN_NONE;
  int code;
  int64_t len;
  void* ptr;
  try {
    const at::Tensor& t = THPVariable_Unpack(a[6]);
    if (!t.is_cuda() || t.device().index() != device || t.layout() != at::kStrided || !t.is_contiguous()) Py_RETURN_NONE;
    code = element_code(t);
    if (code < 0) Py_RETURN_NONE;
    len = t.numel();
    ptr = t.data_ptr();
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
  if (role == kSend) {
    if (len != n) Py_RETURN_NONE;
    for (long i = 0; i < count; ++i) {
      ops[i].g = ptr;
      ops[i].dtype = code;
    }
  } else if (role == kApply) {
    if (len < n) Py_RETURN_NONE;
    ops[0].apply.out = ptr;
    ops[0].apply.out_dtype = code;
  } else if (role == kRleRead) {
    if (len != n || code != CX_F32) Py_RETURN_NONE;
    ops[0].out = ptr;
  } else {
    if (len > n || code != ops[0].dtype) Py_RETURN_NONE;
    ops[0].n = len;
    if (role == kDenseSend) ops[0].g = ptr;
    else ops[0].out = ptr;
    if (role == kDenseAdd) ops[0].own = ptr;
  }
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = run(ops, static_cast<int>(count), seq, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// install(pairs): `v.grad = g` for every (g, v); the checks of the attribute are left to it whenever
// the pair is not plainly two tensors of the same kind.
PyObject* install(PyObject*, PyObject* pairs) {
  PyObject* it = PyObject_GetIter(pairs);
  if (!it) return nullptr;
  while (PyObject* pair = PyIter_Next(it)) {
    PyObject* two = PySequence_Fast(pair, "install: (gradient, variable) pairs");
    Py_DECREF(pair);
    bool ok = two && PySequence_Fast_GET_SIZE(two) == 2;
    if (two && !ok) PyErr_SetString(PyExc_ValueError, "install: (gradient, variable) pairs");
    if (ok) {
      PyObject* g = PySequence_Fast_GET_ITEM(two, 0);
      PyObject* v = PySequence_Fast_GET_ITEM(two, 1);
      bool done = false;
      if (THPVariable_Check(g) && THPVariable_Check(v) && g != v) {
        try {
          const at::Tensor& gt = THPVariable_Unpack(g);
          const at::Tensor& vt = THPVariable_Unpack(v);
          if (gt.defined() && vt.defined() && vt.is_leaf() && gt.layout() == at::kStrided && vt.layout() == at::kStrided &&
              gt.scalar_type() == vt.scalar_type() && vt.grad_dtype() == vt.scalar_type() && gt.device() == vt.device() && gt.sizes() == vt.sizes()) {
            vt.mutable_grad() = gt;
            done = true;
          }
        } catch (const std::exception&) {
          done = false;
        }
      }
      ok = done || PyObject_SetAttrString(v, "grad", g) == 0;
    }
    Py_XDECREF(two);
    if (!ok) break;
  }
  Py_DECREF(it);
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// the value `collect` wants for a dtype, from a tensor of that dtype
PyObject* scalar_type(PyObject*, PyObject* o) {
  if (!THPVariable_Check(o)) {
    PyErr_SetString(PyExc_TypeError, "scalar_type: not a tensor");
    return nullptr;
  }
  return PyLong_FromLong(static_cast<long>(THPVariable_Unpack(o).scalar_type()));      // (does not throw)
}

PyMethodDef methods[] = {{"collect", collect, METH_VARARGS, nullptr},
                         {"layout", layout, METH_O, nullptr},
                         {"addresses", addresses, METH_VARARGS, nullptr},
                         {"graded", graded, METH_O, nullptr},
                         {"stepped", stepped, METH_VARARGS, nullptr},
                         {"run_vector", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(run_vector)),
                          METH_FASTCALL, nullptr},
                         {"install", install, METH_O, nullptr},
                         {"scalar_type", scalar_type, METH_O, nullptr},
                         {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(cx_py_linear)), METH_FASTCALL, nullptr},
                         {"vocab_loss", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(cx_py_vocab_loss)), METH_FASTCALL, nullptr},
                         {"bind_operators", cx_py_bind_operators, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_cxhost", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__cxhost(void) { return PyModule_Create(&module); }
