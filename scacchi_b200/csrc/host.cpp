// The calls of the operators around a policy step from Python, where their
// arguments are plain: a call of them takes the host longer in Python (its
// checks, result tensors and bindings) than the GPU takes for a small one.
//
// Each function returns None where anything is not plain (another type,
// layout, device or size, a value to refuse), and the caller's Python goes on
// with its own checks, copies and errors; no argument is written then.  What
// fails in the library's launches is an error at once: some of a call's
// launches may have run, and the call may not be made again.  The library's
// entry points come as addresses (bind).
//
// 66 small tensors' AdamW step takes 56 us without this and 13 us with it,
// the norm of 73 gradients 47 and 10, log-probabilities of 64 x 82 24 and 11.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <memory>
#include <vector>

#include "../../include/scacchi_b200.h"

namespace {

struct Entries {
  decltype(&scacchi_log_probs) log_probs = nullptr;
  decltype(&scacchi_log_probs_gradient) gradient = nullptr;
  decltype(&scacchi_gradient_norm) norm = nullptr;
  decltype(&scacchi_gradient_norm_workspace_bytes) norm_bytes = nullptr;
  decltype(&scacchi_adamw_step) step = nullptr;
  decltype(&scacchi_adamw_moments) moments = nullptr;
  PyObject *error = nullptr;  // the class of what is raised
} g;

struct Failed {};  // thrown with a Python error set

// Whether the library took the call; false where it refused it, before any launch
bool taken(int status, const char *what) {
  if (status == SCACCHI_OK) return true;
  if (status == SCACCHI_EINVAL) return false;
  PyErr_Format(g.error, "%s: CUDA launch failed (status %d)", what, status);
  throw Failed{};
}

int code_of(at::ScalarType t) {
  return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1;
}

// A dense tensor on device `index`, or nullptr
const at::Tensor *plain(PyObject *o, int index) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor &t = THPVariable_Unpack(o);
  return t.is_cuda() && t.get_device() == index && t.layout() == at::kStrided && t.is_contiguous() ? &t : nullptr;
}

void *stream_of(int index) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream(); }

at::Tensor empty(at::IntArrayRef size, at::ScalarType type, int index) {
  return at::empty(size, at::TensorOptions().dtype(type).device(at::kCUDA, (c10::DeviceIndex)index));
}

// What both calls over rows of logits take.  False where it is not plain.
struct Rows {
  const at::Tensor *logits = nullptr, *action = nullptr, *legal = nullptr;
  scacchi_log_prob_rows rows;
  int64_t num_rows;
  int32_t actions, dtype;
  int index;

  bool read(PyObject *x, PyObject *a, PyObject *mask) {
    if (!THPVariable_Check(x)) return false;
    logits = &THPVariable_Unpack(x);
    if (!logits->is_cuda() || logits->dim() < 1) return false;
    index = logits->get_device();
    dtype = code_of(logits->scalar_type());
    if (index != c10::cuda::current_device() || dtype < 0 || !plain(x, index)) return false;
    const int64_t last = logits->size(-1);
    if (last < 1 || last > SCACCHI_MAX_ACTIONS) return false;
    actions = (int32_t)last;
    num_rows = logits->numel() / last;
    action = plain(a, index);
    if (!action || action->scalar_type() != at::kInt || action->sizes() != lead()) return false;
    if (mask != Py_None) {
      legal = plain(mask, index);
      if (!legal || legal->scalar_type() != at::kBool || legal->sizes() != logits->sizes()) return false;
    }
    rows = {logits->data_ptr(), legal ? static_cast<const uint8_t *>(legal->data_ptr()) : nullptr,
            static_cast<const int32_t *>(action->data_ptr()), last};
    return true;
  }
  at::IntArrayRef lead() const { return logits->sizes().slice(0, logits->dim() - 1); }
  // float32 of the rows' shape; *out stays nullptr for None
  bool per_row(PyObject *o, const float **out) const {
    if (o == Py_None) return true;
    const at::Tensor *t = plain(o, index);
    if (!t || t->scalar_type() != at::kFloat || t->sizes() != lead()) return false;
    *out = static_cast<const float *>(t->data_ptr());
    return true;
  }
};

// (logits, action, legal, temperature, top) -> (log_prob, entropy, max_logit, log_sum, top_log_prob, top_action)
PyObject *log_probs(PyObject *, PyObject *const *args, Py_ssize_t n) {
  try {
    Rows r;
    if (n != 5 || !PyFloat_CheckExact(args[3]) || !PyLong_CheckExact(args[4]) || !r.read(args[0], args[1], args[2]))
      Py_RETURN_NONE;
    const double temperature = PyFloat_AS_DOUBLE(args[3]);
    int over = 0;
    const long top = PyLong_AsLongAndOverflow(args[4], &over);
    if (over || top < 0 || top > SCACCHI_MAX_TOP) Py_RETURN_NONE;
    at::Tensor out[6];
    for (int i = 0; i < 4; ++i) out[i] = empty(r.lead(), at::kFloat, r.index);
    if (top) {
      auto size = r.lead().vec();
      size.push_back(top);
      out[4] = empty(size, at::kFloat, r.index);
      out[5] = empty(size, at::kInt, r.index);
    }
    const scacchi_log_prob_out at = {
        static_cast<float *>(out[0].data_ptr()), static_cast<float *>(out[1].data_ptr()),
        static_cast<float *>(out[2].data_ptr()), static_cast<float *>(out[3].data_ptr()),
        top ? static_cast<float *>(out[4].data_ptr()) : nullptr, top ? static_cast<int32_t *>(out[5].data_ptr()) : nullptr};
    if (!taken(g.log_probs(&r.rows, &at, r.num_rows, r.actions, r.dtype, temperature, (int32_t)top,
                           stream_of(r.index)), "log_probs"))
      Py_RETURN_NONE;
    PyObject *tuple = PyTuple_New(6);
    if (!tuple) return nullptr;
    for (int i = 0; i < 6; ++i) {
      PyObject *o = i < 4 || top ? THPVariable_Wrap(out[i]) : Py_NewRef(Py_None);
      if (!o) {
        Py_DECREF(tuple);
        return nullptr;
      }
      PyTuple_SET_ITEM(tuple, i, o);
    }
    return tuple;
  } catch (const Failed &) {
    return nullptr;
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// (logits, action, legal, temperature, max_logit, log_sum, entropy, grad_log_prob, grad_entropy) -> gradient
PyObject *log_probs_gradient(PyObject *, PyObject *const *args, Py_ssize_t n) {
  try {
    Rows r;
    const float *at[5] = {};
    if (n != 9 || !PyFloat_CheckExact(args[3]) || !r.read(args[0], args[1], args[2])) Py_RETURN_NONE;
    for (int i = 0; i < 5; ++i)
      if (!r.per_row(args[4 + i], &at[i])) Py_RETURN_NONE;
    if (args[4] == Py_None || args[5] == Py_None || (args[7] == Py_None && args[8] == Py_None) ||
        (args[8] != Py_None && args[6] == Py_None))
      Py_RETURN_NONE;
    at::Tensor out = empty(r.logits->sizes(), r.logits->scalar_type(), r.index);
    if (!taken(g.gradient(&r.rows, at[0], at[1], at[2], at[3], at[4], r.num_rows, r.actions, r.dtype,
                          PyFloat_AS_DOUBLE(args[3]), out.data_ptr(), stream_of(r.index)), "log_probs_gradient"))
      Py_RETURN_NONE;
    return THPVariable_Wrap(out);
  } catch (const Failed &) {
    return nullptr;
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// The norm of a table's gradients on device `index`; undefined where the library refuses
at::Tensor norm_of(const scacchi_adamw_tensor *table, int32_t n, int index) {
  at::Tensor out = empty({}, at::kFloat, index);
  at::Tensor workspace = empty({(int64_t)(g.norm_bytes(n) + 7) / 8}, at::kDouble, index);
  if (!taken(g.norm(table, n, static_cast<float *>(out.data_ptr()), workspace.data_ptr(), stream_of(index)),
             "gradient_norm"))
    return at::Tensor();
  return out;
}

// (list or tuple of gradients) -> norm
PyObject *gradient_norm(PyObject *, PyObject *list) {
  try {
    if (!PyList_CheckExact(list) && !PyTuple_CheckExact(list)) Py_RETURN_NONE;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(list);
    PyObject **items = PySequence_Fast_ITEMS(list);
    if (n == 0 || n > 0x7fffffff) Py_RETURN_NONE;
    const int index = c10::cuda::current_device();
    std::vector<scacchi_adamw_tensor> table((size_t)n);
    for (Py_ssize_t i = 0; i < n; ++i) {
      const at::Tensor *t = plain(items[i], index);
      const int dtype = t ? code_of(t->scalar_type()) : -1;
      if (dtype < 0) Py_RETURN_NONE;
      table[i] = {nullptr, t->data_ptr(), t->numel(), 0, 0.0, 0, dtype};
    }
    at::Tensor out = norm_of(table.data(), (int32_t)n, index);
    if (!out.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(out);
  } catch (const Failed &) {
    return nullptr;
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// One float32 on device `index`, or nullptr
const at::Tensor *scalar(PyObject *o, int index) {
  const at::Tensor *t = plain(o, index);
  return t && t->scalar_type() == at::kFloat && t->numel() == 1 ? t : nullptr;
}

// (names, weights, gradients, address of the table, address of the parameters, device, max_norm or None, norm or None,
// learning_rate or None) -> (norm or None,)
PyObject *adamw_step(PyObject *, PyObject *const *args, Py_ssize_t n) {
  try {
    if (n != 9 || !PyTuple_CheckExact(args[0]) || !PyTuple_CheckExact(args[1]) || !PyDict_CheckExact(args[2]))
      Py_RETURN_NONE;
    const Py_ssize_t count = PyTuple_GET_SIZE(args[0]);
    auto *shared = static_cast<const scacchi_adamw_tensor *>(PyLong_AsVoidPtr(args[3]));
    auto *settings = static_cast<const scacchi_adamw *>(PyLong_AsVoidPtr(args[4]));
    const int index = (int)PyLong_AsLong(args[5]);
    if (PyErr_Occurred() || PyTuple_GET_SIZE(args[1]) != count || index != c10::cuda::current_device()) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    std::vector<scacchi_adamw_tensor> table(shared, shared + count), given;
    Py_ssize_t found = 0;
    for (Py_ssize_t i = 0; i < count; ++i) {
      const at::Tensor *w = plain(PyTuple_GET_ITEM(args[1], i), index);
      if (!w || w->numel() != table[i].count || code_of(w->scalar_type()) != table[i].weight_dtype) Py_RETURN_NONE;
      table[i].weight = w->data_ptr();
      table[i].gradient = nullptr;
      PyObject *o = PyDict_GetItemWithError(args[2], PyTuple_GET_ITEM(args[0], i));
      if (!o) {
        if (PyErr_Occurred()) {
          PyErr_Clear();
          Py_RETURN_NONE;
        }
        continue;
      }
      ++found;
      if (o == Py_None) continue;
      const at::Tensor *t = plain(o, index);
      const int dtype = t ? code_of(t->scalar_type()) : -1;
      if (dtype < 0 || t->sizes() != w->sizes()) Py_RETURN_NONE;
      table[i].gradient = t->data_ptr();
      table[i].gradient_dtype = dtype;
    }
    if (found != PyDict_GET_SIZE(args[2])) Py_RETURN_NONE;
    scacchi_adamw params = *settings;
    at::Tensor norm;
    if (args[6] != Py_None) {
      if (!PyFloat_CheckExact(args[6])) Py_RETURN_NONE;
      params.max_norm = PyFloat_AS_DOUBLE(args[6]);
    }
    if (args[7] != Py_None) {
      const at::Tensor *t = scalar(args[7], index);
      if (!t || args[6] == Py_None) Py_RETURN_NONE;
      norm = *t;
    }
    if (PyFloat_CheckExact(args[8])) {
      params.learning_rate = PyFloat_AS_DOUBLE(args[8]);
    } else if (args[8] != Py_None) {
      const at::Tensor *t = scalar(args[8], index);
      if (!t) Py_RETURN_NONE;
      params.learning_rate_at = static_cast<const float *>(t->data_ptr());
    }
    if (args[6] != Py_None && !norm.defined()) {
      for (const scacchi_adamw_tensor &t : table)
        if (t.gradient) given.push_back(t);
      norm = norm_of(given.data(), (int32_t)given.size(), index);
      if (!norm.defined()) Py_RETURN_NONE;
    }
    params.norm = norm.defined() ? static_cast<const float *>(norm.data_ptr()) : nullptr;
    // (made before the step: nothing behind it may fail)
    PyObject *o = norm.defined() ? THPVariable_Wrap(norm) : Py_NewRef(Py_None);
    if (!o) return nullptr;
    const auto release = [](PyObject *p) { Py_XDECREF(p); };
    std::unique_ptr<PyObject, decltype(release)> tuple(PyTuple_New(1), release);
    if (!tuple) {
      Py_DECREF(o);
      return nullptr;
    }
    PyTuple_SET_ITEM(tuple.get(), 0, o);
    if (!taken(g.step(&params, table.data(), (int32_t)count, stream_of(index)), "adamw_step")) Py_RETURN_NONE;
    // a graph recorded before the step refuses to run backward through it
    for (Py_ssize_t i = 0; i < count; ++i) {
      if (!table[i].gradient) continue;
      const at::Tensor &w = THPVariable_Unpack(PyTuple_GET_ITEM(args[1], i));
      if (!w.is_inference()) w.unsafeGetTensorImpl()->bump_version();
    }
    return tuple.release();
  } catch (const Failed &) {
    return nullptr;
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// (first, second, first_exponent, second_exponent) of 8 bits -> (first, root)
PyObject *adamw_moments(PyObject *, PyObject *const *args, Py_ssize_t n) {
  try {
    const int index = c10::cuda::current_device();
    const uint8_t *at[4];
    int64_t size[4];
    if (n != 4) Py_RETURN_NONE;
    for (int i = 0; i < 4; ++i) {
      const at::Tensor *t = plain(args[i], index);
      if (!t || t->scalar_type() != at::kByte) Py_RETURN_NONE;
      at[i] = static_cast<const uint8_t *>(t->data_ptr());
      size[i] = t->numel();
    }
    if (size[1] != size[0] || size[2] != size[0] / SCACCHI_ADAMW_BLOCK || size[3] != size[2]) Py_RETURN_NONE;
    at::Tensor first = empty({size[0]}, at::kBFloat16, index), root = empty({size[0]}, at::kBFloat16, index);
    if (!taken(g.moments(at[0], at[1], at[2], at[3], size[0], first.data_ptr(), root.data_ptr(), stream_of(index)),
               "adamw_moments"))
      Py_RETURN_NONE;
    PyObject *a = THPVariable_Wrap(first), *b = a ? THPVariable_Wrap(root) : nullptr;
    PyObject *tuple = b ? PyTuple_New(2) : nullptr;
    if (!tuple) {
      Py_XDECREF(a);
      Py_XDECREF(b);
      return nullptr;
    }
    PyTuple_SET_ITEM(tuple, 0, a);
    PyTuple_SET_ITEM(tuple, 1, b);
    return tuple;
  } catch (const Failed &) {
    return nullptr;
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// (six addresses of the library's entry points, the class of errors)
PyObject *bind(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 7 || !PyExceptionClass_Check(args[6])) {
    PyErr_SetString(PyExc_TypeError, "bind takes six addresses and an exception's class");
    return nullptr;
  }
  void *at[6];
  for (int i = 0; i < 6; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind takes addresses");
      return nullptr;
    }
  }
  g.log_probs = reinterpret_cast<decltype(g.log_probs)>(at[0]);
  g.gradient = reinterpret_cast<decltype(g.gradient)>(at[1]);
  g.norm = reinterpret_cast<decltype(g.norm)>(at[2]);
  g.norm_bytes = reinterpret_cast<decltype(g.norm_bytes)>(at[3]);
  g.step = reinterpret_cast<decltype(g.step)>(at[4]);
  g.moments = reinterpret_cast<decltype(g.moments)>(at[5]);
  Py_XSETREF(g.error, Py_NewRef(args[6]));
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void *)bind, METH_FASTCALL, "The library's entry points."},
    {"log_probs", (PyCFunction)(void *)log_probs, METH_FASTCALL, "policy_log_probs of plain arguments, or None."},
    {"log_probs_gradient", (PyCFunction)(void *)log_probs_gradient, METH_FASTCALL,
     "policy_log_probs_gradient of plain arguments, or None."},
    {"gradient_norm", (PyCFunction)gradient_norm, METH_O, "gradient_norm of plain gradients, or None."},
    {"adamw_step", (PyCFunction)(void *)adamw_step, METH_FASTCALL, "AdamW.step of plain gradients, or None."},
    {"adamw_moments", (PyCFunction)(void *)adamw_moments, METH_FASTCALL, "The values of 8-bit moments, or None."},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
