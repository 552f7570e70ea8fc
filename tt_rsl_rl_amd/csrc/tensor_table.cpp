// Host code that reads torch's objects: the table of tensors that ppo_adamw_step takes, made from Python lists of tensors in one
// call, and the mark that autograd expects on tensors written behind its back.  Reading each tensor's pointer, size, type and
// device through Python's attributes takes about 2 us a tensor: 300 us for a model of 170 tensors whose step takes the GPU 15.
// A module of CPython's (tt_rsl_rl_amd._tensor_table).
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/Tensor.h>

#include <cmath>
#include <cstring>
#include <vector>

#include "../../include/ppo_hip.h"

namespace {

// A list that may be absent (None), or hold None for a tensor that is.
struct Tensors {
  const char* name;
  PyObject* fast = nullptr;
  explicit Tensors(const char* name_) : name(name_) {}
  ~Tensors() { Py_XDECREF(fast); }
  Tensors(const Tensors&) = delete;
  Tensors& operator=(const Tensors&) = delete;

  bool take(PyObject* list, Py_ssize_t n, bool optional) {
    if (optional && list == Py_None) return true;
    fast = PySequence_Fast(list, "adamw_step: lists of tensors");
    if (fast == nullptr) return false;
    const Py_ssize_t have = PySequence_Fast_GET_SIZE(fast);
    if (n >= 0 && have != n) {
      PyErr_Format(PyExc_ValueError, "adamw_step: %zd %s for %zd params", have, name, n);
      return false;
    }
    return true;
  }
  // The i-th tensor; null without one, or with an error set.
  const at::Tensor* at(Py_ssize_t i, bool optional) const {
    PyObject* item = fast == nullptr ? Py_None : PySequence_Fast_GET_ITEM(fast, i);
    if (THPVariable_Check(item)) return &THPVariable_Unpack(item);
    if (!(optional && item == Py_None)) PyErr_Format(PyExc_ValueError, "adamw_step: %s[%zd] must be a tensor", name, i);
    return nullptr;
  }
};

// A number, or one for each tensor.
struct Numbers {
  const char* name;
  PyObject* fast = nullptr;
  double one = 0.0;
  explicit Numbers(const char* name_) : name(name_) {}
  ~Numbers() { Py_XDECREF(fast); }
  Numbers(const Numbers&) = delete;
  Numbers& operator=(const Numbers&) = delete;

  bool take(PyObject* x, Py_ssize_t n) {
    if (!PyList_Check(x) && !PyTuple_Check(x)) {
      one = PyFloat_AsDouble(x);
      return !(one == -1.0 && PyErr_Occurred());
    }
    fast = PySequence_Fast(x, "adamw_step: numbers");
    if (fast == nullptr) return false;
    if (PySequence_Fast_GET_SIZE(fast) != n) {
      PyErr_Format(PyExc_ValueError, "adamw_step: %zd %s for %zd params", PySequence_Fast_GET_SIZE(fast), name, n);
      return false;
    }
    return true;
  }
  bool at(Py_ssize_t i, double& x) const {
    x = fast == nullptr ? one : PyFloat_AsDouble(PySequence_Fast_GET_ITEM(fast, i));
    return !(fast != nullptr && x == -1.0 && PyErr_Occurred());
  }
};

bool fits(const at::Tensor& t, const char* name, Py_ssize_t i, int64_t count, int device) {
  if (t.layout() == at::kStrided && t.is_cuda() && t.get_device() == device && t.numel() == count && t.is_contiguous()) return true;
  PyErr_Format(PyExc_ValueError,
               "adamw_step: %s[%zd] must be contiguous, of %lld elements, on the current GPU (%d; no CPU path exists): it has %lld on %s",
               name, i, static_cast<long long>(count), device, static_cast<long long>(t.numel()), t.device().str().c_str());
  return false;
}

int type_of(at::ScalarType t) { return t == at::kFloat ? PPO_TYPE_F32 : t == at::kBFloat16 ? PPO_TYPE_BF16 : -1; }

bool entry(const Tensors (&lists)[7], const Numbers& lr, const Numbers& weight_decay, Py_ssize_t i, int device, ppo_adamw_tensor& e) {
  const at::Tensor* t[7];
  for (int k = 0; k < 7; ++k) {
    t[k] = lists[k].at(i, k == 2 || k >= 5);
    if (PyErr_Occurred()) return false;
  }
  const int64_t count = t[0]->numel(), blocks = (count + PPO_ADAMW_BLOCK - 1) / PPO_ADAMW_BLOCK;
  for (int k = 0; k < 7; ++k)
    if (t[k] != nullptr && !fits(*t[k], lists[k].name, i, k >= 5 ? blocks : count, device)) return false;
  const at::ScalarType p = t[0]->scalar_type(), g = t[1]->scalar_type(), m = t[3]->scalar_type(), v = t[4]->scalar_type();
  if (type_of(p) < 0 || (g != at::kFloat && g != p)) {
    PyErr_Format(PyExc_ValueError, "adamw_step: tensor %zd: parameter %s, gradient %s", i, at::toString(p), at::toString(g));
    return false;
  }
  if (t[2] != nullptr && (t[2]->scalar_type() != at::kFloat || p != at::kBFloat16)) {
    PyErr_Format(PyExc_ValueError, "adamw_step: masters[%zd] must be float32, of a bfloat16 parameter", i);
    return false;
  }
  const bool wide = m == at::kFloat && v == at::kFloat;
  if (!wide && !(m == at::kChar && v == at::kByte && t[5] != nullptr && t[6] != nullptr && t[5]->scalar_type() == at::kFloat &&
                 t[6]->scalar_type() == at::kFloat)) {
    PyErr_Format(PyExc_ValueError, "adamw_step: tensor %zd: states %s, %s (float32, or int8 and uint8 with float32 scales)", i,
                 at::toString(m), at::toString(v));
    return false;
  }
  auto data = [](const at::Tensor* x) { return x == nullptr ? nullptr : x->data_ptr(); };
  e = ppo_adamw_tensor{};
  e.param = data(t[0]);
  e.grad = data(t[1]);
  e.master = static_cast<float*>(data(t[2]));
  e.exp_avg = data(t[3]);
  e.exp_avg_sq = data(t[4]);
  e.m_scale = static_cast<float*>(data(t[5]));
  e.v_scale = static_cast<float*>(data(t[6]));
  e.count = count;
  e.param_type = type_of(p);
  e.grad_type = type_of(g);
  e.state_bits = wide ? 32 : 8;
  return lr.at(i, e.lr) && weight_decay.at(i, e.weight_decay);
}

// Whether a parameter comes a second time: two blocks would step it at once.  An open hash table of twice as many places or more.
struct Seen {
  std::vector<const void*> places;
  explicit Seen(Py_ssize_t n) {
    size_t size = 2;
    while (size < 2 * static_cast<size_t>(n)) size *= 2;
    places.resize(size);
  }
  bool again(const void* p) {
    size_t at = (reinterpret_cast<uintptr_t>(p) >> 4) * 0x9e3779b97f4a7c15u >> 20;
    for (;; ++at) {
      const void*& place = places[at & (places.size() - 1)];
      if (place == p) return true;
      if (place == nullptr) {
        place = p;
        return false;
      }
    }
  }
};

// adamw_table(params, grads, masters, exp_avg, exp_avg_sq, m_scales, v_scales, step, lr, weight_decay, beta1, beta2, dither, device)
// -> bytes
PyObject* adamw_table(PyObject*, PyObject* const* args, Py_ssize_t num) {
  if (num != 14) return PyErr_Format(PyExc_TypeError, "adamw_table: 14 arguments, got %zd", num);
  try {
    Tensors lists[7] = {Tensors("params"), Tensors("grads"), Tensors("masters"), Tensors("exp_avg"), Tensors("exp_avg_sq"),
                        Tensors("scales"), Tensors("scales")};
    Numbers step("step"), lr("lr"), weight_decay("weight_decay");
    Py_ssize_t n = -1;
    for (int k = 0; k < 7; ++k) {
      if (!lists[k].take(args[k], n, k == 2 || k >= 5)) return nullptr;
      if (k == 0) n = PySequence_Fast_GET_SIZE(lists[0].fast);
    }
    if (!step.take(args[7], n) || !lr.take(args[8], n) || !weight_decay.take(args[9], n)) return nullptr;
    const double beta1 = PyFloat_AsDouble(args[10]), beta2 = PyFloat_AsDouble(args[11]);
    const int dither = PyObject_IsTrue(args[12]);
    const long device = PyLong_AsLong(args[13]);
    if (PyErr_Occurred()) return nullptr;
    Seen seen(n);
    PyObject* out = PyBytes_FromStringAndSize(nullptr, n * static_cast<Py_ssize_t>(sizeof(ppo_adamw_tensor)));
    if (out == nullptr) return nullptr;
    auto* e = reinterpret_cast<ppo_adamw_tensor*>(PyBytes_AS_STRING(out));
    double last = 0.0, bc1 = 0.0, bc2_sqrt = 0.0;  // (0 is no step)
    for (Py_ssize_t i = 0; i < n; ++i) {
      double s = 0.0;
      bool ok = step.at(i, s);
      if (ok && !(s >= 1.0)) {
        PyErr_Format(PyExc_ValueError, "adamw_step: step of tensor %zd must be 1 or more", i);
        ok = false;
      }
      ppo_adamw_tensor x;
      if (!ok || !entry(lists, lr, weight_decay, i, static_cast<int>(device), x)) {
        Py_DECREF(out);
        return nullptr;
      }
      if (x.count > 0 && seen.again(x.param)) {
        PyErr_Format(PyExc_ValueError, "adamw_step: params[%zd] comes a second time", i);
        Py_DECREF(out);
        return nullptr;
      }
      if (s != last) {
        last = s;
        bc1 = 1.0 - std::pow(beta1, s);
        bc2_sqrt = std::sqrt(1.0 - std::pow(beta2, s));
      }
      x.dither = dither != 0 && x.state_bits == 8 ? static_cast<int64_t>(std::fmin(s, 0x1p62)) : 0;
      x.bc1 = bc1;
      x.bc2_sqrt = bc2_sqrt;
      std::memcpy(e + i, &x, sizeof(x));
    }
    return out;
  } catch (const std::exception& ex) {  // none may leave a C entry
    return PyErr_Format(PyExc_RuntimeError, "adamw_step: %s", ex.what());
  }
}

// A tensor, or None; false for anything else.
bool mark(PyObject* x) {
  if (x == Py_None) return true;
  if (!THPVariable_Check(x)) return false;
  const at::Tensor& t = THPVariable_Unpack(x);
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();  // (an inference tensor has no counter, and autograd none of it)
  return true;
}

bool mark_all(PyObject* x) {
  if (mark(x)) return true;
  Tensors list("");
  if (!list.take(x, -1, false)) return false;
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(list.fast); ++i)
    if (!mark(PySequence_Fast_GET_ITEM(list.fast, i))) {
      PyErr_SetString(PyExc_TypeError, "written: tensors or sequences of them");
      return false;
    }
  return true;
}

// written(*tensors): their version counters go up, as by torch's own in-place operations, so that a backward pass which has kept
// one of them for itself says so instead of using what was written since.
PyObject* written(PyObject*, PyObject* const* args, Py_ssize_t num) {
  try {
    for (Py_ssize_t i = 0; i < num; ++i)
      if (!mark_all(args[i])) return nullptr;
  } catch (const std::exception& ex) {
    return PyErr_Format(PyExc_RuntimeError, "written: %s", ex.what());
  }
  Py_RETURN_NONE;
}

// Whether x is a tensor of the GPU `device`, laid out by strides.
const at::Tensor* on_gpu(PyObject* x, int64_t device) {
  if (!THPVariable_Check(x)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(x);
  return t.layout() == at::kStrided && t.is_cuda() && t.get_device() == device ? &t : nullptr;
}

// head_views(device, tensor, tokens, heads, elements, ...): the bytes of their ppo_head_views, or None unless all are of those shapes, of the first one's
// type, of unit stride in their elements and on the device: then the caller's own checks say what is wrong.
PyObject* head_views(PyObject*, PyObject* const* args, Py_ssize_t num) {
  try {
    constexpr Py_ssize_t most = 8;
    ppo_head_view views[most];
    const Py_ssize_t n = (num - 1) / 4;
    if (n < 1 || n > most || num != 1 + 4 * n) return PyErr_Format(PyExc_TypeError, "head_views: a device and up to 8 tensors with their sizes");
    const int64_t device = PyLong_AsLongLong(args[0]);
    at::ScalarType type{};
    for (Py_ssize_t i = 0; i < n; ++i) {
      const at::Tensor* t = on_gpu(args[1 + 4 * i], device);
      if (t == nullptr || t->dim() != 3 || (i > 0 && t->scalar_type() != type)) Py_RETURN_NONE;
      type = t->scalar_type();
      for (int k = 0; k < 3; ++k)
        if (t->size(k) != PyLong_AsLongLong(args[2 + 4 * i + k])) Py_RETURN_NONE;
      if (t->stride(2) != 1 && t->size(2) > 1) Py_RETURN_NONE;
      views[i] = ppo_head_view{t->data_ptr(), t->stride(0), t->stride(1)};
    }
    if (PyErr_Occurred()) return nullptr;
    return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(views), n * static_cast<Py_ssize_t>(sizeof(ppo_head_view)));
  } catch (const std::exception& ex) {
    return PyErr_Format(PyExc_RuntimeError, "head_views: %s", ex.what());
  }
}

// addresses(device, tensor, elements, ...): their addresses (0 for None), or None unless all are contiguous, of so many elements and on the device.
PyObject* addresses(PyObject*, PyObject* const* args, Py_ssize_t num) {
  try {
    constexpr Py_ssize_t most = 8;
    const Py_ssize_t n = (num - 1) / 2;
    if (n < 1 || n > most || num != 1 + 2 * n) return PyErr_Format(PyExc_TypeError, "addresses: a device and up to 8 tensors with their sizes");
    const int64_t device = PyLong_AsLongLong(args[0]);
    void* at[most];
    for (Py_ssize_t i = 0; i < n; ++i) {
      at[i] = nullptr;
      if (args[1 + 2 * i] == Py_None) continue;
      const at::Tensor* t = on_gpu(args[1 + 2 * i], device);
      if (t == nullptr || !t->is_contiguous() || t->numel() != PyLong_AsLongLong(args[2 + 2 * i])) Py_RETURN_NONE;
      at[i] = t->data_ptr();
    }
    if (PyErr_Occurred()) return nullptr;
    PyObject* out = PyTuple_New(n);
    for (Py_ssize_t i = 0; out != nullptr && i < n; ++i) {
      PyObject* x = PyLong_FromVoidPtr(at[i]);
      if (x == nullptr) {
        Py_DECREF(out);
        return nullptr;
      }
      PyTuple_SET_ITEM(out, i, x);
    }
    return out;
  } catch (const std::exception& ex) {
    return PyErr_Format(PyExc_RuntimeError, "addresses: %s", ex.what());
  }
}

PyMethodDef methods[] = {{"adamw_table", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(adamw_table)), METH_FASTCALL,
                          "The bytes of ppo_adamw_step's table (ops.adamw_step)."},
                         {"head_views", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(head_views)), METH_FASTCALL,
                          "The bytes of tensors' ppo_head_views, or None where one is not as it should be."},
                         {"addresses", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(addresses)), METH_FASTCALL,
                          "Contiguous tensors' addresses, or None where one is not as it should be."},
                         {"written", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(written)), METH_FASTCALL,
                          "Raises the version counters of tensors and of sequences of them; None is skipped."},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_table", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_table() { return PyModule_Create(&module); }
