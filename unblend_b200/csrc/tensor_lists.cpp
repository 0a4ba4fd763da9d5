// Checks of lists of tensors and their tables for the entry points that take many tensors at once (unblend_adamw_step,
// unblend_grad_norm), as a Python extension: a model has hundreds of parameters, and a dozen attributes of each cost 1.5
// us a tensor from Python (675 parameters: 1.0 ms, twice what the update takes on the GPU), 0.1 us from here.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <cstdint>
#include <cstring>
#include <string>
#include <vector>

#include "../../include/unblend_b200.h"

namespace {

constexpr int64_t BLOCK = 256;  // elements per block of the moments

// Raises ValueError.
PyObject* refuse(const std::string& what) {
  PyErr_SetString(PyExc_ValueError, what.c_str());
  return nullptr;
}

bool raised(const std::string& what) {
  refuse(what);
  return false;
}

std::string text(at::IntArrayRef v) {
  std::string s = "(";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + (v.size() == 1 ? ",)" : ")");
}

int type_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return UNBLEND_F32;
    case at::kBFloat16: return UNBLEND_BF16;
    case at::kHalf: return UNBLEND_F16;
    default: return -1;
  }
}

// Whether element i of the list `name` will do; raises ValueError if not. `device`: of the lists' first tensor, set by it.
bool fine(const char* name, Py_ssize_t i, PyObject* o, const at::Tensor*& out, const at::Device*& device,
          at::Device& room) {
  const auto at = [&] { return std::string(name) + "[" + std::to_string(i) + "]"; };
  if (!THPVariable_Check(o)) return raised(at() + " must be a tensor, got " + Py_TYPE(o)->tp_name);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.layout() != at::kStrided) return raised(at() + " must be a dense tensor");
  if (type_of(t) < 0)
    return raised(at() + " must be float32, bfloat16 or float16, got " + std::string(toString(t.scalar_type())));
  if (!t.is_contiguous())
    return raised(at() + " must be contiguous, got shape " + text(t.sizes()) + " with strides " + text(t.strides()));
  if (t.is_neg()) return raised(at() + " is a lazily negated view: give its resolve_neg()");
  if (device == nullptr) {
    room = t.device();
    device = &room;
  } else if (t.device() != *device) {
    return raised(at() + " is on " + t.device().str() + ", expected " + device->str() + " like the others");
  }
  out = &t;
  return true;
}

bool listed(PyObject* o) { return PyList_Check(o); }

// sizes(name, tensors) -> [number of elements of each]
PyObject* sizes(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  if (n_args != 2 || !PyUnicode_Check(args[0]) || !listed(args[1])) return refuse("sizes(name, list of tensors)");
  const char* name = PyUnicode_AsUTF8(args[0]);
  if (!name) return nullptr;
  try {
    const Py_ssize_t n = PyList_GET_SIZE(args[1]);
    PyObject* out = PyList_New(n);
    if (!out) return nullptr;
    at::Device room(at::kCPU);
    const at::Device* device = nullptr;
    for (Py_ssize_t i = 0; i < n; ++i) {
      const at::Tensor* t = nullptr;
      const bool ok = fine(name, i, PyList_GET_ITEM(args[1], i), t, device, room);
      PyObject* x = ok ? PyLong_FromLongLong(t->numel()) : nullptr;
      if (!x) {
        Py_DECREF(out);
        return nullptr;
      }
      PyList_SET_ITEM(out, i, x);
    }
    return out;
  } catch (const std::exception& e) {
    return refuse(std::string(name) + ": " + e.what());
  }
}

// table(params or None, grads) -> (table, [(type of params, type of grads, tensors), ...], blocks, grads' device index)
//
// The table holds an UnblendAdamWTensor for every gradient that is not None and has elements, sorted by the types (by the
// gradients' alone without params) and in the lists' order within them; blocks counts all params, whatever their
// gradients.
PyObject* table(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  if (n_args != 2 || !listed(args[1]) || !(args[0] == Py_None || listed(args[0]))) return refuse("table(params, grads)");
  const bool with = args[0] != Py_None;
  const Py_ssize_t n = PyList_GET_SIZE(args[1]);
  if (with && PyList_GET_SIZE(args[0]) != n)
    return refuse("params and grads must be lists of one length, got " + std::to_string(PyList_GET_SIZE(args[0])) +
                  " and " + std::to_string(n));
  try {
    std::vector<UnblendAdamWTensor> rows[9];
    at::Device room(at::kCPU);
    const at::Device* device = nullptr;
    int64_t blocks = 0;
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* go = PyList_GET_ITEM(args[1], i);
      const at::Tensor *p = nullptr, *g = nullptr;
      const int64_t first = blocks;
      if (with) {
        if (!fine("params", i, PyList_GET_ITEM(args[0], i), p, device, room)) return nullptr;
        blocks += (p->numel() + BLOCK - 1) / BLOCK;
      }
      if (go == Py_None) continue;
      if (!fine("grads", i, go, g, device, room)) return nullptr;
      if (with && p->sizes() != g->sizes())
        return refuse("grads[" + std::to_string(i) + "] must have its parameter's shape " + text(p->sizes()) + ", got " +
                      text(g->sizes()));
      if (g->numel() == 0) continue;
      UnblendAdamWTensor row;
      row.param = with ? p->data_ptr() : nullptr;
      row.grad = g->const_data_ptr();
      row.n = g->numel();
      row.block = first;
      rows[(with ? 3 * type_of(*p) : 0) + type_of(*g)].push_back(row);
    }
    size_t count = 0;
    for (const auto& r : rows) count += r.size();
    PyObject* bytes = PyBytes_FromStringAndSize(nullptr, (Py_ssize_t)(count * sizeof(UnblendAdamWTensor)));
    PyObject* kinds = PyList_New(0);
    char* to = bytes ? PyBytes_AS_STRING(bytes) : nullptr;
    bool ok = bytes && kinds;
    for (int k = 0; ok && k < 9; ++k) {
      if (rows[k].empty()) continue;
      const size_t len = rows[k].size() * sizeof(UnblendAdamWTensor);
      std::memcpy(to, rows[k].data(), len);
      to += len;
      PyObject* kind = Py_BuildValue("(iin)", k / 3, k % 3, (Py_ssize_t)rows[k].size());
      ok = kind && PyList_Append(kinds, kind) == 0;
      Py_XDECREF(kind);
    }
    if (!ok) {
      Py_XDECREF(bytes);
      Py_XDECREF(kinds);
      return nullptr;
    }
    return Py_BuildValue("(NNL)", bytes, kinds, (long long)blocks);
  } catch (const std::exception& e) {
    return refuse(std::string("params and grads: ") + e.what());
  }
}

// changed(params, grads): the parameters that have a gradient were written in place
PyObject* changed(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  if (n_args != 2 || !listed(args[0]) || !listed(args[1]) || PyList_GET_SIZE(args[0]) != PyList_GET_SIZE(args[1]))
    return refuse("changed(params, grads)");
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(args[0]); ++i) {
    PyObject* o = PyList_GET_ITEM(args[0], i);
    if (PyList_GET_ITEM(args[1], i) == Py_None || !THPVariable_Check(o)) continue;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"sizes", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(sizes)), METH_FASTCALL, nullptr},
    {"table", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(table)), METH_FASTCALL, nullptr},
    {"changed", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(changed)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "tensor_lists", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_tensor_lists() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
