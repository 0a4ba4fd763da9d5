// The host side of operators whose arguments take longer to check from Python than the GPU takes to work on them, as a Python
// extension. Lists of tensors (unblend_adamw_step, unblend_grad_norm): a model has hundreds of parameters, and a dozen
// attributes of each cost 1.5 us a tensor from Python (675 parameters: 1.0 ms, twice the update's time on the GPU), 0.05 us
// from here. Heads of queries and keys (the rotary operators): the checks, outputs and parameters of a call.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <cstdint>
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include "../../include/unblend_b200.h"

namespace {

constexpr int64_t BLOCK = 256, RUN = 1024;  // elements per block of the moments, and per run of the norm

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

PyObject* wrap(const at::Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}

// The interpreter is free meanwhile: an allocation can wait for the GPU.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

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
  HANDLE_TH_ERRORS  // torch's exceptions as Python's: out of memory stays what it is
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
  END_HANDLE_TH_ERRORS
}

// table(params or None, grads) -> (table, [(type of params, type of grads, tensors), ...], blocks, runs)
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
  HANDLE_TH_ERRORS
  std::vector<UnblendAdamWTensor> rows[9];
  at::Device room(at::kCPU);
  const at::Device* device = nullptr;
  int64_t blocks = 0, runs = 0;
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
    runs += (row.n + RUN - 1) / RUN;
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
  return Py_BuildValue("(NNLL)", bytes, kinds, (long long)blocks, (long long)runs);
  END_HANDLE_TH_ERRORS
}

// norm_outputs(like, with scale, bytes) -> (norm, scale or None, workspace) on like's device
PyObject* norm_outputs(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  if (n_args != 3 || !THPVariable_Check(args[0])) return refuse("norm_outputs(like, with scale, bytes)");
  const long long bytes = PyLong_AsLongLong(args[2]);
  if (bytes < 0) return PyErr_Occurred() ? nullptr : refuse("norm_outputs: bytes below 0");
  HANDLE_TH_ERRORS
  const at::TensorOptions options = at::TensorOptions().device(THPVariable_Unpack(args[0]).device());
  at::Tensor norm, scale, work;
  {
    const Unlocked unlocked;
    norm = at::empty({}, options.dtype(at::kFloat));
    if (args[1] == Py_True) scale = at::empty({}, options.dtype(at::kFloat));
    work = at::empty({bytes}, options.dtype(at::kByte));
  }
  return Py_BuildValue("(NNN)", wrap(norm), wrap(scale), wrap(work));
  END_HANDLE_TH_ERRORS
}

// Whether x is a number in [low, high); its value.
bool number(const char* name, PyObject* x, double low, double high, double& value) {
  if (!PyBool_Check(x) && (PyFloat_Check(x) || PyLong_Check(x))) {
    value = PyFloat_AsDouble(x);
    if (value >= low && value < high) return true;
    PyErr_Clear();  // an integer beyond all floats
  }
  char range[64];
  std::snprintf(range, sizeof range, " must be a number in [%g, %g), got ", low, high);
  PyObject* shown = PyObject_Repr(x);
  if (!shown) return false;
  const char* got = PyUnicode_AsUTF8(shown);
  if (got) refuse(std::string(name) + range + got);
  Py_DECREF(shown);
  return false;
}

// Whether o is a tensor of one element on `device`.
bool scalar_ok(const char* name, PyObject* o, at::ScalarType type, const at::Device& device) {
  if (THPVariable_Check(o)) {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.scalar_type() == type && t.device() == device && t.layout() == at::kStrided && t.numel() == 1 && !t.is_neg())
      return true;
  }
  return raised(std::string(name) + " must be a " + (type == at::kLong ? "int64" : "float32") +
                " tensor of one element on " + device.str());
}

// Memory from one address up to another, which is above it where two are compared.
struct Span {
  uintptr_t from, to;
  bool meets(const Span& o) const { return (from < o.to) & (o.from < to); }
};

Span span_of(const at::Tensor& t) {  // of a contiguous tensor
  const uintptr_t at = reinterpret_cast<uintptr_t>(t.const_data_ptr());
  return Span{at, at + (uintptr_t)t.numel() * t.element_size()};
}

// The blocks of a state's moments; -1 after a ValueError.
int64_t state_blocks(PyObject* const* o) {
  const bool eight = o[2] != Py_None;
  static const char* const names[2] = {"exp_avg", "exp_avg_sq"};
  for (int i = 0; i < 2; ++i) {
    const at::Tensor* t = THPVariable_Check(o[i]) ? &THPVariable_Unpack(o[i]) : nullptr;
    if (!t || t->layout() != at::kStrided || t->scalar_type() != (eight ? at::kByte : at::kFloat) || t->dim() != 1 ||
        t->numel() % BLOCK || !t->is_contiguous() || t->is_neg() ||
        reinterpret_cast<uintptr_t>(t->const_data_ptr()) % 16) {
      refuse(std::string("state.") + names[i] + " must be contiguous " + (eight ? "uint8" : "float32") +
             " from a 16-byte boundary on, whole blocks of " + std::to_string(BLOCK) +
             (eight ? " (with scales)" : " (without scales)"));
      return -1;
    }
  }
  const at::Tensor &m = THPVariable_Unpack(o[0]), &v = THPVariable_Unpack(o[1]);
  const int64_t blocks = m.numel() / BLOCK;
  if (m.numel() != v.numel() || m.device() != v.device()) {
    refuse("state.exp_avg and state.exp_avg_sq must have one shape and device");
    return -1;
  }
  if (blocks && span_of(m).meets(span_of(v))) {
    refuse("state.exp_avg and state.exp_avg_sq must not share memory");
    return -1;
  }
  if (eight) {
    const at::Tensor* t = THPVariable_Check(o[2]) ? &THPVariable_Unpack(o[2]) : nullptr;
    if (!t || t->layout() != at::kStrided || t->scalar_type() != at::kFloat || t->dim() != 2 || t->size(0) != blocks ||
        t->size(1) != 2 || !t->is_contiguous() || t->is_neg() || t->device() != m.device() ||
        reinterpret_cast<uintptr_t>(t->const_data_ptr()) % 8) {
      refuse("state.scales must be contiguous float32 (" + std::to_string(blocks) + ", 2) on " + m.device().str());
      return -1;
    }
    if (blocks && (span_of(*t).meets(span_of(m)) || span_of(*t).meets(span_of(v)))) {
      refuse("state.scales must not share memory with the moments");
      return -1;
    }
  }
  return blocks;
}

// state(exp_avg, exp_avg_sq, scales or None) -> blocks
PyObject* state(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  if (n_args != 3) return refuse("state(exp_avg, exp_avg_sq, scales)");
  HANDLE_TH_ERRORS
  const int64_t blocks = state_blocks(args);
  return blocks < 0 ? nullptr : PyLong_FromLongLong(blocks);
  END_HANDLE_TH_ERRORS
}

// Whether a step's tensors, the state and the numbers on the device (null: not given) share no memory: the state with any
// tensor, a parameter or the state with a number. Parameters and gradients among themselves are left to the entry point.
bool state_apart(PyObject* table, PyObject* kinds, PyObject* const* state, const UnblendAdamWParams& p) {
  static const uintptr_t SIZE[3] = {4, 2, 2};  // by UnblendDtype
  static_assert(UNBLEND_F32 == 0 && UNBLEND_BF16 < 3 && UNBLEND_F16 < 3, "SIZE");
  Span held[3], number[3];
  int n_held = 0, n_number = 0;
  for (int i = 0; i < 3; ++i)
    if (state[i] != Py_None) held[n_held++] = span_of(THPVariable_Unpack(state[i]));
  if (held[0].from == held[0].to) return true;  // nothing is written
  const auto add = [&](const void* x, uintptr_t bytes) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x);
    if (a) number[n_number++] = Span{a, a + bytes};
  };
  add(p.step_device, sizeof(long long));
  add(p.lr_device, sizeof(float));
  add(p.grad_scale, sizeof(float));
  for (int i = 0; i < n_number; ++i)
    for (int j = 0; j < n_held; ++j)
      if (number[i].meets(held[j])) return raised("step, lr and grad_scale must not share memory with the state");
  const char* row_at = PyBytes_AS_STRING(table);
  for (Py_ssize_t k = 0; k < PyList_GET_SIZE(kinds); ++k) {
    PyObject* const kind = PyList_GET_ITEM(kinds, k);
    const long types[2] = {PyLong_AsLong(PyTuple_GET_ITEM(kind, 0)), PyLong_AsLong(PyTuple_GET_ITEM(kind, 1))};
    const Py_ssize_t n = PyLong_AsSsize_t(PyTuple_GET_ITEM(kind, 2));
    for (Py_ssize_t i = 0; i < n; ++i, row_at += sizeof(UnblendAdamWTensor)) {
      UnblendAdamWTensor row;
      std::memcpy(&row, row_at, sizeof row);
      const uintptr_t w = reinterpret_cast<uintptr_t>(row.param), g = reinterpret_cast<uintptr_t>(row.grad);
      const Span param{w, w + (uintptr_t)row.n * SIZE[types[0]]}, grad{g, g + (uintptr_t)row.n * SIZE[types[1]]};
      bool meet = false, meet_number = false;
      for (int j = 0; j < n_held; ++j) meet |= param.meets(held[j]) | grad.meets(held[j]);
      for (int j = 0; j < n_number; ++j) meet_number |= param.meets(number[j]);
      if (meet) return raised("params and grads must not share memory with the state");
      if (meet_number) return raised("step, lr and grad_scale must not share memory with params");
    }
  }
  return true;
}

// adamw(params, grads, exp_avg, exp_avg_sq, scales, step, lr, beta1, beta2, eps, weight_decay, grad_scale)
//   -> (table, kinds, UnblendAdamWParams, addresses of the state's tensors)
PyObject* adamw(PyObject* self, PyObject* const* args, Py_ssize_t n_args) {
  if (n_args != 12) return refuse("adamw: wrong number of arguments");
  HANDLE_TH_ERRORS
  PyObject* got = table(self, args, 2);
  if (!got) return nullptr;
  const auto fail = [&] {
    Py_DECREF(got);
    return nullptr;
  };
  if (PyList_GET_SIZE(args[0]) == 0) {
    refuse("params must hold at least one tensor");
    return fail();
  }
  const at::Device device = THPVariable_Unpack(PyList_GET_ITEM(args[0], 0)).device();
  const int64_t have = state_blocks(args + 2), want = PyLong_AsLongLong(PyTuple_GET_ITEM(got, 2));
  if (have < 0) return fail();
  if (have != want) {
    refuse("state holds " + std::to_string(have) + " blocks of " + std::to_string(BLOCK) + " moments, params need " +
           std::to_string(want));
    return fail();
  }
  const at::Tensor& m = THPVariable_Unpack(args[2]);
  if (m.device() != device) {
    refuse("state is on " + m.device().str() + ", expected " + device.str());
    return fail();
  }
  UnblendAdamWParams p{};
  if (!number("betas[0]", args[7], 0, 1, p.beta1) || !number("betas[1]", args[8], 0, 1, p.beta2) ||
      !number("eps", args[9], 0, 1e30, p.eps) || !number("weight_decay", args[10], 0, 1e18, p.weight_decay))
    return fail();
  if (p.eps > 0 && p.eps < 1.17549435e-38) {
    refuse("eps must be 0 or a normal float32");
    return fail();
  }
  PyObject* const step = args[5];
  if (THPVariable_Check(step)) {
    if (!scalar_ok("step", step, at::kLong, device)) return fail();
    p.step_device = static_cast<const long long*>(THPVariable_Unpack(step).const_data_ptr());
  } else {
    p.step = PyLong_Check(step) && !PyBool_Check(step) ? PyLong_AsLongLong(step) : 0;
    PyErr_Clear();
    if (p.step < 1) {
      refuse("step must be the update's number from 1 on, an int or an int64 tensor");
      return fail();
    }
  }
  if (THPVariable_Check(args[6])) {
    if (!scalar_ok("lr", args[6], at::kFloat, device)) return fail();
    p.lr_device = THPVariable_Unpack(args[6]).const_data_ptr<float>();
  } else if (!number("lr", args[6], 0, 1e18, p.lr)) {
    return fail();
  }
  if (args[11] != Py_None) {
    if (!scalar_ok("grad_scale", args[11], at::kFloat, device)) return fail();
    p.grad_scale = THPVariable_Unpack(args[11]).const_data_ptr<float>();
  }
  if (!state_apart(PyTuple_GET_ITEM(got, 0), PyTuple_GET_ITEM(got, 1), args + 2, p)) return fail();
  const auto address = [](PyObject* o) {
    return o == Py_None ? 0LL : (long long)reinterpret_cast<uintptr_t>(THPVariable_Unpack(o).const_data_ptr());
  };
  PyObject* out = Py_BuildValue("(OOy#(LLL))", PyTuple_GET_ITEM(got, 0), PyTuple_GET_ITEM(got, 1),
                                reinterpret_cast<const char*>(&p), (Py_ssize_t)sizeof(p), address(args[2]),
                                address(args[3]), address(args[4]));
  Py_DECREF(got);
  return out;
  END_HANDLE_TH_ERRORS
}

// changed(params, grads, state): the parameters that have a gradient, and the state's tensors, were written in place
PyObject* changed(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  if (n_args != 3 || !listed(args[0]) || !listed(args[1]) || PyList_GET_SIZE(args[0]) != PyList_GET_SIZE(args[1]) ||
      !PyTuple_Check(args[2]))
    return refuse("changed(params, grads, state)");
  const auto bump = [](PyObject* o) {
    if (!THPVariable_Check(o)) return;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  };
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(args[0]); ++i)
    if (PyList_GET_ITEM(args[1], i) != Py_None) bump(PyList_GET_ITEM(args[0], i));
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[2]); ++i) bump(PyTuple_GET_ITEM(args[2], i));
  Py_RETURN_NONE;
}

// ------------------------------------------------------------------------------------------ heads of queries and keys

constexpr int64_t MAX_HD = 256, MOST_ROWS = INT64_C(1) << 31;
constexpr double F32_MAX = 3.4028234663852886e38;

const at::Tensor* tensor(PyObject* o) { return o == Py_None ? nullptr : &THPVariable_Unpack(o); }

std::string shape(const at::Tensor& t) { return text(t.sizes()); }

// A tensor of one of the three types; `like`: on its device.
bool element_ok(const char* name, PyObject* o, const at::Tensor* like) {
  const std::string n(name);
  if (!THPVariable_Check(o)) return raised(n + " must be a tensor, got " + Py_TYPE(o)->tp_name);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.layout() != at::kStrided) return raised(n + " must be a dense tensor");
  if (type_of(t) < 0)
    return raised(n + " must be float32, bfloat16 or float16, got " + std::string(toString(t.scalar_type())));
  if (t.is_neg()) return raised(n + " is a lazily negated view: give " + n + ".resolve_neg()");
  if (like && t.device() != like->device())
    return raised(n + " is on " + t.device().str() + ", expected " + like->device().str());
  return true;
}

bool heads_ok(const char* name, PyObject* o, const at::Tensor* q) {
  if (!element_ok(name, o, q)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.dim() != 4 && t.dim() != 5)
    return raised(std::string(name) +
                  " must be [batch, length, heads, head_dim] or [outer, inner, length, heads, head_dim], got shape " +
                  shape(t));
  if (q && t.scalar_type() != q->scalar_type())
    return raised(std::string(name) + " must be of q's type " + std::string(toString(q->scalar_type())) + ", got " +
                  std::string(toString(t.scalar_type())));
  return true;
}

bool weight_ok(const char* name, PyObject* o, const at::Tensor& q) {
  if (!element_ok(name, o, &q)) return false;
  const at::Tensor& w = THPVariable_Unpack(o);
  if (w.scalar_type() != at::kFloat && w.scalar_type() != q.scalar_type())
    return raised(std::string(name) + " must be float32 or of its input's type, got " +
                  std::string(toString(w.scalar_type())));
  if (w.dim() != 1 || w.size(0) != q.size(-1))
    return raised(std::string(name) + " must have shape (" + std::to_string(q.size(-1)) + ",), got " + shape(w));
  return true;
}

bool is_number(PyObject* o) { return PyFloat_Check(o) || PyLong_Check(o); }

// Arguments of a call, in this order.
enum Arg { Q, K, GAMMA_Q, GAMMA_K, FREQS, POSITIONS, INTERLEAVED, SCALE, EPS, LENS, N_ARGS };

struct Call {
  const at::Tensor *q, *k, *gamma[2], *freqs, *positions, *lens;
  bool half;
  double scale, eps;
};

bool read(PyObject* const* o, const char* const (&names)[2], Call& c) {
  if (!heads_ok(names[0], o[Q], nullptr)) return false;
  c.q = tensor(o[Q]), c.k = nullptr;
  const at::Tensor& q = *c.q;
  const int64_t dims = q.dim(), hd = q.size(-1);
  if (o[K] != Py_None) {
    if (!heads_ok(names[1], o[K], c.q)) return false;
    c.k = tensor(o[K]);
    if (c.k->dim() != dims || c.k->size(-1) != hd || c.k->sizes().slice(0, dims - 2) != q.sizes().slice(0, dims - 2))
      return raised("q " + shape(q) + " and k " + shape(*c.k) + " must agree but for their heads");
  }
  if (hd < 1 || hd > MAX_HD)
    return raised("head_dim must be 1 to " + std::to_string(MAX_HD) + ", got " + std::to_string(hd));
  c.freqs = c.positions = c.lens = nullptr;
  if (o[FREQS] != Py_None) {
    c.freqs = THPVariable_Check(o[FREQS]) ? tensor(o[FREQS]) : nullptr;
    if (!c.freqs || c.freqs->layout() != at::kStrided ||
        (c.freqs->scalar_type() != at::kFloat && c.freqs->scalar_type() != at::kDouble) || c.freqs->dim() != 1 ||
        c.freqs->device() != q.device())
      return raised("freqs must be a float32 or float64 tensor [pairs] on " + q.device().str());
    if (2 * c.freqs->numel() > hd)
      return raised(std::to_string(c.freqs->numel()) + " pairs do not fit into head_dim " + std::to_string(hd));
    if (c.freqs->is_neg()) return raised("freqs is a lazily negated view: give freqs.resolve_neg()");
    if (c.freqs->requires_grad() && at::GradMode::is_enabled())
      return raised("freqs has no gradient here: give freqs.detach()");
  }
  if (o[POSITIONS] != Py_None) {
    c.positions = THPVariable_Check(o[POSITIONS]) ? tensor(o[POSITIONS]) : nullptr;
    if (!c.positions || c.positions->layout() != at::kStrided ||
        (c.positions->scalar_type() != at::kInt && c.positions->scalar_type() != at::kLong) ||
        c.positions->device() != q.device())
      return raised("positions must be an int32 or int64 tensor on " + q.device().str());
    const auto all = q.sizes().slice(0, dims - 2), row = q.sizes().slice(dims - 3, 1);
    if (c.positions->sizes() != all && c.positions->sizes() != row)
      return raised("positions must have shape " + text(row) + " or " + text(all) + ", got " + shape(*c.positions));
  }
  if (!is_number(o[EPS]) || !((c.eps = PyFloat_AsDouble(o[EPS])) >= 0 && c.eps <= F32_MAX)) {
    PyErr_Clear();
    return raised("eps must be >= 0");
  }
  if (THPVariable_Check(o[SCALE]) && THPVariable_Unpack(o[SCALE]).numel() != 1)
    return raised("scale must be a number, got a tensor of shape " + shape(THPVariable_Unpack(o[SCALE])));
  c.scale = PyFloat_AsDouble(o[SCALE]);
  if (c.scale == -1.0 && PyErr_Occurred()) {
    if (!PyErr_ExceptionMatches(PyExc_TypeError) && !PyErr_ExceptionMatches(PyExc_OverflowError)) return false;
    PyErr_Clear();
    return raised(std::string("scale must be a number that fp32 holds, got ") + Py_TYPE(o[SCALE])->tp_name);
  }
  if (!(c.scale >= -F32_MAX && c.scale <= F32_MAX))
    return raised("scale must be finite in float32, got " + std::to_string(c.scale));
  if (q.numel() >= MOST_ROWS * hd || (c.k && c.k->numel() >= MOST_ROWS * hd))
    return raised("q and k must have fewer than 2^31 rows each, got shapes " + shape(q) +
                  (c.k ? " and " + shape(*c.k) : ""));
  static const char* const weights[2] = {"gamma_q", "gamma_k"};
  for (int i = 0; i < 2; ++i) {
    c.gamma[i] = nullptr;
    if (o[GAMMA_Q + i] == Py_None) continue;
    if (!weight_ok(weights[i], o[GAMMA_Q + i], q)) return false;
    c.gamma[i] = tensor(o[GAMMA_Q + i]);
  }
  if (c.gamma[1] && !c.k) return raised("gamma_k needs k");
  if (c.gamma[0] && c.gamma[1] && c.gamma[0]->scalar_type() != c.gamma[1]->scalar_type())
    return raised("gamma_q and gamma_k must share a type");
  if (o[LENS] != Py_None) {
    c.lens = THPVariable_Check(o[LENS]) ? tensor(o[LENS]) : nullptr;
    const int64_t seqs = q.size(0) * (dims == 5 ? q.size(1) : 1);
    if (!c.lens || c.lens->layout() != at::kStrided || c.lens->scalar_type() != at::kInt ||
        c.lens->device() != q.device())
      return raised("lens must be an int32 tensor on " + q.device().str());
    if (c.lens->numel() != seqs)
      return raised("lens must hold one length for each of " + std::to_string(seqs) + " sequences, got " +
                    std::to_string(c.lens->numel()));
  }
  const int truth = PyObject_IsTrue(o[INTERLEAVED]);
  if (truth < 0) return false;
  c.half = !truth;
  return true;
}

// A tensor as the kernels take it: unit last stride.
at::Tensor unit(const at::Tensor& t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

UnblendHeadStrides strides(const at::Tensor& t) {
  const int64_t d = t.dim();
  return UnblendHeadStrides{t.stride(0), d == 5 ? t.stride(1) : 0, t.stride(d - 3), t.stride(d - 2)};
}

long long pointer(const at::Tensor& t) { return (long long)reinterpret_cast<uintptr_t>(t.const_data_ptr()); }

// heads(q, k, gamma_q, gamma_k, freqs, positions, interleaved, scale, eps, lens[, q0, k0, weights, workspace])
//   -> None for a side without elements or tensors off the GPU, after the checks; else
//      (q_out, k_out, dgamma_q, dgamma_k, addresses for the entry point, UnblendRotaryParams, tensors that these point to)
//
// With q0 and k0, q and k are the gradients of the norm's outputs for those inputs; weights: whether gradients of gamma_q and
// gamma_k are wanted; workspace: address of unblend_qk_norm_rotary_grad_workspace.
PyObject* heads(PyObject*, PyObject* const* o, Py_ssize_t n_args) {
  if (n_args != N_ARGS && n_args != N_ARGS + 4) return refuse("heads: wrong number of arguments");
  HANDLE_TH_ERRORS
  Call c;
  const bool backward = n_args > N_ARGS;
  const char* const names[2] = {backward ? "dq" : "q", backward ? "dk" : "k"};
  if (!read(o, names, c)) return nullptr;
  if (backward) {
    for (int i = 0; i < 2; ++i) {
      if ((o[N_ARGS + i] == Py_None) != (o[i] == Py_None))
        return refuse(std::string(names[i]) + " must be given with its input, and only then");
      if (o[i] == Py_None) continue;
      if (!heads_ok(names[i] + 1, o[N_ARGS + i], c.q)) return nullptr;
      if (THPVariable_Unpack(o[N_ARGS + i]).sizes() != THPVariable_Unpack(o[i]).sizes())
        return refuse(std::string(names[i]) + " must have shape " + shape(THPVariable_Unpack(o[N_ARGS + i])) + ", got " +
                      shape(THPVariable_Unpack(o[i])));
    }
  }
  if (!c.q->is_cuda() || c.q->numel() == 0 || (c.k && c.k->numel() == 0)) Py_RETURN_NONE;
  const at::NoGradGuard no_grad;
  const int64_t d = c.q->dim();
  const bool weights = backward && (c.gamma[0] || c.gamma[1]) && PyObject_IsTrue(o[N_ARGS + 2]) > 0;
  int (*workspace)(const UnblendRotaryParams*, long long*) = nullptr;
  if (weights) workspace = reinterpret_cast<decltype(workspace)>(PyLong_AsVoidPtr(o[N_ARGS + 3]));
  const at::Tensor* const inputs[2] = {backward ? &THPVariable_Unpack(o[N_ARGS]) : nullptr,
                                       backward && c.k ? &THPVariable_Unpack(o[N_ARGS + 1]) : nullptr};
  at::Tensor q, k, q0, k0, freqs, positions, gammas[2], lens, q_out, k_out, dgamma[2], work;
  {
    const Unlocked unlocked;
    q = unit(*c.q);
    if (c.k) k = unit(*c.k);
    if (inputs[0]) q0 = unit(*inputs[0]);
    if (inputs[1]) k0 = unit(*inputs[1]);
    if (c.freqs) freqs = c.freqs->contiguous();
    if (c.positions) positions = c.positions->contiguous();
    if (c.lens) lens = c.lens->contiguous();
    for (int i = 0; i < 2; ++i)
      if (c.gamma[i]) gammas[i] = c.gamma[i]->contiguous();
    q_out = at::empty(q.sizes(), q.options());
    if (c.k) k_out = at::empty(k.sizes(), k.options());
    if (weights)
      for (at::Tensor& g : dgamma) g = at::empty({q.size(d - 1)}, gammas[c.gamma[0] ? 0 : 1].options());
  }
  UnblendRotaryParams p{};
  p.dtype = type_of(q);
  p.outer = (int)q.size(0);
  p.inner = d == 5 ? (int)q.size(1) : 1;
  p.length = (int)q.size(d - 3);
  p.heads = (int)q.size(d - 2);
  p.k_heads = c.k ? (int)k.size(d - 2) : 0;
  p.hd = (int)q.size(d - 1);
  p.half = c.half;
  p.scale = (float)c.scale;
  p.eps = (float)c.eps;
  if (c.freqs) {
    p.pairs = (int)freqs.numel();
    p.freqs = freqs.const_data_ptr();
    p.freqs_f64 = freqs.scalar_type() == at::kDouble;
  }
  if (c.positions) {
    p.positions = positions.const_data_ptr();
    p.positions_i64 = positions.scalar_type() == at::kLong;
    p.positions_stride = positions.dim() > 1 ? p.length : 0;
  }
  for (int i = 0; i < 2; ++i) {
    if (!c.gamma[i]) continue;
    p.w_dtype = type_of(gammas[i]);
    (i ? p.gamma_k : p.gamma_q) = gammas[i].const_data_ptr();
  }
  if (c.lens) p.lens = lens.const_data_ptr<int>();
  p.q = strides(q);
  if (c.k) p.k = strides(k);
  if (backward) p.q0 = strides(q0);
  if (backward && c.k) p.k0 = strides(k0);
  if (weights) {
    long long bytes = 0;
    if (!workspace || workspace(&p, &bytes) != 0) return refuse("heads: no workspace for these sizes");
    const Unlocked unlocked;
    work = at::empty({bytes}, q.options().dtype(at::kByte));
  }
  const auto address = [](const at::Tensor& t) { return t.defined() ? pointer(t) : 0LL; };
  PyObject* addresses = backward
                            ? Py_BuildValue("(LLLLLLLLL)", address(q), address(k), address(q0), address(k0),
                                            address(q_out), address(k_out), address(dgamma[0]), address(dgamma[1]),
                                            address(work))
                            : Py_BuildValue("(LLLL)", address(q), address(k), address(q_out), address(k_out));
  return Py_BuildValue("(NNNNNy#(NNNNNNNNNNNN))", wrap(q_out), wrap(k_out), wrap(dgamma[0]), wrap(dgamma[1]), addresses,
                       reinterpret_cast<const char*>(&p), (Py_ssize_t)sizeof(p), wrap(q), wrap(k), wrap(q0), wrap(k0),
                       wrap(freqs), wrap(positions), wrap(gammas[0]), wrap(gammas[1]), wrap(lens), wrap(dgamma[0]),
                       wrap(dgamma[1]), wrap(work));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"sizes", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(sizes)), METH_FASTCALL, nullptr},
    {"table", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(table)), METH_FASTCALL, nullptr},
    {"state", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(state)), METH_FASTCALL, nullptr},
    {"adamw", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(adamw)), METH_FASTCALL, nullptr},
    {"norm_outputs", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(norm_outputs)), METH_FASTCALL, nullptr},
    {"changed", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(changed)), METH_FASTCALL, nullptr},
    {"heads", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(heads)), METH_FASTCALL, nullptr},
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
