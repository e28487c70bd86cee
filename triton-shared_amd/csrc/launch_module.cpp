// The Python side of a launch, natively: what Triton's JIT calls for every `kernel[grid](...)`.
//
// `Launcher` is the base of HIPLauncher (backend/driver.py).  Called with the launcher arguments of the reference
// (backend/driver.py:262-265) it turns the ordinary ones -- exact ints and floats, torch tensors on the GPU, None -- into
// tts_arg records on the stack and calls tts_launch with the GIL released; anything else (hooks, objects with a data_ptr
// method, numpy scalars, empty grids, every error) goes to the Python method `_generic`, before anything has happened, so
// that there is one place that says what such calls do.
// What bounds a small launch is the host.  With this work in Python and ctypes a call of vector add took 12.5 us of it and one
// of LayerNorm (nine arguments) 14.1, now 8.0 and 7.7: 3.8 in tts_launch, the rest Triton's own.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <climits>
#include <cstdint>

#include "../../include/tts_hip.h"

namespace {

using LaunchFn = tts_status (*)(tts_plan *, int, int, int, void *, const tts_arg *, int);
LaunchFn g_launch = nullptr;
PyObject *g_plan_type = nullptr, *g_raise = nullptr;            // _native.PlanHandle, _native._raise
PyObject *g_tensor_type = nullptr, *g_parameter_type = nullptr;  // torch.Tensor, torch.nn.Parameter: no overridden attributes
PyObject *g_chain_type = nullptr;                                // triton.knobs.HookChain, or None
PyObject *s_generic, *s_handle, *s_kinds, *s_is_cuda, *s_data_ptr, *s_calls;

constexpr int MAX_ARGS = 64, FIXED = 9;

struct Launcher {
  PyObject_HEAD
  int n;
  int pos[MAX_ARGS];      // positions of the runtime arguments among the kernel's arguments
  char is_ptr[MAX_ARGS];
};

// _bind(slots): [(position, is a pointer), ...]
PyObject *launcher_bind(PyObject *self, PyObject *slots) {
  Launcher *l = (Launcher *)self;
  l->n = -1;  // (until all is well: every call goes the general way)
  PyObject *seq = PySequence_Fast(slots, "slots");
  if (!seq) return nullptr;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  for (Py_ssize_t i = 0; i < n && i < MAX_ARGS; i++) {
    int p = 0, ptr = 0;
    if (!PyArg_ParseTuple(PySequence_Fast_GET_ITEM(seq, i), "ip", &p, &ptr)) {
      Py_DECREF(seq);
      return nullptr;
    }
    l->pos[i] = p;
    l->is_ptr[i] = (char)ptr;
  }
  if (n <= MAX_ARGS) l->n = (int)n;
  Py_DECREF(seq);
  Py_RETURN_NONE;
}

// a non-negative int that fits a grid extent
bool extent(PyObject *o, int *out) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  const long long v = PyLong_AsLongLongAndOverflow(o, &over);
  if (over || v <= 0 || v > INT_MAX) return false;
  *out = (int)v;
  return true;
}

// the address of a tensor in device memory; false: leave it to `_generic` (no Python error is set)
bool device_address(PyObject *o, void **out) {
  if ((PyObject *)Py_TYPE(o) != g_tensor_type && (PyObject *)Py_TYPE(o) != g_parameter_type) return false;
  PyObject *cuda = PyObject_GetAttr(o, s_is_cuda);
  const bool on_gpu = cuda == Py_True;
  Py_XDECREF(cuda);
  PyObject *p = on_gpu ? PyObject_CallMethodNoArgs(o, s_data_ptr) : nullptr;
  const bool ok = p && PyLong_CheckExact(p);
  if (ok) *out = (void *)(uintptr_t)PyLong_AsUnsignedLongLongMask(p);
  Py_XDECREF(p);
  if (!ok) PyErr_Clear();
  return ok;
}

// Is there nothing to call: None, or Triton's chain of hooks (an exact triton.knobs.HookChain) with none in it?
bool no_hook(PyObject *hook) {
  if (hook == Py_None) return true;
  if ((PyObject *)Py_TYPE(hook) != g_chain_type) return false;
  PyObject *calls = PyObject_GetAttr(hook, s_calls);
  const bool none = calls && PyList_CheckExact(calls) && PyList_GET_SIZE(calls) == 0;
  Py_XDECREF(calls);
  if (!calls) PyErr_Clear();
  return none;
}

PyObject *launcher_call(PyObject *self, PyObject *args, PyObject *kwargs) {
  Launcher *l = (Launcher *)self;
  const Py_ssize_t given = PyTuple_GET_SIZE(args);
  auto general = [&]() -> PyObject * {
    PyObject *f = PyObject_GetAttr(self, s_generic);
    if (!f) return nullptr;
    PyObject *r = PyObject_Call(f, args, kwargs);
    Py_DECREF(f);
    return r;
  };
  if (kwargs || given < FIXED || l->n < 0 || !g_launch) return general();
  PyObject *const *a = &PyTuple_GET_ITEM(args, 0);
  int g[3];
  if (!extent(a[0], &g[0]) || !extent(a[1], &g[1]) || !extent(a[2], &g[2]) || !PyLong_CheckExact(a[3]) || (PyObject *)Py_TYPE(a[4]) != g_plan_type || !no_hook(a[7]) ||
      !no_hook(a[8]))
    return general();
  // the plan: its address and the kinds of its arguments, as PlanHandle keeps them
  PyObject *handle = PyObject_GetAttr(a[4], s_handle), *kinds = handle ? PyObject_GetAttr(a[4], s_kinds) : nullptr;
  tts_plan *plan = nullptr;
  tts_arg packed[MAX_ARGS];
  bool plain = kinds && PyLong_CheckExact(handle) && PyBytes_CheckExact(kinds) && PyBytes_GET_SIZE(kinds) == l->n;
  if (plain) plan = (tts_plan *)(uintptr_t)PyLong_AsUnsignedLongLongMask(handle);
  plain = plain && plan;
  for (int i = 0; plain && i < l->n; i++) {
    if (l->pos[i] < 0 || FIXED + l->pos[i] >= given) { plain = false; break; }
    PyObject *v = a[FIXED + l->pos[i]];
    tts_arg &t = packed[i];
    t.kind = PyBytes_AS_STRING(kinds)[i];
    t.reserved = 0;
    t.v.i = 0;
    if ((t.kind == TTS_ARG_PTR) != (l->is_ptr[i] != 0)) plain = false;
    else if (t.kind == TTS_ARG_PTR) {
      if (PyLong_CheckExact(v)) t.v.ptr = (void *)(uintptr_t)PyLong_AsUnsignedLongLongMask(v);
      else if (v != Py_None) plain = device_address(v, &t.v.ptr);
    } else if (t.kind == TTS_ARG_INT) {
      if (PyLong_Check(v)) t.v.i = (int64_t)PyLong_AsUnsignedLongLongMask(v);  // (bool too)
      else plain = false;
    } else {
      if (PyFloat_CheckExact(v)) t.v.f = PyFloat_AS_DOUBLE(v);
      else plain = false;
    }
  }
  Py_XDECREF(handle);
  Py_XDECREF(kinds);
  if (!plain) {
    PyErr_Clear();
    return general();
  }
  void *stream = (void *)(uintptr_t)PyLong_AsUnsignedLongLongMask(a[3]);
  const int n = l->n;
  tts_status st;
  Py_BEGIN_ALLOW_THREADS  // (args holds a reference to the plan and to every tensor)
  st = g_launch(plan, g[0], g[1], g[2], stream, packed, n);
  Py_END_ALLOW_THREADS
  if (st != TTS_OK) return PyObject_CallFunction(g_raise, "i", (int)st);
  Py_RETURN_NONE;
}

PyMethodDef launcher_methods[] = {{"_bind", launcher_bind, METH_O, "takes the runtime arguments' positions: [(position, is a pointer), ...]"}, {nullptr, nullptr, 0, nullptr}};
PyType_Slot launcher_slots[] = {{Py_tp_call, (void *)launcher_call}, {Py_tp_methods, launcher_methods}, {Py_tp_new, (void *)PyType_GenericNew}, {0, nullptr}};
PyType_Spec launcher_spec = {"tts_launch.Launcher", sizeof(Launcher), 0, Py_TPFLAGS_DEFAULT | Py_TPFLAGS_BASETYPE, launcher_slots};

// setup(address of tts_launch, PlanHandle, _raise, torch.Tensor, torch.nn.Parameter, the type of Triton's hook chains)
PyObject *setup(PyObject *, PyObject *args) {
  unsigned long long address = 0;
  PyObject *o[5];
  if (!PyArg_ParseTuple(args, "KOOOOO", &address, &o[0], &o[1], &o[2], &o[3], &o[4])) return nullptr;
  PyObject **to[5] = {&g_plan_type, &g_raise, &g_tensor_type, &g_parameter_type, &g_chain_type};
  for (int i = 0; i < 5; i++) {
    Py_INCREF(o[i]);
    Py_XSETREF(*to[i], o[i]);
  }
  g_launch = (LaunchFn)(uintptr_t)address;
  Py_RETURN_NONE;
}

// ---- triton_shared_amd.ops, natively
// Each function below is the ordinary call of the function of its name in ops.py -- torch tensors on the current device, no gradients; inside a level
// of forward-mode derivatives ops.py does not come here -- and returns its result; for anything else it returns None before anything has
// happened, and ops.py does the call or raises.
// Host time of a call, in Python and ctypes -> here (us): moe_route 15.0 -> 9.4, moe_experts 27.4 -> 17.8, lora_add 21.8 -> 13.2 (one, three and
// two launches among them).
struct Ops {
  decltype(&tts_moe_route) route;
  decltype(&tts_moe_experts_workspace) experts_workspace;
  decltype(&tts_moe_experts) experts;
  decltype(&tts_lora_add_workspace) lora_workspace;
  decltype(&tts_lora_add) lora;
  PyObject *get_device, *get_stream, *grad_enabled;  // torch._C._cuda_getDevice, _cuda_getCurrentRawStream, torch.is_grad_enabled
  PyObject *dtypes[5];                               // by tts_dtype
};
Ops g_ops = {};
PyObject *s_shape, *s_stride, *s_dtype, *s_get_device, *s_requires_grad, *s_new_empty;

// A reference that is let go of at the end
struct Ref {
  PyObject *o;
  explicit Ref(PyObject *p) : o(p) {}
  ~Ref() { Py_XDECREF(o); }
  Ref(const Ref &) = delete;
  Ref &operator=(const Ref &) = delete;
  explicit operator bool() const { return o != nullptr; }
};

bool to_int64(PyObject *o, int64_t *out) {
  if (!o || !PyLong_Check(o)) return false;
  int over = 0;
  *out = PyLong_AsLongLongAndOverflow(o, &over);
  return !over;
}

// What a call knows of its tensors: they are all on the current device, and none wants a gradient.  `ok` false: not an ordinary call.
struct Operands {
  int64_t device = -1;
  bool grad = false, ok = false;
  void *stream = nullptr;
  explicit Operands(PyObject *first) {
    if (!g_ops.route || ((PyObject *)Py_TYPE(first) != g_tensor_type && (PyObject *)Py_TYPE(first) != g_parameter_type)) return;
    Ref cuda(PyObject_GetAttr(first, s_is_cuda));
    if (cuda.o != Py_True) return;
    Ref d(PyObject_CallNoArgs(g_ops.get_device)), g(PyObject_CallNoArgs(g_ops.grad_enabled));
    if (!d || !g || !to_int64(d.o, &device)) return;
    Ref s(PyObject_CallOneArg(g_ops.get_stream, d.o));
    if (!s || !PyLong_CheckExact(s.o)) return;
    stream = (void *)(uintptr_t)PyLong_AsUnsignedLongLongMask(s.o);
    grad = g.o == Py_True;
    ok = true;
  }
  // null, or &t filled in
  const tts_tensor *describe(PyObject *o, tts_tensor &t) {
    if (o == Py_None || !ok) return nullptr;
    ok = false;
    if ((PyObject *)Py_TYPE(o) != g_tensor_type && (PyObject *)Py_TYPE(o) != g_parameter_type) return nullptr;
    Ref on(PyObject_CallMethodNoArgs(o, s_get_device)), type(PyObject_GetAttr(o, s_dtype)), shape(PyObject_GetAttr(o, s_shape)), stride(PyObject_CallMethodNoArgs(o, s_stride)),
        ptr(PyObject_CallMethodNoArgs(o, s_data_ptr));
    int64_t index = -1;
    if (!on || !type || !shape || !stride || !ptr || !to_int64(on.o, &index) || index != device) return nullptr;
    if (grad) {
      Ref wants(PyObject_GetAttr(o, s_requires_grad));
      if (wants.o != Py_False) return nullptr;
    }
    t.dtype = -1;
    for (int i = 0; i < 5; i++)
      if (type.o == g_ops.dtypes[i]) t.dtype = i;
    if (t.dtype < 0 || !PyTuple_Check(shape.o) || !PyTuple_Check(stride.o) || !PyLong_CheckExact(ptr.o)) return nullptr;
    const Py_ssize_t n = PyTuple_GET_SIZE(shape.o);
    if (n < 1 || n > 3 || PyTuple_GET_SIZE(stride.o) != n) return nullptr;
    t.rank = (int32_t)n;
    for (Py_ssize_t i = 0; i < n; i++)
      if (!to_int64(PyTuple_GET_ITEM(shape.o, i), &t.shape[i]) || !to_int64(PyTuple_GET_ITEM(stride.o, i), &t.stride[i])) return nullptr;
    t.ptr = (void *)(uintptr_t)PyLong_AsUnsignedLongLongMask(ptr.o);
    ok = true;
    return &t;
  }
  // a new tensor on the device of `like`, [rows, cols] or (rows < 0) [cols], described; dtype null: of its type
  PyObject *make(PyObject *like, int64_t rows, int64_t cols, PyObject *dtype, tts_tensor &t) {
    if (!ok) return nullptr;
    Ref size(rows < 0 ? Py_BuildValue("(L)", (long long)cols) : Py_BuildValue("(LL)", (long long)rows, (long long)cols));
    Ref names(dtype ? PyTuple_Pack(1, s_dtype) : nullptr);
    PyObject *args[] = {like, size.o, dtype};
    PyObject *made = size ? PyObject_VectorcallMethod(s_new_empty, args, 2, names.o) : nullptr;
    if (made) describe(made, t);
    ok = ok && made;
    return made;
  }
};

PyObject *not_ordinary() {
  PyErr_Clear();
  Py_RETURN_NONE;
}

// the result of a call, or the exception that its status stands for
PyObject *finish(tts_status st, PyObject *result) {
  if (st == TTS_OK) return result;
  Py_XDECREF(result);
  return PyObject_CallFunction(g_raise, "i", (int)st);
}

// moe_route(logits, k, scoring, bias, renormalize, scale): scoring by its number
PyObject *op_route(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 6) return not_ordinary();
  Operands o(a[0]);
  tts_tensor logits, bias, ids, weights;
  int64_t k = 0, scoring = 0;
  if (!o.ok || !PyLong_CheckExact(a[1]) || !to_int64(a[1], &k) || k < 1 || !to_int64(a[2], &scoring) || !PyBool_Check(a[4]) || !PyFloat_CheckExact(a[5])) return not_ordinary();
  const tts_tensor *l = o.describe(a[0], logits), *b = o.describe(a[3], bias);
  if (!l || !o.ok || l->rank != 2 || k > logits.shape[1]) return not_ordinary();
  Ref made_ids(o.make(a[0], logits.shape[0], k, g_ops.dtypes[TTS_I32], ids)), made_weights(o.make(a[0], logits.shape[0], k, g_ops.dtypes[TTS_F32], weights));
  if (!o.ok) return not_ordinary();
  const bool renormalize = a[4] == Py_True;
  const double scale = PyFloat_AS_DOUBLE(a[5]);
  tts_status st;
  Py_BEGIN_ALLOW_THREADS
  st = g_ops.route(l, b, (int)scoring, renormalize, scale, &ids, &weights, o.stream);
  Py_END_ALLOW_THREADS
  return finish(st, st == TTS_OK ? PyTuple_Pack(2, made_ids.o, made_weights.o) : nullptr);
}

// moe_experts(x, ids, weights, w_up, w_down, s_up, s_down, activation, gated, out): activation by its number
PyObject *op_experts(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 10) return not_ordinary();
  Operands o(a[0]);
  tts_tensor t[8], scratch;
  int64_t activation = 0;
  if (!o.ok || !to_int64(a[7], &activation) || !PyBool_Check(a[8])) return not_ordinary();
  const tts_tensor *p[8] = {};
  for (int i = 0; i < 7; i++) p[i] = o.describe(a[i], t[i]);
  if (!o.ok || !p[0] || !p[1] || !p[3] || !p[4] || p[0]->rank != 2 || p[4]->rank != 3) return not_ordinary();
  const bool gated = a[8] == Py_True;
  size_t bytes = 0;
  tts_status st = g_ops.experts_workspace(p[0], p[1], p[3], p[4], gated, &bytes);
  if (st != TTS_OK) return finish(st, nullptr);
  const bool given = a[9] != Py_None;
  if (given) p[7] = o.describe(a[9], t[7]);
  Ref made(given ? nullptr : o.make(a[0], t[0].shape[0], t[4].shape[2], nullptr, t[7]));
  Ref work(bytes ? o.make(a[0], -1, (int64_t)bytes, g_ops.dtypes[TTS_I8], scratch) : nullptr);
  if (!o.ok) return not_ordinary();
  p[7] = &t[7];
  void *at = bytes ? scratch.ptr : nullptr;
  Py_BEGIN_ALLOW_THREADS
  st = g_ops.experts(p[0], p[1], p[2], p[3], p[5], p[4], p[6], (int)activation, gated, p[7], at, bytes, o.stream);
  Py_END_ALLOW_THREADS
  return finish(st, Py_NewRef(given ? a[9] : made.o));
}

// lora_add(base, x, a, b, ids, scales, out)
PyObject *op_lora(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 7) return not_ordinary();
  Operands o(a[0]);
  tts_tensor t[7], scratch;
  if (!o.ok) return not_ordinary();
  const tts_tensor *p[7] = {};
  for (int i = 0; i < 6; i++) p[i] = o.describe(a[i], t[i]);
  if (!o.ok || !p[0] || !p[1] || !p[3] || p[0]->rank != 2) return not_ordinary();
  size_t bytes = 0;
  tts_status st = g_ops.lora_workspace(p[1], p[3], &bytes);
  if (st != TTS_OK) return finish(st, nullptr);
  const bool given = a[6] != Py_None;
  if (given) p[6] = o.describe(a[6], t[6]);
  Ref made(given ? nullptr : o.make(a[0], t[0].shape[0], t[0].shape[1], nullptr, t[6]));
  Ref work(bytes ? o.make(a[0], -1, (int64_t)bytes, g_ops.dtypes[TTS_I8], scratch) : nullptr);
  if (!o.ok) return not_ordinary();
  p[6] = &t[6];
  void *at = bytes ? scratch.ptr : nullptr;
  Py_BEGIN_ALLOW_THREADS
  st = g_ops.lora(p[0], p[1], p[2], p[3], p[4], p[5], p[6], at, bytes, o.stream);
  Py_END_ALLOW_THREADS
  return finish(st, Py_NewRef(given ? a[6] : made.o));
}

// setup_ops(addresses of the five entries, torch._C._cuda_getDevice, _cuda_getCurrentRawStream, torch.is_grad_enabled, the five dtypes,
// torch.Tensor, torch.nn.Parameter, _raise)
PyObject *setup_ops(PyObject *, PyObject *args) {
  unsigned long long f[5];
  PyObject *o[11];
  if (!PyArg_ParseTuple(args, "KKKKKOOOOOOOOOOO", &f[0], &f[1], &f[2], &f[3], &f[4], &o[0], &o[1], &o[2], &o[3], &o[4], &o[5], &o[6], &o[7], &o[8], &o[9], &o[10])) return nullptr;
  PyObject **to[11] = {&g_ops.get_device, &g_ops.get_stream, &g_ops.grad_enabled, &g_ops.dtypes[0], &g_ops.dtypes[1], &g_ops.dtypes[2], &g_ops.dtypes[3], &g_ops.dtypes[4], &g_tensor_type,
                       &g_parameter_type, &g_raise};
  for (int i = 0; i < 11; i++) {
    Py_INCREF(o[i]);
    Py_XSETREF(*to[i], o[i]);
  }
  g_ops.experts_workspace = (decltype(g_ops.experts_workspace))(uintptr_t)f[1];
  g_ops.experts = (decltype(g_ops.experts))(uintptr_t)f[2];
  g_ops.lora_workspace = (decltype(g_ops.lora_workspace))(uintptr_t)f[3];
  g_ops.lora = (decltype(g_ops.lora))(uintptr_t)f[4];
  g_ops.route = (decltype(g_ops.route))(uintptr_t)f[0];
  Py_RETURN_NONE;
}

PyMethodDef module_methods[] = {{"setup", setup, METH_VARARGS, nullptr},
                                {"setup_ops", setup_ops, METH_VARARGS, nullptr},
                                {"moe_route", (PyCFunction)(void (*)(void))op_route, METH_FASTCALL, nullptr},
                                {"moe_experts", (PyCFunction)(void (*)(void))op_experts, METH_FASTCALL, nullptr},
                                {"lora_add", (PyCFunction)(void (*)(void))op_lora, METH_FASTCALL, nullptr},
                                {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "tts_launch", nullptr, -1, module_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_tts_launch(void) {
  s_generic = PyUnicode_InternFromString("_generic");
  s_handle = PyUnicode_InternFromString("_address");
  s_kinds = PyUnicode_InternFromString("_kinds");
  s_is_cuda = PyUnicode_InternFromString("is_cuda");
  s_calls = PyUnicode_InternFromString("calls");
  s_data_ptr = PyUnicode_InternFromString("data_ptr");
  s_shape = PyUnicode_InternFromString("shape");
  s_stride = PyUnicode_InternFromString("stride");
  s_dtype = PyUnicode_InternFromString("dtype");
  s_get_device = PyUnicode_InternFromString("get_device");
  s_requires_grad = PyUnicode_InternFromString("requires_grad");
  s_new_empty = PyUnicode_InternFromString("new_empty");
  PyObject *m = PyModule_Create(&module_def);
  if (!m) return nullptr;
  PyObject *type = PyType_FromSpec(&launcher_spec);
  if (!type || PyModule_AddObject(m, "Launcher", type) < 0) {
    Py_XDECREF(type);
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
