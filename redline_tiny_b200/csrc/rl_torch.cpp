// The hot calls of ops.py in one step each: arguments checked, outputs and workspaces taken from torch's allocator and the
// C ABI called, without the interpreter's share of that (12 - 15 us a call through ctypes, most of a small kernel's time).
//
// A Python extension module, `_rl_torch`. Every function returns None, having done nothing, where an argument is not
// exactly what it expects (another type, shape, stride or device): ops.py then takes its own path, which accepts what is
// acceptable and says what is wrong with the rest. Otherwise it returns the outputs, or the C ABI's negative status.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>

#include "../../include/redline_b200.h"

namespace {

// A tensor argument, or null.
const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool on(const at::Tensor& t, int64_t dev) { return t.is_cuda() && t.get_device() == dev; }
bool ints(const at::Tensor& t, int64_t dev) { return on(t, dev) && t.scalar_type() == at::kInt && t.is_contiguous(); }

// A tuple of integers (a pool's layer, a weight).
template <int N>
bool unpack(PyObject* o, int64_t (&v)[N]) {
  if (!PyTuple_CheckExact(o) || PyTuple_GET_SIZE(o) != N) return false;
  for (int i = 0; i < N; ++i) {
    PyObject* e = PyTuple_GET_ITEM(o, i);
    if (!PyLong_CheckExact(e)) return false;
    v[i] = PyLong_AsLongLong(e);
    if (v[i] == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      return false;
    }
  }
  return true;
}

template <typename T>
T* ptr(int64_t v) { return reinterpret_cast<T*>(static_cast<uintptr_t>(v)); }
template <typename T>
T* ptr(const at::Tensor& t) { return static_cast<T*>(t.data_ptr()); }

struct Pool {   // (k, v, k_exp, v_exp, pages, kv_heads, page, device)
  int64_t v[8];
  int64_t pages() const { return v[4]; }
  int hkv() const { return static_cast<int>(v[5]); }
  int page() const { return static_cast<int>(v[6]); }
  int64_t dev() const { return v[7]; }
};

// Page tables, lengths and row ranges (or first positions) of a batch on the current device.
struct Batch {
  const at::Tensor *table, *len, *start;
  int64_t B, width;
  bool take(PyObject* a, PyObject* b, PyObject* c, int64_t dev, int extra) {
    table = tensor(a), len = tensor(b), start = tensor(c);
    if (!table || !len || !start || !ints(*table, dev) || !ints(*len, dev) || !ints(*start, dev)) return false;
    if (table->dim() != 2 || len->dim() != 1 || start->dim() != 1) return false;
    B = table->size(0), width = table->size(1);
    return width > 0 && B <= 4096 && len->size(0) == B && start->size(0) == B + extra;
  }
};

bool current(int64_t dev) { return c10::cuda::current_device() == dev; }
rl_stream_t stream() { return reinterpret_cast<rl_stream_t>(c10::cuda::getCurrentCUDAStream().stream()); }

// kv_append(pool, k, v, table, kv_len, q_start) -> status
PyObject* kv_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Pool p;
  Batch b;
  if (n != 6 || !unpack(a[0], p.v)) Py_RETURN_NONE;
  const at::Tensor *k = tensor(a[1]), *v = tensor(a[2]);
  if (!k || !v || !on(*k, p.dev()) || !on(*v, p.dev()) || !current(p.dev()) || !b.take(a[3], a[4], a[5], p.dev(), 1)) Py_RETURN_NONE;
  if (k->dim() != 3 || v->dim() != 3 || k->sizes() != v->sizes() || k->size(1) != p.hkv() || k->size(2) != 128) Py_RETURN_NONE;
  const auto dt = k->scalar_type();
  if (dt != v->scalar_type() || (dt != at::kBFloat16 && dt != at::kFloat)) Py_RETURN_NONE;
  const int st = rl_kv_append(k->data_ptr(), k->stride(0), k->stride(1), k->stride(2), v->data_ptr(), v->stride(0),
                              v->stride(1), v->stride(2), dt == at::kFloat ? RL_F32 : RL_BF16, k->size(0),
                              ptr<uint8_t>(p.v[0]), ptr<uint8_t>(p.v[1]), ptr<uint8_t>(p.v[2]), ptr<uint8_t>(p.v[3]),
                              p.pages(), p.hkv(), p.page(), ptr<int32_t>(*b.table), b.width, ptr<int32_t>(*b.len),
                              ptr<int32_t>(*b.start), static_cast<int>(b.B), stream());
  return PyLong_FromLong(st);
  END_HANDLE_TH_ERRORS
}

// kv_read(pool, table, kv_len, start, count) -> (k, v) or status
PyObject* kv_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Pool p;
  Batch b;
  if (n != 5 || !unpack(a[0], p.v) || !PyLong_CheckExact(a[4])) Py_RETURN_NONE;
  if (!b.take(a[1], a[2], a[3], p.dev(), 0) || !current(p.dev())) Py_RETURN_NONE;
  const int64_t count = PyLong_AsLongLong(a[4]);
  if (count <= 0 || count > (1 << 27)) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  const auto opt = b.table->options().dtype(at::kBFloat16);
  const at::Tensor k = at::empty({b.B, count, p.hkv(), 128}, opt), v = at::empty({b.B, count, p.hkv(), 128}, opt);
  const int st = rl_kv_read(ptr<uint8_t>(p.v[0]), ptr<uint8_t>(p.v[1]), ptr<uint8_t>(p.v[2]), ptr<uint8_t>(p.v[3]), p.pages(),
                            p.hkv(), p.page(), ptr<int32_t>(*b.table), b.width, ptr<int32_t>(*b.len), ptr<int32_t>(*b.start),
                            static_cast<int>(b.B), count, ptr<uint16_t>(k), ptr<uint16_t>(v), stream());
  if (st != RL_OK) return PyLong_FromLong(st);
  PyObject* kv = PyTuple_New(2);
  if (!kv) return nullptr;
  PyTuple_SET_ITEM(kv, 0, THPVariable_Wrap(k));
  PyTuple_SET_ITEM(kv, 1, THPVariable_Wrap(v));
  return kv;
  END_HANDLE_TH_ERRORS
}

// kv_attention(q, pool, table, kv_len, q_start, row_limit or None, scale_log2, out or None) -> out or status
PyObject* kv_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Pool p;
  Batch b;
  if (n != 8 || !unpack(a[1], p.v) || !PyFloat_CheckExact(a[6])) Py_RETURN_NONE;
  const at::Tensor *q = tensor(a[0]), *lim = nullptr, *given = nullptr;
  if (!q || !on(*q, p.dev()) || !current(p.dev()) || !b.take(a[2], a[3], a[4], p.dev(), 1)) Py_RETURN_NONE;
  if (q->dim() != 3 || q->scalar_type() != at::kBFloat16 || q->size(2) != 128 || q->stride(2) != 1) Py_RETURN_NONE;
  const int64_t T = q->size(0), H = q->size(1);
  if (T <= 0 || H <= 0 || H > 65535) Py_RETURN_NONE;
  if (a[5] != Py_None) {
    lim = tensor(a[5]);
    if (!lim || !ints(*lim, p.dev()) || lim->dim() != 1 || lim->size(0) != T) Py_RETURN_NONE;
  }
  if (a[7] != Py_None) {
    given = tensor(a[7]);
    if (!given || !on(*given, p.dev()) || given->scalar_type() != at::kBFloat16 || given->dim() != 2 || given->size(0) != T ||
        given->size(1) != H * 128 || given->stride(1) != 1)
      Py_RETURN_NONE;
  }
  const at::Tensor out = given ? *given : at::empty({T, H * 128}, q->options());
  const int64_t need = static_cast<int64_t>(rl_kv_attention_workspace(T, static_cast<int>(b.B), static_cast<int>(H), p.hkv()));
  const at::Tensor ws = at::empty({need < 16 ? 16 : need}, q->options().dtype(at::kByte));
  // (a single row's stride, or a single head's, says nothing)
  const int st = rl_kv_attention(ptr<uint16_t>(*q), T == 1 ? 0 : q->stride(0), H == 1 ? 0 : q->stride(1), T, static_cast<int>(H),
                                 ptr<uint8_t>(p.v[0]), ptr<uint8_t>(p.v[1]), ptr<uint8_t>(p.v[2]), ptr<uint8_t>(p.v[3]),
                                 p.pages(), p.hkv(), p.page(), ptr<int32_t>(*b.table), b.width, ptr<int32_t>(*b.len),
                                 ptr<int32_t>(*b.start), static_cast<int>(b.B), lim ? ptr<int32_t>(*lim) : nullptr,
                                 static_cast<float>(PyFloat_AS_DOUBLE(a[6])), ptr<uint16_t>(out),
                                 T == 1 ? H * 128 : out.stride(0), ws.data_ptr(), static_cast<size_t>(ws.numel()), stream());
  if (st != RL_OK) return PyLong_FromLong(st);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// linear_w4(x, (codes, scales, K, N, group, device), bias or None, epilogue, cols, fp32 output) -> out or status
PyObject* linear_w4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t w[6];
  if (n != 6 || !unpack(a[1], w) || !PyLong_CheckExact(a[3]) || !PyLong_CheckExact(a[4])) Py_RETURN_NONE;
  const at::Tensor *x = tensor(a[0]), *bias = nullptr;
  if (!x || !on(*x, w[5]) || !current(w[5])) Py_RETURN_NONE;
  if (x->dim() != 2 || x->scalar_type() != at::kBFloat16 || x->size(1) != w[2] || !x->is_contiguous() || x->size(0) <= 0)
    Py_RETURN_NONE;
  if (a[2] != Py_None) {
    bias = tensor(a[2]);
    if (!bias || !on(*bias, w[5]) || bias->scalar_type() != at::kBFloat16 || bias->dim() != 1 || bias->size(0) != w[3] ||
        !bias->is_contiguous())
      Py_RETURN_NONE;
  }
  const bool f32 = a[5] == Py_True;
  const at::Tensor out = at::empty({x->size(0), PyLong_AsLongLong(a[4])}, f32 ? x->options().dtype(at::kFloat) : x->options());
  const int st = rl_linear_w4(ptr<uint16_t>(*x), x->size(0), w[2], ptr<uint8_t>(w[0]), ptr<uint8_t>(w[1]), w[3],
                              static_cast<int>(w[4]), bias ? ptr<uint16_t>(*bias) : nullptr,
                              static_cast<int>(PyLong_AsLong(a[3])), out.data_ptr(), f32 ? RL_F32 : RL_BF16, stream());
  if (st != RL_OK) return PyLong_FromLong(st);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

#define RL_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {RL_METHOD(kv_append), RL_METHOD(kv_read), RL_METHOD(kv_attention), RL_METHOD(linear_w4),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_rl_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

#define RL_STR_(x) #x
#define RL_STR(x) RL_STR_(x)
constexpr char kPython[] = RL_STR(PY_MAJOR_VERSION) "." RL_STR(PY_MINOR_VERSION) ".";

}  // namespace

// Refuses to load beside another torch or Python than it was built for: tensors are reached through their headers.
PyMODINIT_FUNC PyInit__rl_torch() {
  PyObject* m = PyImport_ImportModule("torch.version");
  PyObject* v = m ? PyObject_GetAttrString(m, "__version__") : nullptr;
  PyObject* s = v ? PyObject_Str(v) : nullptr;
  const char* have = s ? PyUnicode_AsUTF8(s) : nullptr;
  const bool same = have && std::strcmp(have, RL_TORCH_VERSION) == 0 &&
                    std::strncmp(Py_GetVersion(), kPython, sizeof(kPython) - 1) == 0;
  if (have && !same)
    PyErr_Format(PyExc_ImportError, "_rl_torch is built for torch %s and Python %s, not for torch %s and Python %s",
                 RL_TORCH_VERSION, kPython, have, Py_GetVersion());
  Py_XDECREF(s), Py_XDECREF(v), Py_XDECREF(m);
  return same ? PyModule_Create(&kModule) : nullptr;
}
