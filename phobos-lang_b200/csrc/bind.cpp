// The short calls of serve.py without ctypes: a CPython module that reads a tensor's address, type, sizes and strides
// through torch's own Python methods and calls the C ABI.  (A decode step makes these calls for every layer; with struct
// and ctypes a gemv_q4 call took 5.7 us on the host, of which the launch is 1.7.)  It links against neither torch nor CUDA:
// serve.py hands it the entry points' addresses, torch's types and the exception to raise.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <pthread.h>

#include <cstdint>

#include "../../include/phobos_leaf.h"

namespace {

PyObject *s_data_ptr, *s_get_device, *s_shape, *s_stride, *s_dtype, *s_is_contiguous, *s_numel, *s_cuda_stream, *s_element_size;
PyObject *g_error, *g_get_device, *g_get_stream;  // PhobosError, torch's getters
PyObject* g_types[5];                             // f16, f32, i8, u8, i32
constexpr int32_t TYPE_CODES[5] = {PH_F16, PH_F32, PH_I8, PH_I8, PH_I32};

// The entry points, in the order serve.py lists them.
enum Entry { GEMV_Q4, KV4_APPEND, KV4_READ, KV4_ATTENTION, KV4_EXTEND, KV4_FORK, KV4_FREE, KV4_COMPACT, N_ENTRIES };
void* g_entry[N_ENTRIES];

bool refuse(int code, const char* format, const char* name) {
  PyObject* text = PyUnicode_FromFormat(format, name);
  PyObject* error = text ? PyObject_CallFunction(g_error, "iO", code, text) : nullptr;
  if (error) PyErr_SetObject(g_error, error);
  Py_XDECREF(text);
  Py_XDECREF(error);
  return false;
}

// A method without arguments whose result is an integer.
bool integer(PyObject* of, PyObject* method, long long* out) {
  PyObject* r = PyObject_CallMethodNoArgs(of, method);
  if (!r) return false;
  *out = PyLong_AsLongLong(r);
  Py_DECREF(r);
  return !(*out == -1 && PyErr_Occurred());
}

struct Call {
  long device;
  void* stream;
};

bool begin(PyObject* stream, Call* c) {
  PyObject* device = PyObject_CallNoArgs(g_get_device);
  if (!device) return false;
  c->device = PyLong_AsLong(device);
  PyObject* handle;
  if (stream == Py_None) {
    handle = PyObject_CallOneArg(g_get_stream, device);
  } else if (PyLong_Check(stream)) {
    Py_INCREF(stream);
    handle = stream;
  } else {
    handle = PyObject_GetAttr(stream, s_cuda_stream);
  }
  Py_DECREF(device);
  if (!handle) return false;
  c->stream = PyLong_AsVoidPtr(handle);
  Py_DECREF(handle);
  return !PyErr_Occurred();
}

bool on_device(PyObject* t, const char* name, const Call& c) {
  long long device;
  if (!integer(t, s_get_device, &device)) return false;
  if (device == c.device) return true;
  return refuse(PH_ERR_INVALID, device < 0 ? "%s is not on a CUDA device" : "%s does not live on the current device", name);
}

// PhTensor of a rank-1/2 CUDA tensor (no copy).
bool describe(PyObject* t, const char* name, const Call& c, PhTensor* d) {
  if (!on_device(t, name, c)) return false;
  PyObject* type = PyObject_GetAttr(t, s_dtype);
  if (!type) return false;
  Py_DECREF(type);  // torch keeps its types
  int k = 0;
  while (k < 5 && g_types[k] != type) k++;
  if (k == 5) return refuse(PH_ERR_UNSUPPORTED, "%s: element type", name);
  long long at;
  if (!integer(t, s_data_ptr, &at)) return false;
  PyObject* shape = PyObject_GetAttr(t, s_shape);
  PyObject* stride = shape ? PyObject_CallMethodNoArgs(t, s_stride) : nullptr;
  bool ok = stride != nullptr && PyTuple_Check(shape) && PyTuple_Check(stride);
  if (ok) {
    const Py_ssize_t rank = PyTuple_GET_SIZE(shape);
    *d = PhTensor{reinterpret_cast<void*>(at), TYPE_CODES[k], static_cast<int32_t>(rank), {0, 0}, {0, 0}, 0};
    if (rank != 1 && rank != 2) {
      ok = refuse(PH_ERR_INVALID, "%s: expected rank 1 or 2", name);
    } else {
      for (Py_ssize_t i = 0; i < rank; i++) {
        d->sizes[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i));
        d->strides[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(stride, i));
      }
      ok = !PyErr_Occurred();
    }
  } else if (!PyErr_Occurred()) {
    refuse(PH_ERR_INVALID, "%s: not a tensor", name);
  }
  Py_XDECREF(shape);
  Py_XDECREF(stride);
  return ok;
}

// Address of a contiguous int32 tensor of at least n values, and its length where that is asked for; None is a null
// address, but refused where the length counts.
bool integers(PyObject* t, const char* name, const Call& c, long long n, int32_t** at, long long* count = nullptr) {
  *at = nullptr;
  if (t == Py_None) return count == nullptr || refuse(PH_ERR_INVALID, "%s: expected a contiguous int32 tensor", name);
  if (!on_device(t, name, c)) return false;
  PyObject* type = PyObject_GetAttr(t, s_dtype);
  if (!type) return false;
  Py_DECREF(type);
  PyObject* contiguous = PyObject_CallMethodNoArgs(t, s_is_contiguous);
  if (!contiguous) return false;
  const bool ok = type == g_types[4] && contiguous == Py_True;
  Py_DECREF(contiguous);
  if (!ok) return refuse(PH_ERR_INVALID, "%s: expected a contiguous int32 tensor", name);
  long long have, address;
  if (!integer(t, s_numel, &have) || !integer(t, s_data_ptr, &address)) return false;
  if (have < n) return refuse(PH_ERR_INVALID, "%s: too few values", name);
  if (have > 0x7fffffffLL) return refuse(PH_ERR_INVALID, "%s: too many values", name);
  *at = reinterpret_cast<int32_t*>(address);
  if (count) *count = have;
  return true;
}

bool space(PyObject* t, const Call& c, void** at, size_t* bytes) {
  *at = nullptr;
  *bytes = 0;
  if (t == Py_None) return true;
  PyObject* contiguous = PyObject_CallMethodNoArgs(t, s_is_contiguous);
  if (!contiguous) return false;
  Py_DECREF(contiguous);  // True and False stay
  // (a view that repeats its elements has more of them than bytes of memory)
  if (contiguous != Py_True) return refuse(PH_ERR_WORKSPACE, "%s: not contiguous", "workspace");
  long long address, n, each;
  if (!on_device(t, "workspace", c) || !integer(t, s_data_ptr, &address) || !integer(t, s_numel, &n) || !integer(t, s_element_size, &each)) return false;
  *at = reinterpret_cast<void*>(address);
  *bytes = static_cast<size_t>(n) * static_cast<size_t>(each);
  return true;
}

bool real(PyObject* v, float* out) {
  const double d = PyFloat_AsDouble(v);
  *out = static_cast<float>(d);
  return !(d == -1.0 && PyErr_Occurred());
}
bool whole(PyObject* v, int32_t* out) {
  const long long n = PyLong_AsLongLong(v);
  if (n == -1 && PyErr_Occurred()) return false;
  if (n < INT32_MIN || n > INT32_MAX) return refuse(PH_ERR_INVALID, "%s does not fit 32 bits", "an argument");
  *out = static_cast<int32_t>(n);
  return true;
}
// The address of a PhKv4Cache and the device it was made on, as Kv4Cache keeps them in a pair.
bool cache_of(PyObject* pair, const Call& c, const PhKv4Cache** cache) {
  if (!PyTuple_Check(pair) || PyTuple_GET_SIZE(pair) != 2) return refuse(PH_ERR_INVALID, "%s: not a cache", "cache");
  *cache = static_cast<const PhKv4Cache*>(PyLong_AsVoidPtr(PyTuple_GET_ITEM(pair, 0)));
  if (PyLong_AsLong(PyTuple_GET_ITEM(pair, 1)) == c.device && !PyErr_Occurred()) return true;
  return !PyErr_Occurred() && refuse(PH_ERR_INVALID, "%s does not live on the current device", "the cache");
}

// Calls an entry point without the interpreter's lock: a launch waits where the stream's queue is full, and what it waits for
// may be a host function of the stream that needs the lock.  A lock of its own keeps the launches of one call together, so
// that threads which share a stream and a workspace still make their calls one after another.
pthread_mutex_t g_calls = PTHREAD_MUTEX_INITIALIZER;

template <typename F>
PyObject* unlocked(F call) {
  PyThreadState* state = PyEval_SaveThread();
  pthread_mutex_lock(&g_calls);
  const int rc = call();
  pthread_mutex_unlock(&g_calls);
  PyEval_RestoreThread(state);
  return PyLong_FromLong(rc);
}

bool args_are(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
  return false;
}

// gemv_q4(X, packed, Y, group, alpha, beta, stream)
PyObject* gemv_q4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Call c;
  PhTensor x, w, y;
  int32_t group;
  float alpha, beta;
  if (!args_are(n, 7) || !begin(a[6], &c) || !describe(a[0], "X", c, &x) || !describe(a[1], "packed", c, &w) || !describe(a[2], "Y", c, &y) ||
      !whole(a[3], &group) || !real(a[4], &alpha) || !real(a[5], &beta))
    return nullptr;
  return unlocked([&] {
    return reinterpret_cast<decltype(&phobos_gemv_q4)>(g_entry[GEMV_Q4])(&x, &w, &y, alpha, beta, group, c.stream);
  });
}

// rows(read, cache, layer, K, V, slots, indptr, stream)
PyObject* rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Call c;
  const PhKv4Cache* cache;
  PhTensor k, v;
  int32_t read, layer, *slots, *indptr;
  long long count;
  if (!args_are(n, 8) || !begin(a[7], &c) || !whole(a[0], &read) || !cache_of(a[1], c, &cache) || !whole(a[2], &layer) || !describe(a[3], "K", c, &k) ||
      !describe(a[4], "V", c, &v) || !integers(a[5], "slots", c, 0, &slots, &count) || !integers(a[6], "indptr", c, count + 1, &indptr))
    return nullptr;
  return unlocked([&] {
    return reinterpret_cast<decltype(&phobos_kv4_append)>(g_entry[read ? KV4_READ : KV4_APPEND])(
        cache, layer, &k, &v, slots, indptr, static_cast<int32_t>(count), c.stream);
  });
}

// attention(cache, layer, Q, O, lse, scale, window, slots, indptr, workspace, stream)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Call c;
  const PhKv4Cache* cache;
  PhTensor q, o, lse;
  int32_t layer, window, *slots, *indptr;
  long long count;
  float scale;
  void* ws;
  size_t bytes;
  if (!args_are(n, 11) || !begin(a[10], &c) || !cache_of(a[0], c, &cache) || !whole(a[1], &layer) || !describe(a[2], "Q", c, &q) ||
      !describe(a[3], "O", c, &o) || (a[4] != Py_None && !describe(a[4], "lse", c, &lse)) || !real(a[5], &scale) || !whole(a[6], &window) ||
      !integers(a[7], "slots", c, 0, &slots, &count) || !integers(a[8], "indptr", c, count + 1, &indptr) || !space(a[9], c, &ws, &bytes))
    return nullptr;
  return unlocked([&] {
    return reinterpret_cast<decltype(&phobos_kv4_attention)>(g_entry[KV4_ATTENTION])(
        cache, layer, &q, &o, a[4] != Py_None ? &lse : nullptr, scale, window, slots, indptr, static_cast<int32_t>(count), ws, bytes, c.stream);
  });
}

// extend(cache, slots, counts, shortfall, workspace, stream)
PyObject* extend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Call c;
  const PhKv4Cache* cache;
  int32_t *slots, *counts, *shortfall;
  long long count;
  void* ws;
  size_t bytes;
  if (!args_are(n, 6) || !begin(a[5], &c) || !cache_of(a[0], c, &cache) || !integers(a[1], "slots", c, 0, &slots, &count) ||
      !integers(a[2], "counts", c, count, &counts) || !integers(a[3], "shortfall", c, 1, &shortfall) || !space(a[4], c, &ws, &bytes))
    return nullptr;
  return unlocked([&] {
    return reinterpret_cast<decltype(&phobos_kv4_extend)>(g_entry[KV4_EXTEND])(cache, slots, counts, static_cast<int32_t>(count), shortfall,
        ws, bytes, c.stream);
  });
}

// fork(cache, src, dst, deep, shortfall, workspace, stream)
PyObject* fork(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Call c;
  const PhKv4Cache* cache;
  int32_t *src, *dst, *shortfall, deep;
  long long count;
  void* ws;
  size_t bytes;
  if (!args_are(n, 7) || !begin(a[6], &c) || !cache_of(a[0], c, &cache) || !integers(a[1], "src", c, 0, &src, &count) ||
      !integers(a[2], "dst", c, count, &dst) || !whole(a[3], &deep) || !integers(a[4], "shortfall", c, 1, &shortfall) || !space(a[5], c, &ws, &bytes))
    return nullptr;
  return unlocked([&] {
    return reinterpret_cast<decltype(&phobos_kv4_fork)>(g_entry[KV4_FORK])(cache, src, dst, static_cast<int32_t>(count), deep, shortfall, ws,
        bytes, c.stream);
  });
}

// free(cache, slots, keep, stream)
PyObject* free_(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Call c;
  const PhKv4Cache* cache;
  int32_t *slots, *keep;
  long long count;
  if (!args_are(n, 4) || !begin(a[3], &c) || !cache_of(a[0], c, &cache) || !integers(a[1], "slots", c, 0, &slots, &count) ||
      !integers(a[2], "keep", c, count, &keep))
    return nullptr;
  return unlocked([&] {
    return reinterpret_cast<decltype(&phobos_kv4_free)>(g_entry[KV4_FREE])(cache, slots, keep, static_cast<int32_t>(count), c.stream);
  });
}

// compact(cache, live, workspace, stream)
PyObject* compact(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Call c;
  const PhKv4Cache* cache;
  int32_t* live;
  void* ws;
  size_t bytes;
  if (!args_are(n, 4) || !begin(a[3], &c) || !cache_of(a[0], c, &cache) || !integers(a[1], "live", c, 1, &live) || !space(a[2], c, &ws, &bytes)) return nullptr;
  return unlocked([&] {
    return reinterpret_cast<decltype(&phobos_kv4_compact)>(g_entry[KV4_COMPACT])(cache, live, ws, bytes, c.stream);
  });
}

// setup(entries, types, error, get_device, get_stream): addresses in the order of Entry, torch's types in the order of g_types
PyObject* setup(PyObject*, PyObject* args) {
  PyObject *entries, *types, *error, *device, *stream;
  if (!PyArg_ParseTuple(args, "O!O!OOO", &PyTuple_Type, &entries, &PyTuple_Type, &types, &error, &device, &stream)) return nullptr;
  if (PyTuple_GET_SIZE(entries) != N_ENTRIES || PyTuple_GET_SIZE(types) != 5) {
    PyErr_SetString(PyExc_ValueError, "setup: entries or types");
    return nullptr;
  }
  for (int i = 0; i < N_ENTRIES; i++) {
    g_entry[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(entries, i));
    if (!g_entry[i]) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "setup: entry %d", i);
  }
  for (int i = 0; i < 5; i++) Py_XSETREF(g_types[i], Py_NewRef(PyTuple_GET_ITEM(types, i)));
  Py_XSETREF(g_error, Py_NewRef(error));
  Py_XSETREF(g_get_device, Py_NewRef(device));
  Py_XSETREF(g_get_stream, Py_NewRef(stream));
  Py_RETURN_NONE;
}

using Fast = PyObject* (*)(PyObject*, PyObject* const*, Py_ssize_t);
PyMethodDef fast(const char* name, Fast f) { return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}; }

PyMethodDef methods[] = {{"setup", setup, METH_VARARGS, nullptr},
                         fast("gemv_q4", gemv_q4),
                         fast("rows", rows),
                         fast("attention", attention),
                         fast("extend", extend),
                         fast("fork", fork),
                         fast("free", free_),
                         fast("compact", compact),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind(void) {
  PyObject** names[] = {&s_data_ptr, &s_get_device, &s_shape, &s_stride, &s_dtype, &s_is_contiguous, &s_numel, &s_cuda_stream, &s_element_size};
  const char* texts[] = {"data_ptr", "get_device", "shape", "stride", "dtype", "is_contiguous", "numel", "cuda_stream", "element_size"};
  for (int i = 0; i < 9; i++)
    if (!(*names[i] = PyUnicode_InternFromString(texts[i]))) return nullptr;
  return PyModule_Create(&module);
}
