// calls.cpp — CPython module `_calls`: the step operators' entry points without
// ctypes.  A small launch takes the GPU two or three microseconds, while building
// ctypes descriptors for a call's tensors takes ten; here each tensor is one C
// call into its producer (DLPack's C exchange API, a public struct of function
// pointers on the producer's type) or one attribute of a DeviceArray.
//
// Every function takes its arguments by position and returns the library's
// status code, or -1 when some argument needs the general path (host data, a
// producer without the exchange API, a tensor that requires a gradient, which
// __dlpack__ refuses, or, for a call without a stream, a producer whose current
// stream is not the legacy default stream): nothing has run then.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>
#include <string.h>

#include "kvcache.h"

namespace {

typedef int (*FromObject)(void*, kvc_dltensor*);
typedef int (*WorkStream)(int, int32_t, void**);

struct ExchangeAPI {  // DLPackExchangeAPI (DLPack 1.x)
  uint32_t major, minor;
  void* prev_api;
  void* allocator;
  void* managed_from_object;
  void* managed_to_object;
  FromObject dltensor_from_object;
  WorkStream current_work_stream;
};

struct Producer {
  PyTypeObject* type;
  const ExchangeAPI* api;  // nullptr: none
};
constexpr int kProducers = 16;
Producer g_producers[kProducers];
int g_num_producers = 0;
PyTypeObject* g_device_array = nullptr;
PyObject* g_name_dltensor = nullptr;
PyObject* g_name_handle = nullptr;
PyObject* g_name_requires_grad = nullptr;

enum Fn { kWindowDecode, kWindowPrefill, kStepTables, kRope, kRopeAppend, kNumFns };
const char* const kNames[kNumFns] = {"kvc_paged_attention_window", "kvc_paged_prefill_window", "kvc_step_tables",
                                     "kvc_qk_norm_rope", "kvc_qk_norm_rope_append"};
void* g_fn[kNumFns];

const ExchangeAPI* exchange_api(PyTypeObject* type) {
  for (int i = 0; i < g_num_producers; ++i)
    if (g_producers[i].type == type) return g_producers[i].api;
  const ExchangeAPI* api = nullptr;
  PyObject* cap = PyObject_GetAttrString(reinterpret_cast<PyObject*>(type), "__dlpack_c_exchange_api__");
  if (cap && PyCapsule_IsValid(cap, "dlpack_exchange_api")) {
    api = static_cast<const ExchangeAPI*>(PyCapsule_GetPointer(cap, "dlpack_exchange_api"));
    if (api->major != 1 || !api->dltensor_from_object || !api->current_work_stream) api = nullptr;
  }
  Py_XDECREF(cap);
  PyErr_Clear();
  if (g_num_producers < kProducers) {
    Py_INCREF(type);  // (kept: the address may not come to mean another type)
    g_producers[g_num_producers++] = {type, api};
  }
  return api;
}

// One call's arguments.
struct Call {
  kvc_dltensor storage[12];
  kvc_dltensor* t[12];
  int n = 0;
  void* stream = nullptr;
  bool default_stream = true, checked = false;

  bool set_stream(PyObject* s) {
    if (s == Py_None) return true;
    default_stream = false;
    PyObject* h = nullptr;
    if (!PyLong_Check(s)) {
      s = h = PyObject_GetAttr(s, g_name_handle);
      if (!h) {
        PyErr_Clear();
        return false;
      }
    }
    stream = PyLong_AsVoidPtr(s);
    Py_XDECREF(h);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return false;
    }
    return true;
  }

  bool tensor(PyObject* o) {
    if (o == Py_None) {
      t[n++] = nullptr;
      return true;
    }
    kvc_dltensor* d = &storage[n];
    PyTypeObject* type = Py_TYPE(o);
    if (type == g_device_array) {
      PyObject* dl = PyObject_CallMethodNoArgs(o, g_name_dltensor);
      Py_buffer buf;
      if (!dl || PyObject_GetBuffer(dl, &buf, PyBUF_SIMPLE) != 0) {
        PyErr_Clear();
        Py_XDECREF(dl);
        return false;
      }
      const bool ok = buf.len == (Py_ssize_t)sizeof(kvc_dltensor);
      if (ok) memcpy(d, buf.buf, sizeof(*d));  // (shape and strides live as long as the array does)
      PyBuffer_Release(&buf);
      Py_DECREF(dl);
      if (!ok) return false;
    } else {
      const ExchangeAPI* api = exchange_api(type);
      if (!api) return false;
      PyObject* grad = PyObject_GetAttr(o, g_name_requires_grad);
      if (!grad) PyErr_Clear();
      const bool plain = !grad || grad == Py_False;
      Py_XDECREF(grad);
      if (!plain) return false;
      if (api->dltensor_from_object(o, d) != 0) {
        PyErr_Clear();
        return false;
      }
      if (default_stream && !checked) {
        void* cur = nullptr;
        if (d->device.device_type != 2 || api->current_work_stream(2, d->device.device_id, &cur) != 0 || cur) {
          PyErr_Clear();
          return false;
        }
        checked = true;
      }
    }
    t[n++] = d;
    return true;
  }

  bool tensors(PyObject* const* a, int count) {
    for (int i = 0; i < count; ++i)
      if (!tensor(a[i])) return false;
    return true;
  }
};

bool get_int(PyObject* o, int* v) {
  if (!PyLong_Check(o)) return false;
  int over = 0;
  const long long x = PyLong_AsLongLongAndOverflow(o, &over);
  if (over || x < INT32_MIN || x > INT32_MAX) return false;
  *v = (int)x;
  return true;
}

bool get_float(PyObject* o, float* v) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  *v = (float)x;
  return true;
}

PyObject* general() { return PyLong_FromLong(-1); }

template <typename F>
PyObject* run(F f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS  //
  rc = f();
  Py_END_ALLOW_THREADS  //
  return PyLong_FromLong(rc);
}

// (out, query, key_cache, value_cache, block_tables, context_lens, num_kv_heads,
//  scale, block_size, max_seq_len, window_size, sink_size, stream)
PyObject* window_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Call c;
  int hkv, bs, msl, w, s;
  float scale;
  if (n != 13 || !g_fn[kWindowDecode] || !c.set_stream(a[12]) || !c.tensors(a, 6) || !get_int(a[6], &hkv) ||
      !get_float(a[7], &scale) || !get_int(a[8], &bs) || !get_int(a[9], &msl) || !get_int(a[10], &w) ||
      !get_int(a[11], &s))
    return general();
  return run([&] {
    return reinterpret_cast<decltype(&kvc_paged_attention_window)>(g_fn[kWindowDecode])(
        c.t[0], c.t[1], c.t[2], c.t[3], c.t[4], c.t[5], hkv, scale, bs, msl, w, s, c.stream);
  });
}

// (out, query, key_cache, value_cache, block_tables, qo_indptr, kv_lens, num_kv_heads,
//  scale, block_size, max_q_len, window_size, sink_size, stream)
PyObject* window_prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Call c;
  int hkv, bs, mq, w, s;
  float scale;
  if (n != 14 || !g_fn[kWindowPrefill] || !c.set_stream(a[13]) || !c.tensors(a, 7) || !get_int(a[7], &hkv) ||
      !get_float(a[8], &scale) || !get_int(a[9], &bs) || !get_int(a[10], &mq) || !get_int(a[11], &w) ||
      !get_int(a[12], &s))
    return general();
  return run([&] {
    return reinterpret_cast<decltype(&kvc_paged_prefill_window)>(g_fn[kWindowPrefill])(
        c.t[0], c.t[1], c.t[2], c.t[3], c.t[4], c.t[5], c.t[6], hkv, scale, bs, mq, w, s, c.stream);
  });
}

// (block_tables, kv_lens, qo_indptr, positions, slot_mapping, blocks_used, prefix_lens,
//  new_lens, free_blocks, block_size, stream)
PyObject* step_tables(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Call c;
  int bs;
  if (n != 11 || !g_fn[kStepTables] || !c.set_stream(a[10]) || !c.tensors(a, 9) || !get_int(a[9], &bs))
    return general();
  return run([&] {
    return reinterpret_cast<decltype(&kvc_step_tables)>(g_fn[kStepTables])(
        c.t[0], c.t[1], c.t[2], c.t[3], c.t[4], c.t[5], c.t[6], c.t[7], c.t[8], bs, c.stream);
  });
}

// (q_out, k_out, q, k, positions, cos_sin, q_weight, k_weight, eps, interleaved, stream)
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Call c;
  int inter;
  float eps;
  if (n != 11 || !g_fn[kRope] || !c.set_stream(a[10]) || !c.tensors(a, 8) || !get_float(a[8], &eps) ||
      !get_int(a[9], &inter))
    return general();
  return run([&] {
    return reinterpret_cast<decltype(&kvc_qk_norm_rope)>(g_fn[kRope])(c.t[0], c.t[1], c.t[2], c.t[3], c.t[4], c.t[5],
                                                                      c.t[6], c.t[7], eps, inter, c.stream);
  });
}

// (q_out, key_cache, value_cache, q, k, v, positions, cos_sin, q_weight, k_weight, slot_mapping,
//  eps, interleaved, stream)
PyObject* rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Call c;
  int inter;
  float eps;
  if (n != 14 || !g_fn[kRopeAppend] || !c.set_stream(a[13]) || !c.tensors(a, 11) || !get_float(a[11], &eps) ||
      !get_int(a[12], &inter))
    return general();
  return run([&] {
    return reinterpret_cast<decltype(&kvc_qk_norm_rope_append)>(g_fn[kRopeAppend])(
        c.t[0], c.t[1], c.t[2], c.t[3], c.t[4], c.t[5], c.t[6], c.t[7], c.t[8], c.t[9], eps, inter, c.t[10], c.stream);
  });
}

// bind(DeviceArray type, {symbol: address}): the library's functions, from the
// ctypes handle, so that both paths call the same library.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2 || !PyType_Check(a[0]) || !PyDict_Check(a[1])) {
    PyErr_SetString(PyExc_TypeError, "bind(type, dict)");
    return nullptr;
  }
  Py_INCREF(a[0]);
  Py_XDECREF(reinterpret_cast<PyObject*>(g_device_array));
  g_device_array = reinterpret_cast<PyTypeObject*>(a[0]);
  for (int i = 0; i < kNumFns; ++i) {
    PyObject* v = PyDict_GetItemString(a[1], kNames[i]);
    if (!v) {
      PyErr_Format(PyExc_KeyError, "%s", kNames[i]);
      return nullptr;
    }
    g_fn[i] = PyLong_AsVoidPtr(v);
    if (PyErr_Occurred()) return nullptr;
  }
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL, nullptr
PyMethodDef g_methods[] = {{"bind", FAST(bind)},
                           {"paged_attention_window", FAST(window_decode)},
                           {"paged_prefill_window", FAST(window_prefill)},
                           {"step_tables", FAST(step_tables)},
                           {"qk_norm_rope", FAST(rope)},
                           {"qk_norm_rope_append", FAST(rope_append)},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) {
  g_name_dltensor = PyUnicode_InternFromString("_dltensor");
  g_name_handle = PyUnicode_InternFromString("handle");
  g_name_requires_grad = PyUnicode_InternFromString("requires_grad");
  if (!g_name_dltensor || !g_name_handle || !g_name_requires_grad) return nullptr;
  return PyModule_Create(&g_module);
}
