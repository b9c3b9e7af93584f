// A Python module between the operators of ops/paged.py and ops/sampling.py and their entry points: it looks at a call's tensors, says whether the
// kernels take them, and launches. An operator on a token or two is all host time: us of the host for an append / one token's attention / logits, with the
// tensors' properties asked for one by one in Python and a foreign call of 25 packed numbers 13.3 / 11.3 / 12.2, with this 7.2 / 7.0 / 6.1, of which 2.5 are the
// launch and 1.4 to 1.8 the allocation of the result.
//
// Tensors are seen through the DLPack C exchange interface (version 1), by which a tensor describes itself without a Python object for every size:
// 0.07 us each. Nothing is owned: what a look returns holds addresses, and the caller keeps the tensors until it has launched.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>
#include <cstring>
#include <initializer_list>

#include "calls.h"

namespace {

struct DLTensor {                // of the DLPack specification, as the interface below
  void* data;
  int32_t device_type, device;
  int32_t ndim;
  uint8_t code, bits;
  uint16_t lanes;
  int64_t *shape, *strides;
  uint64_t byte_offset;
};
struct DLPackExchangeAPI {
  uint32_t major, minor;
  void* previous;
  void *allocate, *from_object, *to_object;
  int (*tensor_from_object)(void* object, DLTensor* out);
  int (*current_stream)(int32_t device_type, int32_t device, void** out);
};
enum { INT = 0, FLOAT = 2, BFLOAT = 4, CUDA = 2 };
constexpr long long MOST = 0x7fffffff;

const DLPackExchangeAPI* api;
int (*f_append)(const gf::PagedCall*, const float*, const float*, int, int, void*);
int (*f_attn)(const gf::PagedCall*, float, void*, long long, int, float*, void*);
int (*f_attn_one)(const gf::PagedCall*, float, int, float*, void*);
int (*f_logits)(const gf::LogitsCall*, void*);
// what the operators' `_observed` asks (ops/fused.py), here without its Python frames (0.15 us instead of 0.6), and whether gradients are recorded
PyObject *tracing, *transforms, *dispatch_modes, *function_modes, *only_device_contexts, *forward_ad, *grad_enabled, *requires_grad, *current_level;

// What a Python function of no arguments says; -1, and no exception, where it raises.
long said(PyObject* f) {
  PyObject* r = PyObject_CallNoArgs(f);
  const long v = !r ? -1 : r == Py_None ? 0 : PyLong_Check(r) ? PyLong_AsLong(r) : 1;       // truth values are numbers
  Py_XDECREF(r);
  if (PyErr_Occurred()) PyErr_Clear();
  return v;
}
// Whether something follows the operations of this call, or would record one on these tensors.
bool followed(std::initializer_list<PyObject*> tensors) {
  if (said(tracing) || said(transforms) || said(dispatch_modes)) return true;
  const long modes = said(function_modes);
  if (modes && (modes < 0 || said(only_device_contexts) != 1)) return true;
  PyObject* level = PyDict_GetItemWithError(forward_ad, current_level);      // borrowed
  if (!level || !PyLong_Check(level) || PyLong_AsLong(level) >= 0) {
    PyErr_Clear();
    return true;
  }
  if (!said(grad_enabled)) return false;
  for (PyObject* t : tensors) {
    if (t == Py_None || PyFloat_CheckExact(t)) continue;
    PyObject* r = PyObject_GetAttr(t, requires_grad);
    const bool yes = r == Py_True;
    Py_XDECREF(r);
    PyErr_Clear();                                 // not a tensor: not recorded
    if (yes) return true;
  }
  return false;
}

// A tensor's description; false, and no exception, for what is none.
struct View : DLTensor {
  bool of(PyObject* o) {
    if (api->tensor_from_object(o, this)) {
      PyErr_Clear();
      return false;
    }
    data = static_cast<char*>(data) + byte_offset;
    return true;
  }
  bool is(int code_, int bits_, int ndim_, int on) const {
    return code == code_ && bits == bits_ && lanes == 1 && ndim == ndim_ && device_type == CUDA && device == on;
  }
  // the stride of dimension i; `packed` where nothing goes by it
  long long stride(int i, long long packed) const {
    if (shape[i] <= 1) return packed;
    if (strides) return strides[i];
    long long s = 1;
    for (int j = ndim - 1; j > i; --j) s *= shape[j];
    return s;
  }
  bool ints(PyObject* o, long long n, int on) { return of(o) && is(INT, 32, 1, on) && shape[0] == n && stride(0, 1) == 1; }
  bool floats(PyObject* o, long long n, int on) { return of(o) && is(FLOAT, 32, 1, on) && shape[0] == n && stride(0, 1) == 1; }
  uintptr_t at() const { return reinterpret_cast<uintptr_t>(data); }
};

// x [T, heads, D], kpages, vpages, page_table, lens, cu or None: the call but for H and what is only known at its launch. `packed`: rows of x are dense and
// lie on 16-byte boundaries.
bool paged(PyObject* const* a, PyObject* pages_k, PyObject* pages_v, PyObject* table, PyObject* lens_, PyObject* cu_, gf::PagedCall& c, int& device,
           long long& heads, bool& packed) {
  View x, k, v, t, n, cu;
  if (!x.of(a[0])) return false;
  device = x.device;
  if (!x.is(BFLOAT, 16, 3, device) || !k.of(pages_k) || !k.is(BFLOAT, 16, 4, device) || !v.of(pages_v) || !v.is(BFLOAT, 16, 4, device) ||
      !t.of(table) || !t.is(INT, 32, 2, device) || std::memcmp(k.shape, v.shape, 4 * sizeof(int64_t)))
    return false;
  const long long P = k.shape[0], page = k.shape[1], Hk = k.shape[2], D = k.shape[3], B = t.shape[0], width = t.shape[1], T = x.shape[0];
  if (!n.ints(lens_, B, device) || B == 0 || T == 0 || x.shape[2] != D || D % 8 || D == 0 || t.stride(1, 1) != 1) return false;
  if (cu_ == Py_None ? T != B : !cu.ints(cu_, B + 1, device)) return false;
  if (P == 0 || Hk == 0 || page < 16 || page & (page - 1) || page > MOST || P > MOST / page || width > MOST / page || k.stride(3, 1) != 1 ||
      v.stride(3, 1) != 1 || ((k.at() | v.at()) & 15))
    return false;
  long long* st = c.strides;
  for (const View* w : {&k, &v}) {
    st[2] = w->stride(2, D);
    st[1] = w->stride(1, Hk * D);
    st[0] = w->stride(0, page * st[1]);
    if ((st[0] | st[1] | st[2]) & 7) return false;
    st += 3;
  }
  heads = x.shape[1];
  c.x = x.data;
  c.ldx = x.stride(0, heads * D);
  packed = x.stride(2, 1) == 1 && x.stride(1, D) == D && c.ldx % 8 == 0 && c.ldx >= heads * D && (x.at() & 15) == 0;
  c.kpages = k.data;
  c.vpages = v.data;
  c.table = (const int*)t.data;
  c.ld_table = t.stride(0, width);
  c.width = width;
  c.lens = (const int*)n.data;
  c.cu = cu_ == Py_None ? nullptr : (const int*)cu.data;
  c.B = B; c.T = T; c.Hk = Hk; c.D = D; c.page = page; c.pages = P;
  return true;
}

struct Append {
  gf::PagedCall c;
  const float *cos, *sin;
  int positions;
};

bool arguments(const char* what, Py_ssize_t got, Py_ssize_t want) {
  if (got != want) PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, not %zd", what, want, got);
  return got == want;
}

// append(qkv, H, Hk, kpages, vpages, page_table, lens, cu, cos, sin): (call, device, T, D, whether qkv is packed, the pools where they are not simply
// dense and apart), None for what the kernel does not take
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments("append", n, 10)) return nullptr;
  const long long H = PyLong_AsLongLong(a[1]), Hk = PyLong_AsLongLong(a[2]);
  if (PyErr_Occurred()) return nullptr;
  Append r{};
  int device;
  long long heads;
  bool packed;
  View cs, sn;
  if (followed({a[0], a[3], a[4], a[8], a[9]})) Py_RETURN_NONE;
  if (!paged(a, a[3], a[4], a[5], a[6], a[7], r.c, device, heads, packed) || H <= 0 || H > MOST || r.c.Hk != Hk || heads != H + 2 * Hk ||
      r.c.D % 16 || r.c.D > 4096 || !cs.of(a[8]) || !sn.of(a[9]))
    Py_RETURN_NONE;
  for (const View* t : {&cs, &sn})
    if (!t->is(FLOAT, 32, 2, device) || 2 * t->shape[1] != r.c.D || t->shape[0] != cs.shape[0] || t->shape[0] > MOST || t->stride(1, 1) != 1 ||
        t->stride(0, r.c.D / 2) != r.c.D / 2 || (t->at() & 15) || !t->data)
      Py_RETURN_NONE;
  r.c.H = H;
  r.cos = (const float*)cs.data;
  r.sin = (const float*)sn.data;
  r.positions = (int)cs.shape[0];
  const long long *k = r.c.strides, *v = k + 3, row = Hk * r.c.D, all = r.c.pages * r.c.page * row;
  const uintptr_t k0 = reinterpret_cast<uintptr_t>(r.c.kpages), v0 = reinterpret_cast<uintptr_t>(r.c.vpages);
  const bool apart = k[2] == r.c.D && v[2] == r.c.D && k[1] == row && v[1] == row && k[0] == r.c.page * row && v[0] == k[0] &&
                     (k0 > v0 ? k0 - v0 : v0 - k0) >= (uintptr_t)(2 * all);
  PyObject* pools = apart ? Py_NewRef(Py_None)
                          : Py_BuildValue("(KKLLLLLL)", (unsigned long long)k0, (unsigned long long)v0, k[0], k[1], k[2], v[0], v[1], v[2]);
  return pools ? Py_BuildValue("(y#iLLON)", (const char*)&r, (Py_ssize_t)sizeof r, device, r.c.T, r.c.D, packed ? Py_True : Py_False, pools) : nullptr;
}

// attention(q, kpages, vpages, page_table, lens, cu): (call, device, B, T, H, Hk, D, keys of a sequence at most, whether q is packed), None as above
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments("attention", n, 6)) return nullptr;
  gf::PagedCall c{};
  int device;
  bool packed;
  if (followed({a[0], a[1], a[2]})) Py_RETURN_NONE;
  if (!paged(a, a[1], a[2], a[3], a[4], a[5], c, device, c.H, packed) || (c.D != 64 && c.D != 128) || c.H == 0 || c.H > MOST || c.H % c.Hk ||
      c.H / c.Hk > 128)
    Py_RETURN_NONE;
  for (long long st : c.strides)
    if (st == 0) Py_RETURN_NONE;
  return Py_BuildValue("(y#iLLLLLLO)", (const char*)&c, (Py_ssize_t)sizeof c, device, c.B, c.T, c.H, c.Hk, c.D, c.width * c.page,
                       packed ? Py_True : Py_False);
}

// What a look returned, to be completed.
template <typename T>
bool call_of(PyObject* o, T& c) {
  if (!PyBytes_Check(o) || PyBytes_GET_SIZE(o) != (Py_ssize_t)sizeof(T)) {
    PyErr_SetString(PyExc_TypeError, "not a call");
    return false;
  }
  std::memcpy(&c, PyBytes_AS_STRING(o), sizeof(T));
  return true;
}
bool memory_of(PyObject* o, View& v) {           // None: no memory
  if (o == Py_None) {
    v.data = nullptr;
    return true;
  }
  if (api->tensor_from_object(o, &v)) return false;
  v.data = static_cast<char*>(v.data) + v.byte_offset;
  return true;
}

// run_append(call, q, interleaved, status, stream)
PyObject* run_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Append r;
  View y;
  if (!arguments("run_append", n, 5) || !call_of(a[0], r) || !memory_of(a[1], y)) return nullptr;
  r.c.y = y.data;
  r.c.ldy = r.c.H * r.c.D;
  const int interleaved = PyObject_IsTrue(a[2]);
  r.c.status = (int*)PyLong_AsVoidPtr(a[3]);
  void* stream = PyLong_AsVoidPtr(a[4]);
  if (PyErr_Occurred()) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f_append(&r.c, r.cos, r.sin, r.positions, interleaved, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// run_attention(call, out, scale, one, workspace, parts, scratch, status, stream): gf_paged_attn_one where `one`, else gf_paged_attn
PyObject* run_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  gf::PagedCall c;
  View y, ws, few;
  if (!arguments("run_attention", n, 9) || !call_of(a[0], c) || !memory_of(a[1], y) || !memory_of(a[4], ws) || !memory_of(a[6], few)) return nullptr;
  c.y = y.data;
  c.ldy = y.ndim == 3 ? y.stride(0, c.H * c.D) : 0;
  const float scale = (float)PyFloat_AsDouble(a[2]);
  const int one = PyObject_IsTrue(a[3]);
  const long parts = PyLong_AsLong(a[5]);
  c.status = (int*)PyLong_AsVoidPtr(a[7]);
  void* stream = PyLong_AsVoidPtr(a[8]);
  if (PyErr_Occurred()) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = one ? f_attn_one(&c, scale, (int)parts, (float*)few.data, stream)
           : f_attn(&c, scale, ws.data, ws.data ? ws.shape[0] : 0, (int)parts, (float*)few.data, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// A penalty: a number, or 32-bit numbers of every row.
bool penalty(PyObject* o, long long B, int device, double& number, const float*& rows) {
  View v;
  if (PyFloat_Check(o) || PyLong_Check(o) || !v.of(o)) {
    number = PyFloat_AsDouble(o);
    if (!PyErr_Occurred()) return true;
    PyErr_Clear();
    return false;
  }
  if (!v.is(FLOAT, 32, 1, device) || v.shape[0] != B || v.stride(0, 1) != 1) return false;
  rows = (const float*)v.data;
  return true;
}

// logits(logits, tokens, token_lens, generated_from, repetition, presence, frequency, bias, allowed): (call, device, B, V, distance of rows), None as above
PyObject* logits(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments("logits", n, 9)) return nullptr;
  gf::LogitsCall c{};
  View x, t;
  if (followed({a[0], a[4], a[5], a[6], a[7]}) || !x.of(a[0]) || x.ndim != 2) Py_RETURN_NONE;
  const int device = x.device;
  c.dtype = x.is(FLOAT, 32, 2, device) ? 0 : x.is(BFLOAT, 16, 2, device) ? 1 : x.is(FLOAT, 16, 2, device) ? 2 : 3;
  const long long B = c.B = x.shape[0], V = c.V = x.shape[1], words = (V + 31) / 32;
  if (c.dtype == 3 || B == 0 || V == 0 || x.stride(1, 1) != 1) Py_RETURN_NONE;
  c.x = x.data;
  c.ldx = x.stride(0, V);
  if (a[1] != Py_None) {
    if (!t.of(a[1]) || !(t.is(INT, 32, 2, device) || t.is(INT, 64, 2, device)) || t.shape[0] != B || t.stride(1, 1) != 1) Py_RETURN_NONE;
    c.tokens = t.data;
    c.L = t.shape[1];
    c.ldt = t.stride(0, c.L);
    c.tokens64 = t.bits == 64;
    if (a[2] != Py_None && !t.ints(a[2], B, device)) Py_RETURN_NONE;
    c.token_lens = a[2] != Py_None ? (const int*)t.data : nullptr;
    if (a[3] != Py_None && !t.ints(a[3], B, device)) Py_RETURN_NONE;
    c.generated_from = a[3] != Py_None ? (const int*)t.data : nullptr;
  } else if (a[2] != Py_None || a[3] != Py_None) {
    Py_RETURN_NONE;
  }
  if (!penalty(a[4], B, device, c.repetition0, c.repetition) || !penalty(a[5], B, device, c.presence0, c.presence) ||
      !penalty(a[6], B, device, c.frequency0, c.frequency) || !(c.repetition || (c.repetition0 >= 0x1p-126 && c.repetition0 <= 0x1p126)))
    Py_RETURN_NONE;
  // [V] for all rows or [B, V]
  auto rows = [&](PyObject* o, int code, long long wide, const void*& data, long long& ld) {
    if (o == Py_None) return true;
    if (!t.of(o) || !(t.is(code, 32, 1, device) || (t.is(code, 32, 2, device) && t.shape[0] == B)) || t.shape[t.ndim - 1] != wide ||
        t.stride(t.ndim - 1, 1) != 1)
      return false;
    data = t.data;
    ld = t.ndim == 1 ? 0 : t.stride(0, wide);
    return true;
  };
  const void *bias = nullptr, *allowed = nullptr;
  if (!rows(a[7], FLOAT, V, bias, c.ldb) || !rows(a[8], INT, words, allowed, c.lda)) Py_RETURN_NONE;
  c.bias = (const float*)bias;
  c.allowed = (const unsigned*)allowed;
  return Py_BuildValue("(y#iLLL)", (const char*)&c, (Py_ssize_t)sizeof c, device, B, V, c.ldx);
}

// run_logits(call, out, distance of its rows, stream)
PyObject* run_logits(PyObject*, PyObject* const* a, Py_ssize_t n) {
  gf::LogitsCall c;
  View y;
  if (!arguments("run_logits", n, 4) || !call_of(a[0], c) || !memory_of(a[1], y)) return nullptr;
  c.y = y.data;
  c.ldy = PyLong_AsLongLong(a[2]);
  void* stream = PyLong_AsVoidPtr(a[3]);
  if (PyErr_Occurred()) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f_logits(&c, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// bind(exchange interface, addresses of gf_paged_append, gf_paged_attn, gf_paged_attn_one, gf_process_logits, the functions and the module that `followed`
// asks)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments("bind", n, 12)) return nullptr;
  auto* found = (const DLPackExchangeAPI*)PyCapsule_GetPointer(a[0], "dlpack_exchange_api");
  if (!found) return nullptr;
  if (found->major != 1 || !found->tensor_from_object) {
    PyErr_Format(PyExc_RuntimeError, "DLPack exchange interface of version %u, not 1", found->major);
    return nullptr;
  }
  void* f[4];
  for (int i = 0; i < 4; ++i) f[i] = PyLong_AsVoidPtr(a[i + 1]);
  if (PyErr_Occurred()) return nullptr;
  PyObject* const module_dict = PyModule_Check(a[10]) ? PyModule_GetDict(a[10]) : nullptr;
  if (!module_dict || !(requires_grad = PyUnicode_InternFromString("requires_grad")) || !(current_level = PyUnicode_InternFromString("_current_level"))) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "not a module");
    return nullptr;
  }
  PyObject** to[] = {&tracing, &transforms, &dispatch_modes, &function_modes, &only_device_contexts, &forward_ad, &grad_enabled};
  for (int i = 0; i < 7; ++i) {                    // kept for good
    PyObject* o = i == 5 ? module_dict : a[5 + i];
    Py_INCREF(o);
    *to[i] = o;
  }
  f_append = (decltype(f_append))f[0];
  f_attn = (decltype(f_attn))f[1];
  f_attn_one = (decltype(f_attn_one))f[2];
  f_logits = (decltype(f_logits))f[3];
  api = found;
  Py_RETURN_NONE;
}

#define FN(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FN(bind), FN(append), FN(run_append), FN(attention), FN(run_attention), FN(logits), FN(run_logits), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_gf_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__gf_calls() { return PyModule_Create(&module); }
