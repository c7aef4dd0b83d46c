// The calls of the small ops straight from torch tensors: what a Python layer spends on attributes and argument
// conversion (10 us a call) is more than their kernels take. Each function checks its arguments and calls the C entry
// point, whose address ext.py hands over with set_entry; it returns True if the call was made and succeeded. False
// leaves everything to ext.py: its checks name what is wrong, and its call reports the library's error.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/flash_whisper.h"

namespace {

decltype(&fw_prompt_attention) prompt_attention_entry = nullptr;
decltype(&fw_kv_q4_append) kv_q4_append_entry = nullptr;
decltype(&fw_kv_q4_read) kv_q4_read_entry = nullptr;
decltype(&fw_decode_attention_q4) decode_attention_q4_entry = nullptr;

// A tensor argument on GPU `dev`, or null.
const at::Tensor* tensor(PyObject* o, int64_t dev) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.get_device() == dev ? &t : nullptr;
}

int dtype_of(const at::Tensor& t) {
  return t.scalar_type() == at::kHalf ? FW_F16 : t.scalar_type() == at::kBFloat16 ? FW_BF16 : -1;
}

// [rows, heads, dim] with unit element stride, the others multiples of 8 elements, and 16-byte aligned data.
struct View {
  void* p;
  int64_t rows, heads, row, head;
};
bool view(const at::Tensor* t, at::ScalarType type, int64_t dim, View& v) {
  if (!t || t->scalar_type() != type || t->dim() != 3 || t->size(2) != dim || t->stride(2) != 1) return false;
  v.p = t->data_ptr();
  v.rows = t->size(0);
  v.heads = t->size(1);
  v.row = v.rows > 1 ? t->stride(0) : 0;
  v.head = v.heads > 1 ? t->stride(1) : 0;
  return ((v.row | v.head) & 7) == 0 && (reinterpret_cast<uintptr_t>(v.p) & 15) == 0;
}
// A view that is written: no two rows overlap.
bool apart(const View& v, int64_t dim) {
  if (v.rows > 1 && v.heads > 1)
    return v.row >= dim && v.head >= dim && (v.row >= (v.heads - 1) * v.head + dim || v.head >= (v.rows - 1) * v.row + dim);
  return (v.rows <= 1 || v.row >= dim) && (v.heads <= 1 || v.head >= dim);
}

const int64_t* index(const at::Tensor* t, int64_t n) {
  if (!t || t->scalar_type() != at::kLong || t->dim() != 1 || t->size(0) != n || !t->is_contiguous()) return nullptr;
  return static_cast<const int64_t*>(t->data_ptr());
}

struct Cache {
  void* p[4];
  int64_t n, heads, max_len, dim;
};
bool cache(PyObject* o, int64_t dev, Cache& c) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) return false;
  const at::Tensor* t[4];
  for (int i = 0; i < 4; ++i) {
    t[i] = tensor(PyTuple_GET_ITEM(o, i), dev);
    if (!t[i] || !t[i]->is_contiguous() || t[i]->scalar_type() != (i % 2 ? at::kHalf : at::kByte)) return false;
    c.p[i] = t[i]->data_ptr();
  }
  if (t[0]->dim() != 4) return false;
  c.n = t[0]->size(0);
  c.heads = t[0]->size(1);
  c.max_len = t[0]->size(2);
  c.dim = 2 * t[0]->size(3);
  if (c.max_len % 32 || (c.dim != 64 && c.dim != 128)) return false;
  return t[1]->sizes() == at::IntArrayRef({c.n, c.heads, c.max_len, c.dim / 32, 2}) &&
         t[2]->sizes() == at::IntArrayRef({c.n, c.heads, c.max_len / 8, c.dim / 4, 16}) &&
         t[3]->sizes() == at::IntArrayRef({c.n, c.heads, c.max_len / 8, c.dim / 32, 2, 8});
}

bool integer(PyObject* o, int64_t& v) {
  v = PyLong_Check(o) ? PyLong_AsLongLong(o) : -1;
  if (!PyErr_Occurred()) return PyLong_Check(o);
  PyErr_Clear();
  return false;
}
bool number(PyObject* o, float& v) {
  if (!PyFloat_Check(o)) return false;
  v = static_cast<float>(PyFloat_AS_DOUBLE(o));
  return true;
}
hipStream_t stream_of(PyObject* o) { return reinterpret_cast<hipStream_t>(PyLong_AsVoidPtr(o)); }
PyObject* made(int status) { return PyBool_FromLong(status == FW_OK); }
bool fits(int64_t n) { return n >= 0 && n <= 0x7FFFFFFF; }

// prompt_attention(q, k, v, out, cu_q, cu_k, scale, causal, device, stream)
PyObject* prompt_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  int64_t dev;
  float scale;
  if (n != 10 || !prompt_attention_entry || !integer(a[8], dev) || !number(a[6], scale) || !PyBool_Check(a[7])) Py_RETURN_FALSE;
  const at::Tensor *tq = tensor(a[0], dev), *cu_q = tensor(a[4], dev);
  if (!tq || tq->dim() != 3 || !cu_q || cu_q->dim() != 1) Py_RETURN_FALSE;
  const int dtype = dtype_of(*tq);
  const int64_t dim = tq->size(2), seqs = cu_q->size(0);
  const at::ScalarType type = tq->scalar_type();
  View q, k, v, out;
  if (dtype < 0 || (dim != 64 && dim != 128) || !view(tq, type, dim, q) || !view(tensor(a[1], dev), type, dim, k) ||
      !view(tensor(a[2], dev), type, dim, v) || !view(tensor(a[3], dev), type, dim, out) || !apart(out, dim) ||
      out.rows != q.rows || out.heads != q.heads || v.rows != k.rows || v.heads != k.heads)
    Py_RETURN_FALSE;
  const int64_t *q0 = index(cu_q, seqs), *k0 = index(tensor(a[5], dev), seqs);
  if (!q0 || !k0 || !fits(seqs) || !fits(q.heads)) Py_RETURN_FALSE;
  return made(prompt_attention_entry(q.p, q.row, q.head, k.p, k.row, k.head, v.p, v.row, v.head, out.p, out.row, out.head, q0, k0,
                                     static_cast<int>(seqs) - 1, q.rows, k.rows, static_cast<int>(q.heads),
                                     static_cast<int>(k.heads), static_cast<int>(dim), dtype, scale, a[7] == Py_True,
                                     stream_of(a[9])));
}

// The arguments that the append and the read share.
struct Packed {
  Cache c;
  View k, v;
  const int64_t *cu, *pos;
  int dtype;
};
bool packed(PyObject* ok, PyObject* ov, PyObject* ocu, PyObject* opos, PyObject* ocache, PyObject* odev, Packed& r) {
  int64_t dev;
  if (!integer(odev, dev) || !cache(ocache, dev, r.c)) return false;
  const at::Tensor* tk = tensor(ok, dev);
  if (!tk || (r.dtype = dtype_of(*tk)) < 0) return false;
  const at::ScalarType type = tk->scalar_type();
  if (!view(tk, type, r.c.dim, r.k) || !view(tensor(ov, dev), type, r.c.dim, r.v) || r.k.rows != r.v.rows ||
      r.k.heads != r.c.heads || r.v.heads != r.c.heads)
    return false;
  r.cu = index(tensor(ocu, dev), r.c.n + 1);
  r.pos = index(tensor(opos, dev), r.c.n);
  return r.cu && r.pos && fits(r.c.n) && fits(r.c.heads) && fits(r.c.max_len);
}

// kv_q4_append(k, v, cu, pos, cache, device, stream)
PyObject* kv_q4_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Packed r;
  if (n != 7 || !kv_q4_append_entry || !packed(a[0], a[1], a[2], a[3], a[4], a[5], r)) Py_RETURN_FALSE;
  return made(kv_q4_append_entry(r.k.p, r.k.row, r.k.head, r.v.p, r.v.row, r.v.head, r.k.rows, r.cu, r.pos, r.c.p[0], r.c.p[1],
                                 r.c.p[2], r.c.p[3], static_cast<int>(r.c.n), static_cast<int>(r.c.heads),
                                 static_cast<int>(r.c.max_len), static_cast<int>(r.c.dim), r.dtype, stream_of(a[6])));
}

// kv_q4_read(cache, cu, pos, k, v, device, stream)
PyObject* kv_q4_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Packed r;
  if (n != 7 || !kv_q4_read_entry || !packed(a[3], a[4], a[1], a[2], a[0], a[5], r) || !apart(r.k, r.c.dim) ||
      !apart(r.v, r.c.dim))
    Py_RETURN_FALSE;
  return made(kv_q4_read_entry(r.c.p[0], r.c.p[1], r.c.p[2], r.c.p[3], static_cast<int>(r.c.n), static_cast<int>(r.c.heads),
                               static_cast<int>(r.c.max_len), static_cast<int>(r.c.dim), r.cu, r.pos, r.k.rows, r.k.p, r.k.row,
                               r.k.head, r.v.p, r.v.row, r.v.head, r.dtype, stream_of(a[6])));
}

// decode_attention_q4(q, cache, lens, out, ws, scale, k_new, v_new, device, stream)
PyObject* decode_attention_q4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  int64_t dev;
  float scale;
  Cache c;
  if (n != 10 || !decode_attention_q4_entry || !integer(a[8], dev) || !number(a[5], scale) || !cache(a[1], dev, c)) Py_RETURN_FALSE;
  const at::Tensor *tq = tensor(a[0], dev), *ws = tensor(a[4], dev);
  if (!tq || !ws || ws->scalar_type() != at::kFloat || !ws->is_contiguous()) Py_RETURN_FALSE;
  const int dtype = dtype_of(*tq);
  const at::ScalarType type = tq->scalar_type();
  View q, out, k{}, v{};
  if (dtype < 0 || !view(tq, type, c.dim, q) || !view(tensor(a[3], dev), type, c.dim, out) || !apart(out, c.dim) ||
      q.rows != c.n || out.rows != c.n || out.heads != q.heads)
    Py_RETURN_FALSE;
  if ((a[6] == Py_None) != (a[7] == Py_None)) Py_RETURN_FALSE;
  if (a[6] != Py_None && (!view(tensor(a[6], dev), type, c.dim, k) || !view(tensor(a[7], dev), type, c.dim, v) ||
                          k.rows != c.n || v.rows != c.n || k.heads != c.heads || v.heads != c.heads))
    Py_RETURN_FALSE;
  const int64_t* lens = index(tensor(a[2], dev), c.n);
  if (!lens || !fits(c.n) || !fits(q.heads) || !fits(c.max_len)) Py_RETURN_FALSE;
  return made(decode_attention_q4_entry(
      q.p, q.row, q.head, c.p[0], c.p[1], c.p[2], c.p[3], lens, out.p, out.row, out.head, k.p, k.row, k.head, v.p, v.row, v.head,
      static_cast<int>(c.n), static_cast<int>(q.heads), static_cast<int>(c.heads), static_cast<int>(c.max_len),
      static_cast<int>(c.dim), dtype, scale, static_cast<float*>(ws->data_ptr()), ws->numel(), stream_of(a[9])));
}

// set_entry(name, address)
PyObject* set_entry(PyObject*, PyObject* args) {
  const char* name;
  unsigned long long address;
  if (!PyArg_ParseTuple(args, "sK", &name, &address)) return nullptr;
  const auto is = [&](const char* n) { return strcmp(name, n) == 0; };
  if (is("fw_prompt_attention")) prompt_attention_entry = reinterpret_cast<decltype(&fw_prompt_attention)>(address);
  else if (is("fw_kv_q4_append")) kv_q4_append_entry = reinterpret_cast<decltype(&fw_kv_q4_append)>(address);
  else if (is("fw_kv_q4_read")) kv_q4_read_entry = reinterpret_cast<decltype(&fw_kv_q4_read)>(address);
  else if (is("fw_decode_attention_q4")) decode_attention_q4_entry = reinterpret_cast<decltype(&fw_decode_attention_q4)>(address);
  else return PyErr_Format(PyExc_ValueError, "no entry point %s", name);
  Py_RETURN_NONE;
}

// No C++ exception of a tensor accessor (a tensor without storage, say) passes into the interpreter.
template <PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  try {
    return f(self, a, n);
  } catch (...) {
    Py_RETURN_FALSE;
  }
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<f>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(prompt_attention), FAST(kv_q4_append), FAST(kv_q4_read), FAST(decode_attention_q4),
                         {"set_entry", set_entry, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind() { return PyModule_Create(&module); }
