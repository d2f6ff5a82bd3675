// Python binding of the 8-bit operators for the ordinary call: plain CUDA tensors of the documented
// types, shapes and strides on their own device. It checks, allocates the outputs and calls the C ABI
// (include/qwen_asr_ext.h) without leaving C++: 4 to 6 us a call, where the same through ctypes takes
// 9 to 15. A call that does not fit returns None, and ops.py takes it from there: other strides, and the
// errors with their reasons.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstring>

#include "qwen_asr_ext.h"

namespace {

// The tensor of a plain torch.Tensor on a GPU that needs no gradient and has no tangent, or null.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != at::kStrided || (t.requires_grad() && c10::GradMode::is_enabled()) || t.is_neg() ||
      t._fw_grad(0).defined())
    return nullptr;
  return &t;
}

int dtype_of(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat ? QWEN_ASR_F32 : t.scalar_type() == at::kBFloat16 ? QWEN_ASR_BF16 : -1;
}

bool is(const at::Tensor* t, at::ScalarType type, int device, int dims) {
  return t && t->scalar_type() == type && t->get_device() == device && t->dim() == dims;
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

// As ops.py does: RuntimeError where CUDA refused, ValueError for the arguments.
PyObject* failed() {
  const char* why = qwen_asr_last_error();
  const bool cuda = !why || std::strstr(why, "launch failed") || std::strstr(why, "cannot use device");
  PyErr_SetString(cuda ? PyExc_RuntimeError : PyExc_ValueError, why ? why : "unknown");
  return nullptr;
}

template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// (x, weight, eps, residual or None) -> (q, scale, h)
PyObject* rms_norm_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    const at::Tensor *x = plain(a[0]), *w = plain(a[1]), *r = a[3] == Py_None ? nullptr : plain(a[3]);
    if (!x || x->dim() != 2 || (a[3] != Py_None && !r)) Py_RETURN_NONE;
    const int dev = x->get_device(), type = dtype_of(*x);
    const int64_t rows = x->size(0), d = x->size(1);
    if (type < 0 || rows < 1 || d < 1 || d > 32768 || x->stride(1) != 1 || x->stride(0) < d || !is(w, at::kFloat, dev, 1) ||
        w->size(0) != d || w->stride(0) != 1)
      Py_RETURN_NONE;
    if (r && (!is(r, x->scalar_type(), dev, 2) || r->size(0) != rows || r->size(1) != d || r->stride(1) != 1 ||
              r->stride(0) < d))
      Py_RETURN_NONE;
    if (!PyFloat_CheckExact(a[2])) Py_RETURN_NONE;
    const double eps = PyFloat_AS_DOUBLE(a[2]);
    if (!(eps >= 0)) Py_RETURN_NONE;
    const int64_t ld = (d + 15) / 16 * 16;
    at::Tensor q = at::empty({rows, ld}, x->options().dtype(at::kChar));
    at::Tensor scale = at::empty({rows}, x->options().dtype(at::kFloat));
    at::Tensor h;
    if (r) h = at::empty({rows, d}, x->options());
    if (qwen_asr_rms_norm_int8(x->data_ptr(), x->stride(0), r ? r->data_ptr() : nullptr, r ? r->stride(0) : 0,
                               (const float*)w->data_ptr(), (float)eps, type, rows, (int32_t)d, (int8_t*)q.data_ptr(), ld,
                               (float*)scale.data_ptr(), r ? h.data_ptr() : nullptr, d, dev, stream_of(dev)))
      return failed();
    PyObject* out = PyTuple_New(3);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(ld == d ? q : q.narrow(1, 0, d)));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(scale));
    if (r) {
      PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(h));
    } else {
      Py_INCREF(a[0]);
      PyTuple_SET_ITEM(out, 2, a[0]);
    }
    return out;
  });
}

// (xq, xs, wq, ws, residual or None, swiglu, bf16) -> out
PyObject* linear_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    const at::Tensor *xq = plain(a[0]), *xs = plain(a[1]), *wq = plain(a[2]), *ws = plain(a[3]);
    const at::Tensor* r = a[4] == Py_None ? nullptr : plain(a[4]);
    if (!xq || !wq || (a[4] != Py_None && !r)) Py_RETURN_NONE;
    const int dev = xq->get_device();
    if (!is(xq, at::kChar, dev, 2) || !is(wq, at::kChar, dev, 2) || !is(xs, at::kFloat, dev, 1) ||
        !is(ws, at::kFloat, dev, 1))
      Py_RETURN_NONE;
    const int64_t m = xq->size(0), k = xq->size(1), c = wq->size(0);
    const bool swiglu = a[5] == Py_True, bf16 = a[6] == Py_True;
    const at::ScalarType out_type = bf16 ? at::kBFloat16 : at::kFloat;
    if (m < 1 || c < 1 || k < 1 || k > 131071 || c > 0x7FFFFF00 || wq->size(1) != k || xs->size(0) != m ||
        ws->size(0) != c || xs->stride(0) != 1 || ws->stride(0) != 1 || xq->stride(1) != 1 || wq->stride(1) != 1 ||
        xq->stride(0) < k || wq->stride(0) < k || (swiglu && (r || c % 2)))
      Py_RETURN_NONE;
    if (((xq->stride(0) | wq->stride(0) | (int64_t)xq->data_ptr() | (int64_t)wq->data_ptr()) & 15)) Py_RETURN_NONE;
    if (r && (!is(r, out_type, dev, 2) || r->size(0) != m || r->size(1) != c || r->stride(1) != 1 || r->stride(0) < c))
      Py_RETURN_NONE;
    const int64_t width = swiglu ? c / 2 : c;
    at::Tensor out = at::empty({m, width}, xs->options().dtype(out_type));
    if (qwen_asr_linear_int8((const int8_t*)xq->data_ptr(), xq->stride(0), (const float*)xs->data_ptr(),
                             (const int8_t*)wq->data_ptr(), wq->stride(0), (const float*)ws->data_ptr(), m, (int32_t)c,
                             (int32_t)k, swiglu ? QWEN_ASR_LINEAR_SWIGLU : r ? QWEN_ASR_LINEAR_RESID : QWEN_ASR_LINEAR_STORE,
                             r ? r->data_ptr() : nullptr, r ? r->stride(0) : 0, out.data_ptr(), width,
                             bf16 ? QWEN_ASR_BF16 : QWEN_ASR_F32, dev, stream_of(dev)))
      return failed();
    return THPVariable_Wrap(out);
  });
}

// Descriptor of a Kv8Cache (a tuple of four tensors); false where it is none of the ordinary kind.
bool cache_of(PyObject* o, QwenAsrKv8& c, int& dev) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) return false;
  const at::Tensor* t[4];
  for (int i = 0; i < 4; ++i)
    if (!(t[i] = plain(PyTuple_GET_ITEM(o, i)))) return false;
  dev = t[0]->get_device();
  if (!is(t[0], at::kChar, dev, 4) || !is(t[1], at::kChar, dev, 4) || !is(t[2], at::kFloat, dev, 3) ||
      !is(t[3], at::kFloat, dev, 3))
    return false;
  const int64_t n = t[0]->size(0), h = t[0]->size(1), cap = t[0]->size(2), hd = t[0]->size(3), blocks = cap / 16;
  if (n < 1 || h < 1 || n > 65535 || h > 4096 || cap < 16 || cap % 16 || cap > 0x7FFFFFF0 || (hd != 64 && hd != 128)) return false;
  for (int i = 0; i < 4; ++i) {
    const at::Tensor& x = *t[i];
    if (i < 2 ? x.size(0) != n || x.size(1) != h || x.size(2) != cap || x.size(3) != hd || x.stride(1) != cap * hd ||
                    x.stride(2) != hd || x.stride(3) != 1
              : x.size(0) != n || x.size(1) != h || x.size(2) != blocks || x.stride(1) != blocks || x.stride(2) != 1)
      return false;
  }
  if (t[0]->stride(0) != t[1]->stride(0) || t[2]->stride(0) != t[3]->stride(0)) return false;
  c = QwenAsrKv8{(int8_t*)t[0]->data_ptr(), (int8_t*)t[1]->data_ptr(), (float*)t[2]->data_ptr(), (float*)t[3]->data_ptr(),
                 t[0]->stride(0), t[2]->stride(0), (int32_t)n, (int32_t)h, (int32_t)cap, (int32_t)hd};
  return true;
}

// Row positions and counts (None: all rows) with one stride for both.
bool index_of(PyObject* starts, PyObject* counts, int dev, int64_t n, const int32_t*& sp, const int32_t*& cp, int32_t& stride) {
  const at::Tensor *s = plain(starts), *c = counts == Py_None ? nullptr : plain(counts);
  if (!is(s, at::kInt, dev, 1) || s->size(0) != n || (counts != Py_None && (!is(c, at::kInt, dev, 1) || c->size(0) != n)))
    return false;
  const int64_t st = n > 1 ? s->stride(0) : 1;
  if (st < 1 || st > 0x7FFFFFFF || (c && n > 1 && c->stride(0) != st)) return false;
  sp = (const int32_t*)s->data_ptr();
  cp = c ? (const int32_t*)c->data_ptr() : nullptr;
  stride = (int32_t)st;
  return true;
}

// Rows [n][rows][heads][hd] of `type` with contiguous heads.
bool rows_of(const at::Tensor* t, at::ScalarType type, int dev, int64_t n, int64_t rows, int64_t heads, int64_t hd,
             QwenAsrRows& r) {
  if (!is(t, type, dev, 4) || t->size(0) != n || t->size(1) != rows || t->size(2) != heads || t->size(3) != hd ||
      t->stride(3) != 1 || t->stride(2) != hd)
    return false;
  r = QwenAsrRows{t->data_ptr(), t->stride(0), t->stride(1)};
  return true;
}

// (cache, k, v, starts, counts or None) -> True
PyObject* kv8_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    QwenAsrKv8 c;
    QwenAsrRows k, v;
    int dev;
    const int32_t *sp, *cp;
    int32_t stride;
    if (!cache_of(a[0], c, dev)) Py_RETURN_NONE;
    const at::Tensor *kt = plain(a[1]), *vt = plain(a[2]);
    if (!kt || kt->dim() != 4 || dtype_of(*kt) < 0) Py_RETURN_NONE;
    const int64_t rows = kt->size(1);
    if (rows < 1 || rows > 0x7FFFFFFF || !rows_of(kt, kt->scalar_type(), dev, c.n_seq, rows, c.n_kv, c.head_dim, k) ||
        !rows_of(vt, kt->scalar_type(), dev, c.n_seq, rows, c.n_kv, c.head_dim, v) ||
        !index_of(a[3], a[4], dev, c.n_seq, sp, cp, stride))
      Py_RETURN_NONE;
    if (qwen_asr_kv8_append(&c, &k, &v, dtype_of(*kt), (int32_t)rows, sp, cp, stride, dev, stream_of(dev))) return failed();
    for (int i = 0; i < 4; ++i) {  // the cache has changed in place
      const at::Tensor& t = THPVariable_Unpack(PyTuple_GET_ITEM(a[0], i));
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
    Py_RETURN_TRUE;
  });
}

// (cache, starts, rows, counts or None, bf16) -> (k, v)
PyObject* kv8_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    QwenAsrKv8 c;
    int dev;
    const int32_t *sp, *cp;
    int32_t stride;
    if (!cache_of(a[0], c, dev) || !index_of(a[1], a[3], dev, c.n_seq, sp, cp, stride) || !PyLong_CheckExact(a[2]))
      Py_RETURN_NONE;
    const long long rows = PyLong_AsLongLong(a[2]);
    if (PyErr_Occurred()) PyErr_Clear();
    if (rows < 1 || rows > 0x7FFFFFFF) Py_RETURN_NONE;
    const bool bf16 = a[4] == Py_True;
    const auto options = THPVariable_Unpack(a[1]).options().dtype(bf16 ? at::kBFloat16 : at::kFloat);
    at::Tensor k = at::empty({c.n_seq, rows, c.n_kv, c.head_dim}, options);
    at::Tensor v = at::empty({c.n_seq, rows, c.n_kv, c.head_dim}, options);
    const QwenAsrRows kr{k.data_ptr(), k.stride(0), k.stride(1)}, vr{v.data_ptr(), v.stride(0), v.stride(1)};
    if (qwen_asr_kv8_read(&c, &kr, &vr, bf16 ? QWEN_ASR_BF16 : QWEN_ASR_F32, (int32_t)rows, sp, cp, stride, dev, stream_of(dev)))
      return failed();
    PyObject* out = PyTuple_New(2);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(k));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(v));
    return out;
  });
}

// (q, cache, starts, counts or None, scale or None, max_len) -> out
PyObject* kv8_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    QwenAsrKv8 c;
    QwenAsrRows q;
    int dev;
    const int32_t *sp, *cp;
    int32_t stride;
    if (!cache_of(a[1], c, dev)) Py_RETURN_NONE;
    const at::Tensor* t = plain(a[0]);
    if (!t || t->dim() != 4 || dtype_of(*t) < 0) Py_RETURN_NONE;
    const int64_t rows = t->size(1), heads = t->size(2);
    if (rows < 1 || rows > (1 << 22) || heads < 1 || heads % c.n_kv || heads / c.n_kv > 256 ||
        !rows_of(t, t->scalar_type(), dev, c.n_seq, rows, heads, c.head_dim, q) ||
        !index_of(a[2], a[3], dev, c.n_seq, sp, cp, stride))
      Py_RETURN_NONE;
    double scale = 1.0 / std::sqrt((double)c.head_dim);
    if (a[4] != Py_None) {
      if (!PyFloat_CheckExact(a[4])) Py_RETURN_NONE;
      scale = PyFloat_AS_DOUBLE(a[4]);
    }
    if (!PyLong_CheckExact(a[5])) Py_RETURN_NONE;
    const long long max_len = PyLong_AsLongLong(a[5]);
    if (PyErr_Occurred()) PyErr_Clear();
    at::Tensor out = at::empty({c.n_seq, rows, heads, c.head_dim}, t->options());
    const QwenAsrRows o{out.data_ptr(), out.stride(0), out.stride(1)};
    if (qwen_asr_kv8_attention(&c, &q, &o, dtype_of(*t), (int32_t)rows, (int32_t)heads, sp, cp, stride, (float)scale,
                               max_len < 0 || max_len > c.capacity ? 0 : (int32_t)max_len, dev, stream_of(dev)))
      return failed();
    return THPVariable_Wrap(out);
  });
}

PyMethodDef kMethods[] = {
    {"rms_norm_int8", (PyCFunction)(void (*)(void))rms_norm_int8, METH_FASTCALL, nullptr},
    {"linear_int8", (PyCFunction)(void (*)(void))linear_int8, METH_FASTCALL, nullptr},
    {"kv8_append", (PyCFunction)(void (*)(void))kv8_append, METH_FASTCALL, nullptr},
    {"kv8_read", (PyCFunction)(void (*)(void))kv8_read, METH_FASTCALL, nullptr},
    {"kv8_attention", (PyCFunction)(void (*)(void))kv8_attention, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_ops_fast", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops_fast(void) { return PyModule_Create(&kModule); }
