// Python entry of the paged-cache calls: reads the tensors, allocates the outputs and calls the C ABI.
//
// These calls serve steps of one token, where the host's share is what a caller waits for: reading some twenty tensor fields,
// filling the structure and allocating through Python costs 6 to 9 us a call, here about 1 (a launch alone is 3.5).  Only
// calls that are right in every field are taken; any other returns None, and lvar_b200/kernels.py, which checks the same
// things one by one, says what is wrong or takes the rarer forms (a given output, tensors on a device that is not current).
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <exception>

#include "../../include/lvar_b200.h"

namespace {

// A plain tensor, or null.
const at::Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool is(const at::Tensor* t, at::ScalarType type, int64_t dims, int dev) {
  return t && t->is_cuda() && t->scalar_type() == type && t->dim() == dims && t->get_device() == dev;
}
// Optional arguments: None gives null; anything but a fitting tensor makes `ok` false.
const int32_t* ints(PyObject* o, int64_t n, int dev, bool& ok, bool optional) {
  if (optional && o == Py_None) return nullptr;
  const at::Tensor* t = tensor(o);
  ok = ok && is(t, at::kInt, 1, dev) && t->size(0) == n && (n <= 1 || t->stride(0) == 1);
  return ok ? static_cast<const int32_t*>(t->const_data_ptr()) : nullptr;
}
const float* floats(PyObject* o, int64_t n, int dev, bool& ok) {
  if (o == Py_None) return nullptr;
  const at::Tensor* t = tensor(o);
  ok = ok && is(t, at::kFloat, 1, dev) && t->size(0) == n && t->is_contiguous();
  return ok ? static_cast<const float*>(t->const_data_ptr()) : nullptr;
}
int32_t* status_word(PyObject* o, int dev, bool& ok) {
  if (o == Py_None) return nullptr;
  const at::Tensor* t = tensor(o);
  ok = ok && t && t->is_cuda() && t->scalar_type() == at::kInt && t->get_device() == dev && t->numel() >= 1;
  return ok ? static_cast<int32_t*>(t->data_ptr()) : nullptr;
}

bool fill_cache(lvar_paged_cache& c, PyObject* k_, PyObject* v_, PyObject* table_, PyObject* scales_, int& dev) {
  const at::Tensor *k = tensor(k_), *v = tensor(v_), *table = tensor(table_);
  const at::Tensor* s = scales_ == Py_None ? nullptr : tensor(scales_);
  if (!k || !k->is_cuda() || (scales_ != Py_None && !s)) return false;
  dev = static_cast<int>(k->get_device());
  const at::ScalarType type = s ? at::kFloat8_e4m3fn : at::kBFloat16;
  if (dev != c10::cuda::current_device() || !is(k, type, 4, dev) || !is(v, type, 4, dev) || !is(table, at::kInt, 2, dev) ||
      v->sizes() != k->sizes() || k->stride(3) != 1 || v->stride(3) != 1 || (table->size(1) > 1 && table->stride(1) != 1))
    return false;
  for (int i = 0; i < 4; ++i)
    if (k->size(i) < 1 || k->size(i) > INT32_MAX) return false;
  if (table->size(0) < 1 || table->size(0) > INT32_MAX || table->size(1) < 1 || table->size(1) > INT32_MAX) return false;
  c.k = k->data_ptr();
  c.k_sp = k->stride(0), c.k_sh = k->stride(1), c.k_sl = k->stride(2);
  c.v = v->data_ptr();
  c.v_sp = v->stride(0), c.v_sh = v->stride(1), c.v_sl = v->stride(2);
  if (s) {
    if (!is(s, at::kByte, 4, dev) || s->size(0) != k->size(0) || s->size(1) != k->size(1) || s->size(2) != k->size(2) ||
        s->size(3) != 2 || s->stride(2) != 2 || s->stride(3) != 1)
      return false;
    c.scales = static_cast<uint8_t*>(s->data_ptr());
    c.s_sp = s->stride(0), c.s_sh = s->stride(1);
  }
  c.table = static_cast<const int32_t*>(table->const_data_ptr());
  c.t_sb = table->stride(0);
  c.num_pages = (int32_t)k->size(0), c.Hkv = (int32_t)k->size(1), c.page_size = (int32_t)k->size(2), c.D = (int32_t)k->size(3);
  c.B = (int32_t)table->size(0), c.max_pages = (int32_t)table->size(1);
  return true;
}

at::Tensor make(at::IntArrayRef sizes, at::ScalarType type, int dev) {
  return at::empty(sizes, at::TensorOptions().dtype(type).device(at::kCUDA, static_cast<c10::DeviceIndex>(dev)));
}
void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream(); }

// No C++ exception leaves a call: an allocation that fails, say, becomes a Python error.
template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

#define LVAR_COUNT(n, name)                                              \
  if (nargs != (n)) {                                                    \
    PyErr_SetString(PyExc_TypeError, name " takes " #n " arguments");    \
    return nullptr;                                                      \
  }

// attn(q, k_pages, v_pages, table, lens, scale, scales, causal, max_len, return_stats, status, wait_limit_ns)
PyObject* attn(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  LVAR_COUNT(12, "attn");
  return guarded([&]() -> PyObject* {
    lvar_paged_attn_args p{};
    int dev;
    const at::Tensor* q = tensor(a[0]);
    if (!fill_cache(p.cache, a[1], a[2], a[3], a[6], dev) || !is(q, at::kBFloat16, 4, dev)) Py_RETURN_NONE;
    const int64_t B = q->size(0), Hq = q->size(1), T = q->size(2), D = q->size(3);
    if (B != p.cache.B || D != p.cache.D || Hq < 1 || Hq > INT32_MAX || Hq % p.cache.Hkv || T < 1 || T > INT32_MAX || q->stride(3) != 1)
      Py_RETURN_NONE;
    bool ok = true;
    p.lens = ints(a[4], B, dev, ok, false);
    p.dev_status = status_word(a[10], dev, ok);
    double scale = 0.0;
    if (a[5] != Py_None) {
      scale = PyFloat_AsDouble(a[5]);
      if (PyErr_Occurred()) return nullptr;
    }
    const int64_t room = (int64_t)p.cache.max_pages * p.cache.page_size;
    int64_t most = room < 1 << 30 ? room : 1 << 30;
    if (a[8] != Py_None) {
      most = PyLong_AsLongLong(a[8]);
      if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
      }
    }
    if (a[11] == Py_None) {
      p.wait_limit_ns = LVAR_DEFAULT_WAIT_NS;
    } else {
      p.wait_limit_ns = PyLong_AsUnsignedLongLong(a[11]);
      if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
      }
    }
    const int causal = PyObject_IsTrue(a[7]), stats = PyObject_IsTrue(a[9]);
    if (causal < 0 || stats < 0) return nullptr;
    if (!ok || most < 0 || most > 1 << 30) Py_RETURN_NONE;
    p.q = q->const_data_ptr();
    p.q_sb = q->stride(0), p.q_sh = q->stride(1), p.q_sl = q->stride(2);
    p.scale = a[5] == Py_None ? (float)(1.0 / std::sqrt((double)D)) : (float)scale;
    p.Hq = (int32_t)Hq, p.T = (int32_t)T, p.causal = causal, p.max_len = (int32_t)most;
    const int64_t work = lvar_paged_attn_workspace((int32_t)B, p.Hq, p.cache.Hkv, p.T, (int32_t)D, p.cache.scales != nullptr, p.max_len);
    if (work < 0) Py_RETURN_NONE;
    const at::Tensor o = make({B, Hq, T, D}, at::kBFloat16, dev);
    p.o = o.data_ptr();
    p.o_sb = Hq * T * D, p.o_sh = T * D, p.o_sl = D;
    at::Tensor M, L, space;
    if (stats) {
      M = make({B, Hq, T}, at::kFloat, dev);
      L = make({B, Hq, T}, at::kFloat, dev);
      p.M = static_cast<float*>(M.data_ptr());
      p.L = static_cast<float*>(L.data_ptr());
    }
    if (work > 0) {
      space = make({work}, at::kByte, dev);
      p.workspace = space.data_ptr();
      p.workspace_bytes = work;
    }
    if (lvar_paged_attn(&p, stream_of(dev)) != LVAR_OK) Py_RETURN_NONE;
    PyObject* out = THPVariable_Wrap(o);
    if (!stats || !out) return out;
    return Py_BuildValue("(NNN)", out, THPVariable_Wrap(M), THPVariable_Wrap(L));
  });
}

// append(k, v, k_pages, v_pages, table, start, scales, count, status) -> True
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  LVAR_COUNT(9, "append");
  return guarded([&]() -> PyObject* {
    lvar_paged_write_args p{};
    int dev;
    const at::Tensor *k = tensor(a[0]), *v = tensor(a[1]);
    if (!fill_cache(p.cache, a[2], a[3], a[4], a[6], dev) || !is(k, at::kBFloat16, 4, dev) || !is(v, at::kBFloat16, 4, dev) ||
        k->sizes() != v->sizes() || k->size(0) != p.cache.B || k->size(1) != p.cache.Hkv || k->size(3) != p.cache.D ||
        k->size(2) < 1 || k->size(2) > INT32_MAX || k->stride(3) != 1 || v->stride(3) != 1)
      Py_RETURN_NONE;
    bool ok = true;
    p.start = ints(a[5], p.cache.B, dev, ok, false);
    p.count = ints(a[7], p.cache.B, dev, ok, true);
    p.dev_status = status_word(a[8], dev, ok);
    if (!ok) Py_RETURN_NONE;
    p.k = k->const_data_ptr();
    p.k_sb = k->stride(0), p.k_sh = k->stride(1), p.k_sl = k->stride(2);
    p.v = v->const_data_ptr();
    p.v_sb = v->stride(0), p.v_sh = v->stride(1), p.v_sl = v->stride(2);
    p.L = (int32_t)k->size(2);
    if (lvar_paged_write(&p, stream_of(dev)) != LVAR_OK) Py_RETURN_NONE;
    Py_RETURN_TRUE;
  });
}

// prologue(q, k, v, k_pages, v_pages, table, start, scales, scale_mul, q_weight, k_weight, eps, rope_cos, rope_sin,
//          rope_halves, count, status) -> q
PyObject* prologue(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  LVAR_COUNT(17, "prologue");
  return guarded([&]() -> PyObject* {
    lvar_paged_write_args p{};
    int dev;
    const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *v = tensor(a[2]);
    if (!fill_cache(p.cache, a[3], a[4], a[5], a[7], dev) || !is(q, at::kBFloat16, 4, dev) || !is(k, at::kBFloat16, 4, dev) ||
        !is(v, at::kBFloat16, 4, dev))
      Py_RETURN_NONE;
    const int64_t B = q->size(0), L = q->size(1), Hq = q->size(2), D = q->size(3);
    if (B != p.cache.B || D != p.cache.D || L < 1 || L > INT32_MAX || Hq < 1 || Hq > INT32_MAX || Hq % p.cache.Hkv ||
        k->sizes() != v->sizes() || k->size(0) != B || k->size(1) != L || k->size(2) != p.cache.Hkv || k->size(3) != D ||
        q->stride(3) != 1 || k->stride(3) != 1 || v->stride(3) != 1)
      Py_RETURN_NONE;
    bool ok = true;
    p.start = ints(a[6], B, dev, ok, false);
    p.count = ints(a[15], B, dev, ok, true);
    p.dev_status = status_word(a[16], dev, ok);
    p.scale_mul = floats(a[8], Hq, dev, ok);
    p.q_weight = floats(a[9], D, dev, ok);
    p.k_weight = floats(a[10], D, dev, ok);
    if (a[8] != Py_None) {
      p.norm = 1;
      ok = ok && a[11] == Py_None && a[9] == Py_None && a[10] == Py_None;
    } else if (a[11] != Py_None) {
      p.norm = 2;
      p.eps = (float)PyFloat_AsDouble(a[11]);
      if (PyErr_Occurred()) return nullptr;
    } else {
      ok = ok && a[9] == Py_None && a[10] == Py_None;
    }
    if (a[12] != Py_None || a[13] != Py_None) {
      const at::Tensor *c = tensor(a[12]), *s = tensor(a[13]);
      ok = ok && is(c, at::kFloat, 2, dev) && is(s, at::kFloat, 2, dev) && c->sizes() == s->sizes() && c->size(1) == D / 2 &&
           c->size(0) >= 1 && c->size(0) <= INT32_MAX && c->is_contiguous() && s->is_contiguous();
      if (!ok) Py_RETURN_NONE;
      p.rope_cos = static_cast<const float*>(c->const_data_ptr());
      p.rope_sin = static_cast<const float*>(s->const_data_ptr());
      p.rope_rows = (int32_t)c->size(0);
    }
    p.rope_halves = PyObject_IsTrue(a[14]);
    if (p.rope_halves < 0) return nullptr;
    if (!ok) Py_RETURN_NONE;
    p.q = q->const_data_ptr();
    p.q_sb = q->stride(0), p.q_sl = q->stride(1), p.q_sh = q->stride(2);
    p.k = k->const_data_ptr();
    p.k_sb = k->stride(0), p.k_sl = k->stride(1), p.k_sh = k->stride(2);
    p.v = v->const_data_ptr();
    p.v_sb = v->stride(0), p.v_sl = v->stride(1), p.v_sh = v->stride(2);
    p.L = (int32_t)L, p.Hq = (int32_t)Hq;
    const at::Tensor out = make({B, Hq, L, D}, at::kBFloat16, dev);
    p.q_out = out.data_ptr();
    p.qo_sb = Hq * L * D, p.qo_sh = L * D, p.qo_sl = D;
    if (lvar_paged_write(&p, stream_of(dev)) != LVAR_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(out);
  });
}

// read(k_pages, v_pages, table, lens, n, scales, start, status) -> (k, v)
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  LVAR_COUNT(8, "read");
  return guarded([&]() -> PyObject* {
    lvar_paged_read_args p{};
    int dev;
    if (!fill_cache(p.cache, a[0], a[1], a[2], a[5], dev)) Py_RETURN_NONE;
    const int64_t n = PyLong_AsLongLong(a[4]), start = PyErr_Occurred() ? -1 : PyLong_AsLongLong(a[6]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    bool ok = n >= 1 && start >= 0 && n <= 1 << 30 && start <= 1 << 30;
    p.lens = ints(a[3], p.cache.B, dev, ok, false);
    p.dev_status = status_word(a[7], dev, ok);
    if (!ok) Py_RETURN_NONE;
    const int64_t H = p.cache.Hkv, D = p.cache.D;
    const at::Tensor k = make({p.cache.B, H, n, D}, at::kBFloat16, dev), v = make({p.cache.B, H, n, D}, at::kBFloat16, dev);
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.k_sb = p.v_sb = H * n * D, p.k_sh = p.v_sh = n * D, p.k_sl = p.v_sl = D;
    p.start = (int32_t)start, p.n = (int32_t)n;
    if (lvar_paged_read(&p, stream_of(dev)) != LVAR_OK) Py_RETURN_NONE;
    return Py_BuildValue("(NN)", THPVariable_Wrap(k), THPVariable_Wrap(v));
  });
}

PyMethodDef methods[] = {
    {"attn", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attn)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
    {"prologue", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(prologue)), METH_FASTCALL, nullptr},
    {"read", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(read)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_host() {
  PyObject* m = PyModule_Create(&module);
  // the torch and the Python whose classes the code above was compiled against
  if (m && PyModule_AddStringConstant(m, "built_for", LVAR_BUILT_FOR) < 0) Py_CLEAR(m);
  return m;
}
