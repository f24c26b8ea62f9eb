// Host path of the paged-cache operators: checks, output and workspace
// allocation and the launch of one call, in native code.
//
// A decode step calls these operators once per layer, and its kernels take a
// few microseconds: the same work written in Python took the host 17 us a call.
// A call that does not hold returns NotImplemented, and the Python entry names
// what is wrong (or serves what these functions leave to it: status checks, a
// device other than the current one).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <ATen/ATen.h>

#include <cmath>
#include <cstring>

#include "../../../include/moba_hip.h"

namespace {

PyObject* g_stream;   // torch._C._cuda_getCurrentRawStream
PyObject* g_device;   // torch._C._cuda_getDevice
PyObject* g_error;    // MobaHipError
PyObject *s_cos_sin, *s_rotary_dim, *s_interleaved, *s_packed, *s_meta;
PyTypeObject *t_rotary, *t_plan;

// Borrowed tensor of a Python argument, null if it is none.
const at::Tensor* tensor_in(PyObject* o) {
  return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
}
int type_code(at::ScalarType t) {
  return t == at::kBFloat16 ? 0 : t == at::kHalf ? 1 : -1;
}
// A strided device tensor (the only kind whose address is its data).
bool plain(const at::Tensor& t, int idx) {
  return t.is_cuda() && t.get_device() == idx && t.layout() == at::kStrided;
}
bool index_of(const at::Tensor* t, int idx, int64_t n) {
  return t && plain(*t, idx) && t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == n &&
         t->is_contiguous();
}

struct Pool {
  int code, idx;
  int64_t pages, page, hkv, d, slots, width;
  const char *k, *v;
  int64_t bytes;
};
bool pool_of(const at::Tensor* kc, const at::Tensor* vc, const at::Tensor* table, Pool& p) {
  if (!kc || !vc || !table || !kc->is_cuda() || kc->dim() != 4) return false;
  p.idx = kc->get_device();
  p.code = type_code(kc->scalar_type());
  if (p.code < 0 || !plain(*kc, p.idx) || !plain(*vc, p.idx) || vc->scalar_type() != kc->scalar_type() ||
      vc->sizes() != kc->sizes() || !kc->is_contiguous() || !vc->is_contiguous())
    return false;
  if (!plain(*table, p.idx) || table->scalar_type() != at::kInt || table->dim() != 2 ||
      !table->is_contiguous())
    return false;
  p.pages = kc->size(0); p.page = kc->size(1); p.hkv = kc->size(2); p.d = kc->size(3);
  p.slots = table->size(0); p.width = table->size(1);
  p.k = (const char*)kc->data_ptr(); p.v = (const char*)vc->data_ptr();
  p.bytes = kc->numel() * 2;
  return p.bytes > 0 && p.slots > 0 && p.width > 0 && p.pages * p.page < (1ll << 31) &&
         p.width * p.page < (1ll << 31);
}

// [N, heads, D] of the pool, dims contiguous.
bool tokens_of(const at::Tensor* t, const Pool& p, int64_t n) {
  return t && plain(*t, p.idx) && t->dim() == 3 && type_code(t->scalar_type()) == p.code &&
         t->size(0) == n && t->size(1) > 0 && t->size(2) == p.d && t->stride(2) == 1 &&
         t->stride(0) >= 0 && t->stride(1) >= 0 && !t->requires_grad();
}
struct Span {
  const char *lo, *hi;
};
Span span_of(const at::Tensor& t) {
  const char* p = (const char*)t.data_ptr();
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  return {p, p + (last + 1) * t.element_size()};
}
bool meet(const Span& a, const Span& b) { return a.lo < b.hi && b.lo < a.hi; }

// The current stream of the current device `idx`; false: another device is
// current (or an error is set).
bool stream_of(int idx, void*& stream) {
  PyObject* dev = PyObject_CallNoArgs(g_device);
  if (!dev) return false;
  const long cur = PyLong_AsLong(dev);
  Py_DECREF(dev);
  if (cur != idx) return false;
  PyObject* arg = PyLong_FromLong(idx);
  PyObject* s = arg ? PyObject_CallOneArg(g_stream, arg) : nullptr;
  Py_XDECREF(arg);
  if (!s) return false;
  stream = (void*)PyLong_AsUnsignedLongLong(s);
  Py_DECREF(s);
  return !PyErr_Occurred();
}

PyObject* not_here() {
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NOTIMPLEMENTED;
}
PyObject* failed(const char* name, int rc) {
  return PyErr_Format(g_error, "%s failed (%d): %s", name, rc, moba_hip_last_error());
}
bool int_attr(PyObject* o, PyObject* name, int64_t& out) {
  PyObject* v = PyObject_GetAttr(o, name);
  if (!v) return false;
  out = PyLong_AsLongLong(v);
  Py_DECREF(v);
  return !PyErr_Occurred();
}

// append_rotary(k, v, k_cache, v_cache, page_table, token_seq, token_pos,
//               rotary, q, q_out, offsets) -> q_out or None
PyObject* append_rotary(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 11) return PyErr_Format(PyExc_TypeError, "append_rotary takes 11 arguments");
  const at::Tensor *k = tensor_in(a[0]), *v = tensor_in(a[1]), *table = tensor_in(a[4]);
  const at::Tensor *seq = tensor_in(a[5]), *pos = tensor_in(a[6]);
  Pool p;
  if (!pool_of(tensor_in(a[2]), tensor_in(a[3]), table, p) || !k || k->dim() != 3) return not_here();
  const int64_t n = k->size(0);
  if (n < 1 || !tokens_of(k, p, n) || !tokens_of(v, p, n) || k->size(1) != p.hkv ||
      v->size(1) != p.hkv || !index_of(seq, p.idx, n) || !index_of(pos, p.idx, n))
    return not_here();
  const at::Tensor *q = nullptr, *offsets = nullptr;
  if (a[8] != Py_None && !((q = tensor_in(a[8])) && tokens_of(q, p, n))) return not_here();
  if (a[10] != Py_None && !((offsets = tensor_in(a[10])) && index_of(offsets, p.idx, p.slots)))
    return not_here();
  const int64_t hq = q ? q->size(1) : 0;
  if (n * (hq + 2 * p.hkv) * p.d >= (1ll << 31) || Py_TYPE(a[7]) != t_rotary) return not_here();
  int64_t rotary_dim, inter;
  PyObject* cs_obj = PyObject_GetAttr(a[7], s_cos_sin);
  if (!cs_obj) return nullptr;
  THPObjectPtr cs_ref(cs_obj);
  const at::Tensor* cs = tensor_in(cs_obj);
  if (!int_attr(a[7], s_rotary_dim, rotary_dim) || !int_attr(a[7], s_interleaved, inter)) return nullptr;
  // the table is an attribute that a caller may replace
  if (!cs || !plain(*cs, p.idx) || cs->scalar_type() != at::kFloat || cs->dim() != 3 ||
      !cs->is_contiguous() || cs->size(0) < 1 || cs->size(0) >= (1ll << 31) ||
      2 * cs->size(1) != rotary_dim || cs->size(2) != 2 || rotary_dim > p.d ||
      ((uintptr_t)cs->data_ptr() & 15))
    return not_here();

  const Span pools[2] = {{p.k, p.k + p.bytes}, {p.v, p.v + p.bytes}};
  if (meet(pools[0], pools[1])) return not_here();
  const at::Tensor* ins[3] = {k, v, q};
  Span spans[3];
  for (int i = 0; i < (q ? 3 : 2); ++i) {
    spans[i] = span_of(*ins[i]);
    if (meet(spans[i], pools[0]) || meet(spans[i], pools[1])) return not_here();
  }
  at::Tensor out;
  if (a[9] != Py_None) {
    const at::Tensor* given = tensor_in(a[9]);
    if (!q || !given || !tokens_of(given, p, n) || given->size(1) != hq || !given->is_contiguous())
      return not_here();
    const Span o = span_of(*given);
    if (meet(o, pools[0]) || meet(o, pools[1]) || meet(o, spans[0]) || meet(o, spans[1]) ||
        meet(o, spans[2]))
      return not_here();
    out = *given;
  }
  void* stream;
  if (!stream_of(p.idx, stream)) return not_here();
  if (q && !out.defined()) out = at::empty({n, hq, p.d}, q->options().requires_grad(false));
  const int rc = moba_hip_append_rotary(
      q ? q->data_ptr() : nullptr, q ? q->stride(0) : 0, q ? q->stride(1) : 0, k->data_ptr(),
      k->stride(0), k->stride(1), v->data_ptr(), v->stride(0), v->stride(1), p.code, (int)n, (int)hq,
      (int)p.hkv, (int)p.d, (const float*)cs->data_ptr(), (int)cs->size(0), (int)rotary_dim,
      (int)inter, (void*)p.k, (void*)p.v, (int)p.pages, (int)p.page, (const int*)table->data_ptr(),
      (int)p.slots, (int)p.width, (const int*)seq->data_ptr(), (const int*)pos->data_ptr(),
      offsets ? (const int*)offsets->data_ptr() : nullptr, q ? out.data_ptr() : nullptr, nullptr,
      stream);
  if (rc) return failed("moba_hip_append_rotary", rc);
  if (!q) Py_RETURN_NONE;
  if (a[9] != Py_None) {
    Py_INCREF(a[9]);
    return a[9];
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// The numbers of a plan, as SharedPrefixPlan packs them.
struct Plan {
  int64_t rows, hq, hkv, d, max_slot, max_prefix, max_suffix, n_items, rows_at, parts_at, parts,
      max_parts, uneven;
};

// shared_attention(q, k_cache, v_cache, page_table, suffix_lengths, plan, scale,
//                  out, lse) -> (out, lse)
PyObject* shared_attention(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 9) return PyErr_Format(PyExc_TypeError, "shared_attention takes 9 arguments");
  const at::Tensor *q = tensor_in(a[0]), *table = tensor_in(a[3]), *own = tensor_in(a[4]);
  Pool p;
  if (!pool_of(tensor_in(a[1]), tensor_in(a[2]), table, p) || Py_TYPE(a[5]) != t_plan) return not_here();
  THPObjectPtr packed(PyObject_GetAttr(a[5], s_packed)), meta_ref(PyObject_GetAttr(a[5], s_meta));
  if (!packed || !meta_ref) return nullptr;
  const at::Tensor* meta = tensor_in(meta_ref.get());
  if (!PyBytes_Check(packed.get()) || PyBytes_GET_SIZE(packed.get()) != (Py_ssize_t)sizeof(Plan) ||
      !meta || !plain(*meta, p.idx))
    return not_here();
  Plan x;
  memcpy(&x, PyBytes_AS_STRING(packed.get()), sizeof(x));
  if (meta->scalar_type() != at::kInt || meta->dim() != 1 || !meta->is_contiguous() ||
      meta->size(0) != x.parts_at / 4 + 3 * x.rows || ((uintptr_t)meta->data_ptr() & 15))
    return not_here();  // the records are an attribute that a caller may replace
  if (!q || !tokens_of(q, p, x.rows) || !q->is_contiguous() || q->size(1) != x.hq || p.hkv != x.hkv ||
      p.d != x.d || x.max_slot >= p.slots || x.max_prefix > p.width * p.page ||
      !index_of(own, p.idx, x.rows))
    return not_here();
  const double scale = a[6] == Py_None ? 1.0 / std::sqrt((double)x.d)
                       : PyFloat_Check(a[6]) ? PyFloat_AS_DOUBLE(a[6]) : 0.0;
  if (!(scale >= 0x1p-126 && scale < 1e30)) return not_here();
  if ((((uintptr_t)q->data_ptr()) | (uintptr_t)p.k | (uintptr_t)p.v) & 15) return not_here();
  if (a[7] != Py_None || a[8] != Py_None) return not_here();
  void* stream;
  if (!stream_of(p.idx, stream)) return not_here();
  const auto options = q->options().requires_grad(false);
  at::Tensor out = at::empty({x.rows, x.hq, x.d}, options);
  at::Tensor lse = at::empty({x.rows, x.hq}, options.dtype(at::kFloat));
  // partial sums [parts, D], then (max, sum) pairs
  const int64_t parts = x.parts * x.hq;
  at::Tensor work = at::empty({parts * (x.d + 2)}, options.dtype(at::kFloat));
  float* w = (float*)work.data_ptr();
  const char* m = (const char*)meta->data_ptr();
  const int rc = moba_hip_shared_attention(
      q->data_ptr(), p.code, (int)x.rows, (int)x.hq, (int)x.hkv, (int)x.d, (float)scale, p.k, p.v,
      (int)p.pages, (int)p.page, (const int*)table->data_ptr(), (int)p.width,
      (const int*)own->data_ptr(), 0, (int)std::min(x.max_suffix, p.width * p.page), (const int*)m,
      (int)x.n_items, (const int*)(m + x.rows_at), (const int*)(m + x.parts_at), (int)x.max_parts,
      (int)x.uneven, w, w + parts * x.d, out.data_ptr(), (float*)lse.data_ptr(), stream);
  if (rc) return failed("moba_hip_shared_attention", rc);
  THPObjectPtr po(THPVariable_Wrap(std::move(out))), pl(THPVariable_Wrap(std::move(lse)));
  return po && pl ? PyTuple_Pack(2, po.get(), pl.get()) : nullptr;
  END_HANDLE_TH_ERRORS
}

// bind(get_stream, get_device, error class, RotaryTable, SharedPrefixPlan)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  if (nargs != 5 || !PyType_Check(a[3]) || !PyType_Check(a[4]))
    return PyErr_Format(PyExc_TypeError, "bind takes two functions and three classes");
  for (int i = 0; i < 5; ++i) Py_INCREF(a[i]);  // for the life of the process
  g_stream = a[0]; g_device = a[1]; g_error = a[2];
  t_rotary = (PyTypeObject*)a[3];
  t_plan = (PyTypeObject*)a[4];
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
    {"append_rotary", (PyCFunction)(void (*)(void))append_rotary, METH_FASTCALL, nullptr},
    {"shared_attention", (PyCFunction)(void (*)(void))shared_attention, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) {
  s_cos_sin = PyUnicode_InternFromString("cos_sin");
  s_rotary_dim = PyUnicode_InternFromString("rotary_dim");
  s_interleaved = PyUnicode_InternFromString("interleaved");
  s_packed = PyUnicode_InternFromString("_packed");
  s_meta = PyUnicode_InternFromString("meta");
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", MOBA_BUILT_FOR)) Py_CLEAR(m);
  return m;
}
