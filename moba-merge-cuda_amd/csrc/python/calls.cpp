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
PyTypeObject *t_rotary, *t_plan, *t_pages;

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

// The table of a RotaryTable, an attribute that a caller may replace.
struct Angles {
  THPObjectPtr ref;
  const at::Tensor* cs = nullptr;
  int64_t rotary_dim = 0, inter = 0;
};
// 1: it serves heads of d on device idx; 0: not here; -1: an error is set.
int angles_of(PyObject* o, int idx, int64_t d, Angles& x) {
  if (Py_TYPE(o) != t_rotary) return 0;
  x.ref = THPObjectPtr(PyObject_GetAttr(o, s_cos_sin));
  if (!x.ref) return -1;
  if (!int_attr(o, s_rotary_dim, x.rotary_dim) || !int_attr(o, s_interleaved, x.inter)) return -1;
  const at::Tensor* cs = x.cs = tensor_in(x.ref.get());
  return cs && plain(*cs, idx) && cs->scalar_type() == at::kFloat && cs->dim() == 3 &&
         cs->is_contiguous() && cs->size(0) >= 1 && cs->size(0) < (1ll << 31) &&
         2 * cs->size(1) == x.rotary_dim && cs->size(2) == 2 && x.rotary_dim <= d &&
         !((uintptr_t)cs->data_ptr() & 15);
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
  if (n * (hq + 2 * p.hkv) * p.d >= (1ll << 31)) return not_here();
  Angles turn;
  if (angles_of(a[7], p.idx, p.d, turn) != 1) return not_here();

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
      (int)p.hkv, (int)p.d, (const float*)turn.cs->data_ptr(), (int)turn.cs->size(0), (int)turn.rotary_dim,
      (int)turn.inter, (void*)p.k, (void*)p.v, (int)p.pages, (int)p.page, (const int*)table->data_ptr(),
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

// A QuantizedPages and its table.
struct QPool {
  int code, idx;   // format of the codes
  int64_t pages, hkv, page, d, width, slots, table_width;
  const at::Tensor *k, *v, *ks, *vs, *table;
  Span spans[4];
  bool meets(const Span& x) const {
    return meet(x, spans[0]) || meet(x, spans[1]) || meet(x, spans[2]) || meet(x, spans[3]);
  }
};
bool qpool_of(PyObject* o, PyObject* table, QPool& p) {
  if (Py_TYPE(o) != t_pages || PyTuple_GET_SIZE(o) != 5 || !PyLong_CheckExact(PyTuple_GET_ITEM(o, 4))) return false;
  const at::Tensor* t[5];
  for (int i = 0; i < 4; ++i)
    if (!(t[i] = tensor_in(PyTuple_GET_ITEM(o, i)))) return false;
  if (!(t[4] = tensor_in(table))) return false;
  p.k = t[0]; p.v = t[1]; p.ks = t[2]; p.vs = t[3]; p.table = t[4];
  p.d = PyLong_AsLongLong(PyTuple_GET_ITEM(o, 4));
  if (PyErr_Occurred() || p.d < 8 || p.d > 256 || p.d % 8 || !p.k->is_cuda() || p.k->dim() != 4) return false;
  p.idx = p.k->get_device();
  const auto kind = p.k->scalar_type();
  p.code = kind == at::kChar ? 0 : kind == at::kFloat8_e4m3fn ? 1 : -1;
  p.pages = p.k->size(0); p.hkv = p.k->size(1); p.page = p.k->size(2); p.width = p.k->size(3);
  if (p.code < 0 || p.width != (p.d + 15) / 16 * 16 || p.k->numel() == 0) return false;
  for (int i = 0; i < 4; ++i) {
    if (!plain(*t[i], p.idx) || !t[i]->is_contiguous()) return false;
    if (i == 1 && (p.v->scalar_type() != kind || p.v->sizes() != p.k->sizes())) return false;
    if (i > 1 && (t[i]->scalar_type() != at::kFloat || t[i]->dim() != 3 || t[i]->size(0) != p.pages ||
                  t[i]->size(1) != p.hkv || t[i]->size(2) != p.page))
      return false;
    p.spans[i] = span_of(*t[i]);
    for (int j = 0; j < i; ++j)
      if (meet(p.spans[i], p.spans[j])) return false;
  }
  if (((uintptr_t)p.spans[0].lo | (uintptr_t)p.spans[1].lo) & 15) return false;
  if (!plain(*p.table, p.idx) || p.table->scalar_type() != at::kInt || p.table->dim() != 2 ||
      !p.table->is_contiguous() || p.table->numel() == 0)
    return false;
  p.slots = p.table->size(0); p.table_width = p.table->size(1);
  return p.pages * p.page < (1ll << 31) && p.table_width * p.page < (1ll << 31) &&
         p.pages * p.page * p.hkv <= 0xfffffff0ll / (p.width / 16);
}
// [n, heads, d] in 16 bits on the pool's device, dims contiguous.
bool rows_of(const at::Tensor* t, const QPool& p, int64_t n, int type) {
  return t && plain(*t, p.idx) && t->dim() == 3 && type >= 0 && type_code(t->scalar_type()) == type &&
         t->size(0) == n && t->size(1) > 0 && t->size(2) == p.d && t->stride(2) == 1 &&
         t->stride(0) >= 0 && t->stride(1) >= 0 && !t->requires_grad();
}

// quantized_append(k, v, pages, page_table, token_seq, token_pos, rotary, q,
//                  q_out, offsets) -> q_out or None
PyObject* quantized_append(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 10) return PyErr_Format(PyExc_TypeError, "quantized_append takes 10 arguments");
  const at::Tensor *k = tensor_in(a[0]), *v = tensor_in(a[1]), *seq = tensor_in(a[4]), *pos = tensor_in(a[5]);
  QPool p;
  if (!qpool_of(a[2], a[3], p) || !k || k->dim() != 3) return not_here();
  const int64_t n = k->size(0);
  const int type = type_code(k->scalar_type());
  if (n < 1 || !rows_of(k, p, n, type) || !rows_of(v, p, n, type) || k->size(1) != p.hkv ||
      v->size(1) != p.hkv || !index_of(seq, p.idx, n) || !index_of(pos, p.idx, n))
    return not_here();
  const at::Tensor *q = nullptr, *offsets = nullptr;
  Angles turn;
  if (a[6] == Py_None) {
    if (a[7] != Py_None || a[8] != Py_None || a[9] != Py_None) return not_here();
  } else {
    if (angles_of(a[6], p.idx, p.d, turn) != 1) return not_here();
    if (a[7] != Py_None && !((q = tensor_in(a[7])) && rows_of(q, p, n, type))) return not_here();
    if (a[9] != Py_None && !((offsets = tensor_in(a[9])) && index_of(offsets, p.idx, p.slots))) return not_here();
  }
  const int64_t hq = q ? q->size(1) : 0;
  if (n * (hq + 2 * p.hkv) * p.width >= (1ll << 33)) return not_here();
  const at::Tensor* ins[3] = {k, v, q};
  Span spans[3];
  for (int i = 0; i < (q ? 3 : 2); ++i) {
    spans[i] = span_of(*ins[i]);
    if (p.meets(spans[i])) return not_here();
  }
  at::Tensor out;
  if (a[8] != Py_None) {
    const at::Tensor* given = tensor_in(a[8]);
    if (!q || !rows_of(given, p, n, type) || given->size(1) != hq || !given->is_contiguous()) return not_here();
    const Span o = span_of(*given);
    if (p.meets(o) || meet(o, spans[0]) || meet(o, spans[1]) || meet(o, spans[2])) return not_here();
    out = *given;
  }
  void* stream;
  if (!stream_of(p.idx, stream)) return not_here();
  if (q && !out.defined()) out = at::empty({n, hq, p.d}, q->options().requires_grad(false));
  const int rc = moba_hip_quantized_append(
      q ? q->data_ptr() : nullptr, q ? q->stride(0) : 0, q ? q->stride(1) : 0, k->data_ptr(), k->stride(0),
      k->stride(1), v->data_ptr(), v->stride(0), v->stride(1), type, (int)n, (int)hq, (int)p.hkv, (int)p.d,
      turn.cs ? (const float*)turn.cs->data_ptr() : nullptr, turn.cs ? (int)turn.cs->size(0) : 0,
      (int)turn.rotary_dim, (int)turn.inter, p.code, p.k->data_ptr(), p.v->data_ptr(),
      (float*)p.ks->data_ptr(), (float*)p.vs->data_ptr(), (int)p.pages, (int)p.page,
      (const int*)p.table->data_ptr(), (int)p.slots, (int)p.table_width, (const int*)seq->data_ptr(),
      (const int*)pos->data_ptr(), offsets ? (const int*)offsets->data_ptr() : nullptr,
      q ? out.data_ptr() : nullptr, nullptr, stream);
  if (rc) return failed("moba_hip_quantized_append", rc);
  if (!q) Py_RETURN_NONE;
  if (a[8] != Py_None) {
    Py_INCREF(a[8]);
    return a[8];
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// quantized_read(pages, page_table, token_seq, token_pos, 0 bf16 or 1 fp16) -> (k, v)
PyObject* quantized_read(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 5) return PyErr_Format(PyExc_TypeError, "quantized_read takes 5 arguments");
  const at::Tensor *seq = tensor_in(a[2]), *pos = tensor_in(a[3]);
  const long type = PyLong_AsLong(a[4]);
  QPool p;
  if (PyErr_Occurred() || !qpool_of(a[0], a[1], p) || !seq || seq->dim() != 1) return not_here();
  const int64_t n = seq->size(0);
  if (n < 1 || !index_of(seq, p.idx, n) || !index_of(pos, p.idx, n) || n * p.hkv * (p.d / 8) >= (1ll << 31))
    return not_here();
  void* stream;
  if (!stream_of(p.idx, stream)) return not_here();
  const auto options = seq->options().dtype(type == 0 ? at::kBFloat16 : at::kHalf);
  at::Tensor k = at::empty({n, p.hkv, p.d}, options), v = at::empty({n, p.hkv, p.d}, options);
  const int rc = moba_hip_quantized_read(
      p.code, p.k->data_ptr(), p.v->data_ptr(), (const float*)p.ks->data_ptr(), (const float*)p.vs->data_ptr(),
      (int)p.pages, (int)p.page, (int)p.hkv, (int)p.d, (const int*)p.table->data_ptr(), (int)p.slots,
      (int)p.table_width, (const int*)seq->data_ptr(), (const int*)pos->data_ptr(), (int)n, (int)type,
      k.data_ptr(), v.data_ptr(), nullptr, stream);
  if (rc) return failed("moba_hip_quantized_read", rc);
  THPObjectPtr pk(THPVariable_Wrap(std::move(k))), pv(THPVariable_Wrap(std::move(v)));
  return pk && pv ? PyTuple_Pack(2, pk.get(), pv.get()) : nullptr;
  END_HANDLE_TH_ERRORS
}

// A positive int32 of a Python int; 0: none.
int64_t positive_of(PyObject* o) {
  if (!PyLong_CheckExact(o)) return 0;
  int over;
  const int64_t x = PyLong_AsLongLongAndOverflow(o, &over);
  return over || x < 1 || x >= (1ll << 31) ? 0 : x;
}

// quantized_attention(q, pages, page_table, q_seq, lengths, selected, chunk_size,
//                     max_length, scale) -> (out, lse)
PyObject* quantized_attention(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 9) return PyErr_Format(PyExc_TypeError, "quantized_attention takes 9 arguments");
  const at::Tensor *q = tensor_in(a[0]), *seq = tensor_in(a[3]), *lengths = tensor_in(a[4]);
  QPool p;
  if (!qpool_of(a[1], a[2], p) || !q || q->dim() != 3) return not_here();
  const int64_t n = q->size(0), hq = q->size(1);
  const int type = type_code(q->scalar_type());
  if (n < 1 || !rows_of(q, p, n, type) || hq % p.hkv || !q->is_contiguous() || ((uintptr_t)q->data_ptr() & 15) ||
      !index_of(seq, p.idx, n) || !index_of(lengths, p.idx, n))
    return not_here();
  int64_t limit = p.table_width * p.page, slots = 0, chunk = 0;
  if (a[7] != Py_None) {
    const int64_t given = positive_of(a[7]);
    if (!given) return not_here();
    limit = std::min(limit, given);
  }
  const at::Tensor* selected = nullptr;
  if (a[5] != Py_None) {
    selected = tensor_in(a[5]);
    chunk = positive_of(a[6]);
    if (!selected || !chunk || !plain(*selected, p.idx) || selected->scalar_type() != at::kInt ||
        selected->dim() != 3 || !selected->is_contiguous() || selected->size(0) != n || selected->size(1) != hq)
      return not_here();
    slots = selected->size(2);
    if (slots < 1 || slots > 16) return not_here();
    chunk = std::min(chunk, limit);
  } else if (a[6] != Py_None) {
    return not_here();
  }
  const double scale = a[8] == Py_None ? 1.0 / std::sqrt((double)p.d)
                       : PyFloat_Check(a[8]) ? PyFloat_AS_DOUBLE(a[8]) : 0.0;
  if (!(scale >= 0x1p-126 && scale <= 1e30)) return not_here();
  if (n * hq >= (1ll << 31)) return not_here();
  const int64_t size = moba_hip_quantized_attention_work((int)n, (int)hq, (int)p.hkv, (int)p.d, (int)slots, (int)chunk,
                                                         (int)limit);
  if (size < 0) return not_here();
  void* stream;
  if (!stream_of(p.idx, stream)) return not_here();
  const auto options = q->options().requires_grad(false);
  at::Tensor out = at::empty({n, hq, p.d}, options);
  at::Tensor lse = at::empty({n, hq}, options.dtype(at::kFloat));
  at::Tensor work = at::empty({size}, options.dtype(at::kByte));
  const int rc = moba_hip_quantized_attention(
      q->data_ptr(), type, (int)n, (int)hq, (int)p.hkv, (int)p.d, (float)scale, p.code, p.k->data_ptr(),
      p.v->data_ptr(), (const float*)p.ks->data_ptr(), (const float*)p.vs->data_ptr(), (int)p.pages, (int)p.page,
      (const int*)p.table->data_ptr(), (int)p.slots, (int)p.table_width, (const int*)seq->data_ptr(),
      (const int*)lengths->data_ptr(), 0, (int)limit, selected ? (const int*)selected->data_ptr() : nullptr,
      (int)slots, (int)chunk, work.data_ptr(), out.data_ptr(), (float*)lse.data_ptr(), stream);
  if (rc) return failed("moba_hip_quantized_attention", rc);
  THPObjectPtr po(THPVariable_Wrap(std::move(out))), pl(THPVariable_Wrap(std::move(lse)));
  return po && pl ? PyTuple_Pack(2, po.get(), pl.get()) : nullptr;
  END_HANDLE_TH_ERRORS
}

// bind(get_stream, get_device, error class, RotaryTable, SharedPrefixPlan, QuantizedPages)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  if (nargs != 6 || !PyType_Check(a[3]) || !PyType_Check(a[4]) || !PyType_Check(a[5]))
    return PyErr_Format(PyExc_TypeError, "bind takes two functions and four classes");
  for (int i = 0; i < 6; ++i) Py_INCREF(a[i]);  // for the life of the process
  g_stream = a[0]; g_device = a[1]; g_error = a[2];
  t_rotary = (PyTypeObject*)a[3];
  t_plan = (PyTypeObject*)a[4];
  t_pages = (PyTypeObject*)a[5];
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
    {"append_rotary", (PyCFunction)(void (*)(void))append_rotary, METH_FASTCALL, nullptr},
    {"shared_attention", (PyCFunction)(void (*)(void))shared_attention, METH_FASTCALL, nullptr},
    {"quantized_append", (PyCFunction)(void (*)(void))quantized_append, METH_FASTCALL, nullptr},
    {"quantized_read", (PyCFunction)(void (*)(void))quantized_read, METH_FASTCALL, nullptr},
    {"quantized_attention", (PyCFunction)(void (*)(void))quantized_attention, METH_FASTCALL, nullptr},
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
