// Python face of the batch operators for torch tensors (module quickvideo_amd._qp_torch).  These calls run once per layer and token; reading some
// ten tensors' pointers, shapes and strides through Python attributes and handing twenty arguments to ctypes takes 7 us, more than the kernels of a small
// step, and 1 us from here.  A call whose tensors are not what the kernels take is not made: REFUSED is returned and native.py says what was wrong.
// The entry points of libquickprefill.so come in as addresses (the library is loaded by native.py); nothing is kept between calls.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/quickprefill.h"

namespace {

constexpr long kRefused = 1000;      // no qp_status

struct Args {
  PyObject* const* a;
  bool ok = true;
  void *fn, *ctx, *stream;
  int64_t dev;
  explicit Args(PyObject* const* args) : a(args), fn(p(0)), ctx(p(1)), stream(p(3)), dev(i(2)) {}
  int64_t i(int k) {
    const int64_t v = PyLong_AsLongLong(a[k]);
    if (v == -1 && PyErr_Occurred()) ok = false;
    return v;
  }
  void* p(int k) {                                             // an address; above 2^63 too
    void* v = PyLong_AsVoidPtr(a[k]);
    if (!v && PyErr_Occurred()) ok = false;
    return v;
  }
  double f(int k) {
    const double v = PyFloat_AsDouble(a[k]);
    if (v == -1.0 && PyErr_Occurred()) ok = false;
    return v;
  }
  // the tensor at k when it has this type on this device (and is contiguous); NULL for None where that is allowed
  const at::Tensor* t(int k, at::ScalarType type, bool contiguous = true, bool none = false) {
    if (a[k] == Py_None && none) return nullptr;
    if (!THPVariable_Check(a[k])) { ok = false; return nullptr; }
    const at::Tensor& x = THPVariable_Unpack(a[k]);
    if (x.scalar_type() != type || x.get_device() != dev || x.layout() != at::kStrided || (contiguous && !x.is_contiguous())) { ok = false; return nullptr; }
    return &x;
  }
  bool shape(const at::Tensor* x, std::initializer_list<int64_t> want) {
    if (!ok || !x) return ok;
    if (!x->sizes().equals(at::IntArrayRef(want))) ok = false;
    return ok;
  }
};
const void* ptr(const at::Tensor* x) { return x ? x->const_data_ptr() : nullptr; }
void* out_ptr(const at::Tensor* x) { return x ? x->data_ptr() : nullptr; }

struct PageArgs { const at::Tensor *k, *v, *table, *seq_len, *n_new; int64_t stride, n_pages, size, width; };

bool pages(Args& A, int k, int64_t batch, int64_t n_kv, int64_t D, PageArgs& o, int table, int seq_len, int n_new) {
  o.k = A.t(k, at::kBFloat16, false);
  o.v = A.t(k + 1, at::kBFloat16, false);
  o.table = A.t(table, at::kInt);
  o.seq_len = A.t(seq_len, at::kInt);
  o.n_new = A.t(n_new, at::kInt, true, true);
  if (!A.ok || o.k->dim() != 4 || o.table->dim() != 2) return A.ok = false;
  o.n_pages = o.k->size(0); o.size = o.k->size(2); o.width = o.table->size(1);
  A.shape(o.k, {o.n_pages, n_kv, o.size, D});
  A.shape(o.v, {o.n_pages, n_kv, o.size, D});
  A.shape(o.table, {batch, o.width});
  A.shape(o.seq_len, {batch});
  A.shape(o.n_new, {batch});
  if (o.n_pages > INT32_MAX || o.size > INT32_MAX || o.width > INT32_MAX) A.ok = false;
  if (!A.ok || !o.k->strides().equals(o.v->strides()) || o.k->stride(1) != o.size * D || o.k->stride(2) != D || o.k->stride(3) != 1) return A.ok = false;
  o.stride = o.n_pages > 1 ? o.k->stride(0) : n_kv * o.size * D;
  return true;
}

PyObject* refused() {
  if (PyErr_Occurred()) return nullptr;
  return PyLong_FromLong(kRefused);
}

// (fn, ctx, dev, stream, qkv, cos, sin, seq_len, n_new, table, k_pages, v_pages, n_q, n_kv, D, q_out)
PyObject* batch_rope_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 16) { PyErr_SetString(PyExc_TypeError, "batch_rope_append: 16 arguments"); return nullptr; }
  Args A(args);
  const auto fn = reinterpret_cast<decltype(&qp_batch_rope_append)>(A.fn);
  const int64_t hq = A.i(12), hkv = A.i(13), D = A.i(14);
  const at::Tensor *qkv = A.t(4, at::kBFloat16), *cs = A.t(5, at::kBFloat16), *sn = A.t(6, at::kBFloat16), *q = A.t(15, at::kBFloat16);
  if (!A.ok || qkv->dim() != 3) return refused();
  const int64_t B = qkv->size(0), T = qkv->size(1), need = B * T * (D / 2);
  PageArgs pg;
  A.shape(qkv, {B, T, (hq + 2 * hkv) * D});
  A.shape(q, {B, T, hq, D});
  if (!A.ok || cs->numel() != need || sn->numel() != need || B * T > INT32_MAX || !pages(A, 10, B, hkv, D, pg, 9, 7, 8)) return refused();
  return PyLong_FromLong(fn((qp_ctx*)A.ctx, ptr(qkv), ptr(cs), ptr(sn), (int)B, (int)T, (const int32_t*)ptr(pg.seq_len), (const int32_t*)ptr(pg.n_new), (int)hq,
                            (int)hkv, (int)D, out_ptr(q), out_ptr(pg.k), out_ptr(pg.v), pg.stride, (int)pg.n_pages, (int)pg.size, (const int32_t*)ptr(pg.table),
                            (int)pg.width, A.stream));
}

// (fn, ctx, dev, stream, q, k_prefix, v_prefix, prefix_head_stride, prefix_len, k_pages, v_pages, table, seq_len, n_new, n_q, n_kv, D, scale, out, workspace)
PyObject* batch_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 20) { PyErr_SetString(PyExc_TypeError, "batch_attn: 20 arguments"); return nullptr; }
  Args A(args);
  const auto fn = reinterpret_cast<decltype(&qp_batch_attn)>(A.fn);
  const int64_t stride = A.i(7), P = A.i(8), hq = A.i(14), hkv = A.i(15), D = A.i(16);
  const double scale = A.f(17);
  const at::Tensor *q = A.t(4, at::kBFloat16), *out = A.t(18, at::kBFloat16), *kp = nullptr, *vp = nullptr;
  if (!THPVariable_Check(args[19])) return refused();
  const at::Tensor& ws = THPVariable_Unpack(args[19]);
  if (!A.ok || q->dim() != 4 || ws.layout() != at::kStrided || ws.get_device() != A.dev || !ws.is_contiguous()) return refused();
  const int64_t B = q->size(0), T = q->size(1);
  A.shape(q, {B, T, hq, D});
  A.shape(out, {B, T, hq, D});
  if (P > 0) {
    kp = A.t(5, at::kBFloat16, false);
    vp = A.t(6, at::kBFloat16, false);
    if (!A.ok || P > (1LL << 40) || stride < 0 || stride > (1LL << 50)) return refused();
    const int64_t elements = (hkv - 1) * stride + P * D;
    for (const at::Tensor* x : {kp, vp})
      if (!x->has_storage() || (int64_t)(x->storage().nbytes() / 2) - x->storage_offset() < elements) return refused();
  }
  PageArgs pg;
  if (!A.ok || B * T > INT32_MAX || !pages(A, 9, B, hkv, D, pg, 11, 12, 13)) return refused();
  return PyLong_FromLong(fn((qp_ctx*)A.ctx, ptr(q), ptr(kp), ptr(vp), stride, P, ptr(pg.k), ptr(pg.v), pg.stride, (int)pg.n_pages, (int)pg.size,
                            (const int32_t*)ptr(pg.table), (int)pg.width, (const int32_t*)ptr(pg.seq_len), (const int32_t*)ptr(pg.n_new), (int)B, (int)T, (int)hq,
                            (int)hkv, (int)D, (float)scale, out_ptr(out), ws.data_ptr(), ws.nbytes(), A.stream));
}

// (fn, ctx, dev, stream, logits, drafts, n_draft, draft_probs, uniforms, temperature, n_accepted, tokens, workspace)
PyObject* verify_drafts(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 13) { PyErr_SetString(PyExc_TypeError, "verify_drafts: 13 arguments"); return nullptr; }
  Args A(args);
  const auto fn = reinterpret_cast<decltype(&qp_verify_drafts)>(A.fn);
  const double temperature = A.f(9);
  if (!THPVariable_Check(args[4]) || !THPVariable_Check(args[12])) return refused();
  const at::Tensor &lg = THPVariable_Unpack(args[4]), &ws = THPVariable_Unpack(args[12]);
  const bool f32 = lg.scalar_type() == at::kFloat;
  if ((!f32 && lg.scalar_type() != at::kBFloat16) || lg.layout() != at::kStrided || lg.get_device() != A.dev || lg.dim() != 3 || lg.size(1) < 1 ||
      ws.layout() != at::kStrided || ws.get_device() != A.dev || !ws.is_contiguous())
    return refused();
  const int64_t B = lg.size(0), T = lg.size(1) - 1, V = lg.size(2);
  const at::Tensor *drafts = A.t(5, at::kLong), *nd = A.t(6, at::kInt, true, true), *pr = T ? A.t(7, at::kFloat, false, true) : nullptr,
                   *u = A.t(8, at::kFloat, true, true), *acc = A.t(10, at::kInt), *tok = A.t(11, at::kLong);
  A.shape(drafts, {B, T});
  A.shape(nd, {B});
  A.shape(pr, {B, T, V});
  A.shape(u, {B, T + 1});
  A.shape(acc, {B});
  A.shape(tok, {B, T + 1});
  if (!A.ok || (V > 1 && (lg.stride(2) != 1 || (pr && pr->stride(2) != 1))) || B > INT32_MAX || T > INT32_MAX) return refused();
  return PyLong_FromLong(fn((qp_ctx*)A.ctx, lg.const_data_ptr(), f32, lg.stride(0), lg.stride(1), T ? (const int64_t*)ptr(drafts) : nullptr,
                            (const int32_t*)ptr(nd), (const float*)ptr(pr), pr ? pr->stride(0) : 0, pr ? pr->stride(1) : 0, (const float*)ptr(u), (int)B, (int)T, V,
                            (float)temperature, (int32_t*)out_ptr(acc), (int64_t*)out_ptr(tok), ws.data_ptr(), ws.nbytes(), A.stream));
}

// no C++ exception (a tensor without memory of its own, say) leaves through the C entry
template <PyObject* (*kCall)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  try {
    return kCall(self, args, n);
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyMethodDef kMethods[] = {
    {"batch_rope_append", (PyCFunction)(void (*)(void))guarded<batch_rope_append>, METH_FASTCALL, nullptr},
    {"batch_attn", (PyCFunction)(void (*)(void))guarded<batch_attn>, METH_FASTCALL, nullptr},
    {"verify_drafts", (PyCFunction)(void (*)(void))guarded<verify_drafts>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_qp_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" PyObject* PyInit__qp_torch(void) {
  PyObject* m = PyModule_Create(&kModule);
  if (m) PyModule_AddIntConstant(m, "REFUSED", kRefused);
  return m;
}
