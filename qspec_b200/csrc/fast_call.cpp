// The call path in native code of the linear layers, of the operators around the paged caches and of the log probabilities of tokens: checks and one C call, for a product of a few microseconds that a Python path of ten would hide.
// Takes exactly the calls that the Python functions in ops.py take without an error; everything else (another type or layout, sizes that do not
// match, an empty batch, a workspace that is missing or too small) it leaves to them: returns None, nothing launched.
// 4 tokens, 4096 x 4096, W4A4, through nn.Linear4bit in a row of calls: 11.1 -> 6.3 us (the kernel 2.7).
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/qspec_b200.h"
#include "../../include/qspec_b200_seq.h"

namespace {

typedef decltype(&qspec_gemm_w4a4) Int4Fn;                    // (of qspec_gemm_w4a8, too)
typedef decltype(&qspec_gemm_w4a16) Fp16Fn;
static_assert(std::is_same<Int4Fn, decltype(&qspec_gemm_w4a8)>::value, "one call for both");

PyTypeObject* parameter_type = nullptr;

// A plain CUDA tensor, contiguous; subclasses with behaviour of their own are the Python path's business.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o) && Py_TYPE(o) != parameter_type) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous() ? &t : nullptr;
}
bool is_int4(const at::Tensor& t) { return t.scalar_type() == at::kChar || t.scalar_type() == at::kByte; }

// linear(address, kind, x, x_scale, weight, weight_scale, bias, out, workspaces, key): kind 0 W4A4, 1 W4A16, 2 W4A8; workspaces is the table of
// ops.py, key its kind. Returns the status of the call, or None.
PyObject* linear_(PyObject* const* a, Py_ssize_t n) {
  if (n != 10) {
    PyErr_SetString(PyExc_TypeError, "linear takes 10 arguments");
    return nullptr;
  }
  void* fn = PyLong_AsVoidPtr(a[0]);
  const long kind = PyLong_AsLong(a[1]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor *x = plain(a[2]), *w = plain(a[4]), *ws = plain(a[5]), *out = plain(a[7]);
  if (!fn || !x || !w || !ws || !out) Py_RETURN_NONE;
  const at::Tensor *xs = nullptr, *bias = nullptr;
  const auto type = out->scalar_type();
  if (type != at::kHalf && type != at::kBFloat16) Py_RETURN_NONE;
  if (kind == 1) {
    if (x->scalar_type() != type) Py_RETURN_NONE;
  } else {
    xs = plain(a[3]);
    if (!xs || xs->scalar_type() != type || !is_int4(*x) || (kind == 2 && x->scalar_type() != at::kChar)) Py_RETURN_NONE;
  }
  if (a[6] != Py_None) {
    bias = plain(a[6]);
    if (!bias || bias->scalar_type() != type) Py_RETURN_NONE;
  }
  if (!is_int4(*w) || ws->scalar_type() != type || w->dim() != 2 || x->dim() < 1) Py_RETURN_NONE;
  const int64_t N = w->size(0), K = 2 * w->size(1), cols = kind == 0 ? K / 2 : K;
  if (N <= 0 || K <= 0 || x->size(-1) != cols) Py_RETURN_NONE;
  const int64_t M = x->numel() / cols;
  if (M <= 0 || M > INT32_MAX || N > INT32_MAX || K > INT32_MAX || (xs && xs->numel() != M) || ws->numel() != N || out->numel() != M * N ||
      (bias && bias->numel() != N))
    Py_RETURN_NONE;
  PyObject* index = PyLong_FromLong(x->get_device());
  if (!index) return nullptr;
  PyObject* key = PyTuple_Pack(2, a[9], index);
  Py_DECREF(index);
  if (!key) return nullptr;
  PyObject* space = PyDict_GetItemWithError(a[8], key);      // borrowed
  Py_DECREF(key);
  if (!space) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
  const at::Tensor* room = plain(space);
  if (!room) Py_RETURN_NONE;
  void* stream = c10::cuda::getCurrentCUDAStream().stream();
  const void* b = bias ? bias->const_data_ptr() : nullptr;
  const int dtype = type == at::kBFloat16 ? 1 : 0;
  const void *xp = x->const_data_ptr(), *sp = xs ? xs->const_data_ptr() : nullptr, *wp = w->const_data_ptr(), *wsp = ws->const_data_ptr();
  void *op = out->mutable_data_ptr(), *rp = room->mutable_data_ptr();
  const size_t bytes = (size_t)room->nbytes();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = kind == 1 ? ((Fp16Fn)fn)(xp, (const int8_t*)wp, wsp, b, op, (int)M, (int)N, (int)K, dtype, rp, bytes, stream)
                     : ((Int4Fn)fn)((const int8_t*)xp, sp, (const int8_t*)wp, wsp, b, op, (int)M, (int)N, (int)K, dtype, rp, bytes, stream);
  Py_END_ALLOW_THREADS
  if (status == QSPEC_ERR_WORKSPACE) Py_RETURN_NONE;
  return PyLong_FromLong(status);
}

// Tensors without memory of their own (inside a functional transform) throw when asked for it: the Python path's business.
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    return linear_(a, n);
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
}

// ---- the paged caches, the verification of drafts, log probabilities -----------------------------------------------------------------------------
// The same bargain: what ops.py takes without an error, on the current device.
// Host time of a call: page_plan 15.1 -> 5.3 us, kv8_append 11.4 -> 5.0, kv8_attention 16.5 -> 3.9, verify_drafts 10.7 -> 3.9 (the kernels 3 to 12 at the
// smallest sizes).

const at::Tensor* on_device(PyObject* o, c10::DeviceIndex device) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.get_device() == device ? &t : nullptr;
}
// contiguous, of this type and shape
bool is(const at::Tensor* t, at::ScalarType type, at::IntArrayRef shape) { return t && t->scalar_type() == type && t->is_contiguous() && t->sizes() == shape; }
bool overlap(const at::Tensor& a, const at::Tensor& b) {
  const char *p = (const char*)a.const_data_ptr(), *q = (const char*)b.const_data_ptr();
  return p < q + b.nbytes() && q < p + a.nbytes();
}
bool fits(int64_t v) { return v <= INT32_MAX; }
int element(at::ScalarType t) { return t == at::kHalf ? QSPEC_DTYPE_F16 : t == at::kBFloat16 ? QSPEC_DTYPE_BF16 : -1; }
#define QSPEC_NOT_HERE(cond) do { if (cond) Py_RETURN_NONE; } while (0)
template <typename Call> PyObject* called(Call&& call) {
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = call();
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(status);
}
template <PyObject* (*F)(PyObject* const*, Py_ssize_t)> PyObject* guarded(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    return F(a, n);
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
}

// A cache: codes [pages, G, P, D], scales [pages, G].
struct Cache {
  const at::Tensor *k, *v, *ks, *vs;
  int64_t pages, G, P, D;
  bool take(PyObject* const* a, c10::DeviceIndex device) {
    k = on_device(a[0], device), v = on_device(a[1], device), ks = on_device(a[2], device), vs = on_device(a[3], device);
    if (!k || !v || k->dim() != 4) return false;
    pages = k->size(0), G = k->size(1), P = k->size(2), D = k->size(3);
    return is(k, at::kChar, {pages, G, P, D}) && is(v, at::kChar, {pages, G, P, D}) && is(ks, at::kFloat, {pages, G}) && is(vs, at::kFloat, {pages, G}) && fits(pages) && fits(G) &&
           fits(P) && fits(D);
  }
  void *kp() const { return k->mutable_data_ptr(); }
  void *vp() const { return v->mutable_data_ptr(); }
  float *ksp() const { return (float*)ks->mutable_data_ptr(); }
  float *vsp() const { return (float*)vs->mutable_data_ptr(); }
};

// page_plan(address, lengths, counts, table, free_pages, state, page_tokens, q_start, kv_len, positions, seq_ids, slots, state_out)
PyObject* page_plan(PyObject* const* a, Py_ssize_t n) {
  QSPEC_NOT_HERE(n != 13 || !PyLong_Check(a[6]));
  const auto device = c10::cuda::current_device();
  const at::Tensor* t[13] = {};
  for (int i = 1; i < 13; ++i)
    if (i != 6) QSPEC_NOT_HERE(!(t[i] = on_device(a[i], device)) || t[i]->scalar_type() != at::kInt || !t[i]->is_contiguous());
  QSPEC_NOT_HERE(t[1]->dim() != 1 || t[3]->dim() != 2 || t[4]->dim() != 1 || t[9]->dim() != 1);
  const int64_t B = t[1]->size(0), W = t[3]->size(1), T = t[9]->size(0), pages = t[4]->size(0);
  QSPEC_NOT_HERE(!fits(B) || !fits(W) || !fits(T) || !fits(pages) || t[2]->sizes() != at::IntArrayRef{B} || t[3]->size(0) != B || t[5]->sizes() != at::IntArrayRef{B + 1} ||
                 t[7]->sizes() != at::IntArrayRef{B + 1} || t[8]->sizes() != at::IntArrayRef{B} || t[10]->sizes() != at::IntArrayRef{T} ||
                 t[11]->sizes() != at::IntArrayRef{T} || t[12]->sizes() != at::IntArrayRef{B + 2});
  for (int i = 7; i < 13; ++i)
    for (int j = 1; j < i; ++j) QSPEC_NOT_HERE(j != 6 && overlap(*t[i], *t[j]));
  const auto fn = (decltype(&qspec_page_plan))PyLong_AsVoidPtr(a[0]);
  const long P = PyLong_AsLong(a[6]);
  if (PyErr_Occurred()) return nullptr;
  QSPEC_NOT_HERE(!fn || P < 0 || !fits(P));
  int* p[13];
  for (int i = 1; i < 13; ++i) p[i] = i == 6 ? nullptr : (int*)t[i]->mutable_data_ptr();
  void* stream = c10::cuda::getCurrentCUDAStream().stream();
  return called([&] { return fn(p[1], p[2], p[3], p[4], p[5], (int)B, (int)W, (int)pages, (int)P, (int)T, p[7], p[8], p[9], p[10], p[11], p[12], stream); });
}

// kv8_append(address, qkv, cos_sin_cache, positions, slots, k_codes, v_codes, k_scale, v_scale, q_out)
PyObject* kv8_append(PyObject* const* a, Py_ssize_t n) {
  QSPEC_NOT_HERE(n != 10);
  const auto device = c10::cuda::current_device();
  const at::Tensor *qkv = on_device(a[1], device), *cs = on_device(a[2], device), *pos = on_device(a[3], device), *slots = on_device(a[4], device), *q = nullptr;
  Cache c;
  QSPEC_NOT_HERE(!qkv || !cs || !c.take(a + 5, device) || qkv->dim() != 2 || qkv->stride(1) != 1 || element(qkv->scalar_type()) < 0 || c.D < 1);
  const int64_t T = qkv->size(0), H = qkv->size(1) / c.D - 2 * c.G;
  QSPEC_NOT_HERE(!fits(T) || H < 1 || !fits(H) || qkv->size(1) % c.D || cs->dim() != 2 || !fits(cs->size(0)) || !is(cs, qkv->scalar_type(), {cs->size(0), c.D}) ||
                 !is(pos, at::kInt, {T}) || !is(slots, at::kInt, {T}));
  if (a[9] != Py_None) {
    q = on_device(a[9], device);
    QSPEC_NOT_HERE(!q || q->scalar_type() != qkv->scalar_type() || q->sizes() != at::IntArrayRef({T, H, c.D}) || q->stride(2) != 1 || q->stride(1) != c.D);
  }
  const auto fn = (decltype(&qspec_kv8_append))PyLong_AsVoidPtr(a[0]);
  if (PyErr_Occurred()) return nullptr;
  QSPEC_NOT_HERE(!fn);
  void* stream = c10::cuda::getCurrentCUDAStream().stream();
  const void *x = qkv->const_data_ptr(), *table = cs->const_data_ptr();
  const int *pp = (const int*)pos->const_data_ptr(), *sp = (const int*)slots->const_data_ptr();
  void* out = q ? q->mutable_data_ptr() : nullptr;
  return called([&] {
    return fn(x, qkv->stride(0), table, (int)cs->size(0), pp, sp, c.kp(), c.vp(), c.ksp(), c.vsp(), out, q ? q->stride(0) : 0, (int)T, (int)H, (int)c.G, (int)c.D, (int)c.pages,
              (int)c.P, element(qkv->scalar_type()), stream);
  });
}

// kv8_read(address, k_codes, v_codes, k_scale, v_scale, slots, k_out, v_out)
PyObject* kv8_read(PyObject* const* a, Py_ssize_t n) {
  QSPEC_NOT_HERE(n != 8);
  const auto device = c10::cuda::current_device();
  const at::Tensor *slots = on_device(a[5], device), *ko = on_device(a[6], device), *vo = on_device(a[7], device);
  Cache c;
  QSPEC_NOT_HERE(!slots || !ko || !c.take(a + 1, device));
  const int64_t N = slots->numel();
  const auto type = ko->scalar_type();
  QSPEC_NOT_HERE(!fits(N) || element(type) < 0 || !is(slots, at::kInt, {N}) || !is(ko, type, {N, c.G, c.D}) || !is(vo, type, {N, c.G, c.D}));
  const auto fn = (decltype(&qspec_kv8_read))PyLong_AsVoidPtr(a[0]);
  if (PyErr_Occurred()) return nullptr;
  QSPEC_NOT_HERE(!fn);
  void* stream = c10::cuda::getCurrentCUDAStream().stream();
  const int* sp = (const int*)slots->const_data_ptr();
  void *kp = ko->mutable_data_ptr(), *vp = vo->mutable_data_ptr();
  return called([&] { return fn(c.kp(), c.vp(), c.ksp(), c.vsp(), sp, kp, vp, (int)N, (int)c.G, (int)c.D, (int)c.pages, (int)c.P, element(type), stream); });
}

// kv8_attention(address, q, k_codes, v_codes, k_scale, v_scale, table, q_start, kv_len, out, scale, workspace, max_tokens)
PyObject* kv8_attention(PyObject* const* a, Py_ssize_t n) {
  QSPEC_NOT_HERE(n != 13 || !PyFloat_Check(a[10]) || !(a[12] == Py_None || PyLong_Check(a[12])));
  const auto device = c10::cuda::current_device();
  const at::Tensor *q = on_device(a[1], device), *table = on_device(a[6], device), *start = on_device(a[7], device), *lens = on_device(a[8], device), *out = on_device(a[9], device),
                   *work = on_device(a[11], device);
  Cache c;
  QSPEC_NOT_HERE(!q || !table || !out || !work || !c.take(a + 2, device) || q->dim() != 3 || table->dim() != 2);
  const int64_t T = q->size(0), H = q->size(1), B = table->size(0), W = table->size(1);
  const auto type = q->scalar_type();
  QSPEC_NOT_HERE(element(type) < 0 || q->size(2) != c.D || q->stride(2) != 1 || out->scalar_type() != type || out->sizes() != q->sizes() || out->stride(2) != 1 || !fits(T) || T < 1 ||
                 !fits(H) || !fits(B) || !fits(W) || !fits(q->stride(1)) || !fits(out->stride(1)) || !is(table, at::kInt, {B, W}) || !is(start, at::kInt, {B + 1}) ||
                 !is(lens, at::kInt, {B}) || work->scalar_type() != at::kByte || !work->is_contiguous());
  const auto fn = (decltype(&qspec_kv8_attention))PyLong_AsVoidPtr(a[0]);
  const double scale = PyFloat_AsDouble(a[10]);
  const long most = a[12] == Py_None ? (long)T : PyLong_AsLong(a[12]);
  if (PyErr_Occurred()) return nullptr;
  QSPEC_NOT_HERE(!fn || !(scale > 0));
  void* stream = c10::cuda::getCurrentCUDAStream().stream();
  const void* qp = q->const_data_ptr();
  const int *tp = (const int*)table->const_data_ptr(), *sp = (const int*)start->const_data_ptr(), *lp = (const int*)lens->const_data_ptr();
  void *op = out->mutable_data_ptr(), *wp = work->mutable_data_ptr();
  return called([&] {
    return fn(qp, q->stride(0), (int)q->stride(1), c.kp(), c.vp(), c.ksp(), c.vsp(), tp, sp, lp, op, out->stride(0), (int)out->stride(1), (int)T, (int)B, (int)W, (int)H, (int)c.G,
              (int)c.D, (int)c.pages, (int)c.P, (int)(most < T ? most : T), (float)scale, element(type), wp, work->nbytes(), stream);
  });
}

// The cache in 4 bits: codes [pages, G, P, D / 2], words [pages, G, P].
struct Cache4 {
  const at::Tensor *k, *v, *kw, *vw;
  int64_t pages, G, P, D;
  bool take(PyObject* const* a, c10::DeviceIndex device) {
    k = on_device(a[0], device), v = on_device(a[1], device), kw = on_device(a[2], device), vw = on_device(a[3], device);
    if (!k || !v || k->dim() != 4) return false;
    pages = k->size(0), G = k->size(1), P = k->size(2), D = 2 * k->size(3);
    return is(k, at::kByte, {pages, G, P, D / 2}) && is(v, at::kByte, {pages, G, P, D / 2}) && is(kw, at::kShort, {pages, G, P}) && is(vw, at::kShort, {pages, G, P}) && fits(pages) &&
           fits(G) && fits(P) && fits(D);
  }
  void *kp() const { return k->mutable_data_ptr(); }
  void *vp() const { return v->mutable_data_ptr(); }
  void *kwp() const { return kw->mutable_data_ptr(); }
  void *vwp() const { return vw->mutable_data_ptr(); }
};

// kv4_append(address, qkv, cos_sin_cache, positions, slots, k_codes, v_codes, k_words, v_words, q_out, hadamard)
PyObject* kv4_append(PyObject* const* a, Py_ssize_t n) {
  QSPEC_NOT_HERE(n != 11 || !PyBool_Check(a[10]));
  const auto device = c10::cuda::current_device();
  const at::Tensor *qkv = on_device(a[1], device), *cs = on_device(a[2], device), *pos = on_device(a[3], device), *slots = on_device(a[4], device), *q = nullptr;
  Cache4 c;
  QSPEC_NOT_HERE(!qkv || !cs || !c.take(a + 5, device) || qkv->dim() != 2 || qkv->stride(1) != 1 || element(qkv->scalar_type()) < 0 || c.D < 1);
  const int64_t T = qkv->size(0), H = qkv->size(1) / c.D - 2 * c.G;
  QSPEC_NOT_HERE(!fits(T) || H < 1 || !fits(H) || qkv->size(1) % c.D || cs->dim() != 2 || !fits(cs->size(0)) || !is(cs, qkv->scalar_type(), {cs->size(0), c.D}) ||
                 !is(pos, at::kInt, {T}) || !is(slots, at::kInt, {T}));
  if (a[9] != Py_None) {
    q = on_device(a[9], device);
    QSPEC_NOT_HERE(!q || q->scalar_type() != qkv->scalar_type() || q->sizes() != at::IntArrayRef({T, H, c.D}) || q->stride(2) != 1 || q->stride(1) != c.D);
  }
  const auto fn = (decltype(&qspec_kv4_append))PyLong_AsVoidPtr(a[0]);
  if (PyErr_Occurred()) return nullptr;
  QSPEC_NOT_HERE(!fn);
  const int hadamard = a[10] == Py_True;
  void* stream = c10::cuda::getCurrentCUDAStream().stream();
  const void *x = qkv->const_data_ptr(), *table = cs->const_data_ptr();
  const int *pp = (const int*)pos->const_data_ptr(), *sp = (const int*)slots->const_data_ptr();
  void* out = q ? q->mutable_data_ptr() : nullptr;
  return called([&] {
    return fn(x, qkv->stride(0), table, (int)cs->size(0), pp, sp, c.kp(), c.vp(), c.kwp(), c.vwp(), out, q ? q->stride(0) : 0, (int)T, (int)H, (int)c.G, (int)c.D, (int)c.pages,
              (int)c.P, hadamard, element(qkv->scalar_type()), stream);
  });
}

// kv4_read(address, k_codes, v_codes, k_words, v_words, slots, k_out, v_out)
PyObject* kv4_read(PyObject* const* a, Py_ssize_t n) {
  QSPEC_NOT_HERE(n != 8);
  const auto device = c10::cuda::current_device();
  const at::Tensor *slots = on_device(a[5], device), *ko = on_device(a[6], device), *vo = on_device(a[7], device);
  Cache4 c;
  QSPEC_NOT_HERE(!slots || !ko || !c.take(a + 1, device));
  const int64_t N = slots->numel();
  const auto type = ko->scalar_type();
  QSPEC_NOT_HERE(!fits(N) || element(type) < 0 || !is(slots, at::kInt, {N}) || !is(ko, type, {N, c.G, c.D}) || !is(vo, type, {N, c.G, c.D}));
  const auto fn = (decltype(&qspec_kv4_read))PyLong_AsVoidPtr(a[0]);
  if (PyErr_Occurred()) return nullptr;
  QSPEC_NOT_HERE(!fn);
  void* stream = c10::cuda::getCurrentCUDAStream().stream();
  const int* sp = (const int*)slots->const_data_ptr();
  void *kp = ko->mutable_data_ptr(), *vp = vo->mutable_data_ptr();
  return called([&] { return fn(c.kp(), c.vp(), c.kwp(), c.vwp(), sp, kp, vp, (int)N, (int)c.G, (int)c.D, (int)c.pages, (int)c.P, element(type), stream); });
}

// kv4_attention(address, q, k_codes, v_codes, k_words, v_words, table, q_start, kv_len, out, scale, workspace, max_tokens)
PyObject* kv4_attention(PyObject* const* a, Py_ssize_t n) {
  QSPEC_NOT_HERE(n != 13 || !PyFloat_Check(a[10]) || !(a[12] == Py_None || PyLong_Check(a[12])));
  const auto device = c10::cuda::current_device();
  const at::Tensor *q = on_device(a[1], device), *table = on_device(a[6], device), *start = on_device(a[7], device), *lens = on_device(a[8], device), *out = on_device(a[9], device),
                   *work = on_device(a[11], device);
  Cache4 c;
  QSPEC_NOT_HERE(!q || !table || !out || !work || !c.take(a + 2, device) || q->dim() != 3 || table->dim() != 2);
  const int64_t T = q->size(0), H = q->size(1), B = table->size(0), W = table->size(1);
  const auto type = q->scalar_type();
  QSPEC_NOT_HERE(element(type) < 0 || q->size(2) != c.D || q->stride(2) != 1 || out->scalar_type() != type || out->sizes() != q->sizes() || out->stride(2) != 1 || !fits(T) || T < 1 ||
                 !fits(H) || !fits(B) || !fits(W) || !fits(q->stride(1)) || !fits(out->stride(1)) || !is(table, at::kInt, {B, W}) || !is(start, at::kInt, {B + 1}) ||
                 !is(lens, at::kInt, {B}) || work->scalar_type() != at::kByte || !work->is_contiguous());
  const auto fn = (decltype(&qspec_kv4_attention))PyLong_AsVoidPtr(a[0]);
  const double scale = PyFloat_AsDouble(a[10]);
  const long most = a[12] == Py_None ? (long)T : PyLong_AsLong(a[12]);
  if (PyErr_Occurred()) return nullptr;
  QSPEC_NOT_HERE(!fn || !(scale > 0));
  void* stream = c10::cuda::getCurrentCUDAStream().stream();
  const void* qp = q->const_data_ptr();
  const int *tp = (const int*)table->const_data_ptr(), *sp = (const int*)start->const_data_ptr(), *lp = (const int*)lens->const_data_ptr();
  void *op = out->mutable_data_ptr(), *wp = work->mutable_data_ptr();
  return called([&] {
    return fn(qp, q->stride(0), (int)q->stride(1), c.kp(), c.vp(), c.kwp(), c.vwp(), tp, sp, lp, op, out->stride(0), (int)out->stride(1), (int)T, (int)B, (int)W, (int)H, (int)c.G,
              (int)c.D, (int)c.pages, (int)c.P, (int)(most < T ? most : T), (float)scale, element(type), wp, work->nbytes(), stream);
  });
}

// seq_token_logprobs(address, logits, tokens, logprobs, entropy, ranks, top_logprobs, top_tokens, temperature)
PyObject* seq_token_logprobs(PyObject* const* a, Py_ssize_t n) {
  QSPEC_NOT_HERE(n != 9 || !PyFloat_Check(a[8]));
  const auto device = c10::cuda::current_device();
  const at::Tensor* x = on_device(a[1], device);
  QSPEC_NOT_HERE(!x || x->dim() != 2 || x->size(0) < 1 || x->size(1) < 1 || (x->stride(1) != 1 && x->size(1) > 1));
  const auto type = x->scalar_type();
  const int64_t rows = x->size(0), V = x->size(1), stride = rows > 1 ? x->stride(0) : std::max(x->stride(0), V);
  const int dtype = type == at::kFloat ? QSPEC_DTYPE_F32 : element(type);
  const at::Tensor* t[8] = {};
  for (int i = 2; i < 8; ++i)
    if (a[i] != Py_None) QSPEC_NOT_HERE(!(t[i] = on_device(a[i], device)) || !t[i]->is_contiguous());
  const int64_t top = t[6] && t[6]->dim() == 2 ? t[6]->size(1) : 0;
  QSPEC_NOT_HERE(dtype < 0 || !fits(rows) || !fits(V) || !fits(top) || (t[2] && !is(t[2], at::kLong, {rows})) || (t[3] && !is(t[3], at::kFloat, {rows})) ||
                 (t[4] && !is(t[4], at::kFloat, {rows})) || (t[5] && !is(t[5], at::kLong, {rows})) || (t[6] && !is(t[6], at::kFloat, {rows, top})) ||
                 (t[7] && !is(t[7], at::kLong, {rows, top})) || (!t[2] && (t[3] || t[5])) || !t[6] != !t[7]);
  const char* begin = (const char*)x->const_data_ptr();
  const char* end = begin + ((rows - 1) * stride + V) * x->element_size();
  for (int i = 3; i < 8; ++i) {
    if (!t[i] || !t[i]->numel()) continue;
    for (int j = 2; j < i; ++j) QSPEC_NOT_HERE(t[j] && t[j]->numel() && overlap(*t[i], *t[j]));
    const char* p = (const char*)t[i]->const_data_ptr();
    QSPEC_NOT_HERE(p < end && begin < p + t[i]->nbytes());
  }
  const auto fn = (decltype(&qspec_seq_token_logprobs))PyLong_AsVoidPtr(a[0]);
  const double temperature = PyFloat_AsDouble(a[8]);
  if (PyErr_Occurred()) return nullptr;
  QSPEC_NOT_HERE(!fn || !(temperature > 0));
  void* stream = c10::cuda::getCurrentCUDAStream().stream();
  void* p[8] = {};
  for (int i = 2; i < 8; ++i) p[i] = t[i] && t[i]->numel() ? t[i]->mutable_data_ptr() : nullptr;
  return called([&] {
    return fn(begin, stride, (const long long*)p[2], (float*)p[3], (float*)p[4], (long long*)p[5], (float*)p[6], (long long*)p[7], (int)rows, (int)V, (int)top, (float)temperature, dtype,
              stream);
  });
}

// verify_drafts(address, drafted, draft_probs, target_probs, uniform, tokens, emitted, draft_counts)
PyObject* verify_drafts(PyObject* const* a, Py_ssize_t n) {
  QSPEC_NOT_HERE(n != 8);
  const auto device = c10::cuda::current_device();
  const at::Tensor *p = on_device(a[3], device), *u = on_device(a[4], device), *tokens = on_device(a[5], device), *emitted = on_device(a[6], device), *d = nullptr, *q = nullptr,
                   *counts = nullptr;
  QSPEC_NOT_HERE(!p || !u || !tokens || !emitted || p->dim() != 3 || p->scalar_type() != at::kFloat || p->size(1) < 1 || p->stride(2) != 1);
  const int64_t B = p->size(0), k = p->size(1) - 1, V = p->size(2);
  QSPEC_NOT_HERE(B < 1 || V < 1 || !fits(B) || !fits(k) || !fits(V) || !is(u, at::kFloat, {B, k + 1}) || !is(tokens, at::kLong, {B, k + 1}) || !is(emitted, at::kLong, {B}));
  if (k) {
    d = on_device(a[1], device), q = on_device(a[2], device);
    QSPEC_NOT_HERE(!q || !is(d, at::kLong, {B, k}) || q->scalar_type() != at::kFloat || q->sizes() != at::IntArrayRef({B, k, V}) || q->stride(2) != 1);
  } else {
    QSPEC_NOT_HERE(a[1] != Py_None || a[2] != Py_None);
  }
  if (a[7] != Py_None) QSPEC_NOT_HERE(!(counts = on_device(a[7], device)) || !is(counts, at::kInt, {B}));
  for (const at::Tensor* out : {tokens, emitted})
    for (const at::Tensor* t : {d, u, counts}) QSPEC_NOT_HERE(t && overlap(*out, *t));
  QSPEC_NOT_HERE(overlap(*tokens, *emitted));
  const auto fn = (decltype(&qspec_verify_drafts))PyLong_AsVoidPtr(a[0]);
  if (PyErr_Occurred()) return nullptr;
  QSPEC_NOT_HERE(!fn);
  void* stream = c10::cuda::getCurrentCUDAStream().stream();
  const long long* dp = k ? (const long long*)d->const_data_ptr() : nullptr;
  const float *qp = k ? (const float*)q->const_data_ptr() : nullptr, *pp = (const float*)p->const_data_ptr(), *up = (const float*)u->const_data_ptr();
  const int* cp = counts ? (const int*)counts->const_data_ptr() : nullptr;
  long long *tp = (long long*)tokens->mutable_data_ptr(), *ep = (long long*)emitted->mutable_data_ptr();
  return called([&] {
    return fn(dp, qp, k ? q->stride(0) : 0, k ? q->stride(1) : 0, pp, p->stride(0), p->stride(1), up, cp, tp, ep, (int)B, (int)k, (int)V, stream);
  });
}

#define QSPEC_METHOD(name) {#name, (PyCFunction)(void (*)(void))guarded<name>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"linear", (PyCFunction)(void (*)(void))linear, METH_FASTCALL, nullptr}, QSPEC_METHOD(page_plan), QSPEC_METHOD(kv8_append), QSPEC_METHOD(kv8_read),
                         QSPEC_METHOD(kv8_attention), QSPEC_METHOD(kv4_append), QSPEC_METHOD(kv4_read),
                         QSPEC_METHOD(kv4_attention), QSPEC_METHOD(seq_token_logprobs), QSPEC_METHOD(verify_drafts), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast() {
  PyObject* nn = PyImport_ImportModule("torch.nn");
  if (!nn) return nullptr;
  PyObject* type = PyObject_GetAttrString(nn, "Parameter");
  Py_DECREF(nn);
  if (!type) return nullptr;
  parameter_type = (PyTypeObject*)type;                       // kept for the life of the process
  return PyModule_Create(&module);
}
