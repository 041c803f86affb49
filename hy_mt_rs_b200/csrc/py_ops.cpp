// Python entry points of the calls a serving loop makes at every layer and
// step (hy_mt_rs_b200.paged, hy_mt_rs_b200.sampling): argument checks, output
// allocation and the call into libhyq in C++.  The device work of a decode step
// takes a few microseconds; the same checks in Python took 15 to 20.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../include/hyq.h"

namespace {

// Becomes a HyqError(code, message).
struct Refused {
  int code;
  std::string message;
};
[[noreturn]] void refuse(int code, std::string message) { throw Refused{code, std::move(message)}; }

PyObject* raise(int code, const std::string& message) {
  static PyObject* type = nullptr;
  if (!type) {
    PyObject* m = PyImport_ImportModule("hy_mt_rs_b200._native");
    if (!m) return nullptr;
    type = PyObject_GetAttrString(m, "HyqError");
    Py_DECREF(m);
    if (!type) return nullptr;
  }
  PyObject* args = Py_BuildValue("(is)", code, message.c_str());
  if (args) PyErr_SetObject(type, args);
  Py_XDECREF(args);
  return nullptr;
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(HYQ_E_INVALID, std::string(name) + ": expected a CUDA tensor");
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda()) refuse(HYQ_E_INVALID, std::string(name) + ": expected a CUDA tensor");
  return t;
}
const at::Tensor& typed(PyObject* o, const char* name, at::ScalarType type) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != type)
    refuse(HYQ_E_INVALID, std::string(name) + ": expected " + c10::toString(type) + ", got " + c10::toString(t.scalar_type()));
  return t;
}
const at::Tensor& plain(PyObject* o, const char* name, at::ScalarType type) {
  const at::Tensor& t = typed(o, name, type);
  if (!t.is_contiguous()) refuse(HYQ_E_INVALID, std::string(name) + ": expected a contiguous tensor");
  return t;
}
int64_t whole(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused{0, ""};
  return v;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Refused{0, ""};
  return v;
}

// One device for all of a call's tensors.
void same_device(const at::Tensor& a, const at::Tensor& b, const char* name) {
  if (a.device() != b.device()) refuse(HYQ_E_INVALID, std::string(name) + ": on another device");
}

// A contiguous tensor of `n` values on the device of `like`, or null for None.
const void* optional(PyObject* o, const at::Tensor& like, const char* name, at::ScalarType type, int64_t n) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = plain(o, name, type);
  same_device(like, t, name);
  if (t.numel() != n) refuse(HYQ_E_SHAPE, std::string(name) + ": expected " + std::to_string(n) + " values");
  return t.data_ptr();
}

hyq_paged_kv make_kv(const at::Tensor& q, PyObject* k_pages, PyObject* v_pages, PyObject* table) {
  const at::Tensor &k = tensor(k_pages, "k_pages"), &v = tensor(v_pages, "v_pages");
  const at::ScalarType type = k.scalar_type();
  if (type != at::kFloat && type != at::kHalf) refuse(HYQ_E_INVALID, "k_pages: expected a CUDA float32 or float16 tensor");
  if (k.dim() != 4 || k.stride(3) != 1)
    refuse(HYQ_E_SHAPE, "k_pages: expected [pages, kv_heads, page_size, head_dim], contiguous in head_dim");
  if (v.scalar_type() != type || v.sizes() != k.sizes() || v.strides() != k.strides())
    refuse(HYQ_E_SHAPE, "k_pages and v_pages differ in shape, strides or type");
  const at::Tensor& t = plain(table, "table", at::kInt);
  if (t.dim() != 2) refuse(HYQ_E_SHAPE, "table: expected [slots, table_width]");
  same_device(q, k, "k_pages");
  same_device(q, v, "v_pages");
  same_device(q, t, "table");
  for (int i = 1; i < 4; ++i)
    if (k.size(i) > INT32_MAX) refuse(HYQ_E_SHAPE, "k_pages: shape");
  return {k.data_ptr(), v.data_ptr(), type == at::kHalf ? HYQ_KV_F16 : HYQ_KV_F32, (int)k.size(1), (int)k.size(3),
          (int)k.size(2), k.size(0), k.stride(0), k.stride(1), k.stride(2),
          static_cast<const int32_t*>(t.data_ptr()), t.size(0), t.size(1)};
}

hyq_paged_batch make_batch(const at::Tensor& q, PyObject* row_start, PyObject* pos, PyObject* slot, int64_t tokens,
                           int64_t max_new, int64_t max_len) {
  const at::Tensor &r = plain(row_start, "row_start", at::kInt), &p = plain(pos, "pos", at::kInt);
  const int64_t seqs = p.numel();
  if (r.numel() != seqs + 1) refuse(HYQ_E_SHAPE, "row_start takes one more entry than pos");
  same_device(q, r, "row_start");
  same_device(q, p, "pos");
  const void* s = optional(slot, q, "slot", at::kInt, seqs);
  return {static_cast<const int32_t*>(s), static_cast<const int32_t*>(r.data_ptr()),
          static_cast<const int32_t*>(p.data_ptr()), seqs, tokens, max_new, max_len};
}

// [tokens, heads, head_dim] float32 whose heads are contiguous; its row stride.
int64_t row_stride(const at::Tensor& t, const char* name) {
  if (t.dim() != 3 || (t.size(2) > 1 && t.stride(2) != 1) || (t.size(1) > 1 && t.stride(1) != t.size(2)))
    refuse(HYQ_E_SHAPE, std::string(name) + ": expected [tokens, heads, head_dim] with contiguous heads");
  return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2);
}

at::Tensor output(PyObject* given, const at::Tensor& like, at::IntArrayRef shape, at::ScalarType type, const char* name) {
  if (given == Py_None) return at::empty(shape, like.options().dtype(type));
  const at::Tensor& t = typed(given, name, type);
  if (t.sizes() != shape) refuse(HYQ_E_SHAPE, std::string(name) + ": shape");
  same_device(like, t, name);
  return t;
}

void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

void check(int rc) {
  if (rc != HYQ_OK) refuse(rc, hyq_last_error());
}

template <typename F>
PyObject* guarded(Py_ssize_t given, Py_ssize_t wanted, F f) {
  if (given != wanted) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", wanted, given);
    return nullptr;
  }
  try {
    return f();
  } catch (const Refused& r) {
    return PyErr_Occurred() ? nullptr : raise(r.code, r.message);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// q, k_pages, v_pages, table, row_start, pos, max_new, max_len (-1: the table's
// reach), slot, out, workspace
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject* {
    const at::Tensor& q = typed(a[0], "q", at::kFloat);
    const hyq_paged_kv kv = make_kv(q, a[1], a[2], a[3]);
    const int64_t qs = row_stride(q, "q"), max_len = whole(a[7]);
    const hyq_paged_batch batch = make_batch(q, a[4], a[5], a[8], q.size(0), whole(a[6]),
                                             max_len < 0 ? kv.table_width * kv.page_size : max_len);
    if (q.size(2) != kv.head_dim) refuse(HYQ_E_SHAPE, "attention: head_dim of q and the pages");
    const at::Tensor out = output(a[9], q, q.sizes(), at::kFloat, "out");
    const at::Tensor& ws = plain(a[10], "workspace", at::kByte);
    same_device(q, ws, "workspace");
    size_t bytes = 0;
    check(hyq_paged_attention_workspace_bytes((int)q.size(1), kv.head_dim, &bytes));
    if ((size_t)ws.numel() < bytes) refuse(HYQ_E_SHAPE, "attention: the workspace takes " + std::to_string(bytes) + " bytes");
    check(hyq_paged_attention(&kv, &batch, static_cast<const float*>(q.data_ptr()), qs, (int)q.size(1),
                              static_cast<float*>(out.data_ptr()), row_stride(out, "out"), ws.data_ptr(), stream_of(q)));
    return THPVariable_Wrap(out);
  });
}

// q, k, v, k_pages, v_pages, table, row_start, pos, cos, sin, q_norm, k_norm,
// eps, norm_first, slot, out
PyObject* rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 16, [&]() -> PyObject* {
    const at::Tensor &q = typed(a[0], "q", at::kFloat), &k = typed(a[1], "k", at::kFloat), &v = typed(a[2], "v", at::kFloat);
    const hyq_paged_kv kv = make_kv(q, a[3], a[4], a[5]);
    const int64_t qs = row_stride(q, "q"), ks = row_stride(k, "k"), vs = row_stride(v, "v");
    // (positions are checked against the table's reach on the device; max_new
    // and max_len bound attention's work only)
    const hyq_paged_batch batch = make_batch(q, a[6], a[7], a[14], q.size(0), 0, 0);
    const at::Tensor out = output(a[15], q, q.sizes(), at::kFloat, "out");
    if (q.size(2) != kv.head_dim || k.size(0) != q.size(0) || k.size(1) != kv.kv_heads || k.size(2) != kv.head_dim ||
        v.sizes() != k.sizes())
      refuse(HYQ_E_SHAPE, "rope_append: shapes of q, k and v");
    same_device(q, k, "k");
    same_device(q, v, "v");
    const at::Tensor &cos = plain(a[8], "cos", at::kFloat), &sin = plain(a[9], "sin", at::kFloat);
    if (cos.dim() != 2 || cos.sizes() != sin.sizes() || 2 * cos.size(1) != kv.head_dim)
      refuse(HYQ_E_SHAPE, "rope_append: cos and sin are [positions, head_dim / 2]");
    same_device(q, cos, "cos");
    same_device(q, sin, "sin");
    const void* q_norm = optional(a[10], q, "q_norm", at::kFloat, kv.head_dim);
    const void* k_norm = optional(a[11], q, "k_norm", at::kFloat, kv.head_dim);
    check(hyq_paged_rope_append(
        &kv, &batch, static_cast<const float*>(q.data_ptr()), qs, (int)q.size(1), static_cast<const float*>(k.data_ptr()), ks,
        static_cast<const float*>(v.data_ptr()), vs, static_cast<const float*>(cos.data_ptr()),
        static_cast<const float*>(sin.data_ptr()), cos.size(0),
        static_cast<const float*>(q_norm), static_cast<const float*>(k_norm), (float)number(a[12]),
        PyObject_IsTrue(a[13]), static_cast<float*>(out.data_ptr()), row_stride(out, "out"), stream_of(q)));
    return THPVariable_Wrap(out);
  });
}

// logits, u, temperature, top_k, top_p, min_p, token, prob
PyObject* sample(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const at::Tensor& x = typed(a[0], "logits", at::kFloat);
    if (x.dim() != 2 || (x.size(1) > 1 && x.stride(1) != 1)) refuse(HYQ_E_SHAPE, "sample: logits are [rows, n] with contiguous rows");
    const int64_t rows = x.size(0), cols = x.size(1);
    if (a[1] == Py_None) refuse(HYQ_E_INVALID, "u: expected a CUDA tensor");
    const void* u = optional(a[1], x, "u", at::kFloat, rows);
    const void* temperature = optional(a[2], x, "temperature", at::kFloat, rows);
    const void* top_k = optional(a[3], x, "top_k", at::kInt, rows);
    const void* top_p = optional(a[4], x, "top_p", at::kFloat, rows);
    const void* min_p = optional(a[5], x, "min_p", at::kFloat, rows);
    const at::Tensor token = output(a[6], x, {rows}, at::kInt, "token"), prob = output(a[7], x, {rows}, at::kFloat, "prob");
    if (!token.is_contiguous() || !prob.is_contiguous()) refuse(HYQ_E_INVALID, "sample: expected contiguous outputs");
    check(hyq_sample(static_cast<const float*>(x.data_ptr()), cols, rows > 1 ? x.stride(0) : cols, rows,
                     static_cast<const float*>(temperature), static_cast<const int32_t*>(top_k),
                     static_cast<const float*>(top_p), static_cast<const float*>(min_p), static_cast<const float*>(u),
                     static_cast<int32_t*>(token.data_ptr()), static_cast<float*>(prob.data_ptr()), stream_of(x)));
    PyObject *t = THPVariable_Wrap(token), *p = THPVariable_Wrap(prob);
    PyObject* both = t && p ? PyTuple_Pack(2, t, p) : nullptr;
    Py_XDECREF(t);
    Py_XDECREF(p);
    return both;
  });
}

PyMethodDef methods[] = {
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(attention)), METH_FASTCALL, nullptr},
    {"rope_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(rope_append)), METH_FASTCALL, nullptr},
    {"sample", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(sample)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" PyObject* PyInit__ops() { return PyModule_Create(&module); }
