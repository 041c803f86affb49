// Python entry points of the calls a serving loop makes at every layer and
// step (hy_mt_rs_b200.paged, hy_mt_rs_b200.sampling): argument checks, output
// allocation and the call into libhyq in C++.  The device work of a decode step
// takes a few microseconds; the same checks in Python took 15 to 20.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
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

// A layer's pages, and the scales of 8-bit ones (None otherwise).
hyq_paged_kv8 make_kv(const at::Tensor& q, PyObject* k_pages, PyObject* v_pages, PyObject* table, PyObject* k_scale,
                      PyObject* v_scale) {
  const at::Tensor &k = tensor(k_pages, "k_pages"), &v = tensor(v_pages, "v_pages");
  const at::ScalarType type = k.scalar_type();
  const int kv_type = type == at::kFloat  ? HYQ_KV_F32
                      : type == at::kHalf ? HYQ_KV_F16
                      : type == at::kChar ? HYQ_KV_I8
                                          : HYQ_KV_F8;
  const bool coded = kv_type == HYQ_KV_I8 || kv_type == HYQ_KV_F8;
  if (kv_type == HYQ_KV_F8 && type != at::kFloat8_e4m3fn)
    refuse(HYQ_E_INVALID, "k_pages: expected a CUDA float32, float16, int8 or float8_e4m3fn tensor");
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
  hyq_paged_kv8 kv{{k.data_ptr(), v.data_ptr(), kv_type, (int)k.size(1), (int)k.size(3), (int)k.size(2), k.size(0), k.stride(0),
                    k.stride(1), k.stride(2), static_cast<const int32_t*>(t.data_ptr()), t.size(0), t.size(1)},
                   nullptr, nullptr, 0, 0, 0};
  if (!coded) {
    if (k_scale != Py_None || v_scale != Py_None) refuse(HYQ_E_INVALID, "k_scale, v_scale: these pages have none");
    return kv;
  }
  const at::Tensor &ks = typed(k_scale, "k_scale", at::kFloat), &vs = typed(v_scale, "v_scale", at::kFloat);
  same_device(q, ks, "k_scale");
  same_device(q, vs, "v_scale");
  if (ks.dim() != 3 || ks.size(0) != k.size(0) || ks.size(1) != k.size(1) || ks.size(2) != k.size(2))
    refuse(HYQ_E_SHAPE, "k_scale: expected [pages, kv_heads, page_size]");
  if (vs.sizes() != ks.sizes() || vs.strides() != ks.strides()) refuse(HYQ_E_SHAPE, "k_scale and v_scale differ in shape or strides");
  kv.k_scale = static_cast<float*>(ks.data_ptr());
  kv.v_scale = static_cast<float*>(vs.data_ptr());
  kv.scale_page_stride = ks.stride(0);
  kv.scale_head_stride = ks.stride(1);
  kv.scale_row_stride = ks.stride(2);
  return kv;
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

PyObject* pair(const at::Tensor& a, const at::Tensor& b) {
  PyObject *x = THPVariable_Wrap(a), *y = THPVariable_Wrap(b);
  PyObject* both = x && y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return both;
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
// reach), slot, out, workspace, k_scale, v_scale
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 13, [&]() -> PyObject* {
    const at::Tensor& q = typed(a[0], "q", at::kFloat);
    const hyq_paged_kv8 kv8 = make_kv(q, a[1], a[2], a[3], a[11], a[12]);
    const hyq_paged_kv& kv = kv8.kv;
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
    const c10::cuda::CUDAGuard device(q.device());
    check(hyq_paged_attention_kv8(&kv8, &batch, static_cast<const float*>(q.data_ptr()), qs, (int)q.size(1),
                                  static_cast<float*>(out.data_ptr()), row_stride(out, "out"), ws.data_ptr(), stream_of(q)));
    return THPVariable_Wrap(out);
  });
}

// q, k_pages, v_pages, table, row_start, pos, group_start, shared, max_new, max_len
// (-1: the table's reach), max_shared (-1: max_len), slot, out, workspace, k_scale,
// v_scale
PyObject* attention_shared(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 16, [&]() -> PyObject* {
    const at::Tensor& q = typed(a[0], "q", at::kFloat);
    const hyq_paged_kv8 kv8 = make_kv(q, a[1], a[2], a[3], a[14], a[15]);
    const hyq_paged_kv& kv = kv8.kv;
    const int64_t qs = row_stride(q, "q"), given = whole(a[9]), max_len = given < 0 ? kv.table_width * kv.page_size : given;
    const int64_t max_shared = whole(a[10]);
    const hyq_paged_batch batch = make_batch(q, a[4], a[5], a[11], q.size(0), whole(a[8]), max_len);
    if (q.size(2) != kv.head_dim) refuse(HYQ_E_SHAPE, "attention_shared: head_dim of q and the pages");
    const at::Tensor &start = plain(a[6], "group_start", at::kInt), &shared = plain(a[7], "shared", at::kInt);
    same_device(q, start, "group_start");
    same_device(q, shared, "shared");
    if (start.numel() != shared.numel() + 1) refuse(HYQ_E_SHAPE, "group_start takes one more entry than shared");
    const at::Tensor out = output(a[12], q, q.sizes(), at::kFloat, "out");
    const at::Tensor& ws = plain(a[13], "workspace", at::kByte);
    same_device(q, ws, "workspace");
    size_t bytes = 0;
    check(hyq_paged_attention_shared_workspace_bytes((int)q.size(1), kv.head_dim, q.size(0), &bytes));
    if ((size_t)ws.numel() < bytes) refuse(HYQ_E_SHAPE, "attention_shared: the workspace takes " + std::to_string(bytes) + " bytes");
    const c10::cuda::CUDAGuard device(q.device());
    check(hyq_paged_attention_shared(&kv8, &batch, static_cast<const int32_t*>(start.data_ptr()),
                                     static_cast<const int32_t*>(shared.data_ptr()), shared.numel(), max_shared < 0 ? max_len : max_shared,
                                     static_cast<const float*>(q.data_ptr()), qs, (int)q.size(1), static_cast<float*>(out.data_ptr()),
                                     row_stride(out, "out"), ws.data_ptr(), stream_of(q)));
    return THPVariable_Wrap(out);
  });
}

// k_pages, v_pages, table, row_start, pos, tokens, f16, slot, k_out,
// v_out, k_scale, v_scale
PyObject* gather(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 12, [&]() -> PyObject* {
    const at::Tensor& pages = tensor(a[0], "k_pages");
    const hyq_paged_kv8 kv = make_kv(pages, a[0], a[1], a[2], a[10], a[11]);
    const int64_t tokens = whole(a[5]);
    const bool f16 = PyObject_IsTrue(a[6]);
    if (tokens < 0 || tokens > INT32_MAX) refuse(HYQ_E_SHAPE, "gather: tokens");
    const hyq_paged_batch batch = make_batch(pages, a[3], a[4], a[7], tokens, 0, 0);
    const at::ScalarType type = f16 ? at::kHalf : at::kFloat;
    const at::Tensor k = output(a[8], pages, {tokens, kv.kv.kv_heads, kv.kv.head_dim}, type, "k_out"),
                     v = output(a[9], pages, {tokens, kv.kv.kv_heads, kv.kv.head_dim}, type, "v_out");
    const c10::cuda::CUDAGuard device(pages.device());
    check(hyq_paged_gather(&kv, &batch, f16, k.data_ptr(), row_stride(k, "k_out"), v.data_ptr(), row_stride(v, "v_out"),
                           stream_of(pages)));
    return pair(k, v);
  });
}

// q, k, v, k_pages, v_pages, table, row_start, pos, cos, sin, q_norm, k_norm,
// eps, norm_first, slot, out, k_scale, v_scale
PyObject* rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 18, [&]() -> PyObject* {
    const at::Tensor &q = typed(a[0], "q", at::kFloat), &k = typed(a[1], "k", at::kFloat), &v = typed(a[2], "v", at::kFloat);
    const hyq_paged_kv8 kv8 = make_kv(q, a[3], a[4], a[5], a[16], a[17]);
    const hyq_paged_kv& kv = kv8.kv;
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
    const c10::cuda::CUDAGuard device(q.device());
    check(hyq_paged_rope_append_kv8(
        &kv8, &batch, static_cast<const float*>(q.data_ptr()), qs, (int)q.size(1), static_cast<const float*>(k.data_ptr()), ks,
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
    const c10::cuda::CUDAGuard device(x.device());
    check(hyq_sample(static_cast<const float*>(x.data_ptr()), cols, rows > 1 ? x.stride(0) : cols, rows,
                     static_cast<const float*>(temperature), static_cast<const int32_t*>(top_k),
                     static_cast<const float*>(top_p), static_cast<const float*>(min_p), static_cast<const float*>(u),
                     static_cast<int32_t*>(token.data_ptr()), static_cast<float*>(prob.data_ptr()), stream_of(x)));
    return pair(token, prob);
  });
}

// [rows, columns] whose rows are contiguous; their distance.
int64_t matrix_stride(const at::Tensor& t, const char* name) {
  if (t.dim() != 2 || (t.size(1) > 1 && t.stride(1) != 1))
    refuse(HYQ_E_SHAPE, std::string(name) + ": expected a matrix with contiguous rows");
  return t.size(0) > 1 ? t.stride(0) : t.size(1);
}

// logits, history, length, prompt, slot, repetition, presence, frequency,
// bias_start, bias_token, bias_value, mask, mask_row, out
PyObject* adjust(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 14, [&]() -> PyObject* {
    const at::Tensor& x = typed(a[0], "logits", at::kFloat);
    const int64_t stride = matrix_stride(x, "logits"), rows = x.size(0), cols = x.size(1);
    hyq_adjust p{};
    if (a[1] != Py_None) {
      const at::Tensor& h = typed(a[1], "history", at::kInt);
      same_device(x, h, "history");
      p.history_stride = matrix_stride(h, "history");
      p.history = static_cast<const int32_t*>(h.data_ptr());
      p.slots = h.size(0);
      p.history_width = h.size(1);
      if (a[2] == Py_None) refuse(HYQ_E_INVALID, "length: expected a CUDA tensor");
      p.length = static_cast<const int32_t*>(optional(a[2], x, "length", at::kInt, p.slots));
      p.prompt = static_cast<const int32_t*>(optional(a[3], x, "prompt", at::kInt, p.slots));
      p.slot = static_cast<const int32_t*>(optional(a[4], x, "slot", at::kInt, rows));
    } else {
      for (int i = 2; i < 8; ++i)
        if (a[i] != Py_None) refuse(HYQ_E_INVALID, "adjust: lengths and penalties go with a history");
    }
    p.repetition = static_cast<const float*>(optional(a[5], x, "repetition", at::kFloat, rows));
    p.presence = static_cast<const float*>(optional(a[6], x, "presence", at::kFloat, rows));
    p.frequency = static_cast<const float*>(optional(a[7], x, "frequency", at::kFloat, rows));
    if (a[1] != Py_None && p.history_width == 0 && p.slots > 0) {  // no token in any: a tensor without elements has no address
      p.history = nullptr;
      p.repetition = p.presence = p.frequency = nullptr;
    }
    if (a[8] != Py_None) {
      const at::Tensor& t = plain(a[9], "bias tokens", at::kInt);
      same_device(x, t, "bias tokens");
      p.bias_count = t.numel();
      p.bias_start = static_cast<const int32_t*>(optional(a[8], x, "bias starts", at::kInt, rows + 1));
      p.bias_token = static_cast<const int32_t*>(t.data_ptr());
      if (a[10] == Py_None) refuse(HYQ_E_INVALID, "bias values: expected a CUDA tensor");
      p.bias_value = static_cast<const float*>(optional(a[10], x, "bias values", at::kFloat, p.bias_count));
      if (p.bias_count == 0) p.bias_start = nullptr;
    }
    if (a[11] != Py_None) {
      const at::Tensor& m = typed(a[11], "mask", at::kInt);
      same_device(x, m, "mask");
      p.mask_stride = matrix_stride(m, "mask");
      if (m.size(1) < (cols + 31) / 32) refuse(HYQ_E_SHAPE, "mask: expected [masks, (n + 31) / 32]");
      p.mask = static_cast<const int32_t*>(m.data_ptr());
      p.masks = m.size(0);
      p.mask_row = static_cast<const int32_t*>(optional(a[12], x, "mask_row", at::kInt, rows));
    } else if (a[12] != Py_None) {
      refuse(HYQ_E_INVALID, "adjust: mask_row goes with a mask");
    }
    const at::Tensor out = output(a[13], x, x.sizes(), at::kFloat, "out");
    const c10::cuda::CUDAGuard device(x.device());
    check(hyq_logits_adjust(static_cast<const float*>(x.data_ptr()), cols, stride, rows, &p, static_cast<float*>(out.data_ptr()),
                            matrix_stride(out, "out"), stream_of(x)));
    return THPVariable_Wrap(out);
  });
}

PyMethodDef methods[] = {
    {"adjust", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(adjust)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(attention)), METH_FASTCALL, nullptr},
    {"attention_shared", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(attention_shared)), METH_FASTCALL, nullptr},
    {"gather", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(gather)), METH_FASTCALL, nullptr},
    {"rope_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(rope_append)), METH_FASTCALL, nullptr},
    {"sample", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(sample)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" PyObject* PyInit__ops() { return PyModule_Create(&module); }
