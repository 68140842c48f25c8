// xn_torch.cpp - the Python binding's inner part for the paged-cache operators
// and the 8-bit RMSNorm: checks of the torch tensors, outputs, current stream,
// and the call of the C ABI, as one CPython extension module. These calls make
// up a decoding step whose kernels take a few microseconds each; the same
// checks in Python took 15 to 20 (measured: rms_norm_q8 of 16 x 4096 22.7 us a
// call, of which the call through ctypes with its arguments at hand is 5).
// The functions are documented where users see them, in xn_fused.py.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <sstream>
#include <string>

#include "xn_fused.h"

namespace {

PyObject *g_error = nullptr;  // xn_fused.XnError(message, code)

struct Refused {
  std::string text;
  int code;
};
struct PyFailed {};  // a Python exception is set

template <typename... A>
[[noreturn]] void refuse(int code, const A &...parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw Refused{s.str(), code};
}

std::string shape_text(c10::IntArrayRef v) {
  std::ostringstream s;
  s << "(";
  for (size_t i = 0; i < v.size(); ++i) s << (i ? ", " : "") << v[i];
  s << (v.size() == 1 ? ",)" : ")");
  return s.str();
}

// Arguments. A tensor argument may be None where `maybe` reads it.
const at::Tensor &tensor(PyObject *o, const char *op, const char *name) {
  if (!THPVariable_Check(o)) refuse(XN_E_INVALID, op, ": ", name, " must be a tensor");
  return THPVariable_Unpack(o);
}
at::Tensor maybe(PyObject *o, const char *op, const char *name) {
  if (o == Py_None) return at::Tensor();
  return tensor(o, op, name);
}
int64_t integer(PyObject *o) {
  PyObject *i = PyNumber_Index(o);
  if (i == nullptr) throw PyFailed{};
  const long long v = PyLong_AsLongLong(i);
  Py_DECREF(i);
  if (v == -1 && PyErr_Occurred()) throw PyFailed{};
  return v;
}
bool truth(PyObject *o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PyFailed{};
  return v != 0;
}
double real(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PyFailed{};
  return v;
}

// Checks.
int dtype_code(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kHalf:
      return XN_F16;
    case at::kBFloat16:
      return XN_BF16;
    case at::kFloat:
      return XN_F32;
    default:
      refuse(XN_E_DTYPE, "unsupported dtype ", t.scalar_type());
  }
}
void on_device(const char *op, const at::Tensor &ref, const at::Tensor &t) {
  if (!t.defined()) return;
  if (!t.is_cuda()) refuse(XN_E_INVALID, op, ": xn_fused ops take CUDA tensors (there is no CPU path)");
  if (t.device() != ref.device()) refuse(XN_E_INVALID, op, ": tensors on different devices: ", ref.device(), " and ", t.device());
}
void dense(const char *op, const at::Tensor &ref, const at::Tensor &t) {
  if (!t.defined()) return;
  on_device(op, ref, t);
  if (!t.is_contiguous()) refuse(XN_E_INVALID, op, ": xn_fused ops take contiguous tensors");
}
void same_dtype(const at::Tensor &ref, const at::Tensor &t) {
  if (t.defined() && t.scalar_type() != ref.scalar_type())
    refuse(XN_E_DTYPE, "dtype mismatch: ", ref.scalar_type(), " and ", t.scalar_type());
}
void has_dtype(const char *op, const char *name, const at::Tensor &t, at::ScalarType s) {
  if (t.scalar_type() != s) refuse(XN_E_DTYPE, op, ": ", name, " must be ", s, ", got ", t.scalar_type());
}
void has_shape(const char *op, const char *name, const at::Tensor &t, c10::IntArrayRef shape) {
  if (t.sizes() != shape)
    refuse(XN_E_INVALID, "shape mismatch in ", op, " ", name, ", ", shape_text(t.sizes()), " <> ", shape_text(shape));
}
void err_word(const char *op, const at::Tensor &t) {
  if (t.defined() && (t.scalar_type() != at::kInt || t.numel() < 1)) refuse(XN_E_INVALID, op, ": err_flag must be an int32 CUDA tensor");
}

struct Pool {
  int64_t n_pages, h_kv, page, d, ps, hs, ss;
};
Pool pool(const char *op, const at::Tensor &k, const at::Tensor &v) {
  has_shape(op, "pools", k, v.sizes());
  if (k.dim() != 4) refuse(XN_E_INVALID, op, ": pools must be [n_pages, h_kv, page_size, d], got ", shape_text(k.sizes()));
  if (k.strides() != v.strides() || k.stride(3) != 1)
    refuse(XN_E_INVALID, op, ": pools must share their strides and have a unit last stride");
  return Pool{k.size(0), k.size(1), k.size(2), k.size(3), k.stride(0), k.stride(1), k.stride(2)};
}

void *ptr(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// The tensors' device (which need not be the current one) and its current stream.
struct On {
  c10::cuda::CUDAGuard guard;
  void *stream;
  explicit On(const at::Tensor &t)
      : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

void called(const char *name, int rc) {
  if (rc != XN_OK) refuse(rc, name, " failed (", rc, "): ", xn_last_error());
}

at::Tensor empty(c10::IntArrayRef shape, at::ScalarType s, const at::Tensor &like) {
  return at::empty(shape, like.options().dtype(s).requires_grad(false).memory_format(c10::MemoryFormat::Contiguous));
}

// The k-th part of a one-dimensional buffer, without a dispatched view.
at::Tensor part(const at::Tensor &buf, int64_t at, int64_t n) {
  at::Tensor t = at::detail::make_tensor<at::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(), buf.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(at);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}

PyObject *wrap(const at::Tensor &t) { return THPVariable_Wrap(t); }

// Runs f, turning what it throws into a Python exception: torch's own (an
// allocation that fails, for one) into those that torch's operators raise.
template <typename F>
PyObject *guarded(F f) {
  try {
    return f();
  } catch (const Refused &e) {
    if (PyObject *x = PyObject_CallFunction(g_error, "si", e.text.c_str(), e.code)) {
      PyErr_SetObject(g_error, x);
      Py_DECREF(x);
    }
  } catch (const PyFailed &) {
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());
  }
  return nullptr;
}

void arity(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
    throw PyFailed{};
  }
}

// (lens, new_len, block_table, free_ring, ring_state, page_size, token_cap, out or None, err_flag or None)
PyObject *paged_plan(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    const char *op = "paged_plan";
    arity(n, 9);
    const at::Tensor &lens = tensor(a[0], op, "lens"), &add = tensor(a[1], op, "new_len"), &table = tensor(a[2], op, "block_table");
    const at::Tensor &ring = tensor(a[3], op, "free_ring"), &state = tensor(a[4], op, "ring_state");
    const int64_t page = integer(a[5]), cap = integer(a[6]);
    const at::Tensor err = maybe(a[8], op, "err_flag");
    if (lens.dim() != 1 || table.dim() != 2 || ring.dim() != 1)
      refuse(XN_E_INVALID, op, ": expected lens [R], block_table [R, blocks], free_ring [n_pages]");
    const int64_t r = table.size(0), blocks = table.size(1);
    has_shape(op, "lens", lens, {r});
    has_shape(op, "new_len", add, {r});
    has_shape(op, "ring_state", state, {2});
    if (cap < 0) refuse(XN_E_INVALID, op, ": negative token_cap");
    for (const at::Tensor *t : {&lens, &add, &table, &ring, &state, &err}) dense(op, lens, *t);
    has_dtype(op, "lens", lens, at::kLong);
    has_dtype(op, "new_len", add, at::kLong);
    has_dtype(op, "ring_state", state, at::kLong);
    has_dtype(op, "block_table", table, at::kInt);
    has_dtype(op, "free_ring", ring, at::kInt);
    err_word(op, err);
    const int64_t sizes[5] = {r + 1, r, cap, cap, 2};
    const char *names[5] = {"q_start", "kv_len", "positions", "slots", "ring_state"};
    On on(lens);
    at::Tensor out[5];
    if (a[7] == Py_None) {
      // Five parts of one buffer, each on a 16-byte boundary.
      int64_t at[6] = {0};
      for (int i = 0; i < 5; ++i) at[i + 1] = at[i] + (sizes[i] + 1) / 2 * 2;
      const at::Tensor buf = empty({at[5]}, at::kLong, lens);
      for (int i = 0; i < 5; ++i) out[i] = part(buf, at[i], sizes[i]);
    } else {
      if (!PyTuple_Check(a[7]) || PyTuple_GET_SIZE(a[7]) != 5) refuse(XN_E_INVALID, op, ": out must be a PagedPlan");
      for (int i = 0; i < 5; ++i) {
        out[i] = tensor(PyTuple_GET_ITEM(a[7], i), op, names[i]);
        has_shape(op, names[i], out[i], {sizes[i]});
        dense(op, lens, out[i]);
        has_dtype(op, names[i], out[i], at::kLong);
      }
    }
    auto p = [](const at::Tensor &t) { return static_cast<int64_t *>(ptr(t)); };
    called("xn_paged_plan",
           xn_paged_plan(p(out[0]), p(out[1]), p(out[2]), p(out[3]), p(out[4]), static_cast<int32_t *>(ptr(table)),
                         static_cast<int32_t *>(ptr(ring)), p(lens), p(add), p(state), r, blocks, ring.numel(), page, cap,
                         static_cast<int *>(ptr(err)), on.stream));
    if (a[7] != Py_None) return Py_NewRef(a[7]);
    PyObject *t = PyTuple_New(5);
    for (int i = 0; i < 5; ++i) PyTuple_SET_ITEM(t, i, wrap(out[i]));
    return t;
  });
}

// (qkv, heads, kv_heads, cos, sin, k_pages, v_pages, positions, slots, interleaved, err_flag or None, q_out or None)
PyObject *paged_append_rope(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    const char *op = "paged_append_rope";
    arity(n, 12);
    const at::Tensor &qkv = tensor(a[0], op, "qkv"), &cos = tensor(a[3], op, "cos"), &sin = tensor(a[4], op, "sin");
    const at::Tensor &k = tensor(a[5], op, "k_pages"), &v = tensor(a[6], op, "v_pages");
    const at::Tensor &pos = tensor(a[7], op, "positions"), &slots = tensor(a[8], op, "slots");
    const int64_t h = integer(a[1]), hk = integer(a[2]);
    const bool interleaved = truth(a[9]);
    const at::Tensor err = maybe(a[10], op, "err_flag");
    at::Tensor q = maybe(a[11], op, "q_out");
    const Pool c = pool(op, k, v);
    const int64_t tokens = pos.numel();
    if (c.h_kv != hk || h <= 0 || qkv.dim() < 1 || qkv.size(0) != tokens || qkv.numel() != tokens * (h + 2 * hk) * c.d)
      refuse(XN_E_INVALID, op, ": expected qkv [", tokens, ", (", h, " + 2 * ", hk, ") * ", c.d, "] and ", hk,
             " kv heads in the pools, got ", shape_text(qkv.sizes()), " and ", c.h_kv);
    has_shape(op, "slots", slots, pos.sizes());
    has_shape(op, "cos/sin", cos, sin.sizes());
    if (cos.dim() != 2 || cos.size(1) * 2 != c.d)
      refuse(XN_E_INVALID, op, ": cos/sin must be [max_pos, ", c.d / 2, "], got ", shape_text(cos.sizes()));
    for (const at::Tensor *t : {&qkv, &cos, &sin, &pos, &slots, &err}) dense(op, qkv, *t);
    on_device(op, qkv, k);
    on_device(op, qkv, v);
    for (const at::Tensor *t : {&cos, &sin, &k, &v}) same_dtype(qkv, *t);
    has_dtype(op, "positions", pos, at::kLong);
    has_dtype(op, "slots", slots, at::kLong);
    err_word(op, err);
    const int dtype = dtype_code(qkv);
    On on(qkv);
    if (!q.defined()) {
      q = empty({tokens, h, c.d}, qkv.scalar_type(), qkv);
    } else {
      has_shape(op, "q_out", q, {tokens, h, c.d});
      dense(op, qkv, q);
      same_dtype(qkv, q);
    }
    called("xn_paged_append_rope",
           xn_paged_append_rope(ptr(q), ptr(k), ptr(v), ptr(qkv), ptr(cos), ptr(sin), static_cast<int64_t *>(ptr(pos)),
                                static_cast<int64_t *>(ptr(slots)), tokens, h, hk, c.d, cos.size(0), c.n_pages, c.page, c.ps,
                                c.hs, c.ss, interleaved, dtype, static_cast<int *>(ptr(err)), on.stream));
    return wrap(q);
  });
}

// (q, k_pages, v_pages, block_table, q_start, kv_len, scale, max_new, window, workspace or None, err_flag or None, out or None)
PyObject *paged_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    const char *op = "paged_attention";
    arity(n, 12);
    const at::Tensor &q = tensor(a[0], op, "q"), &k = tensor(a[1], op, "k_pages"), &v = tensor(a[2], op, "v_pages");
    const at::Tensor &table = tensor(a[3], op, "block_table"), &start = tensor(a[4], op, "q_start"), &kv = tensor(a[5], op, "kv_len");
    const float scale = static_cast<float>(real(a[6]));
    const int64_t max_new = integer(a[7]), window = integer(a[8]);
    at::Tensor ws = maybe(a[9], op, "workspace"), out = maybe(a[11], op, "out");
    const at::Tensor err = maybe(a[10], op, "err_flag");
    const Pool c = pool(op, k, v);
    if (q.dim() != 3 || q.size(2) != c.d || c.h_kv == 0 || q.size(1) % c.h_kv != 0)
      refuse(XN_E_INVALID, op, ": q must be [N, H, ", c.d, "] with H a multiple of ", c.h_kv, ", got ", shape_text(q.sizes()));
    const int64_t tokens = q.size(0), h = q.size(1);
    if (tokens > 0 && (q.stride(2) != 1 || (h > 1 && q.stride(1) != c.d)))
      refuse(XN_E_INVALID, op, ": the rows of q must be contiguous");
    if (table.dim() != 2) refuse(XN_E_INVALID, op, ": block_table must be [R, blocks], got ", shape_text(table.sizes()));
    const int64_t r = table.size(0), blocks = table.size(1);
    has_shape(op, "kv_len", kv, {r});
    has_shape(op, "q_start", start, {r + 1});
    on_device(op, q, q);
    on_device(op, q, k);
    on_device(op, q, v);
    for (const at::Tensor *t : std::initializer_list<const at::Tensor *>{&table, &start, &kv, &ws, &err}) dense(op, q, *t);
    same_dtype(q, k);
    same_dtype(q, v);
    has_dtype(op, "q_start", start, at::kLong);
    has_dtype(op, "kv_len", kv, at::kLong);
    has_dtype(op, "block_table", table, at::kInt);
    err_word(op, err);
    const int dtype = dtype_code(q);
    On on(q);
    if (!out.defined()) {
      out = empty({tokens, h * c.d}, q.scalar_type(), q);
    } else {
      if (out.numel() != tokens * h * c.d) refuse(XN_E_INVALID, op, ": out must hold [N, H * D]");
      dense(op, q, out);
      same_dtype(q, out);
    }
    if (!ws.defined()) {
      int64_t bytes = 0;
      called("xn_paged_attention_workspace", xn_paged_attention_workspace(&bytes, tokens, r, h, c.h_kv, c.d, max_new, dtype));
      ws = empty({bytes}, at::kByte, q);
    }
    called("xn_paged_attention",
           xn_paged_attention(ptr(out), ptr(q), ptr(k), ptr(v), static_cast<int32_t *>(ptr(table)),
                              static_cast<int64_t *>(ptr(start)), static_cast<int64_t *>(ptr(kv)), tokens, r, h, c.h_kv, c.d,
                              c.n_pages, c.page, blocks, tokens > 1 ? q.stride(0) : h * c.d, c.ps, c.hs, c.ss, max_new, window,
                              scale, dtype, ptr(ws), static_cast<int64_t>(ws.nbytes()), static_cast<int *>(ptr(err)), on.stream));
    return wrap(out);
  });
}

// (x, alpha, eps, branch or None, group, out or None, scales or None, residual_out or None)
PyObject *rms_norm_q8(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    const char *op = "rms_norm_q8";
    arity(n, 8);
    const at::Tensor &x = tensor(a[0], op, "x"), &alpha = tensor(a[1], op, "alpha");
    const double eps = real(a[2]);
    const at::Tensor branch = maybe(a[3], op, "branch");
    const int64_t group = integer(a[4]);
    at::Tensor out = maybe(a[5], op, "out"), scales = maybe(a[6], op, "scales"), res = maybe(a[7], op, "residual_out");
    if (!(eps > 0.0)) refuse(XN_E_INVALID, op, " eps must be positive");
    const int64_t cols = x.dim() > 0 ? x.size(-1) : 1;
    int64_t rows = 1;
    for (int64_t i = 0; i + 1 < x.dim(); ++i) rows *= x.size(i);
    if ((group != 0 && group != 32 && group != 64 && group != 128) || (group != 0 && cols % group != 0))
      refuse(XN_E_INVALID, op, ": group ", group, " is not 0, 32, 64 or 128 and a divisor of ", cols);
    has_shape(op, "alpha", alpha, {cols});
    if (branch.defined()) has_shape(op, "branch", branch, x.sizes());
    if (res.defined()) has_shape(op, "residual_out", res, x.sizes());
    for (const at::Tensor *t : std::initializer_list<const at::Tensor *>{&x, &alpha, &branch, &out, &scales, &res}) dense(op, x, *t);
    same_dtype(x, alpha);
    same_dtype(x, branch);
    same_dtype(x, res);
    const int dtype = dtype_code(x);
    c10::DimVector shape(x.sizes());
    if (!shape.empty()) shape.pop_back();
    if (group != 0) shape.push_back(cols / group);
    On on(x);
    if (!out.defined())
      out = empty(x.sizes(), at::kFloat8_e4m3fn, x);
    else
      has_shape(op, "out", out, x.sizes());
    if (!scales.defined())
      scales = empty(shape, at::kFloat, x);
    else
      has_shape(op, "scales", scales, shape);
    if (out.scalar_type() != at::kFloat8_e4m3fn || scales.scalar_type() != at::kFloat)
      refuse(XN_E_DTYPE, op, ": out must be float8_e4m3fn and scales float32");
    if (branch.defined() && !res.defined()) res = empty(x.sizes(), x.scalar_type(), x);
    called("xn_rms_norm_q8", xn_rms_norm_q8(ptr(out), static_cast<float *>(ptr(scales)), ptr(res), ptr(x), ptr(alpha), ptr(branch),
                                            rows, cols, group, static_cast<float>(eps), dtype, on.stream));
    PyObject *t = PyTuple_New(3);
    PyTuple_SET_ITEM(t, 0, wrap(out));
    PyTuple_SET_ITEM(t, 1, wrap(scales));
    PyTuple_SET_ITEM(t, 2, res.defined() ? wrap(res) : Py_NewRef(a[0]));
    return t;
  });
}

// The exception class that failed checks raise: called once, with (message, code) as its arguments.
PyObject *set_error(PyObject *, PyObject *cls) {
  Py_XDECREF(g_error);
  g_error = Py_NewRef(cls);
  Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {FAST(paged_plan), FAST(paged_append_rope), FAST(paged_attention), FAST(rms_norm_q8),
                           {"set_error", set_error, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "xn_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_xn_torch() { return PyModule_Create(&g_module); }
