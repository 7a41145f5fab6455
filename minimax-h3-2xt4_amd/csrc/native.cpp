// Python module _native: whole calls of the package whose device work is short
// enough that the interpreter bounded them (one decode token through a
// projection: 17 us of kernels behind 32 us of argument checks, allocations
// and ctypes structs). Each function takes the plain case - exact tensors or
// parameters on the current device, in the layout the kernels read in place -
// checks it completely, allocates the outputs and calls the C ABI on the
// current stream; for anything else it returns None without having done
// anything, and the Python route (which converts, copies or raises) runs.
// Host time of a call, measured: a one-row projection 32 -> 10 us (the whole
// call 31.2 -> 14.7), a 64-row one with split K 36 -> 14, an attention 45 -> 11
// (16 heads x 353 x 1000 fp32: 45.8 -> 30.4), a modulated norm with 16
// segments 78 -> 25 (its labels came by a copy that waited for the stream).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <initializer_list>
#include <vector>

#include "w8a8.h"

namespace {

PyObject* g_error_class = nullptr;   // _abi.W8A8Error(function, status, message)

// The tensor of a plain torch.Tensor or Parameter on the current GPU, or null.
// Subclasses, functorch wrappers and dispatch modes take the Python route.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckTypeExact(Py_TYPE(o))) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.get_device() != c10::hip::current_device() || t.layout() != at::kStrided ||
      !t.has_storage() || t.is_neg() || t.is_conj())
    return nullptr;
  const auto keys = t.key_set();
  if (keys.has(c10::DispatchKey::Python) || keys.has(c10::DispatchKey::FuncTorchBatched) ||
      keys.has(c10::DispatchKey::FuncTorchGradWrapper) || keys.has(c10::DispatchKey::Functionalize))
    return nullptr;
  return &t;
}

bool modes_active() {
  return c10::impl::dispatch_mode_enabled() || at::impl::torch_function_mode_enabled();
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return W8A8_F16;
    case at::kBFloat16: return W8A8_BF16;
    case at::kFloat: return W8A8_F32;
    default: return 0;
  }
}

void* stream_of(int device) { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream(); }

template <typename T>
T* ptr(const at::Tensor& t) { return reinterpret_cast<T*>(t.data_ptr()); }

PyObject* fail(const char* fn, int rc) {
  PyObject* e = PyObject_CallFunction(g_error_class, "sis", fn, rc, w8a8_last_error());
  if (e) {
    PyErr_SetObject(g_error_class, e);
    Py_DECREF(e);
  }
  return nullptr;
}

// fn(&args) without the interpreter lock, as ctypes calls it.
template <typename Args>
int call(int (*fn)(const Args*), Args& a) {
  a.struct_size = sizeof(Args);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fn(&a);
  Py_END_ALLOW_THREADS
  return rc;
}

// linear(x, weight, weight_scale, bias | None, epilogue, round_rotated,
// out_dtype): ConvRot256 and per-row INT8 of x [.., K], then the GEMM with the
// row- or column-order epilogue.
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || modes_active() || !THPDtype_Check(args[6])) Py_RETURN_NONE;
  const at::Tensor* x = plain(args[0]);
  const at::Tensor* w = plain(args[1]);
  const at::Tensor* ws = plain(args[2]);
  const at::Tensor* bias = args[3] == Py_None ? nullptr : plain(args[3]);
  if (!x || !w || !ws || (args[3] != Py_None && !bias)) Py_RETURN_NONE;
  const int dev = x->get_device();
  const long epilogue = PyLong_AsLong(args[4]), round_rotated = PyLong_AsLong(args[5]);
  const at::ScalarType out_type = reinterpret_cast<THPDtype*>(args[6])->scalar_type;
  const int xt = dtype_code(x->scalar_type()), ot = dtype_code(out_type);
  if (!xt || !ot || x->dim() < 1 || !x->is_contiguous() || w->dim() != 2 || w->scalar_type() != at::kChar ||
      !w->is_contiguous())
    Py_RETURN_NONE;
  const int64_t k = x->size(-1), nn = w->size(0);
  if (k <= 0 || k % 256 || w->size(1) != k || nn <= 0 || x->numel() == 0) Py_RETURN_NONE;
  const int64_t rows = x->numel() / k;
  if (ws->scalar_type() != at::kFloat || !ws->is_contiguous() || (ws->numel() != 1 && ws->numel() != nn))
    Py_RETURN_NONE;
  if (bias && ((bias->scalar_type() != at::kHalf && bias->scalar_type() != at::kFloat) || !bias->is_contiguous() ||
               bias->numel() != nn))
    Py_RETURN_NONE;
  const auto opt = at::TensorOptions().device(x->device());
  const at::Tensor q = at::empty({rows, k}, opt.dtype(at::kChar));
  const at::Tensor scale = at::empty({rows}, opt.dtype(at::kFloat));
  at::DimVector shape(x->sizes().begin(), x->sizes().end());
  shape.back() = nn;
  at::Tensor out = at::empty(shape, opt.dtype(out_type));
  void* const stream = stream_of(dev);

  W8A8QuantArgs qa{};
  qa.x_dtype = xt;
  qa.x = x->data_ptr();
  qa.ldx = k;
  qa.rows = rows;
  qa.cols = k;
  qa.convrot = 256;
  qa.round_rotated = round_rotated ? 1 : 0;
  qa.q = ptr<int8_t>(q);
  qa.ldq = k;
  qa.scale = ptr<float>(scale);
  qa.stream = stream;
  int rc = call(w8a8_quantize_rows, qa);
  if (rc != W8A8_OK) return fail("w8a8_quantize_rows", rc);

  W8A8GemmArgs ga{};
  ga.epilogue = (int32_t)epilogue;
  ga.a = qa.q;
  ga.lda = k;
  ga.b = ptr<int8_t>(*w);
  ga.ldb = k;
  ga.m = rows;
  ga.n = nn;
  ga.k = k;
  ga.row_scale = qa.scale;
  ga.col_scale = ptr<float>(*ws);
  ga.col_scale_stride = ws->numel() == 1 ? 0 : 1;
  if (bias) {
    ga.bias = bias->data_ptr();
    ga.bias_dtype = dtype_code(bias->scalar_type());
  }
  ga.out_dtype = ot;
  ga.out = out.data_ptr();
  ga.ldc = nn;
  at::Tensor workspace;
  ga.workspace_bytes = w8a8_gemm_workspace_size(rows, nn, k);
  if (ga.workspace_bytes > 0) {
    workspace = at::empty({ga.workspace_bytes}, opt.dtype(at::kByte));
    ga.workspace = workspace.data_ptr();
  }
  ga.stream = stream;
  rc = call(w8a8_gemm, ga);
  if (rc != W8A8_OK) return fail("w8a8_gemm", rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// Element strides {batch, head, token} of a [b, h, n, 128] tensor whose rows
// the kernels read in place; false: a copy is needed.
bool row_strides(const at::Tensor& t, int64_t (&st)[3]) {
  const int64_t es = t.element_size();
  if ((t.size(3) != 1 && t.stride(3) != 1) || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  for (int i = 0; i < 3; ++i) {
    st[i] = t.size(i) == 1 ? 0 : t.stride(i);
    if (st[i] < 0 || st[i] * es % 16) return false;
  }
  return true;
}

// int8_attention(q, k, v, sm_scale | None): the preparation and the attention
// of [b, h, n, 128] fp16 or fp32 tensors; the operands live in one buffer for
// the length of the call.
PyObject* int8_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4 || modes_active()) Py_RETURN_NONE;
  const at::Tensor* q = plain(args[0]);
  const at::Tensor* k = plain(args[1]);
  const at::Tensor* v = plain(args[2]);
  if (!q || !k || !v || q->dim() != 4 || k->dim() != 4 || v->dim() != 4) Py_RETURN_NONE;
  if (args[3] != Py_None && !PyFloat_CheckExact(args[3])) Py_RETURN_NONE;
  const at::ScalarType type = q->scalar_type();
  const int64_t b = q->size(0), h = q->size(1), nq = q->size(2), nk = k->size(2), d = 128;
  if ((type != at::kHalf && type != at::kFloat) || k->scalar_type() != type || v->scalar_type() != type ||
      q->size(3) != d || k->size(0) != b || k->size(1) != h || k->size(3) != d || v->sizes() != k->sizes() ||
      b * h == 0 || nq == 0 || nk == 0)
    Py_RETURN_NONE;
  W8A8AttnPrepareArgs pa{};
  if (!row_strides(*q, pa.q_strides) || !row_strides(*k, pa.k_strides) || !row_strides(*v, pa.v_strides)) Py_RETURN_NONE;
  const int64_t nblk = (nk + 127) / 128, nkp = 128 * nblk, bh = b * h;
  int64_t bytes = 0;
  auto take = [&](int64_t size) {
    const int64_t at = bytes;
    bytes += (size + 255) & ~int64_t(255);
    return at;
  };
  const int64_t wsb = w8a8_attention_workspace_size(b, h, nk);
  const int64_t o_q8 = take(bh * nq * d), o_qs = take(bh * nq * 4), o_k8 = take(bh * nkp * d), o_ks = take(bh * nblk * 16),
                o_vt = take(bh * nkp * d), o_vs = take(bh * d * 4), o_vsum = take(bh * nblk * d * 4), o_ws = take(wsb);
  const auto opt = at::TensorOptions().device(q->device());
  const at::Tensor buf = at::empty({bytes}, opt.dtype(at::kByte));
  at::Tensor out = at::empty({b, h, nq, d}, opt.dtype(type));
  char* const base = ptr<char>(buf);
  pa.in_dtype = dtype_code(type);
  pa.q = q->data_ptr();
  pa.k = k->data_ptr();
  pa.v = v->data_ptr();
  pa.b = b;
  pa.h = h;
  pa.nq = nq;
  pa.nk = nk;
  pa.d = (int32_t)d;
  pa.sm_scale = (float)(args[3] == Py_None ? std::pow((double)d, -0.5) : PyFloat_AS_DOUBLE(args[3]));
  pa.q8 = reinterpret_cast<int8_t*>(base + o_q8);
  pa.qs = reinterpret_cast<float*>(base + o_qs);
  pa.k8 = reinterpret_cast<int8_t*>(base + o_k8);
  pa.ks = reinterpret_cast<float*>(base + o_ks);
  pa.vt8 = reinterpret_cast<int8_t*>(base + o_vt);
  pa.vs = reinterpret_cast<float*>(base + o_vs);
  pa.vsum = reinterpret_cast<int32_t*>(base + o_vsum);
  pa.workspace = base + o_ws;
  pa.workspace_bytes = wsb;
  pa.stream = stream_of(q->get_device());
  int rc = call(w8a8_attention_prepare, pa);
  if (rc != W8A8_OK) return fail("w8a8_attention_prepare", rc);
  W8A8AttentionArgs aa{};
  aa.out_dtype = pa.in_dtype;
  aa.q8 = pa.q8;
  aa.qs = pa.qs;
  aa.k8 = pa.k8;
  aa.ks = pa.ks;
  aa.vt8 = pa.vt8;
  aa.vs = pa.vs;
  aa.vsum = pa.vsum;
  aa.b = b;
  aa.h = h;
  aa.nq = nq;
  aa.nk = nk;
  aa.d = (int32_t)d;
  aa.sm_scale = pa.sm_scale;
  aa.out = out.data_ptr();
  row_strides(out, aa.out_strides);
  aa.stream = pa.stream;
  rc = call(w8a8_attention, aa);
  if (rc != W8A8_OK) return fail("w8a8_attention", rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// segment_labels(rows, segments, table_rows, device_index): int32 [rows] with
// each row's table row, when the (a, b, row) segments tile [0, rows) exactly.
PyObject* segment_labels(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4 || modes_active() || !(PyList_CheckExact(args[1]) || PyTuple_CheckExact(args[1]))) Py_RETURN_NONE;
  const int64_t rows = PyLong_AsLongLong(args[0]), table_rows = PyLong_AsLongLong(args[2]);
  const long dev = PyLong_AsLong(args[3]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (rows <= 0 || rows >= (int64_t(1) << 31) || dev != c10::hip::current_device()) Py_RETURN_NONE;
  const Py_ssize_t count = PySequence_Fast_GET_SIZE(args[1]);
  std::vector<std::array<int64_t, 3>> segs((size_t)count);
  for (Py_ssize_t i = 0; i < count; ++i) {
    PyObject* s = PySequence_Fast_GET_ITEM(args[1], i);
    if (!(PyList_CheckExact(s) || PyTuple_CheckExact(s)) || PySequence_Fast_GET_SIZE(s) != 3) Py_RETURN_NONE;
    for (int j = 0; j < 3; ++j) {
      PyObject* v = PySequence_Fast_GET_ITEM(s, j);
      if (!PyLong_CheckExact(v)) Py_RETURN_NONE;
      int overflow = 0;
      segs[(size_t)i][(size_t)j] = PyLong_AsLongLongAndOverflow(v, &overflow);
      if (overflow) Py_RETURN_NONE;
    }
  }
  std::sort(segs.begin(), segs.end());
  std::vector<int32_t> ends, values;
  ends.reserve((size_t)count);
  values.reserve((size_t)count);
  int64_t cursor = 0;
  for (const auto& s : segs) {
    if (s[0] != cursor || s[1] <= s[0] || s[1] > rows || s[2] < 0 || s[2] >= table_rows || s[2] > INT32_MAX)
      Py_RETURN_NONE;
    cursor = s[1];
    ends.push_back((int32_t)s[1]);
    values.push_back((int32_t)s[2]);
  }
  if (cursor != rows) Py_RETURN_NONE;
  at::Tensor out = at::empty({rows}, at::TensorOptions().device(at::kCUDA, (c10::DeviceIndex)dev).dtype(at::kInt));
  void* const stream = stream_of((int)dev);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = w8a8_segment_labels(ends.data(), values.data(), (int64_t)ends.size(), ptr<int32_t>(out), rows, stream);
  Py_END_ALLOW_THREADS
  if (rc != W8A8_OK) return fail("w8a8_segment_labels", rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------- around the projections of a block

// A tensor argument that may be None: `ok` turns false for anything but None or
// a plain tensor.
const at::Tensor* optional(PyObject* o, bool& ok) {
  if (o == Py_None) return nullptr;
  const at::Tensor* t = plain(o);
  if (!t) ok = false;
  return t;
}

// A float argument that may be None.
bool optional_float(PyObject* o, float& v, bool& given) {
  given = o != Py_None;
  if (!given) return true;
  if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
  v = (float)PyFloat_AsDouble(o);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

// Whether a gradient, backward or forward, would be asked of a tensor: the Python
// route refuses it.
bool wants_gradient(std::initializer_list<const at::Tensor*> ts) {
  const bool grad = at::GradMode::is_enabled();
  for (const at::Tensor* t : ts)
    if (t && ((grad && t->requires_grad()) || t->_fw_grad(0).defined())) return true;
  return false;
}

bool aligned(const at::Tensor& t, uintptr_t n) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % n == 0; }

// [rows, cols] with contiguous 16-byte aligned rows; ld its row stride.
bool aligned_rows(const at::Tensor& t, int64_t rows, int64_t cols, int64_t& ld) {
  if (t.dim() != 2 || t.size(0) != rows || t.size(1) != cols || t.stride(1) != 1 || !aligned(t, 16)) return false;
  const int64_t es = t.element_size();
  ld = rows > 1 ? t.stride(0) : (cols * es + 15) / 16 * 16 / es;
  return ld >= cols && ld * es % 16 == 0;
}

bool fp32_vector(const at::Tensor* t, int64_t n) {
  return !t || (t->scalar_type() == at::kFloat && t->numel() == n && t->is_contiguous() && aligned(*t, 16));
}

bool set_item(PyObject* dict, const char* key, at::Tensor t) {
  PyObject* o = THPVariable_Wrap(std::move(t));
  const bool ok = o && PyDict_SetItemString(dict, key, o) == 0;
  Py_XDECREF(o);
  return ok;
}

// Counts a write into a caller's tensor, as torch's own in-place operators do:
// autograd then sees that a tensor it saved has changed.
void written(const at::Tensor* t) {
  if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// residual_norm(x, branch, weight, eps, post_weight, post_eps, gate, shift,
// scale, labels, residual_scale, branch_scale, quantize, convrot,
// round_rotated, want_normalized, out): kernels.residual_norm without signs.
PyObject* residual_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 17 || modes_active()) Py_RETURN_NONE;
  bool ok = true;
  const at::Tensor* x = plain(args[0]);
  const at::Tensor* branch = plain(args[1]);
  const at::Tensor* weight = optional(args[2], ok);
  const at::Tensor* post_weight = optional(args[4], ok);
  const at::Tensor* gate = optional(args[6], ok);
  const at::Tensor* shift = optional(args[7], ok);
  const at::Tensor* mscale = optional(args[8], ok);
  const at::Tensor* labels = optional(args[9], ok);
  const at::Tensor* out = optional(args[16], ok);
  W8A8ResidualNormArgs a{};
  bool pre = false, post = false, given = false;
  if (!x || !branch || !ok || x->dim() != 2 || !optional_float(args[3], a.eps, pre) ||
      !optional_float(args[5], a.post_eps, post) || !optional_float(args[10], a.residual_scale, given) || !given ||
      !optional_float(args[11], a.branch_scale, given) || !given)
    Py_RETURN_NONE;
  for (int i = 12; i < 16; ++i)
    if (!PyBool_Check(args[i])) Py_RETURN_NONE;
  const bool quantize = args[12] == Py_True, convrot = args[13] == Py_True, want = args[15] == Py_True;
  const int64_t rows = x->size(0), cols = x->size(1);
  const at::ScalarType type = x->scalar_type();
  if ((type != at::kHalf && type != at::kBFloat16) ||
      (branch->scalar_type() != type && branch->scalar_type() != at::kFloat) || rows <= 0 || cols <= 0 ||
      cols % (quantize && convrot ? 256 : 16) || !aligned_rows(*x, rows, cols, a.ldx) ||
      !aligned_rows(*branch, rows, cols, a.ldb) || !fp32_vector(weight, cols) || !fp32_vector(post_weight, cols) ||
      (post_weight && !post) || (!pre && (quantize || want || weight || shift || mscale)) ||
      wants_gradient({x, branch, weight, post_weight, gate, shift, mscale}))
    Py_RETURN_NONE;
  if (gate) {
    if (gate->scalar_type() != at::kFloat || gate->dim() != 2 || gate->size(0) < 1 ||
        !aligned_rows(*gate, gate->size(0), cols, a.ld_gate))
      Py_RETURN_NONE;
    a.gate = ptr<float>(*gate);
    a.gate_rows = (int32_t)gate->size(0);
  }
  if (shift || mscale) {
    int64_t ld = 0;
    if (!shift || !mscale || shift->scalar_type() != at::kFloat || mscale->scalar_type() != at::kFloat ||
        shift->dim() != 2 || shift->size(0) < 1 || !aligned_rows(*shift, shift->size(0), cols, a.ld_mod) ||
        !aligned_rows(*mscale, shift->size(0), cols, ld) || ld != a.ld_mod)
      Py_RETURN_NONE;
    a.mod_shift = ptr<float>(*shift);
    a.mod_scale = ptr<float>(*mscale);
    a.mod_rows = (int32_t)shift->size(0);
  }
  if (gate || shift) {
    if (!labels || labels->scalar_type() != at::kInt || labels->numel() != rows || !labels->is_contiguous())
      Py_RETURN_NONE;
    a.labels = ptr<int32_t>(*labels);
  }
  if (out && (out->scalar_type() != type || !aligned_rows(*out, rows, cols, a.ldo) || wants_gradient({out})))
    Py_RETURN_NONE;
  const auto opt = at::TensorOptions().device(x->device());
  at::Tensor fresh, y, q, qs;
  if (!out) {
    fresh = at::empty({rows, cols}, opt.dtype(type));
    a.ldo = cols;
  }
  const bool want_y = pre && (want || !quantize);
  if (want_y) y = at::empty({rows, cols}, opt.dtype(type));
  if (quantize) {
    q = at::empty({rows, cols}, opt.dtype(at::kChar));
    qs = at::empty({rows, 1}, opt.dtype(at::kFloat));
  }
  a.x_dtype = dtype_code(type);
  a.x = x->data_ptr();
  a.rows = rows;
  a.cols = cols;
  a.branch = branch->data_ptr();
  a.branch_dtype = dtype_code(branch->scalar_type());
  a.post = post;
  a.post_weight = post_weight ? ptr<float>(*post_weight) : nullptr;
  a.out = out ? out->data_ptr() : fresh.data_ptr();
  a.weight = weight ? ptr<float>(*weight) : nullptr;
  a.y = want_y ? y.data_ptr() : nullptr;
  a.ldy = cols;
  a.convrot = quantize && convrot ? 256 : 0;
  a.round_rotated = args[14] == Py_True;
  a.q = quantize ? ptr<int8_t>(q) : nullptr;
  a.ldq = cols;
  a.q_scale = quantize ? ptr<float>(qs) : nullptr;
  a.stream = stream_of(x->get_device());
  const int rc = call(w8a8_residual_norm, a);
  if (rc != W8A8_OK) return fail("w8a8_residual_norm", rc);
  written(out);
  PyObject* d = PyDict_New();
  if (!d) return nullptr;
  ok = out ? PyDict_SetItemString(d, "x", args[16]) == 0 : set_item(d, "x", std::move(fresh));
  if (ok && want_y) ok = set_item(d, "y", std::move(y));
  if (ok && quantize) ok = set_item(d, "q", std::move(q)) && set_item(d, "scale", std::move(qs));
  if (!ok) {
    Py_DECREF(d);
    return nullptr;
  }
  return d;
  END_HANDLE_TH_ERRORS
}

// Element strides {row, head} of a [rows, heads, dim] tensor.
bool head_strides(const at::Tensor& t, int64_t (&st)[2]) {
  if (t.dim() != 3 || (t.size(2) > 1 && t.stride(2) != 1)) return false;
  st[1] = t.size(1) > 1 ? t.stride(1) : t.size(2);
  st[0] = t.size(0) > 1 ? t.stride(0) : t.size(1) * st[1];
  return true;
}

// axial_rope(q, k, positions, inv_freq, axis, adjacent, q_gain, k_gain, eps,
// q_out, k_out): kernels.axial_rope; returns (q_out, k_out).
PyObject* axial_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11 || modes_active() || !PyBool_Check(args[5])) Py_RETURN_NONE;
  bool ok = true, given = false;
  const at::Tensor* q = plain(args[0]);
  const at::Tensor* k = optional(args[1], ok);
  const at::Tensor* pos = plain(args[2]);
  const at::Tensor* inv = plain(args[3]);
  const at::Tensor* axis = plain(args[4]);
  const at::Tensor* gq = optional(args[6], ok);
  const at::Tensor* gk = optional(args[7], ok);
  const at::Tensor* qo = optional(args[9], ok);
  const at::Tensor* ko = optional(args[10], ok);
  W8A8AxialRopeArgs a{};
  if (!q || !pos || !inv || !axis || !ok || !optional_float(args[8], a.eps, given) || !given ||
      !head_strides(*q, a.q_strides) || (k && !head_strides(*k, a.k_strides)))
    Py_RETURN_NONE;
  const at::ScalarType type = q->scalar_type();
  const int64_t rows = q->size(0), heads = q->size(1), dim = q->size(2), pairs = inv->numel();
  const int64_t kheads = k ? k->size(1) : 0;
  const auto pt = pos->scalar_type();
  if (!dtype_code(type) || rows <= 0 || heads <= 0 || heads > 4096 || dim < 2 || dim > 256 || dim % 2 ||
      (k && (k->scalar_type() != type || k->size(0) != rows || k->size(2) != dim || kheads <= 0 || kheads > 4096)) ||
      pos->dim() != 2 || pos->size(0) != rows || pos->size(1) < 1 || pos->size(1) > 16 ||
      (pt != at::kInt && pt != at::kLong && pt != at::kFloat) || inv->dim() != 1 || inv->scalar_type() != at::kDouble ||
      !inv->is_contiguous() || pairs < 1 || 2 * pairs > dim || axis->dim() != 1 || axis->numel() != pairs ||
      axis->scalar_type() != at::kInt || !axis->is_contiguous() || !fp32_vector(gq, dim) || !fp32_vector(gk, dim) ||
      (gq && k && !gk) || (gk && !(gq && k)) || wants_gradient({q, k, pos, inv, gq, gk, qo, ko}))
    Py_RETURN_NONE;
  if ((qo || ko) && (!qo || (ko != nullptr) != (k != nullptr))) Py_RETURN_NONE;
  if (qo && (qo->scalar_type() != type || qo->sizes() != q->sizes() || !head_strides(*qo, a.q_out_strides)))
    Py_RETURN_NONE;
  if (ko && (ko->scalar_type() != type || ko->sizes() != k->sizes() || !head_strides(*ko, a.k_out_strides)))
    Py_RETURN_NONE;
  const auto opt = at::TensorOptions().device(q->device()).dtype(type);
  at::Tensor q_new, k_new;
  if (!qo) {
    q_new = at::empty({rows, heads, dim}, opt);
    head_strides(q_new, a.q_out_strides);
    if (k) {
      k_new = at::empty({rows, kheads, dim}, opt);
      head_strides(k_new, a.k_out_strides);
    }
  }
  a.dtype = dtype_code(type);
  a.q = q->data_ptr();
  a.k = k ? k->data_ptr() : nullptr;
  a.q_out = qo ? qo->data_ptr() : q_new.data_ptr();
  a.k_out = !k ? nullptr : ko ? ko->data_ptr() : k_new.data_ptr();
  a.rows = rows;
  a.q_heads = (int32_t)heads;
  a.k_heads = (int32_t)kheads;
  a.dim = (int32_t)dim;
  a.pairs = (int32_t)pairs;
  a.axes = (int32_t)pos->size(1);
  a.pairing = args[5] == Py_True ? W8A8_ROPE_ADJACENT : W8A8_ROPE_HALF;
  a.positions = pos->data_ptr();
  a.pos_strides[0] = pos->stride(0);
  a.pos_strides[1] = pos->stride(1);
  a.pos_type = pt == at::kInt ? W8A8_POS_I32 : pt == at::kLong ? W8A8_POS_I64 : W8A8_POS_F32;
  a.inv_freq = ptr<double>(*inv);
  a.axis = ptr<int32_t>(*axis);
  a.q_gain = gq ? ptr<float>(*gq) : nullptr;
  a.k_gain = gk ? ptr<float>(*gk) : nullptr;
  a.stream = stream_of(q->get_device());
  const int rc = call(w8a8_axial_rope, a);
  if (rc != W8A8_OK) return fail("w8a8_axial_rope", rc);
  written(qo);
  written(ko);
  PyObject* pq = qo ? Py_NewRef(args[9]) : THPVariable_Wrap(std::move(q_new));
  PyObject* pk = !k ? Py_NewRef(Py_None) : ko ? Py_NewRef(args[10]) : THPVariable_Wrap(std::move(k_new));
  PyObject* r = pq && pk ? PyTuple_Pack(2, pq, pk) : nullptr;
  Py_XDECREF(pq);
  Py_XDECREF(pk);
  return r;
  END_HANDLE_TH_ERRORS
}

// linear_w4(x, codes, scales, zeros, bias, residual, gated): kernels.linear_w4
// of contiguous tensors into a new output.
PyObject* linear_w4(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || modes_active() || !PyBool_Check(args[6])) Py_RETURN_NONE;
  bool ok = true;
  const at::Tensor* x = plain(args[0]);
  const at::Tensor* codes = plain(args[1]);
  const at::Tensor* scales = plain(args[2]);
  const at::Tensor* zeros = optional(args[3], ok);
  const at::Tensor* bias = optional(args[4], ok);
  const at::Tensor* residual = optional(args[5], ok);
  const bool gated = args[6] == Py_True;
  if (!x || !codes || !scales || !ok || x->dim() < 1 || !x->is_contiguous() || codes->dim() != 2 ||
      codes->scalar_type() != at::kInt || !codes->is_contiguous() || scales->dim() != 2 || !scales->is_contiguous())
    Py_RETURN_NONE;
  const at::ScalarType type = x->scalar_type();
  const int64_t nn = codes->size(0), k = 8 * codes->size(1), groups = scales->size(0);
  if ((type != at::kHalf && type != at::kBFloat16) || scales->scalar_type() != type || k <= 0 || nn <= 0 ||
      x->size(-1) != k || x->numel() == 0 || groups <= 0 || k % groups || scales->size(1) != nn || !aligned(*x, 16) ||
      !aligned(*codes, 16) || codes->size(1) % 4 || wants_gradient({x, scales, bias, residual}))
    Py_RETURN_NONE;
  const int64_t group = k / groups, m = x->numel() / k, width = gated ? nn / 2 : nn;
  if ((group != 32 && group != 64 && group % 128) || (gated && (nn % 2 || residual)) ||
      (zeros && (zeros->scalar_type() != at::kByte || zeros->sizes() != scales->sizes() || !zeros->is_contiguous())) ||
      (bias && (bias->scalar_type() != type || bias->numel() != nn || !bias->is_contiguous())) ||
      (residual && (residual->scalar_type() != type || !residual->is_contiguous())))
    Py_RETURN_NONE;
  const auto opt = at::TensorOptions().device(x->device());
  at::DimVector shape(x->sizes().begin(), x->sizes().end());
  shape.back() = width;
  if (residual && !residual->sizes().equals(shape) && !residual->sizes().equals({m, nn})) Py_RETURN_NONE;
  at::Tensor out = at::empty(shape, opt.dtype(type));
  W8A8LinearW4Args a{};
  at::Tensor workspace;
  a.workspace_bytes = w8a8_linear_w4_workspace_size(m, nn, k, (int32_t)group, gated);
  if (a.workspace_bytes > 0) {
    workspace = at::empty({a.workspace_bytes}, opt.dtype(at::kByte));
    a.workspace = workspace.data_ptr();
  }
  a.dtype = dtype_code(type);
  a.x = x->data_ptr();
  a.ldx = k;
  a.codes = ptr<int32_t>(*codes);
  a.ldw = k / 8;
  a.scales = scales->data_ptr();
  a.zeros = zeros ? ptr<uint8_t>(*zeros) : nullptr;
  a.m = m;
  a.n = nn;
  a.k = k;
  a.group = (int32_t)group;
  a.gated = gated;
  a.bias = bias ? bias->data_ptr() : nullptr;
  a.residual = residual ? residual->data_ptr() : nullptr;
  a.ldr = nn;
  a.out = out.data_ptr();
  a.ldo = width;
  a.stream = stream_of(x->get_device());
  const int rc = call(w8a8_linear_w4, a);
  if (rc != W8A8_OK) return fail("w8a8_linear_w4", rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyObject* set_error_class(PyObject*, PyObject* cls) {
  Py_INCREF(cls);
  Py_XSETREF(g_error_class, cls);
  Py_RETURN_NONE;
}

template <typename F>
PyCFunction fast(F f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

}  // namespace

PyMODINIT_FUNC PyInit__native() {
  static PyMethodDef methods[] = {
      {"linear", fast(linear), METH_FASTCALL, nullptr},
      {"int8_attention", fast(int8_attention), METH_FASTCALL, nullptr},
      {"segment_labels", fast(segment_labels), METH_FASTCALL, nullptr},
      {"residual_norm", fast(residual_norm), METH_FASTCALL, nullptr},
      {"axial_rope", fast(axial_rope), METH_FASTCALL, nullptr},
      {"linear_w4", fast(linear_w4), METH_FASTCALL, nullptr},
      {"set_error_class", set_error_class, METH_O, nullptr},
      {nullptr, nullptr, 0, nullptr},
  };
  static PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};
  return PyModule_Create(&module);
}
