// The per-call host path of a packed linear, of the 8-bit KV cache's calls and of packed attention, in native code: checks the plain form of a call (contiguous
// tensors of the expected dtypes and shapes on one device), allocates the output and the workspace from
// torch's caching allocator and calls the C ABI on the current stream. The checks run on every call and
// nothing is kept between calls. A call in any other form returns None, and the caller takes the general
// path, which converts, broadcasts or raises as torch would.
//
// Why: at one token the kernel takes 4.8 us, and the same steps in Python (attribute look-ups, checks,
// two ctypes calls) held a 4096 x 4096 call at 18.9 us; 6.9 us with this path. An append to the 8-bit cache, a decode
// step's attention over it and a short packed prompt: 28 / 36 / 17 us in Python, 7.8 / 12.5 / 6.2 here, as kernels
// 4.2 / 8.5 / 6.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

namespace {

using LinearFn = int (*)(const void*, int64_t, int64_t, int64_t, const void*, int64_t, const float*, const float*,
                         const void*, void*, int64_t, int64_t, int, int, int, int, int, void*, size_t, void*, int);
using SwigluFn = int (*)(const void*, int64_t, int64_t, int64_t, const void*, int64_t, const float*, const float*,
                         const void*, void*, int64_t, int64_t, int, int, int, int, int, void*, size_t, void*);
using WorkspaceFn = size_t (*)(int64_t, int64_t, int64_t, int, int, int);

struct Api {
  LinearFn linear = nullptr;
  SwigluFn swiglu = nullptr;
  WorkspaceFn linear_ws = nullptr, swiglu_ws = nullptr;
} g_api;

// attach(linear_ex, linear_workspace_ex, linear_swiglu, linear_swiglu_workspace_ex): the C ABI's addresses.
PyObject* attach(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "attach takes four addresses");
    return nullptr;
  }
  void* p[4];
  for (int i = 0; i < 4; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (!p[i] && PyErr_Occurred()) return nullptr;
  }
  g_api.linear = reinterpret_cast<LinearFn>(p[0]);
  g_api.linear_ws = reinterpret_cast<WorkspaceFn>(p[1]);
  g_api.swiglu = reinterpret_cast<SwigluFn>(p[2]);
  g_api.swiglu_ws = reinterpret_cast<WorkspaceFn>(p[3]);
  Py_RETURN_NONE;
}

const at::Tensor* tensor_of(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// linear(x, qweight, scales, zeros, bias, out_features, in_features, bits, group_size, symmetric, dtype,
// swiglu) -> tensor or None. dtype: 0 fp32, 1 fp16, 2 bf16. swiglu: fused gate/up rows, out_features / 2
// columns come back.
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 12 || !g_api.linear) {
    PyErr_SetString(PyExc_TypeError, "linear takes twelve arguments, after attach");
    return nullptr;
  }
  HANDLE_TH_ERRORS  // torch's own exception types: an allocation that fails is torch.OutOfMemoryError
  if (!THPVariable_CheckExact(args[0])) Py_RETURN_NONE;  // a subclass may see the general path's torch calls
  const at::Tensor *x = tensor_of(args[0]), *qw = tensor_of(args[1]), *sc = tensor_of(args[2]);
  const at::Tensor* zp = tensor_of(args[3]);
  const at::Tensor* bias = tensor_of(args[4]);
  if (!x || !qw || !sc || (!bias && args[4] != Py_None)) Py_RETURN_NONE;
  int64_t v[7];
  for (int i = 0; i < 7; ++i) {
    v[i] = PyLong_AsLongLong(args[5 + i]);
    if (v[i] == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
  }
  const int64_t N = v[0], K = v[1], bits = v[2], group = v[3] > 0 ? v[3] : v[1], dtype = v[5];
  const bool symmetric = v[4] != 0, swiglu = v[6] != 0;
  if (N < 1 || K < 1 || N > INT32_MAX || K > INT32_MAX || bits < 1 || bits > 8 || K % group != 0 || dtype < 0 ||
      dtype > 2 || (swiglu && N % 8 != 0))
    Py_RETURN_NONE;
  const at::ScalarType act = dtype == 0 ? at::kFloat : dtype == 1 ? at::kHalf : at::kBFloat16;
  const at::Device dev = x->device();
  if (!dev.is_cuda() || x->layout() != at::kStrided || x->scalar_type() != act || x->dim() < 1 ||
      x->size(-1) != K || !x->is_contiguous())
    Py_RETURN_NONE;
  const int64_t G = K / group, M = x->numel() / K;
  if (M < 1) Py_RETURN_NONE;
  const bool is_signed = qw->scalar_type() == at::kChar;
  if (qw->device() != dev || !(qw->scalar_type() == at::kByte || (bits == 8 && is_signed)) || qw->dim() != 2 ||
      qw->size(0) != N || qw->size(1) < (bits == 8 ? K : (K + 1) / 2) || !qw->is_contiguous())
    Py_RETURN_NONE;
  auto plain_meta = [&](const at::Tensor* t) {
    return t && t->device() == dev && t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(0) == N &&
           t->size(1) == G && t->is_contiguous();
  };
  if (!plain_meta(sc) || (!symmetric && !plain_meta(zp))) Py_RETURN_NONE;
  if (bias && (bias->device() != dev || bias->scalar_type() != act || bias->dim() != 1 || bias->size(0) != N ||
               !bias->is_contiguous()))
    Py_RETURN_NONE;

  const size_t ws_bytes = (swiglu ? g_api.swiglu_ws : g_api.linear_ws)(M, N, K, int(bits), int(group), int(dtype));
  const int64_t cols = swiglu ? N / 2 : N;
  at::Tensor y, ws;
  {
    const auto options = at::TensorOptions().device(dev);
    c10::SmallVector<int64_t, 6> shape(x->sizes().begin(), x->sizes().end());
    shape.back() = cols;
    y = at::empty(shape, options.dtype(act));
    if (ws_bytes) ws = at::empty({int64_t(ws_bytes)}, options.dtype(at::kByte));
  }
  void* stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  const void *xp = x->const_data_ptr(), *qp = qw->const_data_ptr();
  const float *sp = sc->const_data_ptr<float>(), *zpp = symmetric ? nullptr : zp->const_data_ptr<float>();
  const void* bp = bias ? bias->const_data_ptr() : nullptr;
  void *yp = y.mutable_data_ptr(), *wp = ws_bytes ? ws.mutable_data_ptr() : nullptr;
  int rc;
  {
    pybind11::gil_scoped_release released;  // taken again also where the call throws
    rc = swiglu ? g_api.swiglu(xp, M, K, K, qp, qw->size(1), sp, zpp, bp, yp, N, cols, int(dtype), int(bits),
                               int(group), symmetric, is_signed, wp, ws_bytes, stream)
                : g_api.linear(xp, M, K, K, qp, qw->size(1), sp, zpp, bp, yp, N, cols, int(dtype), int(bits),
                               int(group), symmetric, is_signed, wp, ws_bytes, stream, 0);
  }
  if (rc != 0) Py_RETURN_NONE;  // the general path asks again and reports the error
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// ---- the 8-bit KV cache and packed prompts (include/llmopt_kvq.h) ----

using KvqWriteFn = int (*)(void*, float*, void*, float*, int, int64_t, int64_t, int64_t, int64_t, const int32_t*, int64_t,
                           const int32_t*, const int32_t*, const int32_t*, const void*, int64_t, int64_t, int64_t,
                           const void*, int64_t, int64_t, int64_t, int, int64_t, int64_t, int64_t, void*);
using KvqWorkspaceFn = size_t (*)(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int, int);
using KvqAttentionFn = int (*)(const void*, int, int64_t, int64_t, int64_t, const void*, const float*, const void*,
                               const float*, int, int64_t, int64_t, int64_t, int64_t, const int32_t*, int64_t,
                               const int32_t*, int64_t, int64_t, int64_t, float, float, void*, int64_t, int64_t, int64_t,
                               int, void*, size_t, void*);
using PackedFn = int (*)(const void*, int64_t, int64_t, const void*, int64_t, int64_t, const void*, int64_t, int64_t, int,
                         const int32_t*, int64_t, int64_t, int64_t, int64_t, int64_t, float, float, void*, int64_t,
                         int64_t, int, void*);

struct KvqApi {
  KvqWriteFn write = nullptr;
  KvqWorkspaceFn workspace = nullptr;
  KvqAttentionFn attention = nullptr;
  PackedFn packed = nullptr;
} g_kvq;

// attach_kvq(kvq_write, kvq_attention_workspace, kvq_attention, packed_attention): the C ABI's addresses.
PyObject* attach_kvq(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "attach_kvq takes four addresses");
    return nullptr;
  }
  void* p[4];
  for (int i = 0; i < 4; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (!p[i] && PyErr_Occurred()) return nullptr;
  }
  g_kvq.write = reinterpret_cast<KvqWriteFn>(p[0]);
  g_kvq.workspace = reinterpret_cast<KvqWorkspaceFn>(p[1]);
  g_kvq.attention = reinterpret_cast<KvqAttentionFn>(p[2]);
  g_kvq.packed = reinterpret_cast<PackedFn>(p[3]);
  Py_RETURN_NONE;
}

int dtype_code(const at::Tensor& t) {
  const auto s = t.scalar_type();
  return s == at::kFloat ? 0 : s == at::kHalf ? 1 : s == at::kBFloat16 ? 2 : -1;
}

// An int32 tensor of `dim` dimensions with at least `rows` rows, contiguous and on the device.
bool plain_int32(const at::Tensor* t, const at::Device& dev, int64_t dim, int64_t rows) {
  return t && t->device() == dev && t->scalar_type() == at::kInt && t->dim() == dim && t->size(0) >= rows &&
         t->is_contiguous();
}

// One layer of a QuantizedPagedKVCache's tensors (args: key_codes, key_scales, value_codes, value_scales, layer).
struct Layer {
  char* codes[2];
  float* scales[2];
  int format;
  int64_t blocks, heads, block_size, head_dim;
  at::Device device = at::kCPU;

  const at::Tensor* t[4];

  // Whether the four tensors are a cache (whole, all layers) on one HIP device.
  bool check(PyObject* const* args) {
    for (int i = 0; i < 4; ++i)
      if (!(t[i] = tensor_of(args[i]))) return false;
    device = t[0]->device();
    const auto type = t[0]->scalar_type();
    if (!device.is_cuda() || (type != at::kChar && type != at::kFloat8_e4m3fn) || t[0]->dim() != 5) return false;
    for (int k = 0; k < 2; ++k) {
      const at::Tensor &c = *t[2 * k], &s = *t[2 * k + 1];
      if (c.device() != device || c.scalar_type() != type || c.sizes() != t[0]->sizes() || !c.is_contiguous() ||
          s.device() != device || s.scalar_type() != at::kFloat || s.sizes() != t[0]->sizes().slice(0, 3) ||
          !s.is_contiguous())
        return false;
    }
    format = type == at::kChar ? 0 : 1;
    return true;
  }

  bool from(PyObject* const* args) {
    if (!check(args)) return false;
    const int64_t layer = PyLong_AsLongLong(args[4]);
    if (layer == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      return false;
    }
    if (layer < 0 || layer >= t[0]->size(0)) return false;
    blocks = t[0]->size(1), heads = t[0]->size(2), block_size = t[0]->size(3), head_dim = t[0]->size(4);
    for (int k = 0; k < 2; ++k) {
      codes[k] = static_cast<char*>(t[2 * k]->mutable_data_ptr()) + layer * blocks * heads * block_size * head_dim;
      scales[k] = static_cast<float*>(t[2 * k + 1]->mutable_data_ptr()) + layer * blocks * heads;
    }
    return true;
  }
};

// kvq_cache_shape(key_codes, key_scales, value_codes, value_scales) -> (layers, blocks, kv_heads, block_size, head_dim), or
// None where the general checks have to look.
PyObject* kvq_cache_shape(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "kvq_cache_shape takes four tensors");
    return nullptr;
  }
  HANDLE_TH_ERRORS
  Layer c;
  if (!c.check(args) || c.t[0]->numel() == 0) Py_RETURN_NONE;
  const auto s = c.t[0]->sizes();
  return Py_BuildValue("(LLLLL)", (long long)s[0], (long long)s[1], (long long)s[2], (long long)s[3], (long long)s[4]);
  END_HANDLE_TH_ERRORS
}

bool on_current_device(const at::Device& dev) { return dev.index() == c10::hip::current_device(); }

// kvq_write(key_codes, key_scales, value_codes, value_scales, layer, block_ids, token_offsets, keys, values, cu_seqlens
// or None, query_lens or None) -> True, or None where the general path has to take the call. keys and values
// [seq, kv_heads, head_dim] (one token each) or [seq, q_len, kv_heads, head_dim], with cu_seqlens [tokens, ...].
PyObject* kvq_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 11 || !g_kvq.write) {
    PyErr_SetString(PyExc_TypeError, "kvq_write takes eleven arguments, after attach_kvq");
    return nullptr;
  }
  HANDLE_TH_ERRORS
  Layer c;
  const at::Tensor *table = tensor_of(args[5]), *offsets = tensor_of(args[6]), *k = tensor_of(args[7]);
  const at::Tensor *v = tensor_of(args[8]), *cu = tensor_of(args[9]), *lens = tensor_of(args[10]);
  if (!k || !v || (!cu && args[9] != Py_None) || (!lens && args[10] != Py_None) || !c.from(args)) Py_RETURN_NONE;
  const int dtype = dtype_code(*k);
  const int64_t dim = k->dim();
  if (dtype < 0 || v->scalar_type() != k->scalar_type() || k->device() != c.device || v->device() != c.device ||
      (cu ? dim != 3 : dim != 3 && dim != 4) || k->sizes() != v->sizes() || k->size(dim - 1) != c.head_dim ||
      k->size(dim - 2) != c.heads || k->stride(dim - 1) != 1 || v->stride(dim - 1) != 1 || k->numel() == 0)
    Py_RETURN_NONE;
  if (cu && (lens || !plain_int32(cu, c.device, 1, 2))) Py_RETURN_NONE;
  const int64_t seqs = cu ? cu->size(0) - 1 : k->size(0), q_len = cu ? 0 : dim == 4 ? k->size(1) : 1;
  if (!plain_int32(table, c.device, 2, seqs) || !plain_int32(offsets, c.device, 1, seqs) ||
      (lens && !plain_int32(lens, c.device, 1, seqs)) || !on_current_device(c.device))
    Py_RETURN_NONE;
  auto seq = [&](const at::Tensor* t) { return cu ? 0 : t->stride(0); };
  auto tok = [&](const at::Tensor* t) { return cu ? t->stride(0) : dim == 4 ? t->stride(1) : 0; };
  const int64_t ks = seq(k), kt = tok(k), kh = k->stride(dim - 2), vs = seq(v), vt = tok(v), vh = v->stride(dim - 2);
  const int64_t ldb = table->size(1), tokens = cu ? k->size(0) : 0;
  void* stream = c10::hip::getCurrentHIPStream(c.device.index()).stream();
  const auto* tp = table->const_data_ptr<int32_t>();
  const auto* op = offsets->const_data_ptr<int32_t>();
  const auto* cp = cu ? cu->const_data_ptr<int32_t>() : nullptr;
  const auto* lp = lens ? lens->const_data_ptr<int32_t>() : nullptr;
  const void *kp = k->const_data_ptr(), *vp = v->const_data_ptr();
  int rc;
  {
    pybind11::gil_scoped_release released;
    rc = g_kvq.write(c.codes[0], c.scales[0], c.codes[1], c.scales[1], c.format, c.blocks, c.block_size, c.heads,
                     c.head_dim, tp, ldb, op, cp, lp, kp, ks, kt, kh, vp, vs, vt, vh, dtype, seqs, q_len, tokens, stream);
  }
  if (rc != 0) Py_RETURN_NONE;  // the general path asks again and reports the error
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// kvq_attention(key_codes, key_scales, value_codes, value_scales, layer, block_ids, context_lens, query, q_len, scale,
// softcap) -> [seq, heads, q_len, head_dim], a view of token-major rows, or None.
PyObject* kvq_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 11 || !g_kvq.attention) {
    PyErr_SetString(PyExc_TypeError, "kvq_attention takes eleven arguments, after attach_kvq");
    return nullptr;
  }
  HANDLE_TH_ERRORS
  if (!THPVariable_CheckExact(args[7])) Py_RETURN_NONE;
  Layer c;
  const at::Tensor *table = tensor_of(args[5]), *lens = tensor_of(args[6]), *q = tensor_of(args[7]);
  const int64_t q_len = PyLong_AsLongLong(args[8]);
  const double scale = PyFloat_AsDouble(args[9]), softcap = PyFloat_AsDouble(args[10]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (!q || q->dim() != 4 || !c.from(args)) Py_RETURN_NONE;
  const int dtype = dtype_code(*q);
  const int64_t seqs = q->size(0), heads = q->size(1);
  if (dtype < 0 || q->device() != c.device || q->size(3) != c.head_dim || q->stride(3) != 1 || q_len < 1 ||
      q->size(2) < q_len || seqs < 1 || heads < 1 || heads % c.heads != 0 || !plain_int32(table, c.device, 2, seqs) ||
      !plain_int32(lens, c.device, 1, seqs) || !on_current_device(c.device))
    Py_RETURN_NONE;
  const void* qp = q->const_data_ptr();
  if (dtype && q_len > 1 && (reinterpret_cast<uintptr_t>(qp) % 16 || q->stride(0) % 8 || q->stride(1) % 8 || q->stride(2) % 8))
    Py_RETURN_NONE;
  const int64_t ldb = table->size(1), d = c.head_dim;
  const size_t ws_bytes = g_kvq.workspace(seqs, heads, c.heads, d, q_len, ldb, c.block_size, dtype, 0);
  const auto options = at::TensorOptions().device(c.device);
  at::Tensor ws;
  at::Tensor out = at::empty_strided({seqs, heads, q_len, d}, {q_len * heads * d, d, heads * d, 1}, options.dtype(q->scalar_type()));
  if (ws_bytes) ws = at::empty({int64_t(ws_bytes)}, options.dtype(at::kByte));
  void* stream = c10::hip::getCurrentHIPStream(c.device.index()).stream();
  const auto* tp = table->const_data_ptr<int32_t>();
  const auto* lp = lens->const_data_ptr<int32_t>();
  void *op = out.mutable_data_ptr(), *wp = ws_bytes ? ws.mutable_data_ptr() : nullptr;
  const int64_t q0 = q->stride(0), q1 = q->stride(1), q2 = q->stride(2);
  int rc;
  {
    pybind11::gil_scoped_release released;
    rc = g_kvq.attention(qp, dtype, q0, q1, q2, c.codes[0], c.scales[0], c.codes[1], c.scales[1], c.format, c.blocks,
                         c.block_size, c.heads, d, tp, ldb, lp, seqs, heads, q_len, float(scale), float(softcap), op,
                         q_len * heads * d, d, heads * d, 0, wp, ws_bytes, stream);
  }
  if (rc != 0) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// packed_attention(query, key, value, cu_seqlens, scale, softcap) -> [tokens, heads, head_dim], or None.
PyObject* packed_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 6 || !g_kvq.packed) {
    PyErr_SetString(PyExc_TypeError, "packed_attention takes six arguments, after attach_kvq");
    return nullptr;
  }
  HANDLE_TH_ERRORS
  if (!THPVariable_CheckExact(args[0])) Py_RETURN_NONE;
  const at::Tensor *q = tensor_of(args[0]), *k = tensor_of(args[1]), *v = tensor_of(args[2]), *cu = tensor_of(args[3]);
  const double scale = PyFloat_AsDouble(args[4]), softcap = PyFloat_AsDouble(args[5]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (!q || !k || !v || q->dim() != 3 || k->dim() != 3 || v->sizes() != k->sizes()) Py_RETURN_NONE;
  const int dtype = dtype_code(*q);
  const at::Device dev = q->device();
  const int64_t tokens = q->size(0), heads = q->size(1), d = q->size(2), kvh = k->size(1);
  if (dtype < 1 || !dev.is_cuda() || k->device() != dev || v->device() != dev || k->scalar_type() != q->scalar_type() ||
      v->scalar_type() != q->scalar_type() || k->size(0) != tokens || k->size(2) != d || tokens < 1 || kvh < 1 ||
      heads < 1 || heads % kvh != 0 || q->stride(2) != 1 || k->stride(2) != 1 || v->stride(2) != 1 ||
      !plain_int32(cu, dev, 1, 1) || !on_current_device(dev))
    Py_RETURN_NONE;
  at::Tensor out = at::empty({tokens, heads, d}, q->options());
  void* stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  const void *qp = q->const_data_ptr(), *kp = k->const_data_ptr(), *vp = v->const_data_ptr();
  const auto* cp = cu->const_data_ptr<int32_t>();
  void* op = out.mutable_data_ptr();
  const int64_t seqs = cu->size(0) - 1;
  const int64_t s[6] = {q->stride(0), q->stride(1), k->stride(0), k->stride(1), v->stride(0), v->stride(1)};
  int rc;
  {
    pybind11::gil_scoped_release released;
    rc = g_kvq.packed(qp, s[0], s[1], kp, s[2], s[3], vp, s[4], s[5], dtype, cp, seqs, tokens, heads, kvh, d, float(scale),
                      float(softcap), op, heads * d, d, 1, stream);
  }
  if (rc != 0) Py_RETURN_NONE;  // the general path copies what is not aligned, or reports the error
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"attach", reinterpret_cast<PyCFunction>(attach), METH_FASTCALL, nullptr},
    {"attach_kvq", reinterpret_cast<PyCFunction>(attach_kvq), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(linear), METH_FASTCALL, nullptr},
    {"kvq_cache_shape", reinterpret_cast<PyCFunction>(kvq_cache_shape), METH_FASTCALL, nullptr},
    {"kvq_write", reinterpret_cast<PyCFunction>(kvq_write), METH_FASTCALL, nullptr},
    {"kvq_attention", reinterpret_cast<PyCFunction>(kvq_attention), METH_FASTCALL, nullptr},
    {"packed_attention", reinterpret_cast<PyCFunction>(packed_attention), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_llmopt_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__llmopt_torch(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) != 0) Py_CLEAR(m);
  return m;
}
