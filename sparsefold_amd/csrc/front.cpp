// The serving-step calls from Python straight to the C entries, in their common form: packed tensors on the current device, outputs
// made here.  A small call is bound by the host (a norm of 8 rows: 3.3 us of kernel, 9.9 us through Python's checks, allocations and
// ctypes), so this form is checked and launched here; every function returns None, having done nothing, where a call is
// of any other form, wrong ones included: the Python wrapper then checks, copies, refuses or runs it.  What is accepted
// here the wrapper accepts too, with the same results.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <optional>

#include "sparsefold_hip.h"

namespace {

// The entries of the library that the Python side has loaded (bind), and its class of codes and scales.
struct Entries {
  decltype(&sf_hip_last_error) last_error;
  decltype(&sf_hip_add_rms_norm_fwd) add_rms_norm;
  decltype(&sf_hip_mx_encode_fwd) mx_encode, mx_decode;
  decltype(&sf_hip_mx_linear_workspace_bytes) mx_linear_bytes;
  decltype(&sf_hip_mx_linear_fwd) mx_linear;
  decltype(&sf_hip_paged_write_fwd) paged_write;
  decltype(&sf_hip_paged_attention_workspace_bytes) paged_attention_bytes;
  decltype(&sf_hip_paged_attention_fwd) paged_attention;
} entry;
PyObject* microscaled = nullptr;

struct Other {};                                             // thrown: a call of another form

void need(bool ok) {
  if (!ok) throw Other();
}

// The arguments of a call: tensors of the current device that take no gradient and carry no tangent.
struct Call {
  int device = -1;
  bool grad = c10::GradMode::is_enabled();
  const at::Tensor& tensor(PyObject* o) {
    need(THPVariable_CheckExact(o));
    const at::Tensor& t = THPVariable_Unpack(o);
    need(t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.has_storage());
    need(!t.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::Functionalize, c10::DispatchKey::FuncTorchBatched,
                                                   c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Negative})));
    need(!(grad && t.requires_grad()) && !t._fw_grad(0).defined());
    if (device < 0) {
      device = t.get_device();
      need(device == c10::hip::current_device());
    }
    need(t.get_device() == device);
    return t;
  }
  const at::Tensor* optional(PyObject* o) { return o == Py_None ? nullptr : &tensor(o); }
  void* stream() const { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream(); }
};

int element(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return SF_DTYPE_BF16;
    case at::kHalf: return SF_DTYPE_F16;
    case at::kFloat: return SF_DTYPE_F32;
    default: throw Other();
  }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

const int32_t* int32s(const at::Tensor& t, int64_t n) {      // n < 0: any number
  need(t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() && (n < 0 || t.size(0) == n));
  return t.data_ptr<int32_t>();
}

at::Tensor empty(at::IntArrayRef sizes, const at::Tensor& like, at::ScalarType type) {
  return at::empty(sizes, at::TensorOptions().dtype(type).device(like.device()));
}

PyObject* failed(const char* what, int rc) {
  char text[1024] = "";
  entry.last_error(text, sizeof text);
  return PyErr_Format(PyExc_RuntimeError, "%s failed (status %d): %s", what, rc, text);
}

// Without the interpreter's lock, as ctypes calls the library: allocations and launches may wait for the device (a full queue, whose
// host functions may want the lock).
struct Unlocked {
  PyThreadState* const state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// Codes and scales for rows like x's.
struct Coded {
  at::Tensor codes, scales;
  Coded(const at::Tensor& x, int format) {
    c10::SmallVector<int64_t, 6> s(x.sizes().begin(), x.sizes().end());
    const int64_t K = s.back();
    s.back() = format == SF_FORMAT_MXFP8 ? K : K / 2;
    codes = empty(s, x, format == SF_FORMAT_MXFP8 ? at::kFloat8_e4m3fn : at::kByte);
    s.back() = K / 32;
    scales = empty(s, x, at::kFloat8_e8m0fnu);
  }
  PyObject* wrap() const {
    PyObject *c = THPVariable_Wrap(codes), *s = THPVariable_Wrap(scales);
    PyObject* r = c && s ? PyObject_CallFunctionObjArgs(microscaled, c, s, nullptr) : nullptr;
    Py_XDECREF(c);
    Py_XDECREF(s);
    return r;
  }
};

int format_of(PyObject* o) {
  need(PyUnicode_Check(o));
  if (PyUnicode_CompareWithASCIIString(o, "mxfp8") == 0) return SF_FORMAT_MXFP8;
  need(PyUnicode_CompareWithASCIIString(o, "mxfp4") == 0);
  return SF_FORMAT_MXFP4;
}

// x, residual, weight, eps, output -> (norm, sum)
PyObject* add_rms_norm(PyObject* const* arg) {
  Call call;
  const at::Tensor& x = call.tensor(arg[0]);
  const at::Tensor* const res = call.optional(arg[1]);
  const at::Tensor* const weight = call.optional(arg[2]);
  sf_add_rms_norm_args a{};
  a.dtype = element(x.scalar_type());
  need(x.dim() >= 1 && x.numel() > 0 && x.is_contiguous() && PyFloat_CheckExact(arg[3]));
  const double eps = PyFloat_AS_DOUBLE(arg[3]);
  const int64_t C = x.size(-1);
  need(C < 1 << 30 && eps >= 0.0 && eps <= 1e30);
  need(res == nullptr || (res->scalar_type() == x.scalar_type() && res->sizes() == x.sizes() && res->is_contiguous()));
  need(weight == nullptr || (weight->scalar_type() == at::kFloat && weight->dim() == 1 && weight->size(0) == C && weight->is_contiguous()));
  a.R = x.numel() / C;
  a.C = (int32_t)C;
  a.eps = (float)eps;
  a.x = x.data_ptr();
  a.residual = res ? res->data_ptr() : nullptr;
  a.weight = weight ? weight->data_ptr<float>() : nullptr;
  a.x_rs = a.r_rs = a.h_rs = a.y_rs = C;
  const bool coded = arg[4] != Py_None;
  if (coded) {
    a.format = format_of(arg[4]);
    need(C % 32 == 0 && al16(a.x) && al16(a.residual));
  }
  at::Tensor y, h;
  std::optional<Coded> q;
  int rc;
  {
    const Unlocked unlocked;
    if (coded) {
      q.emplace(x, a.format);
      a.codes = q->codes.data_ptr();
      a.c_rs = q->codes.size(-1);
      a.scales = q->scales.data_ptr();
      a.s_rs = C / 32;
    } else {
      y = empty(x.sizes(), x, x.scalar_type());
      a.y = y.data_ptr();
    }
    if (res) {
      h = empty(x.sizes(), x, x.scalar_type());
      a.sum = h.data_ptr();
    }
    rc = entry.add_rms_norm(&a, call.stream());
  }
  if (rc) return failed("sf_hip_add_rms_norm_fwd", rc);
  PyObject* const first = coded ? q->wrap() : THPVariable_Wrap(y);
  PyObject* const second = res ? THPVariable_Wrap(h) : Py_NewRef(Py_None);
  PyObject* const both = first && second ? PyTuple_Pack(2, first, second) : nullptr;
  Py_XDECREF(first);
  Py_XDECREF(second);
  return both;
}

// x, format -> codes and scales
PyObject* mx_quantize(PyObject* const* arg) {
  Call call;
  const at::Tensor& x = call.tensor(arg[0]);
  sf_mx_convert_args a{};
  a.dtype = element(x.scalar_type());
  a.format = format_of(arg[1]);
  need(x.dim() >= 1 && x.numel() > 0 && x.is_contiguous() && x.size(-1) % 32 == 0 && x.size(-1) <= INT32_MAX && al16(x.data_ptr()));
  a.K = (int32_t)x.size(-1);
  a.R = x.numel() / a.K;
  a.x = x.data_ptr();
  a.x_rs = a.K;
  std::optional<Coded> q;
  int rc;
  {
    const Unlocked unlocked;
    q.emplace(x, a.format);
    a.codes = q->codes.data_ptr();
    a.c_rs = q->codes.size(-1);
    a.scales = q->scales.data_ptr();
    a.s_rs = a.K / 32;
    rc = entry.mx_encode(&a, call.stream());
  }
  if (rc) return failed("sf_hip_mx_encode_fwd", rc);
  return q->wrap();
}

// Checks codes and scales; returns K, and the format and rows.
int64_t operand(const at::Tensor& codes, const at::Tensor& scales, int32_t& format, int64_t& rows) {
  const bool eight = codes.scalar_type() == at::kFloat8_e4m3fn;
  need(eight || codes.scalar_type() == at::kByte);
  need(scales.scalar_type() == at::kFloat8_e8m0fnu || scales.scalar_type() == at::kByte);
  need(codes.dim() >= 1 && scales.dim() == codes.dim() && codes.is_contiguous() && scales.is_contiguous() && al16(codes.data_ptr()));
  const int64_t K = eight ? codes.size(-1) : 2 * codes.size(-1);
  need(K >= 32 && K % 32 == 0 && K <= 1 << 22 && scales.size(-1) * 32 == K);
  for (int64_t d = 0; d + 1 < codes.dim(); ++d) need(codes.size(d) == scales.size(d));
  format = eight ? SF_FORMAT_MXFP8 : SF_FORMAT_MXFP4;
  rows = scales.numel() / scales.size(-1);
  return K;
}

at::ScalarType type_of(PyObject* o) {
  need(THPDtype_Check(o));
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

// codes, scales, type -> numbers
PyObject* mx_dequantize(PyObject* const* arg) {
  Call call;
  const at::Tensor &codes = call.tensor(arg[0]), &scales = call.tensor(arg[1]);
  const at::ScalarType type = type_of(arg[2]);
  sf_mx_convert_args a{};
  a.dtype = element(type);
  a.K = (int32_t)operand(codes, scales, a.format, a.R);
  need(a.R >= 1);
  c10::SmallVector<int64_t, 6> s(codes.sizes().begin(), codes.sizes().end());
  s.back() = a.K;
  a.x_rs = a.K;
  a.codes = codes.data_ptr();
  a.c_rs = codes.size(-1);
  a.scales = scales.data_ptr();
  a.s_rs = a.K / 32;
  at::Tensor x;
  int rc;
  {
    const Unlocked unlocked;
    x = empty(s, codes, type);
    a.x = x.data_ptr();
    rc = entry.mx_decode(&a, call.stream());
  }
  if (rc) return failed("sf_hip_mx_decode_fwd", rc);
  return THPVariable_Wrap(x);
}

// codes and scales of x and w, bias, type -> y
PyObject* mx_linear(PyObject* const* arg) {
  Call call;
  const at::Tensor &xc = call.tensor(arg[0]), &xs = call.tensor(arg[1]), &wc = call.tensor(arg[2]), &ws = call.tensor(arg[3]);
  const at::Tensor* const bias = call.optional(arg[4]);
  sf_mx_linear_args a{};
  int64_t N = 0;
  need(wc.dim() == 2);
  const int64_t K = operand(xc, xs, a.x_format, a.M);
  need(operand(wc, ws, a.w_format, N) == K && N >= 1 && N <= 1 << 24 && a.M >= 1 && a.M <= INT32_MAX);
  need(!(a.x_format == SF_FORMAT_MXFP4 && a.w_format == SF_FORMAT_MXFP8));
  need(bias == nullptr || (bias->scalar_type() == at::kFloat && bias->dim() == 1 && bias->size(0) == N && bias->is_contiguous()));
  a.N = (int32_t)N;
  a.K = (int32_t)K;
  const at::ScalarType type = type_of(arg[5]);
  a.dtype = element(type);
  need(a.dtype != SF_DTYPE_F32);
  a.x = xc.data_ptr();
  a.x_rs = xc.size(-1);
  a.x_scales = xs.data_ptr();
  a.w = wc.data_ptr();
  a.w_rs = wc.size(-1);
  a.w_scales = ws.data_ptr();
  a.xs_rs = a.ws_rs = K / 32;
  a.bias = bias ? bias->data_ptr<float>() : nullptr;
  c10::SmallVector<int64_t, 6> s(xc.sizes().begin(), xc.sizes().end());
  s.back() = N;
  a.y_rs = N;
  at::Tensor y, work;
  int rc;
  {
    const Unlocked unlocked;
    y = empty(s, xc, type);
    a.y = y.data_ptr();
    const size_t bytes = entry.mx_linear_bytes(&a);
    if (bytes > 0) work = empty({(int64_t)bytes}, xc, at::kByte);
    rc = entry.mx_linear(&a, bytes > 0 ? work.data_ptr() : nullptr, bytes, call.stream());
  }
  if (rc) return failed("sf_hip_mx_linear_fwd", rc);
  return THPVariable_Wrap(y);
}

// Strides of [pages, rows, heads, D], those of a single page or head as if packed, in 16-byte aligned rows.
void page_strides(const at::Tensor& t, int64_t (&s)[3]) {
  const int64_t R = t.size(1), H = t.size(2), D = t.size(3);
  s[2] = H > 1 ? t.stride(2) : D;
  s[1] = t.stride(1);
  s[0] = t.size(0) > 1 ? t.stride(0) : std::max(R * s[1], H * s[2]);
  need((s[0] | s[1] | s[2]) % 8 == 0 && s[1] >= D && s[1] < 1 << 24 && t.stride(3) == 1 && al16(t.data_ptr()));
}

// A cache of B sequences, its table and its lengths into the fields that write and attention name alike.
template <class A>
void cache(A& a, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table, const at::Tensor& lens, at::ScalarType type, int64_t (&ks)[3],
           int64_t (&vs)[3]) {
  need(k.dim() == 4 && v.sizes() == k.sizes() && k.scalar_type() == type && v.scalar_type() == type);
  const int64_t P = k.size(0), R = k.size(1), H = k.size(2), D = k.size(3);
  need(P >= 1 && R >= 16 && R % 16 == 0 && H >= 1 && D % 8 == 0 && D > 0 && D <= 128 && H * D <= 1 << 24);
  need(table.scalar_type() == at::kInt && table.dim() == 2 && table.is_contiguous() && table.size(0) == a.B && table.size(1) >= 1);
  need(R <= 1 << 30 && table.size(1) <= (1 << 30) / R);
  a.Hkv = (int32_t)H;
  a.D = (int32_t)D;
  a.pages = P;
  a.page_rows = (int32_t)R;
  a.table_cols = (int32_t)table.size(1);
  a.table = table.data_ptr<int32_t>();
  a.table_s = table.size(1);
  a.len_k = int32s(lens, a.B);
  page_strides(k, ks);
  page_strides(v, vs);
}

// Row and head strides of [T, H, D] in 16-byte aligned rows, those of a single row or head as if packed.
const void* token_rows(const at::Tensor& t, int64_t (&s)[2]) {
  const int64_t T = t.size(0), H = t.size(1), D = t.size(2);
  s[1] = H > 1 ? t.stride(1) : D;
  s[0] = T > 1 ? t.stride(0) : std::max(H * s[1], H * D);
  need(t.stride(2) == 1 && (s[0] | s[1]) % 8 == 0 && al16(t.data_ptr()));
  return t.data_ptr();
}

struct Dim {
  int64_t size, stride;
};

// Whether a view holds every element once: each dim lies outside what the narrower ones span.
template <size_t N>
bool apart(Dim (&d)[N]) {
  std::sort(d, d + N, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
  int64_t reach = 1;
  for (const Dim& x : d) {
    if (x.size <= 1) continue;
    if (x.stride < reach) return false;
    reach += (x.size - 1) * x.stride;
  }
  return true;
}

// k, v, k_pages, v_pages, table, cu, len_k, len_new -> True
PyObject* paged_cache_write(PyObject* const* arg) {
  Call call;
  const at::Tensor &k = call.tensor(arg[0]), &v = call.tensor(arg[1]), &kp = call.tensor(arg[2]), &vp = call.tensor(arg[3]);
  const at::Tensor &table = call.tensor(arg[4]), &cu = call.tensor(arg[5]), &len_k = call.tensor(arg[6]);
  const at::Tensor* const len_new = call.optional(arg[7]);
  need(k.dim() == 3 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && element(k.scalar_type()) != SF_DTYPE_F32);
  sf_paged_write_args a{};
  a.cu = int32s(cu, -1);
  const int64_t B = cu.size(0) - 1;
  a.T = k.size(0);
  need(B >= 1 && B < 1 << 30 && a.T >= 1 && a.T <= 1 << 30);
  a.B = (int32_t)B;
  cache(a, kp, vp, table, len_k, k.scalar_type(), a.kp_s, a.vp_s);
  need(k.size(1) == a.Hkv && k.size(2) == a.D);
  a.len_new = len_new ? int32s(*len_new, B) : nullptr;
  a.k = token_rows(k, a.k_s);
  a.v = token_rows(v, a.v_s);
  a.k_pages = kp.data_ptr();
  a.v_pages = vp.data_ptr();
  // every place is written once, and overlaps nothing that is read
  const auto dims = [&](const int64_t(&st)[3], int64_t n, int64_t between) {
    Dim d[] = {{a.pages, st[0]}, {a.page_rows, st[1]}, {a.Hkv, st[2]}, {a.D, 1}, {n, between}};
    return apart(d);
  };
  const auto span = [&](const int64_t(&st)[3]) { return 2 * ((a.pages - 1) * st[0] + (a.page_rows - 1) * st[1] + (a.Hkv - 1) * st[2] + a.D); };
  const auto from = [](const void* p) { return (int64_t)reinterpret_cast<uintptr_t>(p); };
  const int64_t k0 = from(a.k_pages), v0 = from(a.v_pages), k1 = k0 + span(a.kp_s), v1 = v0 + span(a.vp_s);
  need(dims(a.kp_s, 1, 0) && dims(a.vp_s, 1, 0));
  need(k1 <= v0 || v1 <= k0 || (std::equal(a.kp_s, a.kp_s + 3, a.vp_s) && dims(a.kp_s, 2, std::abs(v0 - k0) / 2)));
  const auto read = [&](const void* rows, const int64_t(&st)[2]) {
    const int64_t p = from(rows), end = p + 2 * ((a.T - 1) * st[0] + (a.Hkv - 1) * st[1] + a.D);
    return (end <= k0 || k1 <= p) && (end <= v0 || v1 <= p);
  };
  need(read(a.k, a.k_s) && read(a.v, a.v_s));
  int rc;
  {
    const Unlocked unlocked;
    rc = entry.paged_write(&a, call.stream());
  }
  if (rc) return failed("sf_hip_paged_write_fwd", rc);
  for (const at::Tensor* t : {&kp, &vp})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return Py_NewRef(Py_True);
}

// q, k_pages, v_pages, table, cu_q, len_k, len_q, causal, scale, max_len -> out
PyObject* paged_attention(PyObject* const* arg) {
  Call call;
  const at::Tensor &q = call.tensor(arg[0]), &kp = call.tensor(arg[1]), &vp = call.tensor(arg[2]);
  const at::Tensor &table = call.tensor(arg[3]), &cu = call.tensor(arg[4]), &len_k = call.tensor(arg[5]);
  const at::Tensor* const len_q = call.optional(arg[6]);
  need(q.dim() == 3 && (arg[7] == Py_True || arg[7] == Py_False) && (arg[8] == Py_None || PyFloat_CheckExact(arg[8])));
  need(arg[9] == Py_None || PyLong_CheckExact(arg[9]));
  sf_paged_attention_args a{};
  a.dtype = element(q.scalar_type());
  need(a.dtype != SF_DTYPE_F32);
  a.cu_q = int32s(cu, -1);
  const int64_t B = cu.size(0) - 1, H = q.size(1);
  a.Tq = q.size(0);
  need(B >= 1 && B < 1 << 30 && a.Tq >= 1 && H >= 1 && H <= 1 << 24);
  a.B = (int32_t)B;
  a.H = (int32_t)H;
  cache(a, kp, vp, table, len_k, q.scalar_type(), a.k_s, a.v_s);
  need(q.size(2) == a.D && H % a.Hkv == 0);
  a.len_q = len_q ? int32s(*len_q, B) : nullptr;
  a.causal = arg[7] == Py_True;
  const double scale = arg[8] == Py_None ? 1.0 / std::sqrt((double)a.D) : PyFloat_AS_DOUBLE(arg[8]);
  need(std::fabs(scale) <= 1e30);
  a.scale = (float)scale;
  if (arg[9] != Py_None) {
    const long long most = PyLong_AsLongLong(arg[9]);
    if (most == -1 && PyErr_Occurred()) PyErr_Clear();
    need(most >= 0 && most < 1ll << 62);
    a.max_keys = std::max(most, 1ll);
  }
  a.q = token_rows(q, a.q_s);
  a.k = kp.data_ptr();
  a.v = vp.data_ptr();
  a.o_s[0] = H * a.D;
  a.o_s[1] = a.D;
  at::Tensor out, work;
  int rc;
  {
    const Unlocked unlocked;
    out = empty(q.sizes(), q, q.scalar_type());
    a.out = out.data_ptr();
    const size_t bytes = entry.paged_attention_bytes(&a);
    if (bytes > 0) work = empty({(int64_t)bytes}, q, at::kByte);
    rc = entry.paged_attention(&a, bytes > 0 ? work.data_ptr() : nullptr, bytes, call.stream());
  }
  if (rc) return failed("sf_hip_paged_attention_fwd", rc);
  return THPVariable_Wrap(out);
}

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* method(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n == N && microscaled != nullptr && !c10::impl::TorchDispatchModeTLS::any_modes_set()) {
    try {
      return F(args);
    } catch (const Other&) {
    } catch (const std::exception&) {                        // (an allocation that fails: raised by the wrapper's own)
    }
    PyErr_Clear();
  }
  Py_RETURN_NONE;
}

// addresses of the entries in the order of Entries, then the class of codes and scales
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  constexpr int kEntries = sizeof(Entries) / sizeof(void*);
  void* p[kEntries];
  if (n != kEntries + 1) return PyErr_Format(PyExc_TypeError, "%d addresses and a class", kEntries);
  for (int i = 0; i < kEntries; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (p[i] == nullptr) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "a null address");
  }
  __builtin_memcpy(&entry, p, sizeof p);
  Py_XSETREF(microscaled, Py_NewRef(args[kEntries]));
  Py_RETURN_NONE;
}

#define METHOD(F, N) {#F, reinterpret_cast<PyCFunction>(method<F, N>), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(add_rms_norm, 5), METHOD(mx_quantize, 2), METHOD(mx_dequantize, 3), METHOD(mx_linear, 6), METHOD(paged_cache_write, 8), METHOD(paged_attention, 10),
                         {"bind", reinterpret_cast<PyCFunction>(bind), METH_FASTCALL, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_front", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__front() {
  PyObject* const m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddIntConstant(m, "abi_version", SF_HIP_ABI_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
