// Python entry of the 8-bit operators: argument checks, outputs and streams in C++.
//
// A call of a small operator takes a few microseconds on the GPU, less than its checks and its two dozen ctypes
// arguments take in Python.  This extension does for them what the Python wrappers do elsewhere - checks with the
// same exception types, an output of torch's allocator, torch's current stream on the tensors' device, that device
// made current for the launch - and calls libnqt's C ABI through the addresses that `init` was given.  A negative
// libnqt code is returned as an int, which the Python side raises.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cfloat>
#include <cmath>
#include <optional>

#include "../../include/nqt.h"

namespace {

constexpr int kBlock = 16;
constexpr int kMaxDevices = 64;

decltype(&nqt_decode_attention8) f_decode8;
decltype(&nqt_prefill_attention8) f_prefill8;
decltype(&nqt_qk_norm_rope_paged_cache8) f_write8;
decltype(&nqt_read_paged_cache8) f_read8;
decltype(&nqt_gemm_int8) f_gemm_int8;
decltype(&nqt_linear_int8) f_linear_int8;
decltype(&nqt_linear_int8_launches) f_linear_int8_launches;
constexpr int kEntryPoints = 7;

int32_t* g_status[kMaxDevices];
long long g_launches;

struct Fail {
  PyObject* type;
  const char* msg;
};

[[noreturn]] void value_error(const char* msg) { throw Fail{PyExc_ValueError, msg}; }
[[noreturn]] void type_error(const char* msg) { throw Fail{PyExc_TypeError, msg}; }

const at::Tensor& tensor(PyObject* o) {
  if (!THPVariable_Check(o)) type_error("libnqt operators take torch tensors");
  return THPVariable_Unpack(o);
}

// None or a tensor.
std::optional<at::Tensor> maybe(PyObject* o) {
  if (o == Py_None) return std::nullopt;
  return tensor(o);
}

long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Fail{nullptr, nullptr};
  return v;
}

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Fail{nullptr, nullptr};
  return v;
}

// The device that all of them live on.
struct Device {
  int index = -1;
  void add(const at::Tensor& t) {
    const int i = t.is_cuda() ? t.get_device() : -1;
    if (i < 0 || i >= kMaxDevices || (index >= 0 && i != index))
      value_error("libnqt kernels require CUDA tensors on one device");
    index = i;
  }
  void add(const std::optional<at::Tensor>& t) {
    if (t) add(*t);
  }
};

// Runs `launch(status, stream)` with the device current.
template <typename F>
int on_device(const Device& dev, F launch) {
  const c10::cuda::OptionalCUDAGuard guard(
      c10::cuda::current_device() == dev.index ? std::nullopt : std::optional<c10::Device>(c10::Device(
                                                                    c10::kCUDA, static_cast<c10::DeviceIndex>(dev.index))));
  // the Python side makes the device's status word and calls again
  if (g_status[dev.index] == nullptr) return -1000 - dev.index;
  ++g_launches;
  return launch(g_status[dev.index], c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev.index)).stream());
}

PyObject* result(int rc, const at::Tensor& out) {
  if (rc < 0) return PyLong_FromLong(rc);
  return THPVariable_Wrap(out);
}

int cache_code(const at::Tensor& cache, const at::Tensor& scales, int64_t hkv, int64_t d) {
  int code;
  if (cache.scalar_type() == at::kChar) code = NQT_I8;
  else if (cache.scalar_type() == at::kFloat8_e4m3fn) code = NQT_E4M3;
  else type_error("an 8-bit KV cache holds int8 or float8_e4m3fn");
  if (cache.dim() != 5 || cache.size(1) != 2 || cache.size(3) != hkv || cache.size(4) != d)
    value_error("8-bit paged cache must be [pages, 2, page_size, kv_heads, head_dim]");
  const int64_t page = cache.size(2);
  if (page % kBlock || page < kBlock || page > 256)
    value_error("8-bit paged cache needs a page size that is a multiple of 16 up to 256");
  if (d != 64 && d != 128) value_error("8-bit paged cache needs head_dim 64 or 128");
  if (scales.scalar_type() != at::kFloat) type_error("8-bit paged cache scales must be float32");
  if (scales.dim() != 4 || scales.size(0) != cache.size(0) || scales.size(1) != 2 ||
      scales.size(2) != page / kBlock || scales.size(3) != hkv)
    value_error("8-bit paged cache scales must be [pages, 2, page_size / 16, kv_heads]");
  if (!cache.is_contiguous() || !scales.is_contiguous()) value_error("8-bit paged cache and its scales must be contiguous");
  if (cache.size(0) > 0x3fffffff) value_error("8-bit paged cache has too many pages");
  return code;
}

bool is_i32_vector(const at::Tensor& t) { return t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous(); }
bool is_i64_vector(const at::Tensor& t, int64_t n) {
  return t.scalar_type() == at::kLong && t.dim() == 1 && t.size(0) == n && t.is_contiguous();
}

void check_attention_out(const at::Tensor& q, const std::optional<at::Tensor>& out) {
  if (out && (out->sizes() != q.sizes() || out->scalar_type() != at::kBFloat16 || out->stride(2) != 1))
    value_error("attention output must be bf16 of the query's shape, contiguous per head");
}

int check_paged8(const at::Tensor& q, const at::Tensor& cache, const at::Tensor& scales, const at::Tensor& indptr,
                 const at::Tensor& indices, const at::Tensor& last, int64_t rows, const std::optional<at::Tensor>& out) {
  if (q.dim() != 3 || cache.dim() != 5)
    value_error("8-bit paged attention takes query [tokens, heads, head_dim] and a rank-five cache");
  const int64_t hq = q.size(1), hkv = cache.size(3);
  if (hkv < 1 || hq < 1 || hq % hkv || hq / hkv > 8) value_error("8-bit paged attention needs 1 to 8 query heads per KV head");
  if (q.scalar_type() != at::kBFloat16) type_error("8-bit paged attention runs on a bf16 query");
  const int code = cache_code(cache, scales, hkv, q.size(2));
  if (q.stride(2) != 1) value_error("query must be contiguous per head");
  if (!is_i32_vector(indptr) || !is_i32_vector(indices) || !is_i32_vector(last))
    type_error("paged KV metadata must be contiguous int32");
  if (rows < 0 || indptr.size(0) < rows + 1 || last.size(0) < rows) value_error("paged KV metadata must cover every row");
  check_attention_out(q, out);
  return code;
}

// No row has a page: the empty table has no address, and nothing reads one.
const int32_t* table(const at::Tensor& indices, const at::Tensor& indptr) {
  return static_cast<const int32_t*>((indices.numel() ? indices : indptr).const_data_ptr());
}

at::Tensor contiguous_like(const at::Tensor& q) { return at::empty(q.sizes(), q.options()); }

// (query, cache, scales, kv_indptr, kv_indices, last_page_len, workspace, batch_capacity, sm_scale, out, flags)
PyObject* decode8(PyObject* const* a) {
  const at::Tensor &q = tensor(a[0]), &cache = tensor(a[1]), &scales = tensor(a[2]), &indptr = tensor(a[3]),
                   &indices = tensor(a[4]), &last = tensor(a[5]), &ws = tensor(a[6]);
  auto out = maybe(a[9]);
  if (q.dim() < 1) value_error("8-bit paged attention takes query [tokens, heads, head_dim] and a rank-five cache");
  const int64_t rows = q.size(0);
  const int code = check_paged8(q, cache, scales, indptr, indices, last, rows, out);
  const long long cap = a[7] == Py_None ? rows : integer(a[7]);
  const double scale = a[8] == Py_None ? 1.0 / std::sqrt(static_cast<double>(q.size(2))) : number(a[8]);
  const long long flags = integer(a[10]);
  if (cap < rows || cap > 0x7fffffff) value_error("batch_capacity must cover the rows");
  if (!ws.is_contiguous()) value_error("the decode workspace must be contiguous");
  Device dev;
  for (int i = 0; i < 7; ++i) dev.add(tensor(a[i]));
  dev.add(out);
  if (!out) out = contiguous_like(q);
  if (rows == 0) return THPVariable_Wrap(*out);
  return result(on_device(dev, [&](int32_t* status, void* stream) {
    return f_decode8(q.const_data_ptr(), q.stride(0), q.stride(1), cache.const_data_ptr(),
                     scales.const_data_ptr<float>(), static_cast<int>(cache.size(0)), static_cast<int>(cache.size(2)),
                     indptr.const_data_ptr<int32_t>(), table(indices, indptr), last.const_data_ptr<int32_t>(),
                     static_cast<int>(rows), static_cast<int>(cap), static_cast<int>(q.size(1)),
                     static_cast<int>(cache.size(3)), static_cast<int>(q.size(2)), static_cast<float>(scale), code,
                     out->data_ptr(), out->stride(0), out->stride(1), ws.data_ptr(), ws.nbytes(),
                     static_cast<int>(flags), status, stream);
  }), *out);
}

// (query, cache, scales, qo_indptr, kv_indptr, kv_indices, last_page_len, batch, sm_scale, out)
PyObject* prefill8(PyObject* const* a) {
  const at::Tensor &q0 = tensor(a[0]), &cache = tensor(a[1]), &scales = tensor(a[2]), &qo = tensor(a[3]),
                   &indptr = tensor(a[4]), &indices = tensor(a[5]), &last = tensor(a[6]);
  auto out = maybe(a[9]);
  if (!is_i32_vector(qo)) type_error("paged KV metadata must be contiguous int32");
  const int64_t rows = a[7] == Py_None ? qo.size(0) - 1 : integer(a[7]);
  const int code = check_paged8(q0, cache, scales, indptr, indices, last, rows, out);
  if (qo.size(0) < rows + 1) value_error("paged KV metadata must cover every row");
  const double scale = a[8] == Py_None ? 1.0 / std::sqrt(static_cast<double>(q0.size(2))) : number(a[8]);
  if (!(scale >= 0)) value_error("prefill attention needs sm_scale >= 0");
  Device dev;
  for (int i = 0; i < 7; ++i) dev.add(tensor(a[i]));
  dev.add(out);
  if (!out) out = contiguous_like(q0);
  if (rows == 0 || q0.size(0) == 0) return THPVariable_Wrap(*out);
  at::Tensor q = q0;  // a tensor map needs 16-byte strides, and none of zero (a broadcast query)
  if (reinterpret_cast<uintptr_t>(q.const_data_ptr()) % 16 || q.stride(0) % 8 || q.stride(1) % 8 || q.stride(0) == 0 ||
      q.stride(1) == 0)
    q = q.clone(at::MemoryFormat::Contiguous);
  return result(on_device(dev, [&](int32_t* status, void* stream) {
    return f_prefill8(q.const_data_ptr(), q.stride(0), q.stride(1), cache.const_data_ptr(),
                      scales.const_data_ptr<float>(), static_cast<int>(cache.size(0)), static_cast<int>(cache.size(2)),
                      qo.const_data_ptr<int32_t>(), indptr.const_data_ptr<int32_t>(), table(indices, indptr),
                      last.const_data_ptr<int32_t>(), static_cast<int>(rows), static_cast<int>(q.size(0)),
                      static_cast<int>(q.size(1)), static_cast<int>(cache.size(3)), static_cast<int>(q.size(2)),
                      static_cast<float>(scale), code, out->data_ptr(), out->stride(0), out->stride(1), status, stream);
  }), *out);
}

// (query, key, value, q_weight, k_weight, position_ids, epsilon, rope_theta, cache, scales, pages, offsets, out)
PyObject* write8(PyObject* const* a) {
  const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]), &pos = tensor(a[5]), &cache = tensor(a[8]),
                   &scales = tensor(a[9]), &pages = tensor(a[10]), &offsets = tensor(a[11]);
  at::Tensor qw = tensor(a[3]), kw = tensor(a[4]);
  auto out = maybe(a[12]);
  if (q.dim() != 3 || k.dim() != 3 || v.dim() != 3) value_error("Qwen3-TTS QKV tensors must have rank three");
  const int64_t tokens = q.size(0), hq = q.size(1), d = q.size(2), hkv = k.size(1);
  if (k.sizes() != v.sizes() || k.size(0) != tokens || k.size(2) != d) value_error("Qwen3-TTS QKV shapes are incompatible");
  if (hq < 1 || hkv < 1) value_error("Qwen3-TTS QKV shapes are incompatible");
  if (q.scalar_type() != at::kBFloat16 || k.scalar_type() != at::kBFloat16 || v.scalar_type() != at::kBFloat16)
    type_error("8-bit paged staging takes bf16 query, key and value");
  const int code = cache_code(cache, scales, hkv, d);
  if (qw.dim() != 1 || qw.size(0) != d || kw.dim() != 1 || kw.size(0) != d)
    value_error("QK norm weights must match the head dimension");
  if (q.stride(2) != 1 || k.stride(2) != 1 || v.stride(2) != 1) value_error("QKV must be contiguous per head");
  if (pos.dim() != 1 || pos.size(0) != tokens || pages.dim() != 1 || pages.size(0) != tokens || offsets.dim() != 1 ||
      offsets.size(0) != tokens)
    value_error("paged QKV metadata must contain one entry per token");
  if (!is_i64_vector(pos, tokens) || !is_i64_vector(pages, tokens) || !is_i64_vector(offsets, tokens))
    type_error("paged QKV metadata must be contiguous int64");
  if (out && (out->sizes() != q.sizes() || out->scalar_type() != at::kBFloat16 || out->stride(2) != 1))
    value_error("the rotated query must be bf16 of the query's shape, contiguous per head");
  const double eps = number(a[6]), theta = number(a[7]);
  // as the float32 that the call takes
  if (!(std::abs(theta) <= FLT_MAX) || !(static_cast<float>(theta) > 0)) value_error("rope_theta must be a positive float32");
  Device dev;
  for (int i : {0, 1, 2, 3, 4, 5, 8, 9, 10, 11}) dev.add(tensor(a[i]));
  dev.add(out);
  if (!out) out = contiguous_like(q);
  if (tokens == 0) return THPVariable_Wrap(*out);
  if (qw.scalar_type() != at::kBFloat16 || !qw.is_contiguous()) qw = qw.to(at::kBFloat16).contiguous();
  if (kw.scalar_type() != at::kBFloat16 || !kw.is_contiguous()) kw = kw.to(at::kBFloat16).contiguous();
  return result(on_device(dev, [&](int32_t* status, void* stream) {
    return f_write8(q.const_data_ptr(), q.stride(0), q.stride(1), k.const_data_ptr(), k.stride(0), k.stride(1),
                    v.const_data_ptr(), v.stride(0), v.stride(1), qw.const_data_ptr(), kw.const_data_ptr(),
                    pos.const_data_ptr<int64_t>(), pages.const_data_ptr<int64_t>(), offsets.const_data_ptr<int64_t>(),
                    out->data_ptr(), out->stride(0), out->stride(1), cache.data_ptr(), scales.data_ptr<float>(),
                    static_cast<int>(cache.size(0)), static_cast<int>(cache.size(2)), static_cast<int>(tokens),
                    static_cast<int>(hq), static_cast<int>(hkv), static_cast<int>(d), static_cast<float>(eps),
                    static_cast<float>(theta), code, status, stream);
  }), *out);
}

// (cache, scales, pages, out)
PyObject* read8(PyObject* const* a) {
  const at::Tensor &cache = tensor(a[0]), &scales = tensor(a[1]), &pages = tensor(a[2]);
  auto out = maybe(a[3]);
  if (cache.dim() != 5) value_error("8-bit paged cache must be [pages, 2, page_size, kv_heads, head_dim]");
  const int code = cache_code(cache, scales, cache.size(3), cache.size(4));
  if (pages.dim() != 1 || pages.scalar_type() != at::kLong || !pages.is_contiguous())
    type_error("page ids must be contiguous int64 [n]");
  const int64_t n = pages.size(0);
  const int64_t shape[5] = {n, 2, cache.size(2), cache.size(3), cache.size(4)};
  if (out && (out->sizes() != at::IntArrayRef(shape, 5) || out->scalar_type() != at::kBFloat16 || !out->is_contiguous()))
    value_error("read_paged_cache8 output must be contiguous bf16 [n, 2, page_size, kv_heads, head_dim]");
  Device dev;
  for (int i = 0; i < 3; ++i) dev.add(tensor(a[i]));
  dev.add(out);
  if (!out) out = at::empty(at::IntArrayRef(shape, 5), cache.options().dtype(at::kBFloat16));
  if (n == 0) return THPVariable_Wrap(*out);
  return result(on_device(dev, [&](int32_t* status, void* stream) {
    return f_read8(cache.const_data_ptr(), scales.const_data_ptr<float>(), static_cast<int>(cache.size(0)),
                   static_cast<int>(cache.size(2)), static_cast<int>(cache.size(3)), static_cast<int>(cache.size(4)),
                   code, pages.const_data_ptr<int64_t>(), static_cast<int>(n), out->data_ptr(), status, stream);
  }), *out);
}

// Row stride of a matrix in elements; a single row's stride says nothing.
int64_t pitch_of(const at::Tensor& t) {
  return t.size(0) > 1 ? t.stride(0) : (t.size(1) + 15) / 16 * 16;
}

// (x, data, data_scale, k, cols, gate_up, bias, xscale, out): data int8 [rows, >= k] as Int8Weight lays it out
PyObject* linear8(PyObject* const* a) {
  const at::Tensor &x = tensor(a[0]), &w = tensor(a[1]), &ws = tensor(a[2]);
  const int64_t k = integer(a[3]), cols = integer(a[4]);
  const bool gate_up = a[5] == Py_True;
  const auto bias = maybe(a[6]), xscale = maybe(a[7]);
  auto out = maybe(a[8]);
  if (x.dim() != 2 || x.size(1) != k || (x.stride(1) != 1 && k > 1))
    value_error("linear_int8 needs x [m, k] matching the weight, with unit stride along k");
  const int64_t m = x.size(0);
  if (bias) {
    if (gate_up) value_error("the silu_mul epilogue takes no bias");
    if (bias->scalar_type() != at::kBFloat16 || bias->dim() != 1 || bias->size(0) != cols || !bias->is_contiguous())
      value_error("linear_int8 bias must be contiguous bf16 [n]");
  }
  if (out && (out->dim() != 2 || out->size(0) != m || out->size(1) != cols || out->scalar_type() != at::kBFloat16 ||
              (out->stride(1) != 1 && cols > 1)))
    value_error("linear_int8 output must be bf16 [m, n] with unit column stride");
  const bool codes = x.scalar_type() == at::kChar;
  if (!codes && x.scalar_type() != at::kBFloat16) type_error("linear_int8 takes bf16 rows, or int8 codes with their xscale");
  if (codes) {
    if (!xscale) type_error("linear_int8 takes bf16 rows, or int8 codes with their xscale");
    if (xscale->scalar_type() != at::kFloat || xscale->dim() != 1 || xscale->size(0) != m || !xscale->is_contiguous())
      value_error("linear_int8 xscale must be contiguous float32 [m]");
    if (pitch_of(x) % 16 || reinterpret_cast<uintptr_t>(x.const_data_ptr()) % 16)
      value_error("linear_int8 codes need 16-byte aligned rows");
  } else if (xscale) {
    value_error("xscale belongs to int8 codes");
  }
  if (m > 0x7fffffff - 127) value_error("linear_int8 takes up to 2^31 - 128 rows");
  Device dev;
  dev.add(x);
  dev.add(w);
  dev.add(ws);
  dev.add(bias);
  dev.add(xscale);
  dev.add(out);
  if (!out) out = at::empty({m, cols}, x.options().dtype(at::kBFloat16));
  if (m == 0) return THPVariable_Wrap(*out);
  const int epilogue = gate_up ? 2 : (bias ? 1 : 0);
  const void* b = bias ? bias->const_data_ptr() : nullptr;
  const int rows = static_cast<int>(w.size(0));
  if (codes)
    return result(on_device(dev, [&](int32_t* status, void* stream) {
      return f_gemm_int8(x.const_data_ptr(), pitch_of(x), xscale->const_data_ptr<float>(), w.const_data_ptr(), pitch_of(w),
                         ws.const_data_ptr<float>(), b, out->data_ptr(), pitch_of(*out), static_cast<int>(m), rows,
                         static_cast<int>(cols), static_cast<int>(k), epilogue, status, stream);
    }), *out);
  const int64_t pitch = (k + 15) / 16 * 16;
  const bool quantises = f_linear_int8_launches(static_cast<int>(m), static_cast<int>(k)) == 2;
  at::Tensor scratch;
  uint8_t* q = nullptr;
  if (quantises) {
    scratch = at::empty({m * (pitch + 4)}, x.options().dtype(at::kByte));
    q = static_cast<uint8_t*>(scratch.data_ptr());
  }
  return result(on_device(dev, [&](int32_t* status, void* stream) {
    if (quantises) ++g_launches;
    return f_linear_int8(x.const_data_ptr(), pitch_of(x), q, pitch, quantises ? reinterpret_cast<float*>(q + m * pitch) : nullptr,
                         w.const_data_ptr(), pitch_of(w), ws.const_data_ptr<float>(), b, out->data_ptr(), pitch_of(*out),
                         static_cast<int>(m), rows, static_cast<int>(cols), static_cast<int>(k), epilogue, status, stream);
  }), *out);
}

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  HANDLE_TH_ERRORS  // torch's own errors, out of memory among them, as torch raises them
  try {
    return F(args);
  } catch (const Fail& f) {
    if (f.type != nullptr) PyErr_SetString(f.type, f.msg);
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// init(addresses of the entry points, in the order below)
PyObject* init(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != kEntryPoints) {
    PyErr_SetString(PyExc_TypeError, "init takes the entry points' addresses");
    return nullptr;
  }
  void* p[kEntryPoints];
  for (int i = 0; i < kEntryPoints; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (p[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null entry point");
      return nullptr;
    }
  }
  f_decode8 = reinterpret_cast<decltype(f_decode8)>(p[0]);
  f_prefill8 = reinterpret_cast<decltype(f_prefill8)>(p[1]);
  f_write8 = reinterpret_cast<decltype(f_write8)>(p[2]);
  f_read8 = reinterpret_cast<decltype(f_read8)>(p[3]);
  f_gemm_int8 = reinterpret_cast<decltype(f_gemm_int8)>(p[4]);
  f_linear_int8 = reinterpret_cast<decltype(f_linear_int8)>(p[5]);
  f_linear_int8_launches = reinterpret_cast<decltype(f_linear_int8_launches)>(p[6]);
  Py_RETURN_NONE;
}

PyObject* set_status(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "set_status takes a device index and an address");
    return nullptr;
  }
  const long i = PyLong_AsLong(args[0]);
  void* p = PyLong_AsVoidPtr(args[1]);
  if (PyErr_Occurred()) return nullptr;
  if (i < 0 || i >= kMaxDevices) {
    PyErr_SetString(PyExc_ValueError, "device index out of range");
    return nullptr;
  }
  g_status[i] = static_cast<int32_t*>(p);
  Py_RETURN_NONE;
}

PyObject* launches(PyObject*, PyObject* const* args, Py_ssize_t n) {
  const long long v = g_launches;
  if (n == 1 && args[0] == Py_True) g_launches = 0;  // read and reset
  return PyLong_FromLongLong(v);
}

#define ENTRY(name, count) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(entry<name, count>)), METH_FASTCALL, nullptr}
#define PLAIN(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(decode8, 11), ENTRY(prefill8, 10), ENTRY(write8, 13),   ENTRY(read8, 4), ENTRY(linear8, 9),
                         PLAIN(init),        PLAIN(set_status),   PLAIN(launches),     {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_nqt_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__nqt_bind() { return PyModule_Create(&module); }
