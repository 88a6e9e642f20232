// spinnv2_b200._lib._torch_ops: torch tensors to the C calls of
// spkv2_transformer.h.
//
// The calls of a decoding step run for 2 to 5 microseconds each; checking and
// unpacking their tensors attribute by attribute in Python takes longer than
// that, so it is done here.  spinnv2_b200/transformer.py has the signatures and
// the documentation; a function here takes all of its arguments by position.
// The library itself does not depend on torch: its entry points are handed over
// once, by bind().
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <optional>
#include <string>

#include "spkv2_transformer.h"

namespace {

// What becomes a Python exception.
struct Bad {
  PyObject *type;
  std::string text;
};

struct Entry {
  int (*rms_norm)(const Spkv2RmsNormI8 *, void *) = nullptr;
  int (*quantize)(const Spkv2QuantizeRowsI8 *, void *) = nullptr;
  int (*dequantize)(const Spkv2DequantizeRowsI8 *, void *) = nullptr;
  int (*linear)(const Spkv2LinearI8 *, void *) = nullptr;
  int (*cross)(const Spkv2CrossAttention *, void *) = nullptr;
  const char *(*text)(int) = nullptr;
  PyObject *error = nullptr;  // spinnv2_b200.runtime.Spkv2Error
} entry;

std::string shape_text(at::IntArrayRef s) {
  std::string t = "(";
  for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
  return t + ")";
}

const at::Tensor &tensor(PyObject *o, const char *name) {
  if (!THPVariable_Check(o))
    throw Bad{PyExc_TypeError, std::string(name) + ": expected a torch tensor, got " + Py_TYPE(o)->tp_name};
  return THPVariable_Unpack(o);
}

// The first tensor of a call: it says on which device the call runs.
const at::Tensor &cuda_tensor(PyObject *o, const char *name) {
  const at::Tensor &t = tensor(o, name);
  if (!t.is_cuda()) throw Bad{PyExc_ValueError, std::string(name) + ": expected a CUDA tensor, got one on " + t.device().str()};
  return t;
}

int dtype_code(const at::Tensor &t, const char *name) {
  switch (t.scalar_type()) {
    case at::kFloat: return SPKV2_DTYPE_FP32;
    case at::kHalf: return SPKV2_DTYPE_FP16;
    case at::kBFloat16: return SPKV2_CUDA_DTYPE_BF16;
    default: throw Bad{PyExc_TypeError, std::string(name) + ": expected float32, float16 or bfloat16, got " + toString(t.scalar_type())};
  }
}

const at::Tensor &typed(PyObject *o, const char *name, at::ScalarType type, c10::Device device) {
  const at::Tensor &t = tensor(o, name);
  if (t.scalar_type() != type)
    throw Bad{PyExc_TypeError, std::string(name) + ": expected " + toString(type) + ", got " + toString(t.scalar_type())};
  if (t.device() != device)
    throw Bad{PyExc_ValueError, std::string(name) + ": expected a tensor on " + device.str() + ", got one on " + t.device().str()};
  return t;
}

const at::Tensor &shaped(PyObject *o, const char *name, at::IntArrayRef shape, at::ScalarType type, c10::Device device) {
  const at::Tensor &t = typed(o, name, type, device);
  if (t.sizes() != shape)
    throw Bad{PyExc_ValueError, std::string(name) + ": expected shape " + shape_text(shape) + ", got " + shape_text(t.sizes())};
  return t;
}

const at::Tensor &vector(PyObject *o, const char *name, int64_t size, at::ScalarType type, c10::Device device) {
  const at::Tensor &t = typed(o, name, type, device);
  if (t.numel() != size || !t.is_contiguous())
    throw Bad{PyExc_ValueError, std::string(name) + ": expected " + std::to_string(size) + " contiguous values, got " + shape_text(t.sizes())};
  return t;
}

// [..., width] as a list of rows.
struct Rows {
  int64_t rows = 1, width = 0, stride = 0;
};
Rows rows_of(const at::Tensor &t, const char *name) {
  const auto size = t.sizes(), stride = t.strides();
  const int64_t dims = t.dim();
  if (dims < 1) throw Bad{PyExc_ValueError, std::string(name) + ": expected [..., width], got a scalar"};
  Rows r;
  r.width = size[dims - 1];
  if (t.numel() == 0) {  // no row is read or written, so its place does not matter
    for (int64_t i = 0; i < dims - 1; ++i) r.rows *= size[i];
    r.stride = r.width;
    return r;
  }
  for (int64_t i = dims - 2; i >= 0; --i) {
    if (size[i] == 1) continue;
    if (r.rows == 1)
      r.stride = stride[i];
    else if (stride[i] != r.stride * r.rows)
      throw Bad{PyExc_ValueError, std::string(name) + ": leading dimensions are not evenly strided; call contiguous()"};
    r.rows *= size[i];
  }
  if (r.width > 1 && stride[dims - 1] != 1) throw Bad{PyExc_ValueError, std::string(name) + ": the last dimension must be contiguous"};
  if (r.rows <= 1) r.stride = r.width;
  return r;
}

// The stream of a call: None is torch's current one, else an int or an object
// with `cuda_stream`.
struct Stream {
  cudaStream_t raw = nullptr;
  bool given = false;
};
Stream stream_of(PyObject *o, c10::DeviceIndex index) {
  if (o == Py_None) return {c10::cuda::getCurrentCUDAStream(index).stream(), false};
  PyObject *value = PyLong_Check(o) ? Py_NewRef(o) : PyObject_GetAttrString(o, "cuda_stream");
  if (!value) throw Bad{nullptr, ""};  // the exception is set
  void *p = PyLong_AsVoidPtr(value);
  Py_DECREF(value);
  if (PyErr_Occurred()) throw Bad{nullptr, ""};
  return {static_cast<cudaStream_t>(p), true};
}

// A new tensor, in the memory pool of the stream that writes it.
at::Tensor make(at::IntArrayRef shape, at::ScalarType type, c10::Device device, const Stream &s) {
  const auto options = at::TensorOptions().dtype(type).device(device);
  if (!s.given) return at::empty(shape, options);
  c10::cuda::CUDAStreamGuard guard(c10::cuda::getStreamFromExternal(s.raw, device.index()));
  return at::empty(shape, options);
}

// New codes, whose rows start on 16-byte boundaries.
at::Tensor make_codes(at::IntArrayRef shape, c10::Device device, const Stream &s) {
  c10::SmallVector<int64_t, 6> padded(shape.begin(), shape.end());
  padded.back() = (padded.back() + 15) / 16 * 16;
  return make(padded, at::kChar, device, s).narrow(-1, 0, shape.back());
}

template <class Args>
void call(const char *name, int (*fn)(const Args *, void *), const Args &args, const Stream &s, c10::DeviceIndex index) {
  if (!fn) throw Bad{PyExc_RuntimeError, "the runtime library is not bound"};
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != index) guard.set_index(index);
  const int code = fn(&args, s.raw);
  if (code == 0) return;
  PyObject *e = PyObject_CallFunction(entry.error, "sis", name, code, entry.text(code));
  if (e) {
    PyErr_SetObject(entry.error, e);
    Py_DECREF(e);
  }
  throw Bad{nullptr, ""};
}

PyObject *given(PyObject *o) { return Py_NewRef(o); }
PyObject *wrapped(const at::Tensor &t) { return THPVariable_Wrap(t); }

template <class F>
PyObject *guarded(Py_ssize_t n, Py_ssize_t want, F &&body) {
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
    return nullptr;
  }
  try {
    return body();
  } catch (const Bad &b) {
    if (b.type) PyErr_SetString(b.type, b.text.c_str());
  } catch (const c10::Error &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// x, weight, residual, eps, out, scale_out, sum_out, stream
PyObject *rms_norm_i8(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject * {
    const at::Tensor &x = cuda_tensor(a[0], "x");
    const c10::Device device = x.device();
    const at::ScalarType type = x.scalar_type();
    Spkv2RmsNormI8 p = {};
    p.dtype = dtype_code(x, "x");
    const Rows rx = rows_of(x, "x");
    p.x = x.data_ptr(), p.rows = rx.rows, p.width = rx.width, p.x_stride = rx.stride;
    p.weight = vector(a[1], "weight", rx.width, type, device).data_ptr();
    p.eps = float(PyFloat_AsDouble(a[3]));
    if (PyErr_Occurred()) throw Bad{nullptr, ""};
    const Stream s = stream_of(a[7], device.index());
    std::optional<at::Tensor> codes, scale, sum;
    if (a[2] != Py_None) {
      const at::Tensor &r = shaped(a[2], "residual", x.sizes(), type, device);
      p.residual = r.data_ptr(), p.residual_stride = rows_of(r, "residual").stride;
      if (a[6] == Py_None) sum = make(x.sizes(), type, device, s);
    }
    if (a[6] != Py_None || sum) {
      const at::Tensor &t = sum ? *sum : shaped(a[6], "sum_out", x.sizes(), type, device);
      p.sum = t.data_ptr(), p.sum_stride = rows_of(t, "sum_out").stride;
    }
    if (a[4] == Py_None) codes = make_codes(x.sizes(), device, s);
    const at::Tensor &q = codes ? *codes : shaped(a[4], "out", x.sizes(), at::kChar, device);
    p.codes = q.data_ptr<int8_t>(), p.codes_stride = rows_of(q, "out").stride;
    if (a[5] == Py_None) scale = make(x.sizes().slice(0, x.dim() - 1), at::kFloat, device, s);
    p.scale = (scale ? *scale : vector(a[5], "scale_out", rx.rows, at::kFloat, device)).data_ptr<float>();
    call("rms_norm_i8", entry.rms_norm, p, s, device.index());
    return Py_BuildValue("NNN", codes ? wrapped(*codes) : given(a[4]), scale ? wrapped(*scale) : given(a[5]),
                         sum ? wrapped(*sum) : given(a[6] != Py_None ? a[6] : a[0]));
  });
}

// x, out, scale_out, stream
PyObject *quantize_rows_i8(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject * {
    const at::Tensor &x = cuda_tensor(a[0], "x");
    const c10::Device device = x.device();
    Spkv2QuantizeRowsI8 p = {};
    p.dtype = dtype_code(x, "x");
    const Rows rx = rows_of(x, "x");
    p.x = x.data_ptr(), p.rows = rx.rows, p.width = rx.width, p.x_stride = rx.stride;
    const Stream s = stream_of(a[3], device.index());
    std::optional<at::Tensor> codes, scale;
    if (a[1] == Py_None) codes = make_codes(x.sizes(), device, s);
    const at::Tensor &q = codes ? *codes : shaped(a[1], "out", x.sizes(), at::kChar, device);
    p.codes = q.data_ptr<int8_t>(), p.codes_stride = rows_of(q, "out").stride;
    if (a[2] == Py_None) scale = make(x.sizes().slice(0, x.dim() - 1), at::kFloat, device, s);
    p.scale = (scale ? *scale : vector(a[2], "scale_out", rx.rows, at::kFloat, device)).data_ptr<float>();
    call("quantize_rows_i8", entry.quantize, p, s, device.index());
    return Py_BuildValue("NN", codes ? wrapped(*codes) : given(a[1]), scale ? wrapped(*scale) : given(a[2]));
  });
}

at::ScalarType out_type(PyObject *dtype) {
  if (!THPDtype_Check(dtype)) throw Bad{PyExc_TypeError, "dtype: expected a torch dtype"};
  return reinterpret_cast<THPDtype *>(dtype)->scalar_type;
}

// codes, scale, dtype, out, stream
PyObject *dequantize_rows_i8(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject * {
    const at::Tensor &q = cuda_tensor(a[0], "codes");
    const c10::Device device = q.device();
    typed(a[0], "codes", at::kChar, device);
    Spkv2DequantizeRowsI8 p = {};
    const Rows rq = rows_of(q, "codes");
    p.codes = q.data_ptr<int8_t>(), p.rows = rq.rows, p.width = rq.width, p.codes_stride = rq.stride;
    p.scale = vector(a[1], "scale", rq.rows, at::kFloat, device).data_ptr<float>();
    const Stream s = stream_of(a[4], device.index());
    std::optional<at::Tensor> made;
    if (a[3] == Py_None) made = make(q.sizes(), out_type(a[2]), device, s);
    const at::Tensor &y = made ? *made : shaped(a[3], "out", q.sizes(), tensor(a[3], "out").scalar_type(), device);
    p.y = y.data_ptr(), p.y_stride = rows_of(y, "out").stride, p.dtype = dtype_code(y, "out");
    call("dequantize_rows_i8", entry.dequantize, p, s, device.index());
    return made ? wrapped(*made) : given(a[3]);
  });
}

// codes, scale, weight, weight_scale, bias, activation code, dtype, out, stream
PyObject *linear_i8(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject * {
    const at::Tensor &q = cuda_tensor(a[0], "codes");
    const c10::Device device = q.device();
    typed(a[0], "codes", at::kChar, device);
    Spkv2LinearI8 p = {};
    const Rows rq = rows_of(q, "codes");
    p.a = q.data_ptr<int8_t>(), p.m = rq.rows, p.k = rq.width, p.a_stride = rq.stride;
    const at::Tensor &w = typed(a[2], "weight", at::kChar, device);
    if (w.dim() != 2 || w.size(1) != rq.width)
      throw Bad{PyExc_ValueError, "weight: expected [n, " + std::to_string(rq.width) + "], got " + shape_text(w.sizes())};
    p.w = w.data_ptr<int8_t>(), p.n = w.size(0), p.w_stride = rows_of(w, "weight").stride;
    p.a_scale = vector(a[1], "scale", p.m, at::kFloat, device).data_ptr<float>();
    p.w_scale = vector(a[3], "weight_scale", p.n, at::kFloat, device).data_ptr<float>();
    if (a[4] != Py_None) p.bias = vector(a[4], "bias", p.n, at::kFloat, device).data_ptr<float>();
    p.activation = int32_t(PyLong_AsLong(a[5]));
    if (PyErr_Occurred()) throw Bad{nullptr, ""};
    const Stream s = stream_of(a[8], device.index());
    c10::SmallVector<int64_t, 6> shape(q.sizes().begin(), q.sizes().end());
    shape.back() = p.n;
    std::optional<at::Tensor> made;
    if (a[7] == Py_None) made = make(shape, out_type(a[6]), device, s);
    const at::Tensor &y = made ? *made : shaped(a[7], "out", shape, tensor(a[7], "out").scalar_type(), device);
    p.y = y.data_ptr(), p.y_stride = rows_of(y, "out").stride, p.dtype = dtype_code(y, "out");
    call("linear_i8", entry.linear, p, s, device.index());
    return made ? wrapped(*made) : given(a[7]);
  });
}

void head_strides(const at::Tensor &t, const char *name, int64_t (&st)[3]) {
  if (t.size(3) > 1 && t.stride(3) != 1) throw Bad{PyExc_ValueError, std::string(name) + ": the last dimension must be contiguous"};
  for (int i = 0; i < 3; ++i) st[i] = t.stride(i);
}

// q, k, v, lengths, key_mask, scale, out, stream
PyObject *cross_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject * {
    const at::Tensor &q = cuda_tensor(a[0], "q");
    const c10::Device device = q.device();
    const at::ScalarType type = q.scalar_type();
    Spkv2CrossAttention p = {};
    p.dtype = dtype_code(q, "q");
    if (q.dim() != 4) throw Bad{PyExc_ValueError, "q: expected [batch, queries, heads, width], got " + shape_text(q.sizes())};
    const at::Tensor &k = typed(a[1], "k", type, device);
    if (k.dim() != 4) throw Bad{PyExc_ValueError, "k: expected [batch, keys, kv_heads, width], got " + shape_text(k.sizes())};
    const int64_t heads = q.size(2), kv_heads = k.size(2);
    if (heads < 1 || kv_heads < 1 || heads % kv_heads != 0)
      throw Bad{PyExc_ValueError, "heads: " + std::to_string(heads) + " query heads are not a multiple of " + std::to_string(kv_heads) + " key heads"};
    p.batch = q.size(0), p.queries = q.size(1), p.keys = k.size(1);
    if (heads > INT32_MAX || q.size(3) > INT32_MAX) throw Bad{PyExc_ValueError, "q: too many heads or too wide"};
    p.heads = int32_t(heads), p.kv_heads = int32_t(kv_heads), p.width = int32_t(q.size(3));
    const int64_t shape[4] = {p.batch, p.keys, kv_heads, q.size(3)};
    if (k.sizes() != at::IntArrayRef(shape, 4))
      throw Bad{PyExc_ValueError, "k: expected shape " + shape_text(at::IntArrayRef(shape, 4)) + ", got " + shape_text(k.sizes())};
    const at::Tensor &v = shaped(a[2], "v", at::IntArrayRef(shape, 4), type, device);
    p.q = q.data_ptr(), p.k = k.data_ptr(), p.v = v.data_ptr();
    head_strides(q, "q", p.q_stride);
    head_strides(k, "k", p.k_stride);
    head_strides(v, "v", p.v_stride);
    if (a[3] != Py_None) p.lengths = vector(a[3], "lengths", p.batch, at::kInt, device).data_ptr<int32_t>();
    if (a[4] != Py_None) {
      const at::Tensor &m = typed(a[4], "key_mask", tensor(a[4], "key_mask").scalar_type() == at::kByte ? at::kByte : at::kBool, device);
      if (m.dim() != 2 || m.size(0) != p.batch || m.size(1) != p.keys)
        throw Bad{PyExc_ValueError, "key_mask: expected [batch, keys], got " + shape_text(m.sizes())};
      if (p.keys > 1 && m.stride(1) != 1) throw Bad{PyExc_ValueError, "key_mask: the last dimension must be contiguous"};
      p.key_mask = static_cast<const uint8_t *>(m.data_ptr()), p.mask_stride = m.stride(0);
    }
    p.scale = a[5] == Py_None ? float(1.0 / std::sqrt(double(std::max<int64_t>(q.size(3), 1)))) : float(PyFloat_AsDouble(a[5]));
    if (PyErr_Occurred()) throw Bad{nullptr, ""};
    const Stream s = stream_of(a[7], device.index());
    std::optional<at::Tensor> made;
    if (a[6] == Py_None) made = make(q.sizes(), type, device, s);
    const at::Tensor &o = made ? *made : shaped(a[6], "out", q.sizes(), type, device);
    for (int i = 0; i < 4; ++i)
      if (o.stride(i) == 0 && o.size(i) > 1) throw Bad{PyExc_ValueError, "out: its elements must not overlap"};
    p.out = o.data_ptr();
    head_strides(o, "out", p.out_stride);
    call("cross_attention", entry.cross, p, s, device.index());
    return made ? wrapped(*made) : given(a[6]);
  });
}

// addresses of the five calls and of the status text, and the exception class
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject * {
    void *p[6];
    for (int i = 0; i < 6; ++i) {
      p[i] = PyLong_AsVoidPtr(a[i]);
      if (PyErr_Occurred()) throw Bad{nullptr, ""};
    }
    entry.rms_norm = reinterpret_cast<decltype(entry.rms_norm)>(p[0]);
    entry.quantize = reinterpret_cast<decltype(entry.quantize)>(p[1]);
    entry.dequantize = reinterpret_cast<decltype(entry.dequantize)>(p[2]);
    entry.linear = reinterpret_cast<decltype(entry.linear)>(p[3]);
    entry.cross = reinterpret_cast<decltype(entry.cross)>(p[4]);
    entry.text = reinterpret_cast<decltype(entry.text)>(p[5]);
    Py_XDECREF(entry.error);
    entry.error = Py_NewRef(a[6]);
    Py_RETURN_NONE;
  });
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(rms_norm_i8),     METHOD(quantize_rows_i8), METHOD(dequantize_rows_i8), METHOD(linear_i8),
                         METHOD(cross_attention), METHOD(bind),             {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() { return PyModule_Create(&module); }
