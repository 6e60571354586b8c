// CPython module behind tracea_b200.ops: turns torch tensors into the C ABI's tensor views and calls the library, without
// building a ctypes object per view.
//
// Why it exists: a small convolution is 5-10 us of GPU time, and through ctypes the calling thread spent 21-32 us per call
// on the GPU machines measured, most of it on the shape / stride arrays of five views.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include "../../include/tracea_b200.h"

namespace {

struct PyError {};   // a Python exception has been set

constexpr int kMaxRank = 8;
struct View {
  uint64_t shape[kMaxRank];
  int64_t stride[kMaxRank];
  TraceaTensorView v;
};

// `order`: dimension d of the view is dimension order[d] of the tensor (nullptr: the same).
void fill(View& o, const at::Tensor& t, const int* order = nullptr) {
  TraceaDType dt;
  switch (t.scalar_type()) {
    case at::kFloat: dt = TRACEA_DTYPE_FLOAT32; break;
    case at::kHalf: dt = TRACEA_DTYPE_FLOAT16; break;
    case at::kBFloat16: dt = TRACEA_DTYPE_BFLOAT16; break;
    case at::kInt: dt = TRACEA_DTYPE_INT32; break;
    case at::kChar: dt = TRACEA_DTYPE_INT8; break;
    default:
      PyErr_Format(PyExc_TypeError, "unsupported dtype %s", c10::toString(t.scalar_type()));
      throw PyError{};
  }
  const int64_t rank = t.dim();
  if (rank > kMaxRank) {
    PyErr_Format(PyExc_ValueError, "tensors of more than %d dimensions are not supported", kMaxRank);
    throw PyError{};
  }
  for (int64_t d = 0; d < rank; ++d) {
    const int64_t s = order != nullptr ? order[d] : d;
    o.shape[d] = static_cast<uint64_t>(t.size(s));
    o.stride[d] = t.stride(s);
  }
  o.v.ptr = t.data_ptr();
  o.v.rank = static_cast<uint32_t>(rank);
  o.v.shape = o.shape;
  o.v.stride = o.stride;
  o.v.dtype = dt;
  o.v.device_id = t.is_cuda() ? static_cast<int32_t>(t.get_device()) : -1;
}

const at::Tensor& tensor_arg(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a torch.Tensor, not %s", name, Py_TYPE(o)->tp_name);
    throw PyError{};
  }
  return THPVariable_Unpack(o);
}
const at::Tensor* optional_tensor(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor_arg(o, name); }

long int_arg(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred() != nullptr) throw PyError{};
  return v;
}

bool bool_arg(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PyError{};
  return v != 0;
}

// Raises tracea_b200.ffi.TraceaError(status, last error text, entry).
[[noreturn]] void raise_status(TraceaStatus st, const char* entry) {
  char text[1024];
  const int32_t n = tracea_get_last_error(reinterpret_cast<uint8_t*>(text), sizeof(text));
  PyObject* mod = PyImport_ImportModule("tracea_b200.ffi");
  PyObject* cls = mod != nullptr ? PyObject_GetAttrString(mod, "TraceaError") : nullptr;
  PyObject* msg = cls != nullptr ? PyUnicode_DecodeUTF8(text, n > 0 ? n : 0, "replace") : nullptr;
  PyObject* exc = msg != nullptr ? PyObject_CallFunction(cls, "iOs", static_cast<int>(st), msg, entry) : nullptr;
  if (exc != nullptr) PyErr_SetObject(cls, exc);
  Py_XDECREF(exc);
  Py_XDECREF(msg);
  Py_XDECREF(cls);
  Py_XDECREF(mod);
  throw PyError{};
}

void* stream_of(const at::Tensor& t) {
  return t.is_cuda() ? static_cast<void*>(c10::cuda::getCurrentCUDAStream(t.get_device()).stream()) : nullptr;
}

// The library call itself, without the GIL: it may allocate, and on host tensors it copies and waits.
template <typename F>
TraceaStatus without_gil(F&& f) {
  PyThreadState* save = PyEval_SaveThread();
  const TraceaStatus st = f();
  PyEval_RestoreThread(save);
  return st;
}

const TraceaTensorView* opt(const at::Tensor* t, View& v, const int* order = nullptr) {
  if (t == nullptr) return nullptr;
  fill(v, *t, order);
  return &v.v;
}

constexpr int kChannelsLast[4] = {0, 3, 1, 2};   // logical NCHW of dimensions (N, H, W, C); KCRS of (K, R, S, C)

template <typename Body>
PyObject* guarded(Body&& body) {
  HANDLE_TH_ERRORS
  try {
    return body();
  } catch (const PyError&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

bool arg_count(Py_ssize_t got, Py_ssize_t want, const char* name) {
  if (got == want) return true;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments (%zd given)", name, want, got);
  return false;
}

// conv2d(x, w, bias, residual, out, channels-last dimensions, epilogue kind, stride_h, stride_w, pad_h, pad_w, dil_h, dil_w,
// groups) -> out
PyObject* py_conv2d(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arg_count(n, 14, "conv2d")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor &x = tensor_arg(a[0], "x"), &w = tensor_arg(a[1], "w"), &out = tensor_arg(a[4], "out");
    const at::Tensor *bias = optional_tensor(a[2], "bias"), *res = optional_tensor(a[3], "residual");
    const int* order = bool_arg(a[5]) ? kChannelsLast : nullptr;
    if (order != nullptr && (x.dim() != 4 || w.dim() != 4 || out.dim() != 4 || (res != nullptr && res->dim() != 4))) {
      PyErr_SetString(PyExc_ValueError, "x, w, residual and out must have four dimensions");
      throw PyError{};
    }
    TraceaConv2dParams p;
    p.epilogue = static_cast<TraceaEpilogueKind>(int_arg(a[6]));
    p.stride_h = static_cast<uint32_t>(int_arg(a[7]));
    p.stride_w = static_cast<uint32_t>(int_arg(a[8]));
    p.padding_h = static_cast<uint32_t>(int_arg(a[9]));
    p.padding_w = static_cast<uint32_t>(int_arg(a[10]));
    p.dilation_h = static_cast<uint32_t>(int_arg(a[11]));
    p.dilation_w = static_cast<uint32_t>(int_arg(a[12]));
    p.groups = static_cast<uint32_t>(int_arg(a[13]));
    p.stream = stream_of(x);
    View vx, vw, vb, vr, vo;
    fill(vx, x, order);
    fill(vw, w, order);
    const TraceaTensorView* pb = opt(bias, vb);
    const TraceaTensorView* pr = opt(res, vr, order);
    fill(vo, out, order);
    const TraceaStatus st = without_gil([&] { return tracea_conv2d(vx.v, vw.v, pb, pr, &vo.v, p); });
    if (st != TRACEA_SUCCESS) raise_status(st, "tracea_conv2d");
    Py_INCREF(a[4]);
    return a[4];
  });
}

// gemm(x, w, bias, residual, out, epilogue kind) -> out
PyObject* py_gemm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arg_count(n, 6, "gemm")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor &x = tensor_arg(a[0], "x"), &w = tensor_arg(a[1], "w"), &out = tensor_arg(a[4], "out");
    const at::Tensor *bias = optional_tensor(a[2], "bias"), *res = optional_tensor(a[3], "residual");
    TraceaGemmParams p;
    p.epilogue = static_cast<TraceaEpilogueKind>(int_arg(a[5]));
    p.stream = stream_of(x);
    View vx, vw, vb, vr, vo;
    fill(vx, x);
    fill(vw, w);
    const TraceaTensorView* pb = opt(bias, vb);
    const TraceaTensorView* pr = opt(res, vr);
    fill(vo, out);
    const TraceaStatus st = without_gil([&] { return tracea_gemm(vx.v, vw.v, pb, pr, &vo.v, p); });
    if (st != TRACEA_SUCCESS) raise_status(st, "tracea_gemm");
    Py_INCREF(a[4]);
    return a[4];
  });
}

// conv_transpose2d(x, w, bias, residual, out, epilogue kind, stride_h, stride_w, pad_h, pad_w, opad_h, opad_w, dil_h, dil_w)
// -> out
PyObject* py_conv_transpose2d(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arg_count(n, 14, "conv_transpose2d")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor &x = tensor_arg(a[0], "x"), &w = tensor_arg(a[1], "w"), &out = tensor_arg(a[4], "out");
    const at::Tensor *bias = optional_tensor(a[2], "bias"), *res = optional_tensor(a[3], "residual");
    TraceaConvTranspose2dParams p;
    p.epilogue = static_cast<TraceaEpilogueKind>(int_arg(a[5]));
    p.stride_h = static_cast<uint32_t>(int_arg(a[6]));
    p.stride_w = static_cast<uint32_t>(int_arg(a[7]));
    p.padding_h = static_cast<uint32_t>(int_arg(a[8]));
    p.padding_w = static_cast<uint32_t>(int_arg(a[9]));
    p.output_padding_h = static_cast<uint32_t>(int_arg(a[10]));
    p.output_padding_w = static_cast<uint32_t>(int_arg(a[11]));
    p.dilation_h = static_cast<uint32_t>(int_arg(a[12]));
    p.dilation_w = static_cast<uint32_t>(int_arg(a[13]));
    p.groups = 1;
    p.stream = stream_of(x);
    View vx, vw, vb, vr, vo;
    fill(vx, x);
    fill(vw, w);
    const TraceaTensorView* pb = opt(bias, vb);
    const TraceaTensorView* pr = opt(res, vr);
    fill(vo, out);
    const TraceaStatus st = without_gil([&] { return tracea_conv_transpose2d(vx.v, vw.v, pb, pr, &vo.v, p); });
    if (st != TRACEA_SUCCESS) raise_status(st, "tracea_conv_transpose2d");
    Py_INCREF(a[4]);
    return a[4];
  });
}

// ------------------------------------------------------------------ 4-bit microscaled matrices and norms
at::ScalarType scalar_type(long code) {
  switch (code) {
    case TRACEA_DTYPE_FLOAT32: return at::kFloat;
    case TRACEA_DTYPE_FLOAT16: return at::kHalf;
    case TRACEA_DTYPE_BFLOAT16: return at::kBFloat16;
    default:
      PyErr_SetString(PyExc_TypeError, "the output type must be float32, float16 or bfloat16");
      throw PyError{};
  }
}

int32_t cuda_index(const at::Tensor& t) { return t.is_cuda() ? static_cast<int32_t>(t.get_device()) : -1; }

// The matrix of two uint8 tensors, whose sizes have to fit it.
TraceaMxMatrix mx_matrix(const at::Tensor& data, const at::Tensor& scales, int64_t rows, int64_t cols, const char* name) {
  if (rows < 0 || cols < 1 || data.scalar_type() != at::kByte || scales.scalar_type() != at::kByte || !data.is_contiguous() ||
      !scales.is_contiguous() || static_cast<uint64_t>(data.numel()) != tracea_mx_data_bytes(rows, cols) ||
      static_cast<uint64_t>(scales.numel()) != tracea_mx_scale_bytes(rows, cols)) {
    PyErr_Format(PyExc_ValueError, "%s: a %lld x %lld matrix takes contiguous uint8 tensors of %llu bytes of data and %llu of scales",
                 name, (long long)rows, (long long)cols, (unsigned long long)tracea_mx_data_bytes(rows, cols),
                 (unsigned long long)tracea_mx_scale_bytes(rows, cols));
    throw PyError{};
  }
  if (data.device() != scales.device()) {
    PyErr_Format(PyExc_ValueError, "%s: data and scales are on different devices", name);
    throw PyError{};
  }
  TraceaMxMatrix m;
  m.data = data.data_ptr();
  m.scales = scales.data_ptr();
  m.rows = static_cast<uint64_t>(rows);
  m.cols = static_cast<uint64_t>(cols);
  m.device_id = cuda_index(data);
  return m;
}

struct NewMx {
  at::Tensor data, scales;
  TraceaMxMatrix m;
  NewMx(int64_t rows, int64_t cols, const at::Tensor& like) {
    if (rows > 0x7fffffffLL || cols < 1 || cols > 0x7fffff00LL) {
      PyErr_Format(PyExc_ValueError, "a %lld x %lld matrix is out of range", (long long)rows, (long long)cols);
      throw PyError{};
    }
    const auto opt = like.options().dtype(at::kByte);
    // one allocation for both: a second one costs a call ~0.7 us of its 5
    const int64_t row = (cols + 31) / 32 * 16, first = (rows * row + 255) / 256 * 256, tiles = (rows + 127) / 128 * ((cols + 127) / 128);
    const at::Tensor whole = at::empty({first + tiles * 512}, opt);
    auto part = [&](int64_t offset, at::IntArrayRef sizes) {
      at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
      t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
      t.unsafeGetTensorImpl()->set_storage_offset(offset);
      return t;
    };
    data = part(0, {rows, row});
    scales = part(first, {(rows + 127) / 128, (cols + 127) / 128, 512});
    m = mx_matrix(data, scales, rows, cols, "output");
  }
  PyObject* release() {
    PyObject* d = THPVariable_Wrap(data);
    PyObject* s = d != nullptr ? THPVariable_Wrap(scales) : nullptr;
    PyObject* pair = s != nullptr ? PyTuple_Pack(2, d, s) : nullptr;
    Py_XDECREF(d);
    Py_XDECREF(s);
    return pair;
  }
};

void rank2(const at::Tensor& t, const char* name) {
  if (t.dim() != 2) {
    PyErr_Format(PyExc_ValueError, "%s must have two dimensions", name);
    throw PyError{};
  }
}

// mx_quantize(x) -> (data, scales)
PyObject* py_mx_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arg_count(n, 1, "mx_quantize")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor& x = tensor_arg(a[0], "x");
    rank2(x, "x");
    NewMx q(x.size(0), x.size(1), x);
    View vx;
    fill(vx, x);
    void* stream = stream_of(x);
    const TraceaStatus st = without_gil([&] { return tracea_mx_quantize(vx.v, &q.m, stream); });
    if (st != TRACEA_SUCCESS) raise_status(st, "tracea_mx_quantize");
    return q.release();
  });
}

// mx_dequantize(data, scales, rows, cols, dtype) -> tensor
PyObject* py_mx_dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arg_count(n, 5, "mx_dequantize")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor &data = tensor_arg(a[0], "data"), &scales = tensor_arg(a[1], "scales");
    const long rows = int_arg(a[2]), cols = int_arg(a[3]);
    const TraceaMxMatrix q = mx_matrix(data, scales, rows, cols, "q");
    at::Tensor out = at::empty({rows, cols}, data.options().dtype(scalar_type(int_arg(a[4]))));
    View vo;
    fill(vo, out);
    void* stream = stream_of(data);
    const TraceaStatus st = without_gil([&] { return tracea_mx_dequantize(q, &vo.v, stream); });
    if (st != TRACEA_SUCCESS) raise_status(st, "tracea_mx_dequantize");
    return THPVariable_Wrap(out);
  });
}

// mx_gemm(a or a.data, a.scales or None, rows, w.data, w.scales, w rows, cols, bias, residual, epilogue kind, dtype or None)
//   -> tensor, or (data, scales) for None
PyObject* py_mx_gemm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arg_count(n, 11, "mx_gemm")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor& x = tensor_arg(a[0], "a");
    const at::Tensor* x_scales = optional_tensor(a[1], "a.scales");
    const long rows = int_arg(a[2]), w_rows = int_arg(a[5]), cols = int_arg(a[6]);
    const TraceaMxMatrix w = mx_matrix(tensor_arg(a[3], "w.data"), tensor_arg(a[4], "w.scales"), w_rows, cols, "w");
    const at::Tensor *bias = optional_tensor(a[7], "bias"), *res = optional_tensor(a[8], "residual");
    TraceaGemmParams p;
    p.epilogue = static_cast<TraceaEpilogueKind>(int_arg(a[9]));
    p.stream = stream_of(x);
    View vx, vb, vr, vo;
    const TraceaTensorView* pb = opt(bias, vb);
    const TraceaTensorView* pr = opt(res, vr);
    TraceaMxMatrix ax;
    if (x_scales != nullptr) ax = mx_matrix(x, *x_scales, rows, cols, "a");
    else fill(vx, x);
    auto call = [&](TraceaTensorView* c, TraceaMxMatrix* c_mx) {
      const TraceaStatus st = without_gil([&] {
        return x_scales != nullptr ? tracea_mx_gemm(ax, w, pb, pr, c, c_mx, p) : tracea_mx_linear(vx.v, w, pb, pr, c, c_mx, p);
      });
      if (st != TRACEA_SUCCESS) raise_status(st, x_scales != nullptr ? "tracea_mx_gemm" : "tracea_mx_linear");
    };
    if (a[10] == Py_None) {
      NewMx out(rows, w_rows, x);
      call(nullptr, &out.m);
      return out.release();
    }
    at::Tensor out = at::empty({rows, w_rows}, x.options().dtype(scalar_type(int_arg(a[10]))));
    fill(vo, out);
    call(&vo.v, nullptr);
    return THPVariable_Wrap(out);
  });
}

// A norm's arguments from position `i`: weight, bias, scale, shift, kind, eps.
struct NormArgs {
  View w, b, sc, sh;
  TraceaNorm norm;
  NormArgs(PyObject* const* a) {
    norm.weight = opt(optional_tensor(a[0], "weight"), w);
    norm.bias = opt(optional_tensor(a[1], "bias"), b);
    norm.scale = opt(optional_tensor(a[2], "scale"), sc);
    norm.shift = opt(optional_tensor(a[3], "shift"), sh);
    norm.kind = static_cast<TraceaNormKind>(int_arg(a[4]));
    norm.eps = static_cast<float>(PyFloat_AsDouble(a[5]));
    if (PyErr_Occurred() != nullptr) throw PyError{};
  }
};

// block_norm(x, weight, bias, scale, shift, kind, eps, quantize) -> tensor, or (data, scales)
PyObject* py_block_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arg_count(n, 8, "block_norm")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor& x = tensor_arg(a[0], "x");
    rank2(x, "x");
    NormArgs args(a + 1);
    View vx, vy;
    fill(vx, x);
    void* stream = stream_of(x);
    auto call = [&](TraceaTensorView* y, TraceaMxMatrix* y_mx) {
      const TraceaStatus st = without_gil([&] { return tracea_block_norm(vx.v, &args.norm, y, y_mx, stream); });
      if (st != TRACEA_SUCCESS) raise_status(st, "tracea_block_norm");
    };
    if (bool_arg(a[7])) {
      NewMx out(x.size(0), x.size(1), x);
      call(nullptr, &out.m);
      return out.release();
    }
    at::Tensor y = at::empty({x.size(0), x.size(1)}, x.options());
    fill(vy, y);
    call(&vy.v, nullptr);
    return THPVariable_Wrap(y);
  });
}

// block_norm_add(h, x, weight, bias, scale, shift, kind, eps, gate, residual_scale, following: 0 none, 1 rows, 2 quantised[, its
// weight, bias, scale, shift, kind, eps]) -> r, or (r, y), or (r, (data, scales))
PyObject* py_block_norm_add(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arg_count(n, n == 11 ? 11 : 17, "block_norm_add")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor &h = tensor_arg(a[0], "h"), &x = tensor_arg(a[1], "x");
    rank2(x, "x");
    NormArgs args(a + 2);
    View vg, vh, vx, vr, vy;
    const TraceaTensorView* gate = opt(optional_tensor(a[8], "gate"), vg);
    const float residual_scale = static_cast<float>(PyFloat_AsDouble(a[9]));
    if (PyErr_Occurred() != nullptr) throw PyError{};
    const long mode = n == 17 ? int_arg(a[10]) : 0;
    fill(vh, h);
    fill(vx, x);
    at::Tensor r = at::empty({x.size(0), x.size(1)}, x.options());
    fill(vr, r);
    void* stream = stream_of(x);
    auto call = [&](const TraceaNorm* following, TraceaTensorView* y, TraceaMxMatrix* y_mx) {
      const TraceaStatus st = without_gil([&] {
        return tracea_block_norm_add(vh.v, vx.v, &args.norm, gate, residual_scale, &vr.v, following, y, y_mx, stream);
      });
      if (st != TRACEA_SUCCESS) raise_status(st, "tracea_block_norm_add");
    };
    if (mode == 0) {
      call(nullptr, nullptr, nullptr);
      return THPVariable_Wrap(r);
    }
    NormArgs following(a + 11);
    PyObject* second = nullptr;
    if (mode == 2) {
      NewMx out(x.size(0), x.size(1), x);
      call(&following.norm, nullptr, &out.m);
      second = out.release();
    } else {
      at::Tensor y = at::empty({x.size(0), x.size(1)}, x.options());
      fill(vy, y);
      call(&following.norm, &vy.v, nullptr);
      second = THPVariable_Wrap(y);
    }
    PyObject* first = second != nullptr ? THPVariable_Wrap(r) : nullptr;
    PyObject* pair = first != nullptr ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return pair;
  });
}

// ------------------------------------------------------------------ rows of heads and the cache of keys and values
float float_arg(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred() != nullptr) throw PyError{};
  return static_cast<float>(v);
}

void heads_rank(const at::Tensor& t, const char* name) {
  if (t.dim() != 3) {
    PyErr_Format(PyExc_ValueError, "%s must have three dimensions: (tokens, heads, columns)", name);
    throw PyError{};
  }
}

// Rows of heads, their weight and, where asked for, a new tensor for the result.
struct HeadsArg {
  View x, w, y;
  at::Tensor out;
  TraceaHeads h;
  HeadsArg(const at::Tensor& t, PyObject* weight, const char* name, const char* weight_name) {
    heads_rank(t, name);
    out = at::empty({t.size(0), t.size(1), t.size(2)}, t.options());
    fill(x, t);
    fill(y, out);
    h.x = x.v;
    h.y = &y.v;
    h.weight = opt(optional_tensor(weight, weight_name), w);
  }
};

// The rotation of `frequencies` (None: none), which have to lie where `like` does.
struct RotationArg {
  TraceaRotation r;
  bool given;
  RotationArg(PyObject* frequencies, bool interleaved, const at::Tensor& like) : given(frequencies != Py_None) {
    if (!given) return;
    const at::Tensor& f = tensor_arg(frequencies, "frequencies");
    if (f.scalar_type() != at::kDouble || f.dim() != 1 || !f.is_contiguous() || f.device() != like.device() || f.size(0) > 0x7fffffff) {
      PyErr_SetString(PyExc_ValueError, "frequencies must be a contiguous float64 vector on the device of the rows");
      throw PyError{};
    }
    r.frequencies = f.data_ptr<double>();
    r.pairs = static_cast<uint32_t>(f.size(0));
    r.interleaved = interleaved ? 1 : 0;
  }
  const TraceaRotation* get() const { return given ? &r : nullptr; }
};

// head_norm_rotate(q or None, k or None, positions, frequencies, interleaved, q_weight, k_weight, kind, eps) -> (q, k)
PyObject* py_head_norm_rotate(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arg_count(n, 9, "head_norm_rotate")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor *q = optional_tensor(a[0], "q"), *k = optional_tensor(a[1], "k"), *pos = optional_tensor(a[2], "positions");
    if (q == nullptr && k == nullptr) {
      PyErr_SetString(PyExc_ValueError, "neither q nor k is given");
      throw PyError{};
    }
    const at::Tensor& first = q != nullptr ? *q : *k;
    c10::optional<HeadsArg> hq, hk;
    if (q != nullptr) hq.emplace(*q, a[5], "q", "q_weight");
    if (k != nullptr) hk.emplace(*k, a[6], "k", "k_weight");
    const RotationArg rot(a[3], bool_arg(a[4]), first);
    View vp;
    const TraceaTensorView* pp = opt(pos, vp);
    const auto kind = static_cast<TraceaNormKind>(int_arg(a[7]));
    const float eps = float_arg(a[8]);
    void* stream = stream_of(first);
    const TraceaStatus st = without_gil([&] {
      return tracea_head_norm_rotate(hq ? &hq->h : nullptr, hk ? &hk->h : nullptr, kind, eps, rot.get(), pp, stream);
    });
    if (st != TRACEA_SUCCESS) raise_status(st, "tracea_head_norm_rotate");
    PyObject* first_out = q != nullptr ? THPVariable_Wrap(hq->out) : Py_NewRef(Py_None);
    PyObject* second = first_out == nullptr ? nullptr : k != nullptr ? THPVariable_Wrap(hk->out) : Py_NewRef(Py_None);
    PyObject* pair = second != nullptr ? PyTuple_Pack(2, first_out, second) : nullptr;
    Py_XDECREF(first_out);
    Py_XDECREF(second);
    return pair;
  });
}

// The cache of four tensors: k, v (pages, heads, P, D), of one-byte elements, and the scales (pages, heads), uint8.
TraceaKvCache cache_arg(PyObject* const* a) {
  const at::Tensor &k = tensor_arg(a[0], "cache.k"), &v = tensor_arg(a[1], "cache.v"), &ks = tensor_arg(a[2], "cache.k_scales"),
                   &vs = tensor_arg(a[3], "cache.v_scales");
  auto bad = [](const at::Tensor& t) { return t.scalar_type() != at::kFloat8_e4m3fn || !t.is_contiguous(); };
  if (bad(k) || bad(v) || k.dim() != 4 || v.sizes() != k.sizes() || ks.scalar_type() != at::kByte || vs.scalar_type() != at::kByte ||
      !ks.is_contiguous() || !vs.is_contiguous() || ks.dim() != 2 || ks.size(0) != k.size(0) || ks.size(1) != k.size(1) ||
      vs.sizes() != ks.sizes() || v.device() != k.device() || ks.device() != k.device() || vs.device() != k.device()) {
    PyErr_SetString(PyExc_ValueError, "a cache is contiguous tensors on one device: k and v float8_e4m3fn (pages, heads, page size, columns), "
                                      "k_scales and v_scales uint8 (pages, heads)");
    throw PyError{};
  }
  for (int d = 1; d < 4; ++d) {
    if (k.size(d) > 0x7fffffff) {
      PyErr_SetString(PyExc_ValueError, "cache: out of range");
      throw PyError{};
    }
  }
  TraceaKvCache c;
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.k_scales = ks.data_ptr<uint8_t>();
  c.v_scales = vs.data_ptr<uint8_t>();
  c.pages = static_cast<uint64_t>(k.size(0));
  c.heads = static_cast<uint32_t>(k.size(1));
  c.page_size = static_cast<uint32_t>(k.size(2));
  c.head_dim = static_cast<uint32_t>(k.size(3));
  c.device_id = cuda_index(k);
  return c;
}

struct SequencesArg {
  View pages, lengths, starts;
  TraceaSequences s;
  SequencesArg(PyObject* const* a) {
    fill(pages, tensor_arg(a[0], "pages"));
    fill(lengths, tensor_arg(a[1], "lengths"));
    s.pages = pages.v;
    s.lengths = lengths.v;
    s.starts = opt(optional_tensor(a[2], "starts"), starts);
  }
};

// kv_append(k cache, v cache, k scales, v scales, pages, lengths, starts, k, v, k_weight, q or None, q_weight, frequencies, interleaved,
// kind, eps) -> q or None
PyObject* py_kv_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arg_count(n, 16, "kv_append")) return nullptr;
  return guarded([&]() -> PyObject* {
    const TraceaKvCache cache = cache_arg(a);
    const SequencesArg seqs(a + 4);
    const at::Tensor &k = tensor_arg(a[7], "k"), &v = tensor_arg(a[8], "v");
    const at::Tensor* q = optional_tensor(a[10], "q");
    heads_rank(k, "k");
    heads_rank(v, "v");
    View vk, vv, vw;
    fill(vk, k);
    fill(vv, v);
    const TraceaTensorView* pw = opt(optional_tensor(a[9], "k_weight"), vw);
    c10::optional<HeadsArg> hq;
    if (q != nullptr) hq.emplace(*q, a[11], "q", "q_weight");
    const RotationArg rot(a[12], bool_arg(a[13]), k);
    const auto kind = static_cast<TraceaNormKind>(int_arg(a[14]));
    const float eps = float_arg(a[15]);
    void* stream = stream_of(k);
    const TraceaStatus st = without_gil([&] {
      return tracea_kv_append(cache, seqs.s, vk.v, vv.v, pw, hq ? &hq->h : nullptr, kind, eps, rot.get(), stream);
    });
    if (st != TRACEA_SUCCESS) raise_status(st, "tracea_kv_append");
    return q != nullptr ? THPVariable_Wrap(hq->out) : Py_NewRef(Py_None);
  });
}

// kv_attention(q, k cache, v cache, k scales, v scales, pages, lengths, starts, scale, causal, window) -> out
PyObject* py_kv_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arg_count(n, 11, "kv_attention")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor& q = tensor_arg(a[0], "q");
    heads_rank(q, "q");
    const TraceaKvCache cache = cache_arg(a + 1);
    const SequencesArg seqs(a + 5);
    TraceaKvAttentionParams p;
    p.scale = float_arg(a[8]);
    p.causal = bool_arg(a[9]) ? 1 : 0;
    const long window = int_arg(a[10]);
    if (window < 0 || window > 0x7fffffffL) {
      PyErr_SetString(PyExc_ValueError, "window must be 0 (none) or a number of tokens");
      throw PyError{};
    }
    p.window = static_cast<uint32_t>(window);
    p.stream = stream_of(q);
    at::Tensor out = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
    View vq, vo;
    fill(vq, q);
    fill(vo, out);
    const TraceaStatus st = without_gil([&] { return tracea_kv_attention(vq.v, cache, seqs.s, &vo.v, p); });
    if (st != TRACEA_SUCCESS) raise_status(st, "tracea_kv_attention");
    return THPVariable_Wrap(out);
  });
}

PyMethodDef kMethods[] = {
    {"conv2d", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_conv2d)), METH_FASTCALL, nullptr},
    {"gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_gemm)), METH_FASTCALL, nullptr},
    {"conv_transpose2d", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_conv_transpose2d)), METH_FASTCALL, nullptr},
    {"mx_quantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_mx_quantize)), METH_FASTCALL, nullptr},
    {"mx_dequantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_mx_dequantize)), METH_FASTCALL, nullptr},
    {"mx_gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_mx_gemm)), METH_FASTCALL, nullptr},
    {"block_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_block_norm)), METH_FASTCALL, nullptr},
    {"block_norm_add", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_block_norm_add)), METH_FASTCALL, nullptr},
    {"head_norm_rotate", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_head_norm_rotate)), METH_FASTCALL, nullptr},
    {"kv_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_kv_append)), METH_FASTCALL, nullptr},
    {"kv_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_kv_attention)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_ops_native", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops_native() {
  PyObject* m = PyModule_Create(&kModule);
  if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) {   // what it was compiled against
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
