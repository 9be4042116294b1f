// Host side of the microscaled FP4 operators for the calls a program makes a thousand times a second:
// plain CUDA tensors whose sizes and types fit.  It looks at what the checks of microscaling.py look at,
// allocates the outputs and calls the C ABI on the current stream; anything else -- another type, a wrong
// shape, a CPU tensor, a call the library refuses -- returns None, and the Python path checks the
// arguments one by one and raises the error.  (A decode call took 9.3 us of host time through ctypes, twice what its
// kernel runs.)
//
// The only translation unit that sees torch.  It does not link the kernel library: the entry points' addresses are
// handed over once it is loaded.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/lowbitlinear_b200.h"

namespace {

struct EntryPoints {
  decltype(&lbl_fp4_quantize) quantize = nullptr;
  decltype(&lbl_fp4_dequantize) dequantize = nullptr;
  decltype(&lbl_fp4_matmul) matmul = nullptr;
  decltype(&lbl_fp4_linear_workspace_bytes) linear_workspace_bytes = nullptr;
  decltype(&lbl_fp4_linear) linear = nullptr;
} g_lib;

constexpr int64_t kMostColumns = int64_t{1} << 30;

// A plain tensor on a GPU (no subclass, which may have its own ideas, and no view that negates), or null.
const at::Tensor* cuda_tensor(PyObject* object) {
  if (!THPVariable_CheckExact(object)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(object);
  return t.is_cuda() && t.layout() == at::kStrided && !t.is_neg() ? &t : nullptr;
}

int format_code(PyObject* object) {
  if (!PyUnicode_CheckExact(object)) return -1;
  if (PyUnicode_CompareWithASCIIString(object, "mxfp4") == 0) return LBL_FP4_MX;
  if (PyUnicode_CompareWithASCIIString(object, "nvfp4") == 0) return LBL_FP4_NV;
  return -1;
}

int type_code(at::ScalarType type) {
  switch (type) {
    case at::kHalf: return LBL_TYPE_F16;
    case at::kBFloat16: return LBL_TYPE_BF16;
    case at::kFloat: return LBL_TYPE_F32;
    default: return -1;
  }
}

int64_t code_columns(int64_t k) { return (k + 31) / 32 * 16; }
int64_t scale_tiles(int64_t columns, int format) {
  const int64_t blocks = columns * 2 / (format == LBL_FP4_NV ? 16 : 32);
  return (blocks + 3) / 4;
}

// The tensor factor's address; false when the argument is neither None nor one FP32 value on the device.
bool factor_address(PyObject* object, int format, c10::Device device, const float** out) {
  *out = nullptr;
  if (object == Py_None) return true;
  const at::Tensor* t = cuda_tensor(object);
  if (t == nullptr || format != LBL_FP4_NV || t->scalar_type() != at::kFloat || t->numel() != 1 || t->device() != device) {
    return false;
  }
  *out = static_cast<const float*>(t->const_data_ptr());
  return true;
}

// Codes [R, columns] and tiled scales of one operand.
bool operand(PyObject* codes_object, PyObject* scales_object, int format, const at::Tensor** codes, const at::Tensor** scales) {
  const at::Tensor* c = cuda_tensor(codes_object);
  const at::Tensor* s = cuda_tensor(scales_object);
  if (c == nullptr || s == nullptr || c->scalar_type() != at::kByte || s->scalar_type() != at::kByte || c->dim() != 2 ||
      s->dim() != 5 || !c->is_contiguous() || !s->is_contiguous() || c->device() != s->device()) {
    return false;
  }
  const int64_t rows = c->size(0), columns = c->size(1);
  if (rows <= 0 || columns <= 0 || columns % 16 != 0 || columns > kMostColumns) return false;
  const auto size = s->sizes();
  if (size[0] != (rows + 127) / 128 || size[1] != scale_tiles(columns, format) || size[2] != 32 || size[3] != 4 || size[4] != 4) {
    return false;
  }
  *codes = c;
  *scales = s;
  return true;
}

// A matrix whose rows are contiguous; `stride` receives the distance between them.
bool row_matrix(const at::Tensor* t, int64_t* stride) {
  if (t == nullptr || t->dim() != 2 || t->size(0) <= 0 || t->size(1) <= 0 || t->size(1) > kMostColumns) return false;
  *stride = t->stride(0);
  return t->stride(1) == 1 && *stride >= 0;
}

void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

at::Tensor empty_like_device(at::IntArrayRef size, const at::Tensor& t, at::ScalarType type) {
  return at::empty(size, at::TensorOptions().dtype(type).device(t.device()));
}

PyObject* quantize(const at::Tensor* x, PyObject* format_object, PyObject* factor_object) {
  const int format = format_code(format_object);
  int64_t stride = 0;
  const float* factor = nullptr;
  if (format < 0 || !row_matrix(x, &stride)) return nullptr;
  const int type = type_code(x->scalar_type());
  if (type < 0 || !factor_address(factor_object, format, x->device(), &factor)) return nullptr;
  const int64_t rows = x->size(0), k = x->size(1), columns = code_columns(k);
  at::Tensor codes = empty_like_device({rows, columns}, *x, at::kByte);
  at::Tensor scales = empty_like_device({(rows + 127) / 128, scale_tiles(columns, format), 32, 4, 4}, *x, at::kByte);
  if (g_lib.quantize(x->const_data_ptr(), type, rows, k, stride, format, factor, codes.mutable_data_ptr(),
                     scales.mutable_data_ptr(), x->get_device(), stream_of(*x)) != LBL_OK) {
    return nullptr;
  }
  PyObject* result = PyTuple_New(2);
  if (result == nullptr) return nullptr;
  PyTuple_SET_ITEM(result, 0, THPVariable_Wrap(std::move(codes)));
  PyTuple_SET_ITEM(result, 1, THPVariable_Wrap(std::move(scales)));
  return result;
}

PyObject* dequantize(PyObject* codes_object, PyObject* scales_object, PyObject* in_features, PyObject* format_object,
                     PyObject* factor_object, PyObject* dtype) {
  const int format = format_code(format_object);
  const at::Tensor *codes, *scales;
  const float* factor;
  if (format < 0 || !THPDtype_Check(dtype) || !operand(codes_object, scales_object, format, &codes, &scales) ||
      !factor_address(factor_object, format, codes->device(), &factor)) {
    return nullptr;
  }
  const at::ScalarType out_type = reinterpret_cast<THPDtype*>(dtype)->scalar_type;
  const int type = type_code(out_type);
  int64_t k = codes->size(1) * 2;
  if (in_features != Py_None) {
    if (!PyLong_CheckExact(in_features)) return nullptr;
    k = PyLong_AsLongLong(in_features);
    if (k == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      return nullptr;
    }
  }
  if (type < 0 || k <= 0 || k > kMostColumns || code_columns(k) != codes->size(1)) return nullptr;
  at::Tensor out = empty_like_device({codes->size(0), k}, *codes, out_type);
  if (g_lib.dequantize(codes->const_data_ptr(), scales->const_data_ptr(), codes->size(0), k, format, factor,
                       out.mutable_data_ptr(), type, codes->get_device(), stream_of(*codes)) != LBL_OK) {
    return nullptr;
  }
  return THPVariable_Wrap(std::move(out));
}

PyObject* matmul(PyObject* const* args) {
  const int format = format_code(args[4]);
  const at::Tensor *ac, *as, *bc, *bs;
  const float *fa, *fb;
  if (format < 0 || !THPDtype_Check(args[7]) || !operand(args[0], args[1], format, &ac, &as) ||
      !operand(args[2], args[3], format, &bc, &bs) || ac->device() != bc->device() || ac->size(1) != bc->size(1) ||
      !factor_address(args[5], format, ac->device(), &fa) || !factor_address(args[6], format, ac->device(), &fb)) {
    return nullptr;
  }
  const at::ScalarType out_type = reinterpret_cast<THPDtype*>(args[7])->scalar_type;
  if (out_type != at::kHalf && out_type != at::kBFloat16) return nullptr;
  const int64_t m = ac->size(0), n = bc->size(0);
  at::Tensor out = empty_like_device({m, n}, *ac, out_type);
  if (g_lib.matmul(ac->const_data_ptr(), as->const_data_ptr(), fa, bc->const_data_ptr(), bs->const_data_ptr(), fb,
                   out.mutable_data_ptr(), m, n, ac->size(1) * 2, format, type_code(out_type),
                   static_cast<unsigned>(PyLong_AsUnsignedLongMask(args[8])), ac->get_device(), stream_of(*ac)) != LBL_OK) {
    return nullptr;
  }
  return THPVariable_Wrap(std::move(out));
}

PyObject* linear(PyObject* const* args) {
  const at::Tensor* x = cuda_tensor(args[0]);
  const int format = format_code(args[3]);
  const at::Tensor *codes, *scales;
  const float *fw, *fx;
  int64_t stride = 0;
  if (format < 0 || !row_matrix(x, &stride) || !operand(args[1], args[2], format, &codes, &scales) ||
      x->device() != codes->device() || !factor_address(args[4], format, x->device(), &fw) ||
      !factor_address(args[5], format, x->device(), &fx)) {
    return nullptr;
  }
  const at::ScalarType type = x->scalar_type();
  const int64_t m = x->size(0), k = x->size(1), n = codes->size(0);
  if ((type != at::kHalf && type != at::kBFloat16) || code_columns(k) != codes->size(1)) return nullptr;
  at::Tensor y = empty_like_device({m, n}, *x, type);
  // Scratch per call: calls on different streams, and graphs captured from them, share nothing.
  const size_t need = g_lib.linear_workspace_bytes(m, n, k, format);
  at::Tensor scratch;
  if (need > 0) scratch = empty_like_device({static_cast<int64_t>(need)}, *x, at::kByte);
  if (g_lib.linear(x->const_data_ptr(), type_code(type), stride, fx, codes->const_data_ptr(), scales->const_data_ptr(), fw,
                   y.mutable_data_ptr(), m, n, k, format, need > 0 ? scratch.mutable_data_ptr() : nullptr, need,
                   static_cast<unsigned>(PyLong_AsUnsignedLongMask(args[6])), x->get_device(), stream_of(*x)) != LBL_OK) {
    return nullptr;
  }
  return THPVariable_Wrap(std::move(y));
}

// No C++ exception may cross into the interpreter; a call that met one is left to the Python path.
template <typename F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F&& f) {
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
    return nullptr;
  }
  PyObject* result = nullptr;
  if (g_lib.linear != nullptr) {
    try {
      result = f();
    } catch (const std::exception&) {
      result = nullptr;
    }
  }
  if (result == nullptr) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  return result;
}

PyObject* py_bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "expected the addresses of five entry points");
    return nullptr;
  }
  void* address[5];
  for (int i = 0; i < 5; ++i) {
    address[i] = PyLong_AsVoidPtr(args[i]);
    if (address[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null entry point");
      return nullptr;
    }
  }
  g_lib.quantize = reinterpret_cast<decltype(g_lib.quantize)>(address[0]);
  g_lib.dequantize = reinterpret_cast<decltype(g_lib.dequantize)>(address[1]);
  g_lib.matmul = reinterpret_cast<decltype(g_lib.matmul)>(address[2]);
  g_lib.linear_workspace_bytes = reinterpret_cast<decltype(g_lib.linear_workspace_bytes)>(address[3]);
  g_lib.linear = reinterpret_cast<decltype(g_lib.linear)>(address[4]);
  Py_RETURN_NONE;
}
PyObject* py_quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 3, [&] { return quantize(cuda_tensor(args[0]), args[1], args[2]); });
}
PyObject* py_dequantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 6, [&] { return dequantize(args[0], args[1], args[2], args[3], args[4], args[5]); });
}
PyObject* py_matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 9, [&] { return matmul(args); });
}
PyObject* py_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 7, [&] { return linear(args); });
}

PyMethodDef g_methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_bind)), METH_FASTCALL, nullptr},
    {"quantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_quantize)), METH_FASTCALL, nullptr},
    {"dequantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_dequantize)), METH_FASTCALL, nullptr},
    {"matmul", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_matmul)), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_linear)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&g_module); }
