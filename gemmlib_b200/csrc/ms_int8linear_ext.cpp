// The 8-bit path of the PyTorch extension `ms_blkq4linear_ext`: tensors are checked, reduced to pointers, byte sizes and
// leading dimensions, and handed to the int8_* calls of the C ABI in include/ms_blkq4gemm.h on PyTorch's current stream.
// CPython's vectorcall signature, as for `linear`: at decode sizes the conversion of the arguments is a good part of a call.
#include "ext_tensors.h"

namespace {

using namespace ext_tensors;

void no_backward(const Tensor& x) { ext_tensors::no_backward(x, "int8"); }

// int8 rows in the shape of `x`, every row beginning on 32 bytes (what the product copies fastest), and their scales.
struct Int8Out {
  Tensor values, scales;
  int64_t ld;
};
Int8Out int8_like(const Tensor& x) {
  const int64_t cols = x.size(-1), pitch = (cols + 31) / 32 * 32, rows = x.numel() / cols;
  Int8Out o;
  o.ld = pitch;
  // One allocation for both, the scales behind the rows: at a token's sizes an allocation (0.7 us) is a good part of a call.
  o.values = at::empty({rows * (pitch + 4)}, at::TensorOptions().dtype(at::kChar).device(x.device()));
  o.scales = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(o.values.storage()), o.values.key_set(), caffe2::TypeMeta::Make<float>());
  auto* scales = o.scales.unsafeGetTensorImpl();
  scales->set_storage_offset(rows * pitch / 4);
  scales->set_sizes_contiguous(x.sizes().slice(0, x.dim() - 1));
  c10::SmallVector<int64_t, 6> strides(x.dim(), 1);
  int64_t s = pitch;
  for (int64_t i = x.dim() - 2; i >= 0; --i) {
    strides[i] = s;
    s *= std::max<int64_t>(x.size(i), 1);
  }
  o.values.unsafeGetTensorImpl()->set_sizes_and_strides(x.sizes(), strides);
  return o;
}
size_t int8_bytes(const Int8Out& o, int rows, int cols) { return size_t(rows - 1) * size_t(o.ld) + size_t(cols); }

Int8Out quantize(const Tensor& x) {
  const int dtype = type_of("int8_quantize: the input", x.scalar_type());
  no_backward(x);
  const Rows a = as_rows("int8_quantize: the input", x, true);
  const c10::cuda::CUDAGuard guard(x.device());
  Int8Out o = int8_like(x);
  if (a.rows == 0) return o;
  std::string err;
  TORCH_CHECK(int8_rows_quant_sm100(dtype, a.rows, a.cols, current_stream(), a.data, a.bytes, a.ld, o.values.data_ptr(),
                                    int8_bytes(o, a.rows, a.cols), o.ld, o.scales.data_ptr(), size_t(a.rows) * 4, &err) == 0,
              err);
  return o;
}

Int8Out rms_norm(const Tensor& x, const Tensor& weight, double eps, const Tensor* residual, Tensor* residual_out) {
  const int dtype = type_of("rms_norm_int8: the input", x.scalar_type());
  no_backward(x);
  no_backward(weight);
  if (residual) {
    no_backward(*residual);
    if (residual_out->defined()) no_backward(*residual_out);
  }
  const Rows a = as_rows("rms_norm_int8: the input", x, true);
  TORCH_CHECK(weight.scalar_type() == x.scalar_type() && weight.dim() == 1 && weight.size(0) == a.cols,
              "rms_norm_int8: the weight must be one row of the input's length and type");
  same_device("rms_norm_int8: the weight", weight, x);
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor w = weight.contiguous();
  Rows r, s;
  const bool brought = residual && residual_out->defined();
  if (residual) {
    TORCH_CHECK(residual->scalar_type() == x.scalar_type() && residual->sizes() == x.sizes(),
                "rms_norm_int8: the residual must have the input's shape and type");
    same_device("rms_norm_int8: the residual", *residual, x);
    r = as_rows("rms_norm_int8: the residual", *residual, true);
    if (brought) {
      TORCH_CHECK(residual_out->scalar_type() == x.scalar_type() && residual_out->sizes() == x.sizes(),
                  "rms_norm_int8: residual_out must have the input's shape and type");
      same_device("rms_norm_int8: residual_out", *residual_out, x);
      s = as_rows("rms_norm_int8: residual_out", *residual_out, false);
      TORCH_CHECK(apart_or_same(s, a) && apart_or_same(s, r),
                  "rms_norm_int8: residual_out may be the input or the residual, but not overlap them otherwise");
      TORCH_CHECK(apart(s, as_row(w)), "rms_norm_int8: residual_out overlaps the weight");
    } else {
      *residual_out = at::empty(x.sizes(), x.options());
      s = as_rows("rms_norm_int8: residual_out", *residual_out, false);
    }
  }
  Int8Out o = int8_like(x);
  if (a.rows == 0) return o;
  if (brought) written(*residual_out);
  std::string err;
  TORCH_CHECK(int8_rows_rms_norm_sm100(dtype, a.rows, a.cols, current_stream(), a.data, a.bytes, a.ld, r.data, r.bytes, r.ld,
                                       w.data_ptr(), w.nbytes(), float(eps), s.data, s.bytes, s.ld, o.values.data_ptr(),
                                       int8_bytes(o, a.rows, a.cols), o.ld, o.scales.data_ptr(), size_t(a.rows) * 4, &err) == 0,
              err);
  return o;
}

Int8Out silu_mul(const Tensor& gate, const Tensor& up) {
  const int dtype = type_of("silu_mul_int8: gate", gate.scalar_type());
  no_backward(gate);
  no_backward(up);
  TORCH_CHECK(up.scalar_type() == gate.scalar_type() && up.sizes() == gate.sizes(),
              "silu_mul_int8: gate and up must have one shape and type");
  const Rows g = as_rows("silu_mul_int8: gate", gate, true);
  same_device("silu_mul_int8: up", up, gate);
  const Rows u = as_rows("silu_mul_int8: up", up, true);
  const c10::cuda::CUDAGuard guard(gate.device());
  Int8Out o = int8_like(gate);
  if (g.rows == 0) return o;
  std::string err;
  TORCH_CHECK(int8_rows_silu_mul_sm100(dtype, g.rows, g.cols, current_stream(), g.data, g.bytes, g.ld, u.data, u.bytes, u.ld,
                                       o.values.data_ptr(), int8_bytes(o, g.rows, g.cols), o.ld, o.scales.data_ptr(),
                                       size_t(g.rows) * 4, &err) == 0,
              err);
  return o;
}

// Scales of `rows` rows, contiguous.
Tensor check_scales(const char* name, const Tensor& scales, const Tensor& values, int64_t rows) {
  TORCH_CHECK(scales.scalar_type() == torch::kFloat && scales.numel() == rows, name, ": one float32 scale a row is wanted");
  same_device(name, scales, values);
  return scales.contiguous();
}

Tensor dequantize(const Tensor& values, const Tensor& scales, torch::ScalarType type) {
  const int dtype = type_of("int8_dequantize: the output's type", type);
  TORCH_CHECK(values.scalar_type() == torch::kChar, "int8_dequantize: the values must be int8");
  no_backward(scales);
  const Rows v = as_rows("int8_dequantize: the values", values, true);
  const c10::cuda::CUDAGuard guard(values.device());
  const Tensor s = check_scales("int8_dequantize: scales", scales, values, v.rows);
  Tensor out = at::empty(values.sizes(), values.options().dtype(type).memory_format(at::MemoryFormat::Contiguous));
  if (v.rows == 0) return out;
  std::string err;
  TORCH_CHECK(int8_rows_dequant_sm100(dtype, v.rows, v.cols, current_stream(), v.data, v.bytes, v.ld, s.data_ptr(), s.nbytes(),
                                      out.data_ptr(), out.nbytes(), v.cols, &err) == 0,
              err);
  return out;
}

Tensor linear(const Tensor& x, const Tensor& x_scales, const Tensor& w, const Tensor& w_scales, const Tensor* bias,
              torch::ScalarType type, int64_t flags, const Tensor* brought) {
  const int dtype = type_of("int8_linear: the output's type", type);
  TORCH_CHECK(x.scalar_type() == torch::kChar && w.scalar_type() == torch::kChar, "int8_linear: input and weight must be int8 rows");
  no_backward(x_scales);
  no_backward(w_scales);
  if (bias) no_backward(*bias);
  if (brought) no_backward(*brought);
  Rows a = as_rows("int8_linear: the input", x, true);
  TORCH_CHECK(w.dim() == 2, "int8_linear: the weight must be [out_features, in_features]");
  const Rows b = as_rows("int8_linear: the weight", w, false);
  same_device("int8_linear: the weight", w, x);
  TORCH_CHECK(a.cols == b.cols, "int8_linear: rows of ", a.cols, " cannot be multiplied with weights of ", b.cols, " in_features");
  TORCH_CHECK(b.rows > 0, "int8_linear: the weight is empty");
  TORCH_CHECK(on_16_bytes(b), "int8_linear: rows of the weight must begin on 16 bytes");
  const c10::cuda::CUDAGuard guard(x.device());
  if (!on_16_bytes(a)) {  // rows that no int8 operator made: laid out as they make them
    Int8Out copy = int8_like(x);
    copy.values.copy_(x);
    a = as_rows("int8_linear: the input", copy.values, false);
  }
  const Tensor xs = check_scales("int8_linear: the input's scales", x_scales, x, a.rows);
  const Tensor ws = check_scales("int8_linear: the weight's scales", w_scales, x, b.rows);
  if (bias) {
    TORCH_CHECK(bias->scalar_type() == type && bias->dim() == 1 && bias->size(0) == b.rows && bias->is_contiguous(),
                "int8_linear: the bias must be a contiguous [out_features] tensor of the output's type");
    same_device("int8_linear: the bias", *bias, x);
  }
  auto shape = x.sizes().vec();
  shape.back() = b.rows;
  Tensor out;
  if (brought) {
    out = *brought;
    TORCH_CHECK(out.scalar_type() == type && out.sizes() == c10::IntArrayRef(shape),
                "int8_linear: out must have the shape and type of the result");
    same_device("int8_linear: out", out, x);
  } else {
    out = at::empty(shape, at::TensorOptions().dtype(type).device(x.device()));
  }
  if (a.rows == 0) return out;
  const Rows o = as_rows("int8_linear: out", out, false);
  if (brought) {
    TORCH_CHECK(apart(o, a) && apart(o, b) && apart(o, as_row(xs)) && apart(o, as_row(ws)) && (!bias || apart(o, as_row(*bias))),
                "int8_linear: out overlaps a tensor that the product reads");
    written(out);
  }
  std::string err;
  TORCH_CHECK(int8_gemm_sm100(dtype, a.rows, b.rows, a.cols, current_stream(), a.data, a.bytes, a.ld, xs.data_ptr(), xs.nbytes(),
                              b.data, b.bytes, b.ld, ws.data_ptr(), ws.nbytes(), bias ? bias->data_ptr() : nullptr,
                              bias ? bias->nbytes() : 0, o.data, o.bytes, o.ld, unsigned(flags), &err) == 0,
              err);
  return out;
}

// Int8Rows, a named tuple of the Python module: made here, since its own constructor is a Python function.
PyTypeObject* g_rows_type = nullptr;

PyObject* wrap(const Int8Out& o) {
  PyObject* pair = PyTuple_New(2);
  if (!pair) throw python_error();
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(o.values));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(o.scales));
  if (!g_rows_type) return pair;
  PyObject* args = PyTuple_Pack(1, pair);
  Py_DECREF(pair);
  if (!args) throw python_error();
  PyObject* rows = PyTuple_Type.tp_new(g_rows_type, args, nullptr);
  Py_DECREF(args);
  if (!rows) throw python_error();
  return rows;
}

PyObject* py_rows_type(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count_args(nargs, 1, "int8_rows_type(cls)");
  TORCH_CHECK_TYPE(PyType_Check(args[0]) && PyType_IsSubtype(reinterpret_cast<PyTypeObject*>(args[0]), &PyTuple_Type),
                   "int8_rows_type: a subclass of tuple is wanted");
  Py_INCREF(args[0]);
  g_rows_type = reinterpret_cast<PyTypeObject*>(args[0]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* py_quantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count_args(nargs, 1, "int8_quantize(x)");
  return wrap(quantize(tensor(args[0], "int8_quantize")));
  END_HANDLE_TH_ERRORS
}

PyObject* py_rms_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count_args(nargs, 5, "rms_norm_int8(x, weight, eps, residual, residual_out)");
  const double eps = PyFloat_AsDouble(args[2]);
  if (eps == -1.0 && PyErr_Occurred()) throw python_error();
  const Tensor* residual = tensor_or_none(args[3], "rms_norm_int8");
  Tensor out;
  if (args[4] != Py_None) {
    TORCH_CHECK(residual, "rms_norm_int8: residual_out without a residual");
    out = tensor(args[4], "rms_norm_int8");
  }
  const Int8Out o = rms_norm(tensor(args[0], "rms_norm_int8"), tensor(args[1], "rms_norm_int8"), eps, residual, &out);
  PyObject* rows = wrap(o);
  if (!residual) return rows;
  PyObject* both = PyTuple_New(2);
  if (!both) throw python_error();
  PyTuple_SET_ITEM(both, 0, rows);
  PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(out));
  return both;
  END_HANDLE_TH_ERRORS
}

PyObject* py_silu_mul(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count_args(nargs, 2, "silu_mul_int8(gate, up)");
  return wrap(silu_mul(tensor(args[0], "silu_mul_int8"), tensor(args[1], "silu_mul_int8")));
  END_HANDLE_TH_ERRORS
}

PyObject* py_dequantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count_args(nargs, 3, "int8_dequantize(values, scales, dtype)");
  return THPVariable_Wrap(dequantize(tensor(args[0], "int8_dequantize"), tensor(args[1], "int8_dequantize"),
                                     dtype_of(args[2], "int8_dequantize")));
  END_HANDLE_TH_ERRORS
}

PyObject* py_linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count_args(nargs, 8, "int8_linear(x, x_scales, weight, weight_scales, bias, dtype, flags, out)");
  const long flags = PyLong_AsLong(args[6]);
  if (flags == -1 && PyErr_Occurred()) throw python_error();
  constexpr const char* call = "int8_linear";
  return THPVariable_Wrap(linear(tensor(args[0], call), tensor(args[1], call), tensor(args[2], call), tensor(args[3], call),
                                 tensor_or_none(args[4], call), dtype_of(args[5], call), flags, tensor_or_none(args[7], call)));
  END_HANDLE_TH_ERRORS
}

PyMethodDef g_methods[] = {
    {"int8_rows_type", fast<py_rows_type>(), METH_FASTCALL, "The tuple's subclass that int8 rows are returned as"},
    {"int8_quantize", fast<py_quantize>(), METH_FASTCALL, "The rows of x in int8"},
    {"rms_norm_int8", fast<py_rms_norm>(), METH_FASTCALL, "The normed rows, or them and the sum where there is a residual"},
    {"silu_mul_int8", fast<py_silu_mul>(), METH_FASTCALL, "The rows of silu(gate) * up"},
    {"int8_dequantize", fast<py_dequantize>(), METH_FASTCALL, "scales * values"},
    {"int8_linear", fast<py_linear>(), METH_FASTCALL, "The product of int8 rows with an int8 weight"},
    {nullptr, nullptr, 0, nullptr}};

}  // namespace

bool add_int8_functions(PyObject* module) { return PyModule_AddFunctions(module, g_methods) == 0; }
