// The 8-bit path of the PyTorch extension `ms_blkq4linear_ext`: tensors are checked, reduced to pointers, byte sizes and
// leading dimensions, and handed to the int8_* calls of the C ABI in include/ms_blkq4gemm.h on PyTorch's current stream.
// CPython's vectorcall signature, as for `linear`: at decode sizes the conversion of the arguments is a good part of a call.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/extension.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <string>
#include <vector>

#include "ms_blkq4gemm.h"

namespace {

using torch::Tensor;

// A tensor as a matrix of its last dimension's rows, one pitch from row to row.
struct Rows {
  Tensor held;
  void* data = nullptr;
  int rows = 0, cols = 0;
  int64_t ld = 0;
  size_t bytes = 0;
};

// Whether the leading dimensions of `x` are rows of one pitch, at least a row long; `ld` is that pitch.
bool one_pitch(const Tensor& x, int64_t rows, int64_t cols, int64_t* ld) {
  const int64_t d = x.dim();
  if (cols > 1 && x.stride(d - 1) != 1) return false;
  *ld = cols;
  int64_t expect = -1;
  for (int64_t i = d - 2; i >= 0; --i) {
    if (x.size(i) == 1) continue;
    if (expect < 0) *ld = x.stride(i);
    else if (x.stride(i) != expect) return false;
    expect = x.stride(i) * x.size(i);
  }
  return rows <= 1 || *ld >= cols;
}

Rows as_rows(const char* name, const Tensor& x, bool may_copy) {
  TORCH_CHECK(x.is_cuda(), name, " must be a CUDA tensor, instead got ", x.device().str());
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, name, " must have rows of at least one element");
  Rows r;
  const int64_t cols = x.size(-1), rows = x.numel() / cols;
  TORCH_CHECK(rows <= (1 << 28) && cols <= (1 << 28), name, " is too large: ", rows, " rows of ", cols);
  r.held = x;
  if (!one_pitch(x, rows, cols, &r.ld)) {
    TORCH_CHECK(may_copy, name, " must have contiguous rows of one pitch");
    r.held = x.contiguous();
    r.ld = cols;
  }
  r.data = r.held.data_ptr();
  r.rows = int(rows);
  r.cols = int(cols);
  r.bytes = rows > 0 ? size_t((rows - 1) * r.ld + cols) * r.held.element_size() : 0;
  return r;
}

int type_of(const char* name, torch::ScalarType t) {
  TORCH_CHECK(t == torch::kFloat16 || t == torch::kBFloat16, name, " must be float16 or bfloat16, instead got ", toString(t));
  return t == torch::kFloat16 ? INT8_FP16 : INT8_BF16;
}

void no_backward(const Tensor& x) {
  TORCH_CHECK(!x.requires_grad() || !at::GradMode::is_enabled(),
              "The int8 operators have no backward pass: call them under torch.no_grad(), or detach the tensor");
  TORCH_CHECK(!x._fw_grad(/*level=*/0).defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode(),
              "The int8 operators have no forward derivatives: take the primal of the dual tensor");
}

// A caller's tensor is about to be written: what autograd has saved of it, or of a view, is not what it was.  (Tensors made under
// inference mode have no versions.)
void written(const Tensor& x) {
  if (!x.is_inference()) torch::autograd::impl::bump_version(x);
}

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

void* current_stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

void same_device(const char* name, const Tensor& t, const Tensor& with) {
  TORCH_CHECK(t.device() == with.device(), name, " must be on the device of the input, ", with.device().str(), ", instead got ",
              t.device().str());
}

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

// Whether two matrices of one shape share no element, or are one and the same.
bool apart_or_same(const Rows& a, const Rows& b) {
  const int64_t elt = a.held.element_size();
  const char *pa = static_cast<const char*>(a.data), *pb = static_cast<const char*>(b.data);
  if (pa + a.bytes <= pb || pb + b.bytes <= pa) return true;
  if (a.rows > 1 && a.ld != b.ld) return false;
  if (pa == pb) return true;
  const int64_t diff = (pa < pb ? pb - pa : pa - pb);
  if (a.rows <= 1 || diff % elt != 0) return false;
  const int64_t d = diff / elt % a.ld;  // two column ranges of one wider matrix
  return d >= a.cols && d + a.cols <= a.ld;
}

// Whether no byte of `a` is one of `b`, whatever their types: column ranges of one wider matrix are apart, for instance.
bool apart(const Rows& a, const Rows& b) {
  const char *pa = static_cast<const char*>(a.data), *pb = static_cast<const char*>(b.data);
  if (a.bytes == 0 || b.bytes == 0 || pa + a.bytes <= pb || pb + b.bytes <= pa) return true;
  const Rows &few = a.rows <= b.rows ? a : b, &many = a.rows <= b.rows ? b : a;
  const int64_t few_elt = few.held.element_size(), elt = many.held.element_size();
  const int64_t pitch = many.rows > 1 ? many.ld * elt : 1, length = many.cols * elt;
  for (int64_t i = 0; i < few.rows; ++i) {  // the last row of `many` that begins before this one's end
    const int64_t begin = static_cast<const char*>(few.data) + i * few.ld * few_elt - static_cast<const char*>(many.data);
    const int64_t end = begin + few.cols * few_elt;
    if (end <= 0) continue;
    const int64_t row = std::min<int64_t>((end - 1) / pitch, many.rows - 1);
    if (row * pitch + length > begin) return false;
  }
  return true;
}
// A vector as one row.
Rows as_row(const Tensor& v) {
  Rows r;
  r.held = v;
  r.data = v.data_ptr();
  r.rows = 1;
  r.cols = int(v.numel());
  r.ld = r.cols;
  r.bytes = v.nbytes();
  return r;
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

bool on_16_bytes(const Rows& r) {
  return reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && (r.rows <= 1 || r.ld % 16 == 0);
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

// ---- the calls' arguments, by position ----
const Tensor& tensor(PyObject* o, const char* call) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), call, ": a tensor is wanted, instead got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
const Tensor* tensor_or_none(PyObject* o, const char* call) { return o == Py_None ? nullptr : &tensor(o, call); }
torch::ScalarType dtype_of(PyObject* o, const char* call) {
  TORCH_CHECK_TYPE(THPDtype_Check(o), call, ": a torch.dtype is wanted, instead got ", Py_TYPE(o)->tp_name);
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}
void count_args(Py_ssize_t nargs, Py_ssize_t wanted, const char* signature) { TORCH_CHECK_TYPE(nargs == wanted, signature); }

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

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
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
