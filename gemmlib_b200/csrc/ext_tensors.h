// What the parts of the PyTorch extension share: tensors as matrices of rows, their checks, and the calls' arguments by position.
#pragma once

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

namespace ext_tensors {

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
inline bool one_pitch(const Tensor& x, int64_t rows, int64_t cols, int64_t* ld) {
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

inline Rows as_rows(const char* name, const Tensor& x, bool may_copy) {
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

inline int type_of(const char* name, torch::ScalarType t) {
  TORCH_CHECK(t == torch::kFloat16 || t == torch::kBFloat16, name, " must be float16 or bfloat16, instead got ", toString(t));
  return t == torch::kFloat16 ? INT8_FP16 : INT8_BF16;
}

inline void no_tangent(const Tensor& x, const char* kind) {
  TORCH_CHECK(!x._fw_grad(/*level=*/0).defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode(),
              "The ", kind, " operators have no forward derivatives: take the primal of the dual tensor");
}
inline void no_backward(const Tensor& x, const char* kind) {
  TORCH_CHECK(!x.requires_grad() || !at::GradMode::is_enabled(),
              "The ", kind, " operators have no backward pass: call them under torch.no_grad(), or detach the tensor");
  no_tangent(x, kind);
}

// A caller's tensor is about to be written: what autograd has saved of it, or of a view, is not what it was.  (Tensors made under
// inference mode have no versions.)
inline void written(const Tensor& x) {
  if (!x.is_inference()) torch::autograd::impl::bump_version(x);
}

inline void* current_stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

inline void same_device(const char* name, const Tensor& t, const Tensor& with) {
  TORCH_CHECK(t.device() == with.device(), name, " must be on the device of the input, ", with.device().str(), ", instead got ",
              t.device().str());
}

// Whether two matrices of one shape share no element, or are one and the same.
inline bool apart_or_same(const Rows& a, const Rows& b) {
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
inline bool apart(const Rows& a, const Rows& b) {
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
inline Rows as_row(const Tensor& v) {
  Rows r;
  r.held = v;
  r.data = v.data_ptr();
  r.rows = 1;
  r.cols = int(v.numel());
  r.ld = r.cols;
  r.bytes = v.nbytes();
  return r;
}

inline bool on_16_bytes(const Rows& r) {
  return reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && (r.rows <= 1 || r.ld % 16 == 0);
}

// ---- the calls' arguments, by position ----
inline const Tensor& tensor(PyObject* o, const char* call) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), call, ": a tensor is wanted, instead got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
inline const Tensor* tensor_or_none(PyObject* o, const char* call) { return o == Py_None ? nullptr : &tensor(o, call); }
inline torch::ScalarType dtype_of(PyObject* o, const char* call) {
  TORCH_CHECK_TYPE(THPDtype_Check(o), call, ": a torch.dtype is wanted, instead got ", Py_TYPE(o)->tp_name);
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}
inline void count_args(Py_ssize_t nargs, Py_ssize_t wanted, const char* signature) { TORCH_CHECK_TYPE(nargs == wanted, signature); }

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}

}  // namespace ext_tensors
