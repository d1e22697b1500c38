// The 8-bit floating-point path of the PyTorch extension `ms_blkq4linear_ext`, and layers of experts: tensors are checked, reduced to pointers,
// byte sizes and leading dimensions, and handed to the fp8_* and experts_* calls of the C ABI on PyTorch's current stream.
#include "ext_tensors.h"

#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>

#include <tuple>
#include <unordered_set>

namespace {

using namespace ext_tensors;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kBlock = 128;
int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }

void no_backward(const Tensor& x) { ext_tensors::no_backward(x, "fp8"); }
void no_backward_here(const Tensor& x) { ext_tensors::no_backward(x, "experts'"); }

void check_e4m3(const char* name, const Tensor& x) {
  TORCH_CHECK(x.scalar_type() == torch::kFloat8_e4m3fn, name, " must be float8_e4m3fn, instead got ", toString(x.scalar_type()));
}
// A tensor that begins `offset` bytes into the storage of `held`.
Tensor piece(const Tensor& held, int64_t offset, caffe2::TypeMeta type, c10::IntArrayRef sizes) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(held.storage()), held.key_set(), type);
  t.unsafeGetTensorImpl()->set_storage_offset(offset / int64_t(type.itemsize()));
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}

// e4m3 rows of these sizes, every row beginning on 32 bytes, and their scales; one allocation for both, the scales behind the rows.
struct Fp8Out {
  Tensor values, scales;
  int64_t ld, lds;
  size_t bytes, scale_bytes;
};
Fp8Out rows_like(c10::IntArrayRef sizes, int64_t rows, const c10::Device& device) {
  const int64_t d = int64_t(sizes.size()), cols = sizes.back(), pitch = (cols + 31) / 32 * 32, blocks = blocks_of(cols);
  Fp8Out o;
  o.ld = pitch;
  o.lds = blocks;
  o.bytes = rows > 0 ? size_t((rows - 1) * pitch + cols) : 0;
  o.scale_bytes = size_t(rows * blocks) * 4;
  o.values = at::empty({rows * (pitch + 4 * blocks)}, at::TensorOptions().dtype(at::kFloat8_e4m3fn).device(device));
  c10::SmallVector<int64_t, 6> scale_sizes(sizes.begin(), sizes.end()), strides(d, 1);
  scale_sizes.back() = blocks;
  o.scales = piece(o.values, rows * pitch, caffe2::TypeMeta::Make<float>(), scale_sizes);
  int64_t s = pitch;
  for (int64_t i = d - 2; i >= 0; --i) {
    strides[i] = s;
    s *= std::max<int64_t>(sizes[i], 1);
  }
  o.values.unsafeGetTensorImpl()->set_sizes_and_strides(sizes, strides);
  return o;
}

// The order of the choices: tensors of sort_by_expert, or their like.
struct Order {
  Tensor source, places, offsets;
  int64_t rows, choices, tokens;
  const void* count;
};
Order check_order(const char* call, const Tensor& source, const Tensor& places, const Tensor& offsets, const Tensor& with) {
  Order o{source, places, offsets, 0, 0, 0, nullptr};
  for (const Tensor* t : {&source, &places, &offsets}) {
    TORCH_CHECK(t->scalar_type() == torch::kInt && t->is_contiguous(), call, ": the order's tensors must be contiguous and int32");
    same_device(call, *t, with);
  }
  TORCH_CHECK(places.dim() >= 1 && places.size(-1) > 0 && source.dim() == 1 && source.numel() == places.numel() && offsets.dim() == 1 &&
                  offsets.numel() >= 2,
              call, ": the order must have source [choices of all tokens], places [..., choices of a token] and offsets [experts + 1]");
  o.rows = source.numel();
  o.choices = places.size(-1);
  o.tokens = o.rows / o.choices;
  TORCH_CHECK(o.rows <= (1 << 28), call, ": too many choices: ", o.rows);
  o.count = offsets.const_data_ptr<int>() + offsets.numel() - 1;
  return o;
}
const char* kOrderText = ": the rows must be those of the order's tokens";

Fp8Out quantize(const Tensor& x, const Tensor* source, const Tensor* places, const Tensor* offsets) {
  const int dtype = type_of("quantize_fp8: the input", x.scalar_type());
  no_backward(x);
  const Rows a = as_rows("quantize_fp8: the input", x, true);
  const c10::cuda::CUDAGuard guard(x.device());
  std::string err;
  if (!source) {
    Fp8Out o = rows_like(x.sizes(), a.rows, x.device());
    if (a.rows == 0) return o;
    TORCH_CHECK(fp8_rows_quant_sm100(dtype, a.rows, a.cols, current_stream(), a.data, a.bytes, a.ld, o.values.data_ptr(), o.bytes, o.ld,
                                     o.scales.data_ptr(), o.scale_bytes, o.lds, &err) == 0,
                err);
    return o;
  }
  const Order order = check_order("quantize_fp8", *source, *places, *offsets, x);
  TORCH_CHECK(a.rows == order.tokens, "quantize_fp8", kOrderText, ", ", order.tokens, ", instead got ", a.rows);
  const int64_t sizes[2] = {order.rows, a.cols};
  Fp8Out o = rows_like(sizes, order.rows, x.device());
  if (order.rows == 0) return o;
  TORCH_CHECK(fp8_rows_gather_quant_sm100(dtype, a.rows, int(order.choices), a.cols, current_stream(), a.data, a.bytes, a.ld,
                                          order.places.data_ptr(), order.places.nbytes(), order.count, o.values.data_ptr(), o.bytes, o.ld,
                                          o.scales.data_ptr(), o.scale_bytes, o.lds, &err) == 0,
              err);
  return o;
}

Fp8Out silu_mul(const Tensor& gate, const Tensor& up) {
  const int dtype = type_of("silu_mul_fp8: gate", gate.scalar_type());
  no_backward(gate);
  no_backward(up);
  TORCH_CHECK(up.scalar_type() == gate.scalar_type() && up.sizes() == gate.sizes(),
              "silu_mul_fp8: gate and up must have one shape and type");
  const Rows g = as_rows("silu_mul_fp8: gate", gate, true);
  same_device("silu_mul_fp8: up", up, gate);
  const Rows u = as_rows("silu_mul_fp8: up", up, true);
  const c10::cuda::CUDAGuard guard(gate.device());
  Fp8Out o = rows_like(gate.sizes(), g.rows, gate.device());
  if (g.rows == 0) return o;
  std::string err;
  TORCH_CHECK(fp8_rows_silu_mul_sm100(dtype, g.rows, g.cols, current_stream(), g.data, g.bytes, g.ld, u.data, u.bytes, u.ld,
                                      o.values.data_ptr(), o.bytes, o.ld, o.scales.data_ptr(), o.scale_bytes, o.lds, &err) == 0,
              err);
  return o;
}

// Weights [..., out_features, in_features]: how many matrices there are.
int64_t matrices_of(const char* name, const Tensor& w) {
  TORCH_CHECK(w.dim() >= 2 && w.size(-1) > 0 && w.size(-2) > 0, name, " must be [..., out_features, in_features]");
  return w.numel() / (w.size(-1) * w.size(-2));
}

Fp8Out quantize_weight(const Tensor& w) {
  const int dtype = type_of("quantize_fp8_weight: the weight", w.scalar_type());
  no_backward(w);
  const int64_t experts = matrices_of("quantize_fp8_weight: the weight", w);
  const Rows a = as_rows("quantize_fp8_weight: the weight", w, true);
  const c10::cuda::CUDAGuard guard(w.device());
  const int64_t n = w.size(-2), k = w.size(-1);
  Fp8Out o = rows_like(w.sizes(), 0, w.device());  // (its strides)
  o.values = at::empty_strided(w.sizes(), o.values.strides(), o.values.options());
  auto sizes = w.sizes().vec();
  sizes[w.dim() - 2] = blocks_of(n);
  sizes[w.dim() - 1] = blocks_of(k);
  o.scales = at::empty(sizes, o.values.options().dtype(at::kFloat));
  if (a.rows == 0) return o;
  std::string err;
  TORCH_CHECK(fp8_weight_quant_sm100(dtype, int(experts), int(n), int(k), current_stream(), a.data, a.bytes, a.ld, o.values.data_ptr(),
                                     size_t((a.rows - 1) * o.ld + k), o.ld, o.scales.data_ptr(), o.scales.nbytes(), o.lds, &err) == 0,
              err);
  return o;
}

// The scales of rows: a matrix of one row of scales a row.
Rows check_scales(const char* name, const Tensor& scales, const Tensor& values) {
  auto sizes = values.sizes().vec();
  sizes.back() = blocks_of(sizes.back());
  TORCH_CHECK(scales.scalar_type() == torch::kFloat && scales.sizes() == c10::IntArrayRef(sizes), name, " must be float32 and of shape ",
              c10::IntArrayRef(sizes));
  same_device(name, scales, values);
  return as_rows(name, scales, true);
}
c10::SmallVector<int64_t, 6> weight_scale_sizes(const Tensor& w) {
  c10::SmallVector<int64_t, 6> sizes(w.sizes().begin(), w.sizes().end());
  const size_t d = sizes.size();
  sizes[d - 2] = blocks_of(sizes[d - 2]);
  sizes[d - 1] = blocks_of(sizes[d - 1]);
  return sizes;
}
void check_weight_scales(const char* name, const Tensor& scales, const Tensor& w) {
  const auto sizes = weight_scale_sizes(w);
  TORCH_CHECK(scales.scalar_type() == torch::kFloat && scales.sizes() == c10::IntArrayRef(sizes), name, " must be float32 and of shape ",
              c10::IntArrayRef(sizes));
  same_device(name, scales, w);
}

Tensor dequantize(const Tensor& values, const Tensor& scales, torch::ScalarType type, bool weight) {
  const int dtype = type_of("fp8_dequantize: the output's type", type);
  check_e4m3("fp8_dequantize: the values", values);
  no_backward(values);
  no_backward(scales);
  const Rows v = as_rows("fp8_dequantize: the values", values, true);
  const c10::cuda::CUDAGuard guard(values.device());
  Tensor out = at::empty(values.sizes(), values.options().dtype(type).memory_format(at::MemoryFormat::Contiguous));
  std::string err;
  if (weight) {
    const int64_t experts = matrices_of("fp8_dequantize: the values", values);
    check_weight_scales("fp8_dequantize: the scales", scales, values);
    if (v.rows == 0) return out;
    const Rows s = as_rows("fp8_dequantize: the scales", scales, true);
    TORCH_CHECK(fp8_weight_dequant_sm100(dtype, int(experts), int(values.size(-2)), v.cols, current_stream(), v.data, v.bytes, v.ld, s.data,
                                         s.bytes, s.ld, out.data_ptr(), out.nbytes(), v.cols, &err) == 0,
                err);
    return out;
  }
  const Rows s = check_scales("fp8_dequantize: the scales", scales, values);
  if (v.rows == 0) return out;
  TORCH_CHECK(fp8_rows_dequant_sm100(dtype, v.rows, v.cols, current_stream(), v.data, v.bytes, v.ld, s.data, s.bytes, s.ld, out.data_ptr(),
                                     out.nbytes(), v.cols, &err) == 0,
              err);
  return out;
}

// Activations that a product reads: rows that no operator of this path made are laid out as they make them.
Rows product_rows(const char* name, const Tensor& x) {
  Rows a = as_rows(name, x, true);
  if (!on_16_bytes(a)) {
    Fp8Out copy = rows_like(x.sizes(), a.rows, x.device());
    copy.values.copy_(x);
    a = as_rows(name, copy.values, false);
  }
  return a;
}
Tensor output_of(const char* name, const Tensor* brought, c10::IntArrayRef shape, torch::ScalarType type, const Tensor& x) {
  if (!brought) return at::empty(shape, at::TensorOptions().dtype(type).device(x.device()));
  TORCH_CHECK(brought->scalar_type() == type && brought->sizes() == shape, name, " must have the shape and type of the result");
  same_device(name, *brought, x);
  return *brought;
}

Tensor linear(const Tensor& x, const Tensor& x_scales, const Tensor& w, const Tensor& w_scales, const Tensor* bias, torch::ScalarType type,
              int64_t flags, const Tensor* brought) {
  const int dtype = type_of("fp8_linear: the output's type", type);
  check_e4m3("fp8_linear: the input", x);
  check_e4m3("fp8_linear: the weight", w);
  for (const Tensor* t : {&x, &x_scales, &w, &w_scales, bias, brought})
    if (t) no_backward(*t);
  TORCH_CHECK(x.is_cuda(), "fp8_linear: the input must be a CUDA tensor, instead got ", x.device().str());
  TORCH_CHECK(w.dim() == 2, "fp8_linear: the weight must be [out_features, in_features]");
  const c10::cuda::CUDAGuard guard(x.device());
  const Rows a = product_rows("fp8_linear: the input", x);
  const Rows b = as_rows("fp8_linear: the weight", w, false);
  same_device("fp8_linear: the weight", w, x);
  TORCH_CHECK(a.cols == b.cols, "fp8_linear: rows of ", a.cols, " cannot be multiplied with weights of ", b.cols, " in_features");
  TORCH_CHECK(b.rows > 0, "fp8_linear: the weight is empty");
  TORCH_CHECK(on_16_bytes(b), "fp8_linear: rows of the weight must begin on 16 bytes");
  const Rows xs = check_scales("fp8_linear: the input's scales", x_scales, x);
  check_weight_scales("fp8_linear: the weight's scales", w_scales, w);
  const Rows ws = as_rows("fp8_linear: the weight's scales", w_scales, true);
  if (bias) {
    TORCH_CHECK(bias->scalar_type() == type && bias->dim() == 1 && bias->size(0) == b.rows && bias->is_contiguous(),
                "fp8_linear: the bias must be a contiguous [out_features] tensor of the output's type");
    same_device("fp8_linear: the bias", *bias, x);
  }
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = b.rows;
  const Tensor out = output_of("fp8_linear: out", brought, shape, type, x);
  if (a.rows == 0) return out;
  const Rows o = as_rows("fp8_linear: out", out, false);
  if (brought) {
    TORCH_CHECK(apart(o, a) && apart(o, b) && apart(o, xs) && apart(o, ws) && (!bias || apart(o, as_row(*bias))),
                "fp8_linear: out overlaps a tensor that the product reads");
    written(out);
  }
  std::string err;
  TORCH_CHECK(fp8_gemm_sm100(dtype, a.rows, b.rows, a.cols, current_stream(), a.data, a.bytes, a.ld, xs.data, xs.bytes, xs.ld, b.data, b.bytes,
                             b.ld, ws.data, ws.bytes, ws.ld, bias ? bias->data_ptr() : nullptr, bias ? bias->nbytes() : 0, o.data, o.bytes,
                             o.ld, unsigned(flags), &err) == 0,
              err);
  return out;
}

// Matrices [experts, rows, cols] as they lie: rows of one pitch, experts a stride apart.
struct Stack {
  void* data;
  int64_t ld, stride;
  size_t bytes;
  Rows extent;  // all that lies between the first element and the last, as one row
};
bool is_stack(const Tensor& w) {
  return (w.size(2) <= 1 || w.stride(2) == 1) && (w.size(1) <= 1 || w.stride(1) >= w.size(2)) &&
         (w.size(0) <= 1 || w.stride(0) >= (w.size(1) - 1) * w.stride(1) + w.size(2));
}
Stack as_stack(const Tensor& w) {
  Stack s;
  s.data = w.data_ptr();
  s.ld = w.size(1) > 1 ? w.stride(1) : w.size(2);
  const int64_t one = (w.size(1) - 1) * s.ld + w.size(2);
  s.stride = w.size(0) > 1 ? w.stride(0) : one;
  s.bytes = size_t((w.size(0) - 1) * s.stride + one) * w.element_size();
  s.extent.held = w;
  s.extent.data = s.data;
  s.extent.rows = 1;
  s.extent.bytes = s.bytes;
  return s;
}
// Whether the two occupy no common range of addresses.
bool ranges_apart(const Rows& a, const Rows& b) {
  const char *pa = static_cast<const char*>(a.data), *pb = static_cast<const char*>(b.data);
  return pa + a.bytes <= pb || pb + b.bytes <= pa;
}

Tensor expert_linear(const Tensor& x, const Tensor& x_scales, const Tensor& w, const Tensor& w_scales, const Tensor& offsets,
                     torch::ScalarType type, int64_t flags, const Tensor* brought) {
  const int dtype = type_of("fp8_expert_linear: the output's type", type);
  check_e4m3("fp8_expert_linear: the input", x);
  check_e4m3("fp8_expert_linear: the weight", w);
  for (const Tensor* t : {&x, &x_scales, &w, &w_scales, brought})
    if (t) no_backward(*t);
  TORCH_CHECK(x.is_cuda(), "fp8_expert_linear: the input must be a CUDA tensor, instead got ", x.device().str());
  TORCH_CHECK(x.dim() == 2, "fp8_expert_linear: the input must be [rows, in_features]");
  TORCH_CHECK(w.dim() == 3 && w.numel() > 0, "fp8_expert_linear: the weight must be [experts, out_features, in_features]");
  same_device("fp8_expert_linear: the weight", w, x);
  TORCH_CHECK(w.size(0) <= 1024 && w.size(1) <= (1 << 28) && w.size(2) <= (1 << 28), "fp8_expert_linear: the weight is too large: ", w.sizes());
  TORCH_CHECK(x.size(1) == w.size(2), "fp8_expert_linear: rows of ", x.size(1), " cannot be multiplied with weights of ", w.size(2),
              " in_features");
  TORCH_CHECK(is_stack(w), "fp8_expert_linear: the weight must have contiguous rows of one pitch, and experts behind one another");
  const Stack b = as_stack(w);
  TORCH_CHECK(reinterpret_cast<uintptr_t>(b.data) % 16 == 0 && (w.size(1) <= 1 || b.ld % 16 == 0) && (w.size(0) <= 1 || b.stride % 16 == 0),
              "fp8_expert_linear: rows of the weight must begin on 16 bytes");
  check_weight_scales("fp8_expert_linear: the weight's scales", w_scales, w);
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor scales = is_stack(w_scales) ? w_scales : w_scales.contiguous();
  const Stack ws = as_stack(scales);
  const Rows a = product_rows("fp8_expert_linear: the input", x);
  const Rows xs = check_scales("fp8_expert_linear: the input's scales", x_scales, x);
  TORCH_CHECK(offsets.scalar_type() == torch::kInt && offsets.dim() == 1 && offsets.size(0) == w.size(0) + 1 && offsets.is_contiguous(),
              "fp8_expert_linear: offsets must be a contiguous int32 tensor of experts + 1 elements");
  same_device("fp8_expert_linear: offsets", offsets, x);
  const int64_t shape[2] = {a.rows, w.size(1)};
  const Tensor out = output_of("fp8_expert_linear: out", brought, shape, type, x);
  if (a.rows == 0) return out;
  const Rows o = as_rows("fp8_expert_linear: out", out, false);
  if (brought) {
    TORCH_CHECK(apart(o, a) && apart(o, xs) && apart(o, as_row(offsets)) && ranges_apart(o, b.extent) && ranges_apart(o, ws.extent),
                "fp8_expert_linear: out overlaps a tensor that the product reads");
    written(out);
  }
  std::string err;
  TORCH_CHECK(fp8_experts_gemm_sm100(dtype, int(w.size(0)), a.rows, int(w.size(1)), a.cols, current_stream(), a.data, a.bytes, a.ld, xs.data,
                                     xs.bytes, xs.ld, b.data, b.bytes, b.ld, b.stride, ws.data, ws.bytes, ws.ld, ws.stride,
                                     offsets.data_ptr(), offsets.nbytes(), o.data, o.bytes, o.ld,
                                     unsigned(flags) | (brought ? 0u : FP8_EXPERTS_ZERO_REST), &err) == 0,
              err);
  return out;
}

// ---- tokens to their experts and back ----
Order sort_choices(const Tensor& experts, int64_t n_experts) {
  TORCH_CHECK(experts.is_cuda(), "sort_by_expert: the experts must be a CUDA tensor, instead got ", experts.device().str());
  TORCH_CHECK(experts.scalar_type() == torch::kInt || experts.scalar_type() == torch::kLong,
              "sort_by_expert: the experts must be int32 or int64, instead got ", toString(experts.scalar_type()));
  TORCH_CHECK(experts.dim() >= 1 && experts.size(-1) > 0, "sort_by_expert: the experts must be [..., choices of a token]");
  TORCH_CHECK(n_experts >= 1 && n_experts <= 1024, "sort_by_expert: 1 to 1024 experts are taken, not ", n_experts);
  const int64_t n = experts.numel();
  TORCH_CHECK(n <= (1 << 28), "sort_by_expert: too many choices: ", n);
  const c10::cuda::CUDAGuard guard(experts.device());
  const Tensor ids = experts.contiguous();
  // one allocation for the three, offsets first
  const int64_t offsets_room = (n_experts + 1 + 3) / 4 * 4, source_room = (n + 3) / 4 * 4;
  const Tensor held = at::empty({offsets_room + source_room + n}, at::TensorOptions().dtype(at::kInt).device(experts.device()));
  const auto type = caffe2::TypeMeta::Make<int>();
  Order o{};
  o.offsets = piece(held, 0, type, {n_experts + 1});
  o.source = piece(held, offsets_room * 4, type, {n});
  o.places = piece(held, (offsets_room + source_room) * 4, type, experts.sizes());
  if (n == 0) {
    o.offsets.zero_();
    return o;
  }
  const size_t need = experts_sort_workspace_size(n, int(n_experts));
  const Tensor workspace = need > 0 ? at::empty({int64_t(need)}, held.options().dtype(at::kByte)) : Tensor();
  std::string err;
  TORCH_CHECK(experts_sort_sm100(n, int(n_experts), int(ids.element_size()), current_stream(), ids.data_ptr(), ids.nbytes(),
                                 o.source.data_ptr(), o.source.nbytes(), o.places.data_ptr(), o.places.nbytes(), o.offsets.data_ptr(),
                                 o.offsets.nbytes(), need > 0 ? workspace.data_ptr() : nullptr, need, &err) == 0,
              err);
  return o;
}

Tensor gather(const Tensor& x, const Tensor& source, const Tensor& places, const Tensor& offsets) {
  const int dtype = type_of("gather_rows: the input", x.scalar_type());
  no_backward_here(x);
  const Rows a = as_rows("gather_rows: the input", x, true);
  const Order order = check_order("gather_rows", source, places, offsets, x);
  TORCH_CHECK(a.rows == order.tokens, "gather_rows", kOrderText, ", ", order.tokens, ", instead got ", a.rows);
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor out = at::empty({order.rows, a.cols}, at::TensorOptions().dtype(x.scalar_type()).device(x.device()));
  if (order.rows == 0) return out;
  std::string err;
  TORCH_CHECK(experts_gather_sm100(dtype, a.rows, int(order.choices), a.cols, current_stream(), a.data, a.bytes, a.ld, source.data_ptr(),
                                   source.nbytes(), order.count, out.data_ptr(), out.nbytes(), a.cols, &err) == 0,
              err);
  return out;
}

int weights_type(const char* name, const Tensor& weights, const Tensor& places) {
  const auto t = weights.scalar_type();
  TORCH_CHECK(t == torch::kFloat || t == torch::kFloat16 || t == torch::kBFloat16, name,
              ": the weights must be float32, float16 or bfloat16, instead got ", toString(t));
  TORCH_CHECK(weights.sizes() == places.sizes(), name, ": the weights must have the shape of the order's places, ", places.sizes(),
              ", instead got ", weights.sizes());
  same_device(name, weights, places);
  return t == torch::kFloat ? EXPERTS_FP32 : t == torch::kFloat16 ? INT8_FP16 : INT8_BF16;
}

Tensor combine(const Tensor& y, const Tensor& source, const Tensor& places, const Tensor& offsets, const Tensor* weights) {
  const int dtype = type_of("combine_rows: the rows", y.scalar_type());
  no_backward_here(y);
  if (weights) no_backward_here(*weights);
  TORCH_CHECK(y.dim() == 2, "combine_rows: the rows must be [rows, features]");
  const Rows a = as_rows("combine_rows: the rows", y, true);
  const Order order = check_order("combine_rows", source, places, offsets, y);
  TORCH_CHECK(a.rows == order.rows, "combine_rows: one row a choice is wanted, ", order.rows, ", instead got ", a.rows);
  const int type = weights ? weights_type("combine_rows", *weights, places) : EXPERTS_FP32;
  const c10::cuda::CUDAGuard guard(y.device());
  const Tensor w = weights ? weights->contiguous() : Tensor();
  c10::SmallVector<int64_t, 6> shape(places.sizes().begin(), places.sizes().end());
  shape.back() = a.cols;
  const Tensor out = at::empty(shape, at::TensorOptions().dtype(y.scalar_type()).device(y.device()));
  if (order.rows == 0) return out;
  std::string err;
  TORCH_CHECK(experts_combine_sm100(dtype, int(order.tokens), int(order.choices), a.cols, current_stream(), a.data, a.bytes, a.ld,
                                    places.data_ptr(), places.nbytes(), weights ? w.data_ptr() : nullptr, weights ? w.nbytes() : 0, type,
                                    out.data_ptr(), out.nbytes(), a.cols, &err) == 0,
              err);
  return out;
}

// Undefined where it is not wanted.
std::pair<Tensor, Tensor> combine_backward(const Tensor& d, const Tensor& y, const Tensor& source, const Tensor& places, const Tensor& offsets,
                                           const Tensor& weights, bool want_y, bool want_weights) {
  const int dtype = type_of("combine_rows: the rows", y.scalar_type());
  no_backward_here(d);
  no_backward_here(y);
  no_backward_here(weights);
  TORCH_CHECK(d.scalar_type() == y.scalar_type() && y.dim() == 2, "combine_rows: the gradient must have the type of the rows");
  same_device("combine_rows: the gradient", d, y);
  const Rows g = as_rows("combine_rows: the gradient", d, true), a = as_rows("combine_rows: the rows", y, true);
  const Order order = check_order("combine_rows", source, places, offsets, y);
  TORCH_CHECK(a.rows == order.rows && g.rows == order.tokens && g.cols == a.cols, "combine_rows: the gradient must have the output's shape");
  const int type = weights_type("combine_rows", weights, places);
  const c10::cuda::CUDAGuard guard(y.device());
  const Tensor w = weights.contiguous();
  Tensor d_y, d_weights;
  if (want_y) d_y = at::empty({order.rows, a.cols}, at::TensorOptions().dtype(y.scalar_type()).device(y.device()));
  if (want_weights) d_weights = at::empty(places.sizes(), at::TensorOptions().dtype(at::kFloat).device(y.device()));
  if (order.rows == 0 || (!want_y && !want_weights)) return {d_y, d_weights};
  std::string err;
  TORCH_CHECK(experts_combine_backward_sm100(dtype, int(order.tokens), int(order.choices), a.cols, current_stream(), g.data, g.bytes, g.ld,
                                             a.data, a.bytes, a.ld, w.data_ptr(), w.nbytes(), type, source.data_ptr(), source.nbytes(),
                                             order.count, want_y ? d_y.data_ptr() : nullptr, want_y ? d_y.nbytes() : 0, a.cols,
                                             want_weights ? d_weights.data_ptr() : nullptr, want_weights ? d_weights.nbytes() : 0, &err) == 0,
              err);
  return {d_y, d_weights};
}

// While a graph is captured: a leaf whose node for its gradient was made on another stream, and lives because an eager graph of the leaf does, makes
// the backward pass wait for that stream, which ends the capture with an error that is not one to go on after.  Refused while it can be.
void check_captured_leaf(const Tensor& x) {
  if (!x.is_cuda() || !x.requires_grad() || !x.is_leaf()) return;
  const c10::cuda::CUDAGuard guard(x.device());
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(x);
  const c10::Stream now = c10::cuda::getCurrentCUDAStream();
  TORCH_CHECK(!node || !node->stream().has_value() || *node->stream() == now,
              "An eager graph of a tensor that requires a gradient lives on another stream than the one that is captured: delete it (its outputs) first, or "
              "make it on this stream");
}

// The same of a leaf that stands behind other operators, or of an input that was computed before the capture: asked in the backward pass, when it is known which
// nodes it will come to.  Those of the legacy default stream are the ones that nothing captured can be waited for on.
void check_captured_backward(const Tensor& d) {
  if (!d.is_cuda()) return;
  const c10::cuda::CUDAGuard guard(d.device());
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  const auto* wanted = torch::autograd::get_current_graph_task_exec_info();  // empty: all of them
  const auto here = torch::autograd::get_current_node();
  if (!here) return;
  std::vector<torch::autograd::Node*> left{here.get()};
  std::unordered_set<torch::autograd::Node*> seen{here.get()};
  while (!left.empty()) {
    torch::autograd::Node* node = left.back();
    left.pop_back();
    for (const auto& edge : node->next_edges()) {
      torch::autograd::Node* next = edge.function.get();
      if (!next || !seen.insert(next).second) continue;
      if (wanted && !wanted->empty()) {
        const auto it = wanted->find(next);
        if (it == wanted->end() || !it->second.should_execute()) continue;
      }
      const auto stream = next->stream();
      TORCH_CHECK(!stream || stream->device_type() != c10::DeviceType::CUDA || c10::cuda::CUDAStream(c10::cuda::CUDAStream::UNCHECKED, *stream).stream() != nullptr,
                  "A backward pass that is captured comes to a node of the default stream (", next->name(),
                  "), which lives on another stream than the one that is captured: compute the input inside the capture, and delete eager graphs of the same leaves (their "
                  "outputs) first, or make them on this stream");
      left.push_back(next);
    }
  }
}

// ---- their backward passes ----
// Gradients that have none of their own: the error is the one of a second differentiation, not of the first with a graph.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list defined;
  for (const Tensor& g : grads)
    if (g.defined()) defined.push_back(g.detach().set_requires_grad(true));
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      "gather_rows and combine_rows cannot be differentiated twice", int64_t(defined.size()));
  const variable_list out = (*error)(std::move(defined));
  size_t i = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = out[i++];
  return grads;
}

struct GatherRows : torch::autograd::Function<GatherRows> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& source, const Tensor& places, const Tensor& offsets) {
    ctx->save_for_backward({source, places, offsets});
    ctx->saved_data["shape"] = x.sizes().vec();
    return gather(x, source, places, offsets);
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    check_captured_backward(d[0]);
    const auto saved = ctx->get_saved_variables();
    variable_list grads(4);
    {
      const at::AutoGradMode off(false);
      grads[0] = combine(d[0], saved[0], saved[1], saved[2], nullptr).view(ctx->saved_data["shape"].toIntVector());
    }
    return once(std::move(grads));
  }
};

struct CombineRows : torch::autograd::Function<CombineRows> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& weights, const Tensor& source, const Tensor& places,
                        const Tensor& offsets) {
    ctx->save_for_backward({y, weights, source, places, offsets});
    return combine(y, source, places, offsets, &weights);
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    check_captured_backward(d[0]);
    const auto saved = ctx->get_saved_variables();
    variable_list grads(5);
    {
      const at::AutoGradMode off(false);
      std::tie(grads[0], grads[1]) = combine_backward(d[0], saved[0], saved[2], saved[3], saved[4], saved[1], ctx->needs_input_grad(0),
                                                      ctx->needs_input_grad(1));
      if (grads[1].defined()) grads[1] = grads[1].to(saved[1].scalar_type());
    }
    return once(std::move(grads));
  }
};

Tensor gather_with_backward(const Tensor& x, const Tensor& source, const Tensor& places, const Tensor& offsets) {
  if (!x.requires_grad() || !at::GradMode::is_enabled()) return gather(x, source, places, offsets);
  no_tangent(x, "experts'");
  check_captured_leaf(x);
  return GatherRows::apply(x, source, places, offsets);
}
Tensor combine_with_backward(const Tensor& y, const Tensor& source, const Tensor& places, const Tensor& offsets, const Tensor& weights) {
  if (!(y.requires_grad() || weights.requires_grad()) || !at::GradMode::is_enabled()) return combine(y, source, places, offsets, &weights);
  for (const Tensor* t : {&y, &weights}) {
    no_tangent(*t, "experts'");
    check_captured_leaf(*t);
  }
  return CombineRows::apply(y, weights, source, places, offsets);
}

// ---- the calls' arguments, by position ----
// Fp8Rows, Fp8Weight and ExpertOrder, named tuples of the Python modules: made here, since their own constructors are Python functions.
PyTypeObject* g_types[3] = {};

PyObject* wrap(int type, std::initializer_list<const Tensor*> tensors) {
  PyObject* plain = PyTuple_New(Py_ssize_t(tensors.size()));
  if (!plain) throw python_error();
  Py_ssize_t i = 0;
  for (const Tensor* t : tensors) PyTuple_SET_ITEM(plain, i++, THPVariable_Wrap(*t));
  if (!g_types[type]) return plain;
  PyObject* args = PyTuple_Pack(1, plain);
  Py_DECREF(plain);
  if (!args) throw python_error();
  PyObject* named = PyTuple_Type.tp_new(g_types[type], args, nullptr);
  Py_DECREF(args);
  if (!named) throw python_error();
  return named;
}
int64_t whole(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

PyObject* py_types(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count_args(nargs, 2, "fp8_types(index, cls)");
  const int64_t i = whole(args[0]);
  TORCH_CHECK_TYPE(i >= 0 && i < 3 && PyType_Check(args[1]) && PyType_IsSubtype(reinterpret_cast<PyTypeObject*>(args[1]), &PyTuple_Type),
                   "fp8_types: 0 to 2 and a subclass of tuple are wanted");
  Py_INCREF(args[1]);
  g_types[i] = reinterpret_cast<PyTypeObject*>(args[1]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* py_quantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count_args(nargs, 4, "fp8_quantize(x, source, places, offsets)");
  constexpr const char* call = "quantize_fp8";
  const Fp8Out o = quantize(tensor(args[0], call), tensor_or_none(args[1], call), args[1] == Py_None ? nullptr : &tensor(args[2], call),
                            args[1] == Py_None ? nullptr : &tensor(args[3], call));
  return wrap(0, {&o.values, &o.scales});
  END_HANDLE_TH_ERRORS
}

PyObject* py_quantize_weight(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count_args(nargs, 1, "fp8_quantize_weight(w)");
  const Fp8Out o = quantize_weight(tensor(args[0], "quantize_fp8_weight"));
  return wrap(1, {&o.values, &o.scales});
  END_HANDLE_TH_ERRORS
}

PyObject* py_silu_mul(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count_args(nargs, 2, "silu_mul_fp8(gate, up)");
  const Fp8Out o = silu_mul(tensor(args[0], "silu_mul_fp8"), tensor(args[1], "silu_mul_fp8"));
  return wrap(0, {&o.values, &o.scales});
  END_HANDLE_TH_ERRORS
}

PyObject* py_dequantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count_args(nargs, 4, "fp8_dequantize(values, scales, dtype, weight)");
  constexpr const char* call = "fp8_dequantize";
  return THPVariable_Wrap(dequantize(tensor(args[0], call), tensor(args[1], call), dtype_of(args[2], call), args[3] == Py_True));
  END_HANDLE_TH_ERRORS
}

PyObject* py_linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count_args(nargs, 8, "fp8_linear(x, x_scales, weight, weight_scales, bias, dtype, flags, out)");
  constexpr const char* call = "fp8_linear";
  return THPVariable_Wrap(linear(tensor(args[0], call), tensor(args[1], call), tensor(args[2], call), tensor(args[3], call),
                                 tensor_or_none(args[4], call), dtype_of(args[5], call), whole(args[6]), tensor_or_none(args[7], call)));
  END_HANDLE_TH_ERRORS
}

PyObject* py_expert_linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count_args(nargs, 8, "fp8_expert_linear(x, x_scales, weight, weight_scales, offsets, dtype, flags, out)");
  constexpr const char* call = "fp8_expert_linear";
  return THPVariable_Wrap(expert_linear(tensor(args[0], call), tensor(args[1], call), tensor(args[2], call), tensor(args[3], call),
                                        tensor(args[4], call), dtype_of(args[5], call), whole(args[6]), tensor_or_none(args[7], call)));
  END_HANDLE_TH_ERRORS
}

PyObject* py_sort(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count_args(nargs, 2, "experts_sort(experts, n_experts)");
  const Order o = sort_choices(tensor(args[0], "sort_by_expert"), whole(args[1]));
  return wrap(2, {&o.source, &o.places, &o.offsets});
  END_HANDLE_TH_ERRORS
}

PyObject* py_gather(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count_args(nargs, 4, "experts_gather(x, source, places, offsets)");
  constexpr const char* call = "gather_rows";
  return THPVariable_Wrap(gather_with_backward(tensor(args[0], call), tensor(args[1], call), tensor(args[2], call), tensor(args[3], call)));
  END_HANDLE_TH_ERRORS
}

PyObject* py_combine(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count_args(nargs, 5, "experts_combine(y, source, places, offsets, weights)");
  constexpr const char* call = "combine_rows";
  return THPVariable_Wrap(combine_with_backward(tensor(args[0], call), tensor(args[1], call), tensor(args[2], call), tensor(args[3], call),
                                                tensor(args[4], call)));
  END_HANDLE_TH_ERRORS
}

PyMethodDef g_methods[] = {
    {"fp8_types", fast<py_types>(), METH_FASTCALL, "The tuple's subclasses that rows, weights and orders are returned as"},
    {"fp8_quantize", fast<py_quantize>(), METH_FASTCALL, "The rows of x in e4m3, in the order of their experts where one is given"},
    {"fp8_quantize_weight", fast<py_quantize_weight>(), METH_FASTCALL, "Weights in e4m3, a scale for each 128 x 128"},
    {"silu_mul_fp8", fast<py_silu_mul>(), METH_FASTCALL, "The rows of silu(gate) * up"},
    {"fp8_dequantize", fast<py_dequantize>(), METH_FASTCALL, "scales * values"},
    {"fp8_linear", fast<py_linear>(), METH_FASTCALL, "The product of e4m3 rows with an e4m3 weight"},
    {"fp8_expert_linear", fast<py_expert_linear>(), METH_FASTCALL, "The product of every expert's rows with its weight"},
    {"experts_sort", fast<py_sort>(), METH_FASTCALL, "The order of the choices by expert"},
    {"experts_gather", fast<py_gather>(), METH_FASTCALL, "Tokens in the order of their experts"},
    {"experts_combine", fast<py_combine>(), METH_FASTCALL, "The weighted sum of each token's rows"},
    {nullptr, nullptr, 0, nullptr}};

}  // namespace

bool add_fp8_functions(PyObject* module) { return PyModule_AddFunctions(module, g_methods) == 0; }
