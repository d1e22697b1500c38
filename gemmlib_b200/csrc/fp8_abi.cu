// extern "C" entry points of the 8-bit floating-point path and of layers of experts: argument validation and dispatch.
#include <cstddef>
#include <cstdint>
#include <string>

#include "abi_checks.cuh"
#include "fp8.cuh"
#include "ms_blkq4gemm.h"

namespace {

using namespace blkq4::abi;
using blkq4::fp8::blocks_of;
using blkq4::int8::Dtype;

constexpr int kMaxRows = 1 << 28;

// The pitch of a matrix, where one of a single row may be anything.
int64_t pitch_of(int64_t ld, int rows, int cols) { return rows > 1 ? ld : cols; }

std::string check_rows(const char* name, int64_t rows) {
  return rows > kMaxRows ? std::string("Too many ") + name + ": " + std::to_string(rows) : std::string();
}
std::string check_experts(int experts) {
  if (experts <= 0) return "Empty problem size: " + std::to_string(experts) + " experts";
  if (experts > blkq4::fp8::kMaxExperts)
    return "Up to " + std::to_string(blkq4::fp8::kMaxExperts) + " experts are taken, not " + std::to_string(experts);
  return std::string();
}
std::string check_choices(int dtype, int tokens, int choices, int cols) {
  std::string e = check_shape(dtype, tokens, cols);
  if (e.empty() && choices <= 0) e = "Empty problem size: " + std::to_string(choices) + " choices";
  if (e.empty()) e = check_rows("choices", (int64_t)tokens * choices);
  return e;
}
bool on_16(const void* ptr, int64_t ld, int rows) { return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && (rows <= 1 || ld % 16 == 0); }

std::string check_count(const void* count) {
  if (!count) return "Null tensor pointer: count";
  return reinterpret_cast<uintptr_t>(count) % 4 != 0 ? "Misaligned tensor: count" : std::string();
}
std::string check_weights(const void* weights, size_t size, int type, int64_t n) {
  if (type != INT8_FP16 && type != INT8_BF16 && type != EXPERTS_FP32) return "Unsupported type of weights: " + std::to_string(type);
  return check_matrix("weights", weights, size, n, 1, (int)n, type == EXPERTS_FP32 ? 4 : 2);
}

}  // namespace

extern "C" int fp8_rows_quant_sm100(int dtype, int rows, int cols, void* stream, void const* x, size_t x_size, int64_t ldx, void* values,
                                    size_t values_size, int64_t ldv, void* scales, size_t scales_size, int64_t lds, void* err) {
  return guarded(
      err,
      [&] {
        std::string e = check_shape(dtype, rows, cols);
        if (e.empty()) e = check_rows("rows", rows);
        return !e.empty() ? e
                          : check_all({{"x", x, x_size, ldx, rows, cols, 2},
                                       {"values", values, values_size, ldv, rows, cols, 1},
                                       {"scales", scales, scales_size, lds, rows, blocks_of(cols), 4}});
      },
      [&] {
        blkq4::fp8::RowsParams p{};
        p.a = x;
        p.lda = pitch_of(ldx, rows, cols);
        p.q = reinterpret_cast<uint8_t*>(values);
        p.ldq = pitch_of(ldv, rows, cols);
        p.scales = reinterpret_cast<float*>(scales);
        p.lds = pitch_of(lds, rows, blocks_of(cols));
        p.rows = rows;
        p.cols = cols;
        return blkq4::fp8::launch_rows(blkq4::fp8::kQuant, Dtype(dtype), p, reinterpret_cast<cudaStream_t>(stream));
      });
}

extern "C" int fp8_rows_gather_quant_sm100(int dtype, int tokens, int choices, int cols, void* stream, void const* x, size_t x_size,
                                           int64_t ldx, void const* places, size_t places_size, void const* count, void* values,
                                           size_t values_size, int64_t ldv, void* scales, size_t scales_size, int64_t lds, void* err) {
  const int rows = tokens > 0 && choices > 0 && (int64_t)tokens * choices <= kMaxRows ? tokens * choices : 0;
  return guarded(
      err,
      [&] {
        std::string e = check_choices(dtype, tokens, choices, cols);
        if (e.empty())
          e = check_all({{"x", x, x_size, ldx, tokens, cols, 2},
                         {"places", places, places_size, rows, 1, rows, 4},
                         {"values", values, values_size, ldv, rows, cols, 1},
                         {"scales", scales, scales_size, lds, rows, blocks_of(cols), 4}});
        return e.empty() ? check_count(count) : e;
      },
      [&] {
        blkq4::fp8::RowsParams p{};
        p.a = x;
        p.lda = pitch_of(ldx, tokens, cols);
        p.choices = choices;
        p.places = reinterpret_cast<const int*>(places);
        p.count = reinterpret_cast<const int*>(count);
        p.q = reinterpret_cast<uint8_t*>(values);
        p.ldq = pitch_of(ldv, rows, cols);
        p.scales = reinterpret_cast<float*>(scales);
        p.lds = pitch_of(lds, rows, blocks_of(cols));
        p.rows = tokens;
        p.cols = cols;
        return blkq4::fp8::launch_rows(blkq4::fp8::kQuant, Dtype(dtype), p, reinterpret_cast<cudaStream_t>(stream));
      });
}

extern "C" int fp8_rows_silu_mul_sm100(int dtype, int rows, int cols, void* stream, void const* gate, size_t gate_size, int64_t ldg,
                                       void const* up, size_t up_size, int64_t ldu, void* values, size_t values_size, int64_t ldv,
                                       void* scales, size_t scales_size, int64_t lds, void* err) {
  return guarded(
      err,
      [&] {
        std::string e = check_shape(dtype, rows, cols);
        if (e.empty()) e = check_rows("rows", rows);
        return !e.empty() ? e
                          : check_all({{"gate", gate, gate_size, ldg, rows, cols, 2},
                                       {"up", up, up_size, ldu, rows, cols, 2},
                                       {"values", values, values_size, ldv, rows, cols, 1},
                                       {"scales", scales, scales_size, lds, rows, blocks_of(cols), 4}});
      },
      [&] {
        blkq4::fp8::RowsParams p{};
        p.a = gate;
        p.lda = pitch_of(ldg, rows, cols);
        p.b = up;
        p.ldb = pitch_of(ldu, rows, cols);
        p.q = reinterpret_cast<uint8_t*>(values);
        p.ldq = pitch_of(ldv, rows, cols);
        p.scales = reinterpret_cast<float*>(scales);
        p.lds = pitch_of(lds, rows, blocks_of(cols));
        p.rows = rows;
        p.cols = cols;
        return blkq4::fp8::launch_rows(blkq4::fp8::kSiluMul, Dtype(dtype), p, reinterpret_cast<cudaStream_t>(stream));
      });
}

namespace {

std::string check_stack(int dtype, int experts, int n, int k) {
  std::string e = check_shape(dtype, n, k);
  if (e.empty() && experts <= 0) e = "Empty problem size: " + std::to_string(experts) + " experts";
  if (e.empty()) e = check_rows("weight rows", (int64_t)experts * n);
  return e;
}

}  // namespace

extern "C" int fp8_weight_quant_sm100(int dtype, int experts, int n, int k, void* stream, void const* w, size_t w_size, int64_t ldw,
                                      void* values, size_t values_size, int64_t ldv, void* scales, size_t scales_size, int64_t lds,
                                      void* err) {
  return guarded(
      err,
      [&] {
        std::string e = check_stack(dtype, experts, n, k);
        return !e.empty() ? e
                          : check_all({{"w", w, w_size, ldw, experts * n, k, 2},
                                       {"values", values, values_size, ldv, experts * n, k, 1},
                                       {"scales", scales, scales_size, lds, experts * blocks_of(n), blocks_of(k), 4}});
      },
      [&] {
        blkq4::fp8::RowsParams p{};
        p.a = w;
        p.lda = pitch_of(ldw, experts * n, k);
        p.q = reinterpret_cast<uint8_t*>(values);
        p.ldq = pitch_of(ldv, experts * n, k);
        p.scales = reinterpret_cast<float*>(scales);
        p.lds = pitch_of(lds, experts * blocks_of(n), blocks_of(k));
        p.rows = experts * n;
        p.cols = k;
        p.expert_rows = n;
        return blkq4::fp8::launch_weights(Dtype(dtype), p, reinterpret_cast<cudaStream_t>(stream));
      });
}

extern "C" int fp8_rows_dequant_sm100(int dtype, int rows, int cols, void* stream, void const* values, size_t values_size, int64_t ldv,
                                      void const* scales, size_t scales_size, int64_t lds, void* out, size_t out_size, int64_t ldo,
                                      void* err) {
  return guarded(
      err,
      [&] {
        std::string e = check_shape(dtype, rows, cols);
        if (e.empty()) e = check_rows("rows", rows);
        return !e.empty() ? e
                          : check_all({{"values", values, values_size, ldv, rows, cols, 1},
                                       {"scales", scales, scales_size, lds, rows, blocks_of(cols), 4},
                                       {"out", out, out_size, ldo, rows, cols, 2}});
      },
      [&] {
        blkq4::fp8::DequantParams p{};
        p.q = reinterpret_cast<const uint8_t*>(values);
        p.ldq = pitch_of(ldv, rows, cols);
        p.scales = reinterpret_cast<const float*>(scales);
        p.lds = pitch_of(lds, rows, blocks_of(cols));
        p.out = out;
        p.ldo = pitch_of(ldo, rows, cols);
        p.rows = rows;
        p.cols = cols;
        return blkq4::fp8::launch_dequant(Dtype(dtype), p, reinterpret_cast<cudaStream_t>(stream));
      });
}

extern "C" int fp8_weight_dequant_sm100(int dtype, int experts, int n, int k, void* stream, void const* values, size_t values_size,
                                        int64_t ldv, void const* scales, size_t scales_size, int64_t lds, void* out, size_t out_size,
                                        int64_t ldo, void* err) {
  return guarded(
      err,
      [&] {
        std::string e = check_stack(dtype, experts, n, k);
        return !e.empty() ? e
                          : check_all({{"values", values, values_size, ldv, experts * n, k, 1},
                                       {"scales", scales, scales_size, lds, experts * blocks_of(n), blocks_of(k), 4},
                                       {"out", out, out_size, ldo, experts * n, k, 2}});
      },
      [&] {
        blkq4::fp8::DequantParams p{};
        p.q = reinterpret_cast<const uint8_t*>(values);
        p.ldq = pitch_of(ldv, experts * n, k);
        p.scales = reinterpret_cast<const float*>(scales);
        p.lds = pitch_of(lds, experts * blocks_of(n), blocks_of(k));
        p.out = out;
        p.ldo = pitch_of(ldo, experts * n, k);
        p.rows = experts * n;
        p.cols = k;
        p.expert_rows = n;
        return blkq4::fp8::launch_dequant(Dtype(dtype), p, reinterpret_cast<cudaStream_t>(stream));
      });
}

extern "C" int fp8_gemm_sm100(int dtype, int m, int n, int k, void* stream, void const* x, size_t x_size, int64_t ldx, void const* x_scales,
                              size_t x_scales_size, int64_t ldxs, void const* w, size_t w_size, int64_t ldw, void const* w_scales,
                              size_t w_scales_size, int64_t ldws, void const* bias, size_t bias_size, void* out, size_t out_size,
                              int64_t ldo, unsigned flags, void* err) {
  return guarded(
      err,
      [&] {
        std::string e = check_shape(dtype, m, n);
        if (e.empty()) e = check_shape(dtype, m, k);
        if (e.empty()) e = check_rows("rows", m);
        if (e.empty())
          e = check_all({{"x", x, x_size, ldx, m, k, 1},
                         {"x_scales", x_scales, x_scales_size, ldxs, m, blocks_of(k), 4},
                         {"w", w, w_size, ldw, n, k, 1},
                         {"w_scales", w_scales, w_scales_size, ldws, blocks_of(n), blocks_of(k), 4},
                         {"out", out, out_size, ldo, m, n, 2}});
        if (e.empty() && bias) e = check_all({{"bias", bias, bias_size, n, 1, n, 2}});
        if (e.empty() && !(on_16(x, ldx, m) && on_16(w, ldw, n))) e = "Misaligned operand: rows of x and w must begin on 16 bytes";
        return e;
      },
      [&] {
        blkq4::fp8::GemmArgs g{};
        g.M = m; g.N = n; g.K = k;
        g.x = reinterpret_cast<const uint8_t*>(x);
        g.ldx = row_pitch(ldx, m, k);
        g.x_scales = reinterpret_cast<const float*>(x_scales);
        g.ldxs = pitch_of(ldxs, m, blocks_of(k));
        g.w = reinterpret_cast<const uint8_t*>(w);
        g.ldw = row_pitch(ldw, n, k);
        g.w_stride = g.ldw * n;
        g.w_scales = reinterpret_cast<const float*>(w_scales);
        g.ldws = pitch_of(ldws, blocks_of(n), blocks_of(k));
        g.bias = bias;
        g.out = out;
        g.ldo = pitch_of(ldo, m, n);
        g.experts = 1;
        return blkq4::fp8::launch_gemm(Dtype(dtype), g, flags, reinterpret_cast<cudaStream_t>(stream));
      });
}

extern "C" int fp8_experts_gemm_sm100(int dtype, int experts, int rows, int n, int k, void* stream, void const* x, size_t x_size,
                                      int64_t ldx, void const* x_scales, size_t x_scales_size, int64_t ldxs, void const* w, size_t w_size,
                                      int64_t ldw, int64_t w_stride, void const* w_scales, size_t w_scales_size, int64_t ldws,
                                      int64_t ws_stride, void const* offsets, size_t offsets_size, void* out, size_t out_size, int64_t ldo,
                                      unsigned flags, void* err) {
  return guarded(
      err,
      [&] {
        std::string e = check_shape(dtype, rows, n);
        if (e.empty()) e = check_shape(dtype, rows, k);
        if (e.empty()) e = check_rows("rows", rows);
        if (e.empty()) e = check_experts(experts);
        if (e.empty())
          e = check_all({{"x", x, x_size, ldx, rows, k, 1},
                         {"x_scales", x_scales, x_scales_size, ldxs, rows, blocks_of(k), 4},
                         {"w", w, w_size, ldw, n, k, 1},
                         {"w_scales", w_scales, w_scales_size, ldws, blocks_of(n), blocks_of(k), 4},
                         {"offsets", offsets, offsets_size, experts + 1, 1, experts + 1, 4},
                         {"out", out, out_size, ldo, rows, n, 2}});
        // all experts: those but the last one begin a stride apart
        auto stacked = [&](const char* name, size_t size, int64_t ld, int64_t stride, int r, int c, int elt) {
          if (!e.empty() || experts == 1) return;
          const int64_t one = (r > 1 ? (int64_t)(r - 1) * ld : 0) + c;
          if (stride < one || stride > INT64_MAX / 4 / elt / experts) {
            e = std::string("Stride of ") + name + " is smaller than an expert, or out of range: " + std::to_string(stride);
          } else if (size < ((uint64_t)(experts - 1) * (uint64_t)stride + (uint64_t)one) * (uint64_t)elt) {
            e = std::string("Unexpected size of ") + name + ": " + std::to_string(size) + " expected: " +
                std::to_string(((uint64_t)(experts - 1) * (uint64_t)stride + (uint64_t)one) * (uint64_t)elt);
          }
        };
        stacked("w", w_size, ldw, w_stride, n, k, 1);
        stacked("w_scales", w_scales_size, ldws, ws_stride, blocks_of(n), blocks_of(k), 4);
        if (e.empty() && !(on_16(x, ldx, rows) && on_16(w, ldw, n) && on_16(w, w_stride, experts)))
          e = "Misaligned operand: rows of x and w must begin on 16 bytes";
        return e;
      },
      [&] {
        blkq4::fp8::GemmArgs g{};
        g.M = rows; g.N = n; g.K = k;
        g.x = reinterpret_cast<const uint8_t*>(x);
        g.ldx = row_pitch(ldx, rows, k);
        g.x_scales = reinterpret_cast<const float*>(x_scales);
        g.ldxs = pitch_of(ldxs, rows, blocks_of(k));
        g.w = reinterpret_cast<const uint8_t*>(w);
        g.ldw = row_pitch(ldw, n, k);
        g.w_stride = experts > 1 ? w_stride : g.ldw * n;
        g.w_scales = reinterpret_cast<const float*>(w_scales);
        g.ldws = pitch_of(ldws, blocks_of(n), blocks_of(k));
        g.ws_stride = experts > 1 ? ws_stride : 0;
        g.out = out;
        g.ldo = pitch_of(ldo, rows, n);
        g.experts = experts;
        g.offsets = reinterpret_cast<const int*>(offsets);
        g.zero_rest = (flags & FP8_EXPERTS_ZERO_REST) != 0;
        return blkq4::fp8::launch_gemm(Dtype(dtype), g, flags, reinterpret_cast<cudaStream_t>(stream));
      });
}

extern "C" size_t experts_sort_workspace_size(int64_t n, int n_experts) {
  if (n <= 0 || n > kMaxRows || n_experts <= 0 || n_experts > blkq4::experts::kMaxExperts) return 0;
  return blkq4::experts::sort_workspace(n, n_experts);
}

extern "C" int experts_sort_sm100(int64_t n, int n_experts, int id_bytes, void* stream, void const* ids, size_t ids_size, void* source,
                                  size_t source_size, void* places, size_t places_size, void* offsets, size_t offsets_size,
                                  void* workspace, size_t workspace_size, void* err) {
  return guarded(
      err,
      [&] {
        std::string e = check_experts(n_experts);
        if (e.empty() && n <= 0) e = "Empty problem size: " + std::to_string(n) + " choices";
        if (e.empty()) e = check_rows("choices", n);
        if (e.empty() && id_bytes != 4 && id_bytes != 8) e = "Unsupported type of ids: " + std::to_string(id_bytes) + " bytes";
        if (e.empty())
          e = check_all({{"ids", ids, ids_size, n, 1, (int)n, id_bytes},
                         {"source", source, source_size, n, 1, (int)n, 4},
                         {"places", places, places_size, n, 1, (int)n, 4},
                         {"offsets", offsets, offsets_size, n_experts + 1, 1, n_experts + 1, 4}});
        const size_t need = e.empty() ? blkq4::experts::sort_workspace(n, n_experts) : 0;
        if (need > 0) e = check_all({{"workspace", workspace, workspace_size, (int64_t)(need / 4), 1, (int)(need / 4), 4}});
        return e;
      },
      [&] {
        return blkq4::experts::launch_sort(ids, id_bytes == 8, n, n_experts, reinterpret_cast<int*>(source), reinterpret_cast<int*>(places),
                                           reinterpret_cast<int*>(offsets), workspace, reinterpret_cast<cudaStream_t>(stream));
      });
}

extern "C" int experts_gather_sm100(int dtype, int tokens, int choices, int cols, void* stream, void const* x, size_t x_size, int64_t ldx,
                                    void const* source, size_t source_size, void const* count, void* out, size_t out_size, int64_t ldo,
                                    void* err) {
  const int rows = tokens > 0 && choices > 0 && (int64_t)tokens * choices <= kMaxRows ? tokens * choices : 0;
  return guarded(
      err,
      [&] {
        std::string e = check_choices(dtype, tokens, choices, cols);
        if (e.empty())
          e = check_all({{"x", x, x_size, ldx, tokens, cols, 2},
                         {"source", source, source_size, rows, 1, rows, 4},
                         {"out", out, out_size, ldo, rows, cols, 2}});
        return e.empty() ? check_count(count) : e;
      },
      [&] {
        blkq4::experts::MoveParams p{};
        p.from = x;
        p.ldf = pitch_of(ldx, tokens, cols);
        p.source = reinterpret_cast<const int*>(source);
        p.count = reinterpret_cast<const int*>(count);
        p.to = out;
        p.ldt = pitch_of(ldo, rows, cols);
        p.tokens = tokens;
        p.choices = choices;
        p.cols = cols;
        return blkq4::experts::launch_gather(Dtype(dtype), p, reinterpret_cast<cudaStream_t>(stream));
      });
}

extern "C" int experts_combine_sm100(int dtype, int tokens, int choices, int cols, void* stream, void const* y, size_t y_size, int64_t ldy,
                                     void const* places, size_t places_size, void const* weights, size_t weights_size, int weights_type,
                                     void* out, size_t out_size, int64_t ldo, void* err) {
  const int rows = tokens > 0 && choices > 0 && (int64_t)tokens * choices <= kMaxRows ? tokens * choices : 0;
  return guarded(
      err,
      [&] {
        std::string e = check_choices(dtype, tokens, choices, cols);
        if (e.empty())
          e = check_all({{"y", y, y_size, ldy, rows, cols, 2},
                         {"places", places, places_size, rows, 1, rows, 4},
                         {"out", out, out_size, ldo, tokens, cols, 2}});
        return e.empty() && weights ? check_weights(weights, weights_size, weights_type, rows) : e;
      },
      [&] {
        blkq4::experts::MoveParams p{};
        p.from = y;
        p.ldf = pitch_of(ldy, rows, cols);
        p.weights = weights;
        p.weights_type = weights_type;
        p.places = reinterpret_cast<const int*>(places);
        p.to = out;
        p.ldt = pitch_of(ldo, tokens, cols);
        p.tokens = tokens;
        p.choices = choices;
        p.cols = cols;
        return blkq4::experts::launch_combine(Dtype(dtype), p, reinterpret_cast<cudaStream_t>(stream));
      });
}

extern "C" int experts_combine_backward_sm100(int dtype, int tokens, int choices, int cols, void* stream, void const* d, size_t d_size,
                                              int64_t ldd, void const* y, size_t y_size, int64_t ldy, void const* weights,
                                              size_t weights_size, int weights_type, void const* source, size_t source_size,
                                              void const* count, void* d_y, size_t d_y_size, int64_t lddy, void* d_weights,
                                              size_t d_weights_size, void* err) {
  const int rows = tokens > 0 && choices > 0 && (int64_t)tokens * choices <= kMaxRows ? tokens * choices : 0;
  return guarded(
      err,
      [&] {
        std::string e = check_choices(dtype, tokens, choices, cols);
        if (e.empty())
          e = check_all({{"d", d, d_size, ldd, tokens, cols, 2},
                         {"y", y, y_size, ldy, rows, cols, 2},
                         {"source", source, source_size, rows, 1, rows, 4}});
        if (e.empty() && d_y) e = check_all({{"d_y", d_y, d_y_size, lddy, rows, cols, 2}});
        if (e.empty() && (d_weights || !d_y)) e = check_all({{"d_weights", d_weights, d_weights_size, rows, 1, rows, 4}});
        if (e.empty()) e = check_weights(weights, weights_size, weights_type, rows);
        return e.empty() ? check_count(count) : e;
      },
      [&] {
        blkq4::experts::MoveParams p{};
        p.from = d;
        p.ldf = pitch_of(ldd, tokens, cols);
        p.y = y;
        p.ldy = pitch_of(ldy, rows, cols);
        p.weights = weights;
        p.weights_type = weights_type;
        p.source = reinterpret_cast<const int*>(source);
        p.count = reinterpret_cast<const int*>(count);
        p.to = d_y;
        p.ldt = pitch_of(lddy, rows, cols);
        p.dots = reinterpret_cast<float*>(d_weights);
        p.tokens = tokens;
        p.choices = choices;
        p.cols = cols;
        return blkq4::experts::launch_weigh(Dtype(dtype), p, reinterpret_cast<cudaStream_t>(stream));
      });
}
