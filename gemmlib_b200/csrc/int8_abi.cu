// extern "C" entry points of the 8-bit path: argument validation and dispatch.
#include <cstddef>
#include <cstdint>
#include <string>

#include "abi_checks.cuh"
#include "int8.cuh"
#include "ms_blkq4gemm.h"

namespace {

using namespace blkq4::abi;
using namespace blkq4::int8;

}  // namespace

extern "C" int int8_rows_quant_sm100(int dtype, int rows, int cols, void* stream, void const* x, size_t x_size, int64_t ldx,
                                     void* values, size_t values_size, int64_t ldv, void* scales, size_t scales_size, void* err) {
  return guarded(
      err,
      [&] {
        std::string e = check_shape(dtype, rows, cols);
        return !e.empty() ? e
                          : check_all({{"x", x, x_size, ldx, rows, cols, 2},
                                       {"values", values, values_size, ldv, rows, cols, 1},
                                       {"scales", scales, scales_size, rows, 1, rows, 4}});
      },
      [&] {
        RowsParams p{};
        p.a = x;
        p.lda = row_pitch(ldx, rows, cols);
        p.q = reinterpret_cast<int8_t*>(values);
        p.ldq = row_pitch(ldv, rows, cols);
        p.scales = reinterpret_cast<float*>(scales);
        p.rows = rows;
        p.cols = cols;
        return launch_rows(kQuant, Dtype(dtype), p, reinterpret_cast<cudaStream_t>(stream));
      });
}

extern "C" int int8_rows_rms_norm_sm100(int dtype, int rows, int cols, void* stream, void const* x, size_t x_size, int64_t ldx,
                                        void const* residual, size_t residual_size, int64_t ldr, void const* weight,
                                        size_t weight_size, float eps, void* residual_out, size_t residual_out_size, int64_t ldo,
                                        void* values, size_t values_size, int64_t ldv, void* scales, size_t scales_size,
                                        void* err) {
  return guarded(
      err,
      [&] {
        std::string e = check_shape(dtype, rows, cols);
        if (e.empty())
          e = check_all({{"x", x, x_size, ldx, rows, cols, 2},
                         {"weight", weight, weight_size, cols, 1, cols, 2},
                         {"values", values, values_size, ldv, rows, cols, 1},
                         {"scales", scales, scales_size, rows, 1, rows, 4}});
        if (e.empty() && residual)
          e = check_all({{"residual", residual, residual_size, ldr, rows, cols, 2},
                         {"residual_out", residual_out, residual_out_size, ldo, rows, cols, 2}});
        if (e.empty() && !(eps >= 0.0f)) e = "eps must not be negative";
        if (e.empty() && residual && rows > 1 &&
            ((residual_out == x && ldo != ldx) || (residual_out == residual && ldo != ldr)))
          e = "residual_out in the place of x or residual must have its leading dimension";
        return e;
      },
      [&] {
        RowsParams p{};
        p.a = x;
        p.lda = row_pitch(ldx, rows, cols);
        p.b = residual;
        p.ldb = row_pitch(ldr, rows, cols);
        p.w = weight;
        p.res_out = residual_out;
        p.ldr = row_pitch(ldo, rows, cols);
        p.q = reinterpret_cast<int8_t*>(values);
        p.ldq = row_pitch(ldv, rows, cols);
        p.scales = reinterpret_cast<float*>(scales);
        p.rows = rows;
        p.cols = cols;
        p.eps = eps;
        return launch_rows(residual ? kNormResidual : kNorm, Dtype(dtype), p, reinterpret_cast<cudaStream_t>(stream));
      });
}

extern "C" int int8_rows_silu_mul_sm100(int dtype, int rows, int cols, void* stream, void const* gate, size_t gate_size,
                                        int64_t ldg, void const* up, size_t up_size, int64_t ldu, void* values,
                                        size_t values_size, int64_t ldv, void* scales, size_t scales_size, void* err) {
  return guarded(
      err,
      [&] {
        std::string e = check_shape(dtype, rows, cols);
        return !e.empty() ? e
                          : check_all({{"gate", gate, gate_size, ldg, rows, cols, 2},
                                       {"up", up, up_size, ldu, rows, cols, 2},
                                       {"values", values, values_size, ldv, rows, cols, 1},
                                       {"scales", scales, scales_size, rows, 1, rows, 4}});
      },
      [&] {
        RowsParams p{};
        p.a = gate;
        p.lda = row_pitch(ldg, rows, cols);
        p.b = up;
        p.ldb = row_pitch(ldu, rows, cols);
        p.q = reinterpret_cast<int8_t*>(values);
        p.ldq = row_pitch(ldv, rows, cols);
        p.scales = reinterpret_cast<float*>(scales);
        p.rows = rows;
        p.cols = cols;
        return launch_rows(kSiluMul, Dtype(dtype), p, reinterpret_cast<cudaStream_t>(stream));
      });
}

extern "C" int int8_rows_dequant_sm100(int dtype, int rows, int cols, void* stream, void const* values, size_t values_size,
                                       int64_t ldv, void const* scales, size_t scales_size, void* out, size_t out_size,
                                       int64_t ldo, void* err) {
  return guarded(
      err,
      [&] {
        std::string e = check_shape(dtype, rows, cols);
        return !e.empty() ? e
                          : check_all({{"values", values, values_size, ldv, rows, cols, 1},
                                       {"scales", scales, scales_size, rows, 1, rows, 4},
                                       {"out", out, out_size, ldo, rows, cols, 2}});
      },
      [&] {
        return launch_dequant(Dtype(dtype), rows, cols, reinterpret_cast<const int8_t*>(values), row_pitch(ldv, rows, cols),
                              reinterpret_cast<const float*>(scales), out, row_pitch(ldo, rows, cols),
                              reinterpret_cast<cudaStream_t>(stream));
      });
}

extern "C" int int8_gemm_sm100(int dtype, int m, int n, int k, void* stream, void const* x, size_t x_size, int64_t ldx,
                               void const* x_scales, size_t x_scales_size, void const* w, size_t w_size, int64_t ldw,
                               void const* w_scales, size_t w_scales_size, void const* bias, size_t bias_size, void* out,
                               size_t out_size, int64_t ldo, unsigned flags, void* err) {
  return guarded(
      err,
      [&] {
        std::string e = check_shape(dtype, m, n);
        if (e.empty() && k <= 0) e = "Empty problem size: " + std::to_string(m) + "x" + std::to_string(n) + "x" + std::to_string(k);
        if (e.empty() && k > kMaxK) e = "int32 sums hold up to " + std::to_string(kMaxK) + " k, not " + std::to_string(k);
        if (e.empty() && m > (1 << 28)) e = "Too many rows: " + std::to_string(m);
        if (e.empty())
          e = check_all({{"x", x, x_size, ldx, m, k, 1},
                         {"x_scales", x_scales, x_scales_size, m, 1, m, 4},
                         {"w", w, w_size, ldw, n, k, 1},
                         {"w_scales", w_scales, w_scales_size, n, 1, n, 4},
                         {"out", out, out_size, ldo, m, n, 2}});
        if (e.empty() && bias) e = check_all({{"bias", bias, bias_size, n, 1, n, 2}});
        if (e.empty() && (reinterpret_cast<uintptr_t>(x) % 16 != 0 || reinterpret_cast<uintptr_t>(w) % 16 != 0 ||
                          (m > 1 && ldx % 16 != 0) || (n > 1 && ldw % 16 != 0)))
          e = "Misaligned operand: rows of x and w must begin on 16 bytes";
        return e;
      },
      [&] {
        GemmArgs g{};
        g.M = m; g.N = n; g.K = k;
        g.x = reinterpret_cast<const int8_t*>(x);
        g.ldx = row_pitch(ldx, m, k);
        g.x_scales = reinterpret_cast<const float*>(x_scales);
        g.w = reinterpret_cast<const int8_t*>(w);
        g.ldw = row_pitch(ldw, n, k);
        g.w_scales = reinterpret_cast<const float*>(w_scales);
        g.bias = bias;
        g.out = out;
        g.ldo = m > 1 ? ldo : n;
        return launch_gemm(Dtype(dtype), g, flags, reinterpret_cast<cudaStream_t>(stream));
      });
}
