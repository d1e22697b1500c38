// Shared definitions of the 8-bit path: int8 rows with one fp32 scale each, and their product.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

namespace blkq4 {
namespace int8 {

// 16-bit types of the activations and outputs (INT8_FP16, INT8_BF16 of the C ABI)
enum Dtype { kFp16 = 0, kBf16 = 1 };

// What produces the rows: see the C ABI.
enum RowsOp { kQuant = 0, kNorm = 1, kNormResidual = 2, kSiluMul = 3 };

struct RowsParams {
  const void* a;     // x, or gate
  const void* b;     // residual, or up
  const void* w;     // norm weight
  void* res_out;     // x + residual
  int8_t* q;
  float* scales;
  int64_t lda, ldb, ldr, ldq;  // elements from row to row
  int rows, cols;
  float eps;
  // set by the launcher
  bool q_vec;  // every row of q begins on 8 bytes
  int parts, part_chunks;  // CTAs a row, chunks of 8 elements of each
};
std::string launch_rows(RowsOp op, Dtype dtype, const RowsParams& p, cudaStream_t stream);
// Status word of the kernels' bounded waits: 0, or the first that gave up.
int read_rows_error();
int clear_rows_error(cudaStream_t stream);
std::string launch_dequant(Dtype dtype, int rows, int cols, const int8_t* q, int64_t ldq, const float* scales, void* out,
                           int64_t ldo, cudaStream_t stream);

struct GemmArgs {
  int M, N, K;
  const int8_t* x;
  int64_t ldx;  // bytes from row to row, a multiple of 16
  const float* x_scales;
  const int8_t* w;
  int64_t ldw;
  const float* w_scales;
  const void* bias;  // [N] of the output's type, or null
  void* out;
  int64_t ldo;  // elements
};
// The kernel of a few activation rows, and the problems it is for.
bool gemv_takes(int M, int N, int K);
std::string launch_gemv(Dtype dtype, const GemmArgs& g, unsigned flags, cudaStream_t stream);
std::string launch_gemm(Dtype dtype, const GemmArgs& g, unsigned flags, cudaStream_t stream);
int read_gemm_error();
int clear_gemm_error(cudaStream_t stream);

// Most k of a product: 2^31 - 1 over 128 * 128, so that int32 sums cannot wrap.
constexpr int kMaxK = 131071;

#ifdef __CUDACC__
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
// Two values rounded and packed, the first one in the low half.
template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack2(uint32_t v, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ float2 unpack2(uint32_t v, __nv_bfloat16) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
// Programmatic dependent launch: nothing that another kernel of the stream wrote is read, and nothing written, before
// griddep_wait, which returns once the kernels ahead in the stream have completed.  The next kernel is let in (griddep_launch_dependents)
// only after that: what it does ahead of its own wait - copies of weights, where the caller vouches for them - then
// comes behind everything that was ahead of this kernel, such as the quantization of those weights.
__device__ __forceinline__ void griddep_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void griddep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
#endif

}  // namespace int8
}  // namespace blkq4
