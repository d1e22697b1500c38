// Shared definitions of the 8-bit floating-point path: e4m3 rows with an fp32 scale for each 128 elements, e4m3 weights with one for
// each 128 x 128, their product, and the operators of a layer of experts around it.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "int8.cuh"

namespace blkq4 {
namespace fp8 {

using int8::Dtype;

constexpr int kBlock = 128;   // elements that share a scale, along k and along n
constexpr int kMaxExperts = 1024;

struct RowsParams {
  const void* a;      // x, or gate
  const void* b;      // up
  const int* places;  // [rows, choices]: the rows of q that row r of x is written to; null: row r
  const int* count;   // with places: how many rows of q are written so, the others are set to zero
  int choices;
  uint8_t* q;
  float* scales;
  int64_t lda, ldb, ldq, lds;  // elements from row to row
  int rows, cols;
  // weights: rows of each expert
  int expert_rows;
};
enum RowsOp { kQuant = 0, kSiluMul = 1 };
std::string launch_rows(RowsOp op, Dtype dtype, const RowsParams& p, cudaStream_t stream);
std::string launch_weights(Dtype dtype, const RowsParams& p, cudaStream_t stream);
struct DequantParams {
  const uint8_t* q;
  const float* scales;
  void* out;
  int64_t ldq, lds, ldo;
  int rows, cols;
  int expert_rows;  // weights: rows of each expert; 0: rows
};
std::string launch_dequant(Dtype dtype, const DequantParams& p, cudaStream_t stream);

struct GemmArgs {
  int M, N, K;
  const uint8_t* x;
  int64_t ldx;  // bytes from row to row, a multiple of 16
  const float* x_scales;
  int64_t ldxs;
  const uint8_t* w;
  int64_t ldw, w_stride;  // bytes from row to row, from expert to expert
  const float* w_scales;
  int64_t ldws, ws_stride;
  const void* bias;  // [N] of the output's type, or null
  void* out;
  int64_t ldo;  // elements
  // a layer of experts: rows [offsets[e], offsets[e + 1]) are multiplied with weight e
  int experts;         // 1 without offsets
  const int* offsets;  // null: all rows are those of one weight
  bool zero_rest;      // rows of no expert are set to zero
};
// The kernel of one or two rows, and the problems it is for (without offsets).
bool gemv_takes(int M, int N, int K);
std::string launch_gemv(Dtype dtype, const GemmArgs& g, unsigned flags, cudaStream_t stream);
std::string launch_gemm(Dtype dtype, const GemmArgs& g, unsigned flags, cudaStream_t stream);
int read_gemm_error();
int clear_gemm_error(cudaStream_t stream);

inline int blocks_of(int n) { return (n + kBlock - 1) / kBlock; }

}  // namespace fp8

namespace experts {

using int8::Dtype;

constexpr int kMaxExperts = fp8::kMaxExperts;

std::string launch_sort(const void* ids, bool wide, int64_t n, int n_experts, int* source, int* places, int* offsets,
                        void* workspace, cudaStream_t stream);
// Bytes of the workspace: 0 where one CTA sorts all.
size_t sort_workspace(int64_t n, int n_experts);

struct MoveParams {
  const void* from;    // gather: x [tokens, cols]; combine: y [places, cols]; weigh: the gradient of combine's output [tokens, cols]
  const void* y;       // weigh: y
  const void* weights; // [tokens, choices] of `weights_type`, or null: ones
  int weights_type;    // Dtype, or 2: float32
  const int* source;
  const int* places;
  const int* count;    // rows that belong to an expert
  void* to;
  float* dots;         // weigh: the weights' gradient
  int64_t ldf, ldy, ldt;
  int tokens, choices, cols;
};
std::string launch_gather(Dtype dtype, const MoveParams& p, cudaStream_t stream);
std::string launch_combine(Dtype dtype, const MoveParams& p, cudaStream_t stream);
std::string launch_weigh(Dtype dtype, const MoveParams& p, cudaStream_t stream);

}  // namespace experts
}  // namespace blkq4
