// Product of one or two e4m3 rows: weight rows streamed once through registers.
//
// Bound by the weights' bytes.  A warp takes R weight rows, 512 consecutive bytes of each per load: a lane's 16 lie within a block of
// 128, so its products, exact in fp32, are added up and the sum is scaled once.  e4m3 is exact in fp16, and the multiply-add of two fp16 numbers
// into fp32 takes them as they are converted: 24 instructions for 16 products.  No shared memory, no barrier: at a token's sizes a call is mostly
// latency.  The loads of the next piece are issued before the products of the present one.  One order of additions for a row, whatever
// the number of CTAs: the lane's pieces in turn, then the lanes by halves.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "blkq4_common.cuh"
#include "fp8.cuh"
#include "ms_blkq4gemm.h"

namespace blkq4 {
namespace fp8 {
namespace {

using namespace blkq4::int8;

constexpr int kWarps = 8;

struct GemvParams {
  int M, N, K, early;
  const uint8_t* x;
  int64_t ldx;
  const float* x_scales;
  int64_t ldxs;
  const uint8_t* w;
  int64_t ldw;
  const float* w_scales;
  int64_t ldws;
  const void* bias;
  void* out;
  int64_t ldo;
};

__device__ __forceinline__ uint4 load_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
// Sixteen e4m3 numbers as pairs of fp16.
__device__ __forceinline__ void to_halves(const uint4& v, uint32_t (&h)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[i]) : "h"((uint16_t)(w[i / 2] >> (i % 2 * 16))));
}
// c + a * b of both halves
__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c) {
  asm("{\n\t.reg .b16 a0, a1, b0, b1;\n\tmov.b32 {a0, a1}, %1;\n\tmov.b32 {b0, b1}, %2;\n\t"
      "fma.rn.f32.f16 %0, a0, b0, %0;\n\tfma.rn.f32.f16 %0, a1, b1, %0;\n\t}"
      : "+f"(c)
      : "r"(a), "r"(b));
  return c;
}

// MR >= M activation rows, R weight rows a warp, U pieces of 512 k of each in flight, CTAS resident on an SM: what is launched.
template <class T, int MR, int R, int U, int CTAS>
__global__ void __launch_bounds__(32 * kWarps, CTAS) fp8_gemv_kernel(const GemvParams p) {
  const int lane = threadIdx.x & 31;
  const int groups = (p.N + R - 1) / R;
  // one for each warp at most; neighbouring groups go to different CTAs, so that every SM has the same number of them (give or take one)
  const int g = (int)(threadIdx.x >> 5) * (int)gridDim.x + (int)blockIdx.x;
  const int whole = p.K & ~15;  // the last K % 16 k are taken one by one
  uint4 w[R][U];
  auto load = [&](int k0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint8_t* row = p.w + (int64_t)min(g * R + r, p.N - 1) * p.ldw;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * 512 + lane * 16;
        w[r][u] = k < whole ? load_stream(row + k) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  if (p.early) {
    if (g < groups) load(0);
  } else if (lane < R && whole > 0 && g < groups) {  // on their way into L2, where a write that is still to come would find them
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.w + (int64_t)min(g * R + lane, p.N - 1) * p.ldw), "r"(whole) : "memory");
  }
  griddep_wait();
  griddep_launch_dependents();
  if (!p.early && g < groups) load(0);

  if (g < groups) {
    float acc[R][MR] = {};
    const int n_l = g * R + lane % R, m_l = lane / R;
    const bool mine = lane < R * MR && n_l < p.N && m_l < p.M;
    const float bias = mine && p.bias ? to_float(reinterpret_cast<const T*>(p.bias)[n_l]) : 0.0f;
    const float* w_scales[R];
#pragma unroll
    for (int r = 0; r < R; ++r) w_scales[r] = p.w_scales + (int64_t)(min(g * R + r, p.N - 1) / kBlock) * p.ldws;
    for (int k0 = 0;;) {
      uint4 now[R][U];
      float ws[R][U], xs[MR][U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * 512 + lane * 16, b = k < whole ? k / kBlock : 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          now[r][u] = w[r][u];
          ws[r][u] = w_scales[r][b];
        }
#pragma unroll
        for (int m = 0; m < MR; ++m) xs[m][u] = p.x_scales[(int64_t)min(m, p.M - 1) * p.ldxs + b];
      }
      const int at = k0;
      k0 += 512 * U;
      const bool last = k0 >= whole;
      if (!last) load(k0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = at + u * 512 + lane * 16;
        if (k < whole) {
          uint32_t x[MR][8];
#pragma unroll
          for (int m = 0; m < MR; ++m) to_halves(*reinterpret_cast<const uint4*>(p.x + (int64_t)min(m, p.M - 1) * p.ldx + k), x[m]);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            uint32_t h[8];
            to_halves(now[r][u], h);
#pragma unroll
            for (int m = 0; m < MR; ++m) {
              float even = 0.0f, odd = 0.0f;
#pragma unroll
              for (int i = 0; i < 8; i += 2) even = dot2(h[i], x[m][i], even), odd = dot2(h[i + 1], x[m][i + 1], odd);
              acc[r][m] = fmaf(even + odd, xs[m][u] * ws[r][u], acc[r][m]);
            }
          }
        }
      }
      if (last) break;
    }
    if (whole + lane < p.K) {
      const int k = whole + lane;
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        const int64_t row = min(m, p.M - 1);
        const uint4 x4 = make_uint4(p.x[row * p.ldx + k], 0u, 0u, 0u);
        uint32_t x[8];
        to_halves(x4, x);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const uint4 w4 = make_uint4(p.w[(int64_t)min(g * R + r, p.N - 1) * p.ldw + k], 0u, 0u, 0u);
          uint32_t h[8];
          to_halves(w4, h);
          acc[r][m] = fmaf(dot2(h[0], x[0], 0.0f), p.x_scales[row * p.ldxs + k / kBlock] * w_scales[r][k / kBlock], acc[r][m]);
        }
      }
    }
    float sum = 0.0f;
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float s = acc[r][m];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (lane == m * R + r) sum = s;
      }
    if (mine) reinterpret_cast<T*>(p.out)[(int64_t)m_l * p.ldo + n_l] = from_float<T>(sum + bias);
  }
}

template <class T, int MR, int R, int U, int CTAS>
std::string launch_instance(const GemvParams& p, cudaStream_t stream) {
  const int groups = (p.N + R - 1) / R, ctas = std::min(CTAS * std::max(1, sm_count()), groups);
  if (groups > ctas * kWarps) return "more weight rows than warps";  // (gemv_takes leaves those to the other kernels)
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(32 * kWarps);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, fp8_gemv_kernel<T, MR, R, U, CTAS>, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? std::string() : std::string(cudaGetErrorString(e));
}

template <class T>
std::string launch_typed(const GemvParams& p, cudaStream_t stream) {
  // Two rows: two weight rows at a time, which share the conversion of the activations.  (gemv_takes goes by these.)  One / two weight rows a warp, us: M = 1, 2048 x 2816
  // 3.1 / 3.2; M = 2 4.3 / 3.6.
  return p.M == 1 ? launch_instance<T, 1, 1, 4, 3>(p, stream) : launch_instance<T, 2, 2, 4, 2>(p, stream);
}

}  // namespace

// This kernel has no set-up, no tensor memory and no exchange of parts, but takes its products' instructions, which the tensor cores do not, and a warp
// has a whole weight row (of two rows' calls: two) to itself.  So it is for weights that have one for each warp on the GPU at most, and whose rows are no long
// chains of loads.  Measured, this one / tensor cores, us, K x N: one row, 1024 x 1024 1.8 / 3.0, 1408 x 2048 2.4 / 3.4, 2048 x 2816 2.9 / 4.2, 4096 x 3552 4.8 /
// 6.5; two, 2048 x 2816 3.6 / 4.2, 2560 x 512 3.4 / 3.9, 512 x 4700 2.6 / 3.2.  With a loop over more rows than warps, or beyond the limits of K: one row, 1024 x
// 4096 3.7 / 3.8, 512 x 5504 3.7 / 3.3, 200 x 28672 17.1 / 4.4, 5504 x 512 4.7 / 4.4, 8192 x 512 6.0 / 4.9, 28672 x 200 17.9 / 10.5; two, 512 x 5504 3.8 / 3.2, 4096 x
// 512 4.2 / 3.7, 2560 x 3500 5.6 / 4.6.  Of 484 such problems (with the loop) the choices are 0.3 % slower than the better kernel on average; as the product N * K alone
// would have it, 17 %.
bool gemv_takes(int M, int N, int K) {
  const int sms = sm_count() > 0 ? sm_count() : 148;
  if (M == 1) return K <= 4096 && N <= sms * 3 * kWarps;
  return M == 2 && K <= 2816 && N <= sms * 2 * kWarps * 2 && (int64_t)N * K <= (6 << 20);
}

std::string launch_gemv(Dtype dtype, const GemmArgs& g, unsigned flags, cudaStream_t stream) {
  const GemvParams p{g.M, g.N, g.K, (flags & BLKQ4_GEMM_EARLY_WEIGHT_FETCH) != 0, g.x, g.ldx, g.x_scales, g.ldxs, g.w, g.ldw,
                     g.w_scales, g.ldws, g.bias, g.out, g.ldo};
  return dtype == kFp16 ? launch_typed<__half>(p, stream) : launch_typed<__nv_bfloat16>(p, stream);
}

}  // namespace fp8
}  // namespace blkq4
