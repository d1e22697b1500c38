// Product of a few int8 rows: up to four activation rows against weight rows streamed once through registers.
//
// Bound by the weights' bytes.  A warp takes R weight rows at a time, 512 consecutive bytes of each per load, and multiplies every 16
// bytes with the same k of all activation rows (from L1) by four dp4a; the int32 sums are exact, so that the order of the lanes
// does not matter, and one warp-wide integer reduction a sum ends a row.  No shared memory, no barrier: at a token's sizes a call is
// mostly latency, and this one is one load, a few hundred instructions and a store.  The loads of the next piece are issued before
// the products of the present one.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "blkq4_common.cuh"
#include "int8.cuh"
#include "ms_blkq4gemm.h"

namespace blkq4 {
namespace int8 {
namespace {

constexpr int kWarps = 8;

struct GemvParams {
  int M, N, K, early;
  const int8_t* x;
  int64_t ldx;
  const float* x_scales;
  const int8_t* w;
  int64_t ldw;
  const float* w_scales;
  const void* bias;
  void* out;
  int64_t ldo;
};

__device__ __forceinline__ uint4 load_stream(const int8_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ int dot16(const uint4& a, const uint4& b, int c) {
  c = __dp4a((int)a.x, (int)b.x, c);
  c = __dp4a((int)a.y, (int)b.y, c);
  c = __dp4a((int)a.z, (int)b.z, c);
  return __dp4a((int)a.w, (int)b.w, c);
}

// MR >= M activation rows, R weight rows a warp, U pieces of 512 k of each in flight, CTAS resident on an SM: what is launched.
template <class T, int MR, int R, int U, int CTAS>
__global__ void __launch_bounds__(32 * kWarps, CTAS) gemv_kernel(const GemvParams p) {
  const int lane = threadIdx.x & 31;
  const int groups = (p.N + R - 1) / R, step = (int)gridDim.x * kWarps;
  // neighbouring groups go to different CTAs, so that every SM has the same number of them (give or take one)
  int g = (int)(threadIdx.x >> 5) * (int)gridDim.x + (int)blockIdx.x;
  const int whole = p.K & ~15;  // the last K % 16 k are taken one by one
  uint4 w[R][U];
  auto load = [&](int group, int k0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int8_t* row = p.w + (int64_t)min(group * R + r, p.N - 1) * p.ldw;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * 512 + lane * 16;
        w[r][u] = k < whole ? load_stream(row + k) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  if (p.early) {
    if (g < groups) load(g, 0);
  } else if (lane < R && whole > 0) {  // on their way into L2, where a write that is still to come would find them
    for (int i = 0; i < 2; ++i)
      if ((int64_t)g + (int64_t)i * step < groups)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.w + (int64_t)min((g + i * step) * R + lane, p.N - 1) * p.ldw),
                     "r"(whole)
                     : "memory");
  }
  griddep_wait();
  griddep_launch_dependents();
  if (!p.early && g < groups) load(g, 0);

  for (; g < groups; g += step) {
    int acc[R][MR] = {};
    // what the result needs, fetched under the products
    const int n_l = g * R + lane % R, m_l = lane / R;
    const bool mine = lane < R * MR && n_l < p.N && m_l < p.M;
    const float w_scale = mine ? p.w_scales[n_l] : 0.0f, x_scale = mine ? p.x_scales[m_l] : 0.0f;
    const float bias = mine && p.bias ? to_float(reinterpret_cast<const T*>(p.bias)[n_l]) : 0.0f;
    for (int k0 = 0;;) {
      uint4 now[R][U];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int u = 0; u < U; ++u) now[r][u] = w[r][u];
      const int at = k0;
      k0 += 512 * U;
      const bool last = k0 >= whole;
      if (!last) load(g, k0);
      else if (g + step < groups) load(g + step, 0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = at + u * 512 + lane * 16;
        if (k < whole) {
#pragma unroll
          for (int m = 0; m < MR; ++m) {
            const uint4 x = *reinterpret_cast<const uint4*>(p.x + (int64_t)min(m, p.M - 1) * p.ldx + k);
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r][m] = dot16(now[r][u], x, acc[r][m]);
          }
        }
      }
      if (last) break;
    }
    if (whole + lane < p.K) {
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        const int x = p.x[(int64_t)min(m, p.M - 1) * p.ldx + whole + lane];
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r][m] += x * p.w[(int64_t)min(g * R + r, p.N - 1) * p.ldw + whole + lane];
      }
    }
    int sum = 0;
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int s = __reduce_add_sync(0xffffffffu, acc[r][m]);
        if (lane == m * R + r) sum = s;
      }
    if (mine) reinterpret_cast<T*>(p.out)[(int64_t)m_l * p.ldo + n_l] = from_float<T>(fmaf((float)sum * x_scale, w_scale, bias));
  }
}

template <class T, int MR, int R, int U, int CTAS>
std::string launch_instance(const GemvParams& p, cudaStream_t stream) {
  const int groups = (p.N + R - 1) / R;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min(CTAS * std::max(1, sm_count()), groups));
  cfg.blockDim = dim3(32 * kWarps);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, gemv_kernel<T, MR, R, U, CTAS>, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? std::string() : std::string(cudaGetErrorString(e));
}

template <class T>
std::string launch_typed(const GemvParams& p, cudaStream_t stream) {
  // One activation row: single weight rows, so that the last ones are shared evenly.  More: two at a time, since the products, not the
  // loads, take the issue slots.  Short rows: more of them at a time, as many pieces as a row has.  Measured on B200, back to back
  // in a graph, us, one / two / four weight rows a warp with four pieces each: M = 1, 4096 x 4096 3.9 / 4.4 / 5.0, 8192 x 28672
  // 36.7 / 38.5 / 44; M = 2, 4096 x 11008 11.7 / 9.7 / -; M = 4, 4096 x 4096 9.3 / 5.3 / 5.8.  M = 1, 512 x 20000: one row, four pieces
  // 5.7; two, two 4.2; four, one 3.2; 1024 x 20000: 6.2, 5.3, 5.6.
  if (p.M <= 2 && p.K <= 1024) {
    if (p.M == 1) return p.K <= 512 ? launch_instance<T, 1, 4, 1, 4>(p, stream) : launch_instance<T, 1, 2, 2, 4>(p, stream);
    return p.K <= 512 ? launch_instance<T, 2, 4, 1, 4>(p, stream) : launch_instance<T, 2, 2, 2, 4>(p, stream);
  }
  if (p.M == 1) return launch_instance<T, 1, 1, 4, 4>(p, stream);
  if (p.M == 2) return launch_instance<T, 2, 2, 4, 2>(p, stream);
  return launch_instance<T, 4, 2, 4, 2>(p, stream);
}

}  // namespace

// The tensor-core kernel's calls have some 2 us more of set-up and hand-overs, this one's products take 30 us a GB and row, and a
// warp has a whole row of weights to itself, however few and long they are.  Measured, this one / tensor cores, us: M = 2, 4096 x
// 11008 9.7 / 9.9; M = 4, 2048 x 2048 2.8 / 8.1, 4096 x 4096 5.3 / 6.8, 4096 x 11008 11.3 / 10.0; M = 8, 1024 x 1024 4.7 / 3.8; M = 1,
// 8192 x 1024 5.4 / 4.5, 28672 x 1024 17.3 / 9.4, 11008 x 4096 9.6 / 10.5.
bool gemv_takes(int M, int N, int K) {
  if (K >= 8192 && N <= 2048) return false;
  return M <= 2 || (M <= 4 && (int64_t)N * K <= (24 << 20));
}

std::string launch_gemv(Dtype dtype, const GemmArgs& g, unsigned flags, cudaStream_t stream) {
  const GemvParams p{g.M, g.N, g.K, (flags & BLKQ4_GEMM_EARLY_WEIGHT_FETCH) != 0, g.x, g.ldx, g.x_scales, g.w, g.ldw, g.w_scales,
                     g.bias, g.out, g.ldo};
  return dtype == kFp16 ? launch_typed<__half>(p, stream) : launch_typed<__nv_bfloat16>(p, stream);
}

}  // namespace int8
}  // namespace blkq4
