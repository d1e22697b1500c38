// Rows of int8 with one scale each, from 16-bit rows: plain quantization, the RMS norm (with the residual's addition) and the
// gated activation, each in one pass over its inputs.
//
//   t[k]   quantize: x[k]      silu_mul: g[k] / (1 + exp(-g[k])) * u[k]      norm: h[k] * w[k], h = T(x + residual)
//   q[k] = round(t[k] * (127 / max|t|)), half to even          scale = max|t| / 127, for the norm times r = 1 / sqrt(mean(h^2) + eps)
//
// The norm's factor r is positive and common to the row, so it cancels in t / max|t|: the largest |t| and the sum of squares
// are taken in the same pass and one reduction serves both; q does not depend on the rounding of r.
//
// A row is read once and held in registers between the reduction and its quantization; rows of more than 32768 columns are
// read a second time (from L2).  Bound by HBM: 3 bytes an element for the quantization, 5 for the gate, 7 for the norm with a
// residual (read x and residual, write the sum and q).
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

#include "blkq4_common.cuh"
#include "int8.cuh"

namespace blkq4 {
namespace int8 {
namespace {

// A chunk is 8 consecutive elements of a row, a thread's step.  VEC: every row begins on 16 bytes.
__device__ __forceinline__ uint32_t pick(bool second, uint32_t a, uint32_t b) { return second ? b : a; }

template <class T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int chunk, int cols, float (&v)[8]) {
  const T* src = row + (int64_t)chunk * 8;
  // bytes by which the chunk lies behind a multiple of 16
  const uint32_t behind = VEC ? 0u : (uint32_t)(reinterpret_cast<uintptr_t>(src) & 15u);
  uint32_t r[4];
  if (behind == 0 && chunk * 8 + 8 <= cols) {
    const uint4 u = *reinterpret_cast<const uint4*>(src);
    r[0] = u.x, r[1] = u.y, r[2] = u.z, r[3] = u.w;
  } else if (!VEC && chunk > 0 && chunk * 8 + 16 <= cols) {
    // the two aligned vectors that it lies in, inside the row both of them, and the bytes in question moved to the front
    const uint4* at = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(src) - behind);
    const uint4 lo = at[0], hi = at[1];
    const bool by8 = behind & 8u, by4 = behind & 4u, by2 = behind & 2u;
    const uint32_t a[6] = {pick(by8, lo.x, lo.z), pick(by8, lo.y, lo.w), pick(by8, lo.z, hi.x),
                           pick(by8, lo.w, hi.y), pick(by8, hi.x, hi.z), pick(by8, hi.y, hi.w)};
    uint32_t b[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) b[i] = pick(by4, a[i], a[i + 1]);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __funnelshift_r(b[i], b[i + 1], by2 ? 16u : 0u);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = chunk * 8 + e < cols ? to_float(src[e]) : 0.0f;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2(r[i], T());
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

template <class T, bool VEC>
__device__ __forceinline__ void store8(T* row, int chunk, int cols, const float (&v)[8]) {
  T* dst = row + (int64_t)chunk * 8;
  if (VEC && chunk * 8 + 8 <= cols) {
    *reinterpret_cast<uint4*>(dst) =
        make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
  } else if (chunk * 8 + 8 <= cols) {  // words, between two halves of one where they do not begin on 4 bytes
    if (reinterpret_cast<uintptr_t>(dst) & 2u) {
      dst[0] = from_float<T>(v[0]);
#pragma unroll
      for (int e = 1; e < 7; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack2<T>(v[e], v[e + 1]);
      dst[7] = from_float<T>(v[7]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack2<T>(v[e], v[e + 1]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (chunk * 8 + e < cols) dst[e] = from_float<T>(v[e]);
  }
}

// t of one chunk; adds its squares (norm) to `sum`.  `again`: the second pass over a long row, whose sums are already in
// res_out (which may be x or the residual itself).
template <int OP, class T, bool VEC>
__device__ __forceinline__ void row_values(const RowsParams& p, int64_t row, int chunk, bool again, float (&t)[8],
                                           float& sum) {
  const T* a = reinterpret_cast<const T*>(p.a) + row * p.lda;
  if constexpr (OP == kQuant) {
    load8<T, VEC>(a, chunk, p.cols, t);
  } else if constexpr (OP == kSiluMul) {
    float u[8];
    load8<T, VEC>(a, chunk, p.cols, t);
    load8<T, VEC>(reinterpret_cast<const T*>(p.b) + row * p.ldb, chunk, p.cols, u);
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = __fdividef(t[e], 1.0f + __expf(-t[e])) * u[e];
  } else {
    float w[8];
    T* res_out = reinterpret_cast<T*>(p.res_out) + row * p.ldr;
    if (OP == kNormResidual && again) {
      load8<T, VEC>(res_out, chunk, p.cols, t);
    } else {
      load8<T, VEC>(a, chunk, p.cols, t);
      if constexpr (OP == kNormResidual) {
        float r[8];
        load8<T, VEC>(reinterpret_cast<const T*>(p.b) + row * p.ldb, chunk, p.cols, r);
        // the sum is rounded to T once, and the norm reads what the next layer's residual will be
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = to_float(from_float<T>(t[e] + r[e]));
        store8<T, VEC>(res_out, chunk, p.cols, t);
      }
    }
    load8<T, VEC>(reinterpret_cast<const T*>(p.w), chunk, p.cols, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sum = fmaf(t[e], t[e], sum);
      t[e] *= w[e];  // exact in fp32 where w has 8 or 11 bits
    }
  }
}

// round(t * inverse), half to even, of |t * inverse| < 2^22: the sum's low mantissa bits are the integer.  The product is rounded
// by itself: 16-bit inputs often stand exactly half-way between two integers (t = max / 2 is 63.5 steps), and a product of the
// rounded inverse falls back on the tie where a fused one would always leave it to the side of the inverse's own error.
__device__ __forceinline__ uint32_t rounded(float t, float inverse) {
  return __float_as_uint(__fadd_rn(__fmul_rn(t, inverse), 12582912.0f));
}

__device__ __forceinline__ void store_q(int8_t* row, bool vec, int chunk, int cols, const float (&t)[8], float inverse) {
  uint32_t b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) b[e] = rounded(t[e], inverse);
  int8_t* dst = row + (int64_t)chunk * 8;
  if (vec && chunk * 8 + 8 <= cols) {
    uint2 v;
    v.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    v.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
    *reinterpret_cast<uint2*>(dst) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (chunk * 8 + e < cols) dst[e] = (int8_t)(b[e] & 0xffu);
  }
}

// blockDim.x threads a row, NV chunks of 8 elements a thread (0: any number, two passes); WARP: a warp a row, four rows a CTA.
template <int OP, class T, bool VEC, int NV, int MAXT, bool WARP>
__global__ void __launch_bounds__(MAXT) rows_kernel(const RowsParams p) {
  griddep_launch_dependents();
  griddep_wait();
  const int threads = WARP ? 32 : (int)blockDim.x, tid = WARP ? (int)threadIdx.x % 32 : (int)threadIdx.x;
  const int64_t row = WARP ? (int64_t)blockIdx.x * 4 + threadIdx.x / 32 : (int64_t)blockIdx.x;
  if (WARP && row >= p.rows) return;  // whole warps

  float t[NV > 0 ? NV : 1][8];
  float sum = 0.0f;
  uint32_t top = 0;  // bits of max|t|: their order as integers puts infinities and NaN last
  auto take_top = [&](const float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      row_values<OP, T, VEC>(p, row, i * threads + tid, false, t[i], sum);
      take_top(t[i]);
    }
  } else {
    for (int c = tid; c * 8 < p.cols; c += threads) {
      row_values<OP, T, VEC>(p, row, c, false, t[0], sum);
      take_top(t[0]);
    }
  }

  constexpr bool kSums = OP == kNorm || OP == kNormResidual;
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (kSums) {
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
  }
  if constexpr (!WARP) {
    __shared__ uint32_t tops[32];
    __shared__ float sums[32];
    const int lane = tid % 32, warps = threads / 32;
    if (lane == 0) {
      tops[tid / 32] = top;
      sums[tid / 32] = sum;
    }
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < warps ? tops[lane] : 0u);
    if constexpr (kSums) {
      sum = lane < warps ? sums[lane] : 0.0f;
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    }
  }

  // A row with an infinity or NaN has no scale that its other values could be told by: it is NaN as a whole.
  const bool finite = top < 0x7f800000u;
  const float amax = finite ? __uint_as_float(top) : 0.0f;
  // 127 / amax is no float below 2^-121: such rows are scaled up by 2^64 first
  const float up = amax < 0x1p-64f ? 0x1p64f : 1.0f;
  const float inverse = amax > 0.0f ? __fdiv_rn(127.0f, amax * up) : 0.0f;
  if (tid == 0) {
    float scale = __fdiv_rn(amax, 127.0f);
    if (kSums && amax > 0.0f) scale *= __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(sum, (float)p.cols) + p.eps));
    p.scales[row] = finite ? scale : __uint_as_float(0x7fc00000u);
  }
  int8_t* q = p.q + row * p.ldq;
  auto write = [&](int chunk, float (&v)[8]) {
    if (!finite || up != 1.0f) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = finite ? v[e] * up : 0.0f;
    }
    store_q(q, p.q_vec, chunk, p.cols, v, inverse);
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) write(i * threads + tid, t[i]);
  } else {
    for (int c = tid; c * 8 < p.cols; c += threads) {
      row_values<OP, T, VEC>(p, row, c, true, t[0], sum);
      write(c, t[0]);
    }
  }
}

template <int OP, class T, bool VEC, int NV, int MAXT, bool WARP>
std::string launch_instance(const RowsParams& p, cudaStream_t stream) {
  const int per = 8 * (NV > 0 ? NV : 1);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(WARP ? (p.rows + 3) / 4 : p.rows));
  cfg.blockDim = dim3((unsigned)(WARP ? 128 : NV > 0 ? ((p.cols + per - 1) / per + 31) / 32 * 32 : MAXT));
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, rows_kernel<OP, T, VEC, NV, MAXT, WARP>, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? std::string() : std::string(cudaGetErrorString(e));
}

template <int OP, class T, bool VEC>
std::string launch_by_width(const RowsParams& p, cudaStream_t stream) {
  if (p.cols <= 1024) return launch_instance<OP, T, VEC, 4, 128, true>(p, stream);
  if (p.cols <= 8192 && p.rows <= 2 * sm_count()) return launch_instance<OP, T, VEC, 1, 1024, false>(p, stream);
  if (p.cols <= 8192) return launch_instance<OP, T, VEC, 4, 256, false>(p, stream);
  if (p.cols <= 16384) return launch_instance<OP, T, VEC, 4, 512, false>(p, stream);
  if (p.cols <= 32768) return launch_instance<OP, T, VEC, 4, 1024, false>(p, stream);
  return launch_instance<OP, T, VEC, 0, 1024, false>(p, stream);
}

inline bool aligned(const void* p, int64_t ld, int bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && ld % 8 == 0;
}

template <int OP, class T>
std::string launch_typed(RowsParams p, cudaStream_t stream) {
  p.q_vec = aligned(p.q, p.ldq, 8);
  bool vec = aligned(p.a, p.lda, 16);
  if (OP == kNormResidual || OP == kSiluMul) vec = vec && aligned(p.b, p.ldb, 16);
  if (OP == kNormResidual) vec = vec && aligned(p.res_out, p.ldr, 16);
  if (OP == kNorm || OP == kNormResidual) vec = vec && aligned(p.w, 0, 16);
  return vec ? launch_by_width<OP, T, true>(p, stream) : launch_by_width<OP, T, false>(p, stream);
}

template <class T>
std::string launch_op(RowsOp op, const RowsParams& p, cudaStream_t stream) {
  switch (op) {
    case kQuant: return launch_typed<kQuant, T>(p, stream);
    case kNorm: return launch_typed<kNorm, T>(p, stream);
    case kNormResidual: return launch_typed<kNormResidual, T>(p, stream);
    default: return launch_typed<kSiluMul, T>(p, stream);
  }
}

// T(scale * q): 16 values a thread and step; `lanes` (a power of two) threads of a CTA share a row.
template <class T, bool VEC>
__global__ void __launch_bounds__(256) dequant_kernel(int rows, int cols, int lanes, const int8_t* q, int64_t ldq,
                                                      const float* scales, T* out, int64_t ldo) {
  griddep_launch_dependents();
  griddep_wait();
  const int64_t row = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
  if (row >= rows) return;
  const float scale = scales[row];
  q += row * ldq;
  out += row * ldo;
  for (int c = threadIdx.x % lanes; c * 16 < cols; c += lanes) {
    if (VEC && c * 16 + 16 <= cols) {
      const uint4 u = *reinterpret_cast<const uint4*>(q + c * 16);
      const uint32_t r[4] = {u.x, u.y, u.z, u.w};
      uint32_t o[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const char4 b = *reinterpret_cast<const char4*>(&r[i]);
        o[2 * i] = pack2<T>(scale * (float)b.x, scale * (float)b.y);
        o[2 * i + 1] = pack2<T>(scale * (float)b.z, scale * (float)b.w);
      }
      uint4* dst = reinterpret_cast<uint4*>(out + c * 16);
      dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
      dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
    } else {
      for (int k = c * 16; k < min(c * 16 + 16, cols); ++k) out[k] = from_float<T>(scale * (float)q[k]);
    }
  }
}

template <class T>
std::string launch_dequant_typed(int rows, int cols, const int8_t* q, int64_t ldq, const float* scales, T* out, int64_t ldo,
                                 cudaStream_t stream) {
  const bool vec = reinterpret_cast<uintptr_t>(q) % 16 == 0 && ldq % 16 == 0 && aligned(out, ldo, 16);
  int lanes = 1;
  while (lanes < 256 && lanes * 16 < cols) lanes *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((rows + 256 / lanes - 1) / (256 / lanes)));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, vec ? dequant_kernel<T, true> : dequant_kernel<T, false>, rows, cols, lanes, q, ldq,
                                     scales, out, ldo);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? std::string() : std::string(cudaGetErrorString(e));
}

}  // namespace

std::string launch_rows(RowsOp op, Dtype dtype, const RowsParams& p, cudaStream_t stream) {
  return dtype == kFp16 ? launch_op<__half>(op, p, stream) : launch_op<__nv_bfloat16>(op, p, stream);
}

std::string launch_dequant(Dtype dtype, int rows, int cols, const int8_t* q, int64_t ldq, const float* scales, void* out,
                           int64_t ldo, cudaStream_t stream) {
  return dtype == kFp16 ? launch_dequant_typed(rows, cols, q, ldq, scales, reinterpret_cast<__half*>(out), ldo, stream)
                        : launch_dequant_typed(rows, cols, q, ldq, scales, reinterpret_cast<__nv_bfloat16*>(out), ldo, stream);
}

}  // namespace int8
}  // namespace blkq4
