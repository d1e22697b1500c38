// Rows and weights of e4m3 with fp32 scales, from 16-bit ones; and back.
//
//   t[k]   rows, weights: x[k]        gate: g[k] / (1 + exp(-g[k])) * u[k]
//   values = e4m3(t * (448 / max|t|)), half to even         scale = max|t| / 448
//
// with the largest magnitude taken over 128 elements of a row, or over 128 x 128 of a weight.  One pass: a block is held in registers
// between its reduction and its conversion.  Rows: a block is 16 lanes of 8 elements, so that half a warp reads and reduces it without
// shared memory, and a half-warp takes up to four blocks of a row at a time to have their loads in flight together.  Weights: a CTA a block.
// Bound by HBM: 3 bytes an element, 5 for the gate.
//
// Halves: 16-bit inputs often stand exactly half-way between two e4m3 numbers (wherever max|t| is a multiple of 7, for one), and the rounded
// factor 448 / max|t| would put them to one side.  The quotient 448 x / max of numbers of 11 bits is either half-way between two numbers of 4
// bits or at least 2^-16 of itself away from it (the difference is a fraction of integers over max times a number of 5 bits).  So the product,
// which is off by less than 2^-21, is made a little too large and cut to 18 bits first: what is half-way lies there then, and nothing else does.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <type_traits>

#include "fp8.cuh"
#include "rows_io.cuh"

namespace blkq4 {
namespace fp8 {
namespace {

using namespace blkq4::int8;

constexpr int kThreads = 128;

// What a block's largest |t| (its bits) says.  `up`: blocks whose factor is no float are moved by 2^64 first.
struct Scale {
  float inverse, up;
  bool plain;  // finite, and up is 1
};
__device__ __forceinline__ float reciprocal(float v) {  // 2^-23 off, of 2^-125 to 2^125
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// SHORT: t are 16-bit numbers; the factor is 2^-20 too large for them (see short_of).
template <bool SHORT>
__device__ __forceinline__ Scale scale_of(uint32_t top) {
  constexpr float kTop = SHORT ? 448.0f * (1.0f + 0x1p-20f) : 448.0f;
  Scale s;
  s.plain = top - 0x20000000u < 0x40000000u;  // 2^-63 .. 2^65
  s.up = 1.0f;
  if (s.plain) {
    s.inverse = kTop * reciprocal(__uint_as_float(top));
  } else {
    // A block with an infinity or NaN has no scale that its other values could be told by: it is NaN as a whole, with zeros for values.  448 / max
    // is no float below 2^-119, and the reciprocal none beyond 2^126.
    const float amax = top < 0x7f800000u ? __uint_as_float(top) : 0.0f;
    s.up = top >= 0x7f800000u ? 0.0f : amax < 1.0f ? 0x1p64f : 0x1p-64f;
    s.inverse = amax > 0.0f ? kTop * reciprocal(amax * s.up) : 0.0f;
  }
  return s;
}
// max / 448, rounded once: the quotient by the rounded reciprocal, put right by its remainder.
__device__ __forceinline__ float scale_value(uint32_t top) {
  const float amax = __uint_as_float(top);
  if (top - 0x20000000u >= 0x40000000u) return top < 0x7f800000u ? __fdiv_rn(amax, 448.0f) : __uint_as_float(0x7fc00000u);
  constexpr float kInverse = 1.0f / 448.0f;
  const float q = amax * kInverse;
  return fmaf(fmaf(-448.0f, q, amax), kInverse, q);
}
// v * (1 + 2^-20), give or take 2^-21, cut to 18 bits: what is half-way between two e4m3 numbers (a number of 5 bits) becomes just that; what is not
// is at least 2^-16 away and stays on its side.
__device__ __forceinline__ float short_of(float v) { return __uint_as_float(__float_as_uint(v) & 0xffffffc0u); }
__device__ __forceinline__ uint32_t e4m3x4(const float* v) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]));
  return r;
}
template <bool SHORT>
__device__ __forceinline__ uint2 convert8(const Scale& s, float (&v)[8]) {
  if (!s.plain) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = s.up > 0.0f ? v[e] * s.up : 0.0f;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] *= s.inverse;
    if (SHORT) v[e] = short_of(v[e]);
  }
  return make_uint2(e4m3x4(v), e4m3x4(v + 4));
}
// Rows of 8-bit values: 8 of them, `chunk` times 8 behind the beginning of the row.
__device__ __forceinline__ void store_q8(uint8_t* row, bool vec, int chunk, int cols, uint2 o) {
  uint8_t* dst = row + (int64_t)chunk * 8;
  if (vec && chunk * 8 + 8 <= cols) {
    *reinterpret_cast<uint2*>(dst) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (chunk * 8 + e < cols) dst[e] = (uint8_t)((e < 4 ? o.x : o.y) >> (e % 4 * 8));
  }
}
// Bits of the largest magnitude, NaN last.
template <class T>
__device__ __forceinline__ uint32_t top_of(const uint32_t (&r)[4]) {
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) t = as_word(__hmax2_nan(as_pair<T>(t), __habs2(as_pair<T>(r[i]))));
  const float2 f = unpack2(t, T());
  return __float_as_uint(max_abs(f.x, f.y, 0.0f)) & 0x7fffffffu;
}
__device__ __forceinline__ uint32_t top_of(const float (&v)[8]) {
  float t = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; e += 2) t = max_abs(t, v[e], v[e + 1]);
  return __float_as_uint(t) & 0x7fffffffu;
}
__device__ __forceinline__ uint32_t half_warp_max(uint32_t v) {
#pragma unroll
  for (int s = 8; s > 0; s >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, s));
  return v;
}
// The part of a row that a half-warp takes: U blocks from `block` on.
struct Part {
  int64_t row;
  int block;
};
__device__ __forceinline__ Part part_of(int parts, int U) {
  const int64_t i = (int64_t)blockIdx.x * (kThreads / 16) + (threadIdx.x >> 4);
  Part p;
  if (i < 0xffffffffll) {
    p.row = (uint32_t)i / (uint32_t)parts;
    p.block = (int)((uint32_t)i % (uint32_t)parts) * U;
  } else {
    p.row = i / parts;
    p.block = (int)(i % parts) * U;
  }
  return p;
}

// SCATTER: a row is written to the places of its choices, so that it is read and converted once, whatever their number; the rows behind the
// last place are set to zero by all half-warps in turn.
// ONCE: large inputs make room in L2 for what is written (16000 x 2752 25.6 -> 24.7 us); others are kept, since they may be read again.
template <int OP, class T, bool VEC, bool SCATTER, int U, bool ONCE>
__global__ void __launch_bounds__(kThreads) rows_kernel(const RowsParams p, int parts, bool q_vec) {
  griddep_wait();
  griddep_launch_dependents();
  const Part at = part_of(parts, U);
  const int lane = threadIdx.x & 15;
  const bool in = at.row < p.rows;
  const int places = SCATTER ? p.rows * p.choices : 0;
  int first_zero = places;
  if constexpr (SCATTER) first_zero = max(0, *p.count);
  const T *row_a = reinterpret_cast<const T*>(p.a) + at.row * p.lda, *row_b = reinterpret_cast<const T*>(p.b) + (OP == kSiluMul ? at.row * p.ldb : 0);
  uint32_t a[U][4] = {}, b[U][4] = {};
  uint32_t wa[VEC ? 1 : U][5], wb[VEC ? 1 : U][5];
  const int off_a = off_word(row_a), off_b = off_word(row_b), cols = in ? p.cols : 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int chunk = (at.block + u) * 16 + lane;
    if constexpr (VEC) {
      if (chunk * 8 < cols) {
        load8<T, VEC, OP == kSiluMul || ONCE ? kOnce : kKept>(row_a, chunk, p.cols, a[u]);
        if constexpr (OP == kSiluMul) load8<T, VEC, kOnce>(row_b, chunk, p.cols, b[u]);
      }
    } else {
      load_words(row_a, off_a, chunk, cols, wa[u]);
      if constexpr (OP == kSiluMul) load_words(row_b, off_b, chunk, cols, wb[u]);
    }
  }
  if constexpr (!VEC) {  // all of them ahead of the first use: 16000 x 2747 quantized 32.6 -> 31.4 us
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int chunk = (at.block + u) * 16 + lane;
      take_words(row_a, off_a, chunk, cols, wa[u], a[u]);
      if constexpr (OP == kSiluMul) take_words(row_b, off_b, chunk, cols, wb[u], b[u]);
    }
  }
  auto write = [&](auto far) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int chunk = (at.block + u) * 16 + lane;
      float v[8];
      uint32_t top;
      if constexpr (OP == kSiluMul) {
        silu_mul8<T, decltype(far)::value>(a[u], b[u], v);
        top = top_of(v);
      } else {
        top = top_of<T>(a[u]);
        unpack8<T>(a[u], v);
      }
      top = half_warp_max(top);
      if (!in || chunk * 8 >= p.cols) continue;
      const uint2 q = convert8<OP == kQuant>(scale_of<OP == kQuant>(top), v);
      const float scale = scale_value(top);
      if constexpr (SCATTER) {
        for (int j = 0; j < p.choices; ++j) {
          const int place = p.places[at.row * p.choices + j];
          if (place < 0 || place >= places) continue;  // of no expert (or of an order that is none)
          store_q8(p.q + place * p.ldq, q_vec, chunk, p.cols, q);
          if (lane == 0) p.scales[place * p.lds + at.block + u] = scale;
        }
      } else {
        store_q8(p.q + at.row * p.ldq, q_vec, chunk, p.cols, q);
        if (lane == 0) p.scales[at.row * p.lds + at.block + u] = scale;
      }
    }
  };
  if (OP == kSiluMul && __any_sync(0xffffffffu, far_gates<T>(a))) write(std::true_type());
  else write(std::false_type());
  if constexpr (SCATTER) {
    const int64_t halves = (int64_t)gridDim.x * (kThreads / 16), blocks = (p.cols + kBlock - 1) / kBlock;
    const int64_t end = ((int64_t)places - first_zero) * blocks;
    for (int64_t i = (int64_t)blockIdx.x * (kThreads / 16) + (threadIdx.x >> 4); i < end; i += halves) {
      const int64_t row = first_zero + i / blocks;
      const int block = (int)(i % blocks), chunk = block * 16 + lane;
      if (chunk * 8 < p.cols) store_q8(p.q + row * p.ldq, q_vec, chunk, p.cols, make_uint2(0u, 0u));
      if (lane == 0) p.scales[row * p.lds + block] = 0.0f;
    }
  }
}

// A CTA a block of 128 x 128: 16 lanes a row, 16 rows at a time.
constexpr int kWeightThreads = 256;
template <class T, bool VEC>
__global__ void __launch_bounds__(kWeightThreads) weights_kernel(const RowsParams p, int k_blocks, int n_blocks, bool q_vec) {
  __shared__ uint32_t tops[kWeightThreads / 32];
  griddep_wait();
  griddep_launch_dependents();
  const int64_t block = blockIdx.x;
  const int kb = (int)(block % k_blocks);
  const int64_t eb = block / k_blocks;
  const int nb = (int)(eb % n_blocks);
  const int64_t expert = eb / n_blocks;
  const int chunk = kb * 16 + (threadIdx.x & 15), n0 = nb * kBlock + (threadIdx.x >> 4);
  const bool in_cols = chunk * 8 < p.cols;
  const int64_t row0 = expert * p.expert_rows + n0;
  uint32_t a[8][4] = {};
  const T* first = reinterpret_cast<const T*>(p.a) + row0 * p.lda;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (in_cols && n0 + 16 * i < p.expert_rows) load8<T, VEC, kOnce>(first + 16 * i * p.lda, chunk, p.cols, a[i]);
  } else {
    uint32_t w[8][5];
    const int off = off_word(first);  // (of all eight: sixteen rows are a multiple of 32 bytes)
#pragma unroll
    for (int i = 0; i < 8; ++i) load_words(first + 16 * i * p.lda, off, chunk, n0 + 16 * i < p.expert_rows ? p.cols : 0, w[i]);
#pragma unroll
    for (int i = 0; i < 8; ++i) take_words(first + 16 * i * p.lda, off, chunk, n0 + 16 * i < p.expert_rows ? p.cols : 0, w[i], a[i]);
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, top_of<T>(a[i]));
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWeightThreads / 32; ++i) top = max(top, tops[i]);
  const Scale s = scale_of<true>(top);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (!in_cols || n0 + 16 * i >= p.expert_rows) continue;
    float v[8];
    unpack8<T>(a[i], v);
    store_q8(p.q + (row0 + 16 * i) * p.ldq, q_vec, chunk, p.cols, convert8<true>(s, v));
  }
  if (threadIdx.x == 0) p.scales[(expert * n_blocks + nb) * p.lds + kb] = scale_value(top);
}

// out = scale * values.  Rows of the output that begin anywhere are written by 16 aligned bytes, whose values lie in two pieces of 8 and may have
// two scales.
template <class T, bool WEIGHTS, bool VEC, int U>
__global__ void __launch_bounds__(kThreads) dequant_kernel(const DequantParams p, int parts, bool q_vec) {
  griddep_wait();
  griddep_launch_dependents();
  const Part at = part_of(parts, U);
  if (at.row >= p.rows) return;
  int64_t scale_row = at.row;
  if (WEIGHTS) {
    const int64_t expert = at.row / p.expert_rows, n_blocks = (p.expert_rows + kBlock - 1) / kBlock;
    scale_row = expert * n_blocks + (at.row - expert * p.expert_rows) / kBlock;
  }
  const uint8_t* q = p.q + at.row * p.ldq;
  const float* scales = p.scales + scale_row * p.lds;
  T* out = reinterpret_cast<T*>(p.out) + at.row * p.ldo;
  const int before = VEC ? 0 : (int)(reinterpret_cast<uintptr_t>(out) & 15u) / 2;  // elements that the row's first 16 bytes lack
  const uint32_t shift = (uint32_t)(8 - before) % 8u * 8u;                         // bits of q to drop from the 16 bytes it is read by
  const int last = (p.cols - 1) / kBlock;
  uint64_t v[U];
  float s0[U], s1[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int c = (at.block + u) * 16 + (threadIdx.x & 15), k0 = c * 8 - before;
    v[u] = 0, s0[u] = s1[u] = 0.0f;
    if (k0 >= p.cols) continue;
    s0[u] = scales[max(k0, 0) / kBlock];
    s1[u] = VEC ? s0[u] : scales[min((k0 + 7) / kBlock, last)];
    if (q_vec && k0 >= 0 && c * 8 + 8 <= p.cols) {
      const uint64_t hi = *reinterpret_cast<const uint64_t*>(q + (int64_t)c * 8);
      if (VEC || before == 0) v[u] = hi;
      else v[u] = *reinterpret_cast<const uint64_t*>(q + (int64_t)(c - 1) * 8) >> shift | hi << (64u - shift);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k0 + e >= 0 && k0 + e < p.cols) v[u] |= (uint64_t)q[(int64_t)k0 + e] << (e * 8);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int c = (at.block + u) * 16 + (threadIdx.x & 15), k0 = c * 8 - before;
    if (k0 >= p.cols) continue;
    const int turn = VEC || k0 < 0 ? 8 : kBlock - (k0 & (kBlock - 1));  // elements of the first scale, from k0 on
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t h;  // e4m3 is exact in fp16
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(v[u] >> (16 * i))));
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      o[i] = pack2<T>(f.x * (2 * i < turn ? s0[u] : s1[u]), f.y * (2 * i + 1 < turn ? s0[u] : s1[u]));
    }
    if (k0 >= 0 && k0 + 8 <= p.cols) {
      *reinterpret_cast<uint4*>(out + (int64_t)k0) = make_uint4(o[0], o[1], o[2], o[3]);
    } else {
      uint16_t* one = reinterpret_cast<uint16_t*>(out) + (int64_t)k0;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k0 + e >= 0 && k0 + e < p.cols) one[e] = (uint16_t)(o[e / 2] >> (e % 2 * 16));
    }
  }
}

template <class... Params, class... Args>
std::string launch(void (*kernel)(Params...), int64_t ctas, int threads, cudaStream_t stream, Args... args) {
  if (ctas > 0x7fffffffll) return "too many rows";
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? std::string() : std::string(cudaGetErrorString(e));
}
bool rows_on(const void* ptr, int64_t pitch_bytes, int rows, int bytes) {
  return reinterpret_cast<uintptr_t>(ptr) % bytes == 0 && (rows <= 1 || pitch_bytes % bytes == 0);
}

// Blocks that a half-warp takes at a time: what hides the latency of many rows, one where they are few.
int blocks_at_a_time(int rows, int cols) {
  const int64_t blocks = (int64_t)rows * blocks_of(cols);
  const int most = blocks_of(cols);
  return blocks >= 8 * 148 * 16 && most >= 4 ? 4 : blocks >= 4 * 148 * 16 && most >= 2 ? 2 : 1;
}
template <int OP, class T, bool VEC, bool SCATTER>
std::string launch_rows_u(const RowsParams& p, cudaStream_t stream) {
  const int U = blocks_at_a_time(p.rows, p.cols), parts = (blocks_of(p.cols) + U - 1) / U;
  const int64_t ctas = ((int64_t)p.rows * parts + kThreads / 16 - 1) / (kThreads / 16);
  const bool q_vec = rows_on(p.q, p.ldq, SCATTER ? p.rows * p.choices : p.rows, 8);
  if constexpr (OP == kQuant && VEC && !SCATTER) {
    if (U == 4 && (int64_t)p.rows * p.cols * 2 > (32 << 20)) return launch(rows_kernel<OP, T, VEC, SCATTER, 4, true>, ctas, kThreads, stream, p, parts, q_vec);
  }
  if (U == 4) return launch(rows_kernel<OP, T, VEC, SCATTER, 4, false>, ctas, kThreads, stream, p, parts, q_vec);
  if (U == 2) return launch(rows_kernel<OP, T, VEC, SCATTER, 2, false>, ctas, kThreads, stream, p, parts, q_vec);
  return launch(rows_kernel<OP, T, VEC, SCATTER, 1, false>, ctas, kThreads, stream, p, parts, q_vec);
}
template <class T>
std::string launch_rows_t(RowsOp op, const RowsParams& p, cudaStream_t stream) {
  if (op == kSiluMul) {
    const bool vec = rows_on(p.a, p.lda * 2, p.rows, 16) && rows_on(p.b, p.ldb * 2, p.rows, 16);
    return vec ? launch_rows_u<kSiluMul, T, true, false>(p, stream) : launch_rows_u<kSiluMul, T, false, false>(p, stream);
  }
  const bool vec = rows_on(p.a, p.lda * 2, p.rows, 16);
  if (p.places) return vec ? launch_rows_u<kQuant, T, true, true>(p, stream) : launch_rows_u<kQuant, T, false, true>(p, stream);
  return vec ? launch_rows_u<kQuant, T, true, false>(p, stream) : launch_rows_u<kQuant, T, false, false>(p, stream);
}
template <class T>
std::string launch_weights_t(const RowsParams& p, cudaStream_t stream) {
  const int k_blocks = blocks_of(p.cols), n_blocks = blocks_of(p.expert_rows);
  const int64_t ctas = (int64_t)(p.rows / p.expert_rows) * n_blocks * k_blocks;
  const bool q_vec = rows_on(p.q, p.ldq, p.rows, 8);
  return rows_on(p.a, p.lda * 2, p.rows, 16) ? launch(weights_kernel<T, true>, ctas, kWeightThreads, stream, p, k_blocks, n_blocks, q_vec)
                                             : launch(weights_kernel<T, false>, ctas, kWeightThreads, stream, p, k_blocks, n_blocks, q_vec);
}
template <class T, bool WEIGHTS, bool VEC>
std::string launch_dequant_u(const DequantParams& p, cudaStream_t stream) {
  // (outputs that begin inside 16 bytes: up to 7 elements more)
  const int U = blocks_at_a_time(p.rows, p.cols), blocks = blocks_of(p.cols + (VEC ? 0 : 7)), parts = (blocks + U - 1) / U;
  const int64_t ctas = ((int64_t)p.rows * parts + kThreads / 16 - 1) / (kThreads / 16);
  const bool q_vec = rows_on(p.q, p.ldq, p.rows, 8);
  if (U == 4) return launch(dequant_kernel<T, WEIGHTS, VEC, 4>, ctas, kThreads, stream, p, parts, q_vec);
  if (U == 2) return launch(dequant_kernel<T, WEIGHTS, VEC, 2>, ctas, kThreads, stream, p, parts, q_vec);
  return launch(dequant_kernel<T, WEIGHTS, VEC, 1>, ctas, kThreads, stream, p, parts, q_vec);
}
template <class T, bool WEIGHTS>
std::string launch_dequant_t(const DequantParams& p, cudaStream_t stream) {
  return rows_on(p.out, p.ldo * 2, p.rows, 16) ? launch_dequant_u<T, WEIGHTS, true>(p, stream) : launch_dequant_u<T, WEIGHTS, false>(p, stream);
}

}  // namespace

std::string launch_rows(RowsOp op, Dtype dtype, const RowsParams& p, cudaStream_t stream) {
  return dtype == kFp16 ? launch_rows_t<__half>(op, p, stream) : launch_rows_t<__nv_bfloat16>(op, p, stream);
}
std::string launch_weights(Dtype dtype, const RowsParams& p, cudaStream_t stream) {
  return dtype == kFp16 ? launch_weights_t<__half>(p, stream) : launch_weights_t<__nv_bfloat16>(p, stream);
}
std::string launch_dequant(Dtype dtype, const DequantParams& p, cudaStream_t stream) {
  if (p.expert_rows > 0)
    return dtype == kFp16 ? launch_dequant_t<__half, true>(p, stream) : launch_dequant_t<__nv_bfloat16, true>(p, stream);
  return dtype == kFp16 ? launch_dequant_t<__half, false>(p, stream) : launch_dequant_t<__nv_bfloat16, false>(p, stream);
}

}  // namespace fp8
}  // namespace blkq4
