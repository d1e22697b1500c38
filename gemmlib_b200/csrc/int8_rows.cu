// Rows of int8 with one scale each, from 16-bit rows: plain quantization, the RMS norm (with the residual's addition) and the
// gated activation, each in one pass over its inputs.
//
//   t[k]   quantize: x[k]      silu_mul: g[k] / (1 + exp(-g[k])) * u[k]      norm: h[k] * w[k], h = T(x + residual)
//   q[k] = round(t[k] * (127 / max|t|)), half to even          scale = max|t| / 127, for the norm times r = 1 / sqrt(mean(h^2) + eps)
//
// The norm's factor r is positive and common to the row, so it cancels in t / max|t|: the largest |t| and the sum of squares
// are taken in the same pass and one reduction serves both; q does not depend on the rounding of r.
//
// A row is read once and held in registers between the reduction and its quantization; rows of more than 65536 columns are
// read a second time (from L2).  Bound by HBM: 3 bytes an element for the quantization, 5 for the gate, 7 for the norm with a
// residual (read x and residual, write the sum and q) - as long as an element takes few instructions: at 20 of them the issue
// slots were 79 % busy and set the pace (11008 x 4096: 33 us).  So what can be done to two values at once is: the largest |x| of a
// plain row and the residual's sum in packed halves, three values a maximum in fp32, the integers by a magic addend instead of a
// conversion, four bytes a permutation.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <string>

#include "blkq4_common.cuh"
#include "blkq4_tc.cuh"
#include "blkq4_tma.cuh"
#include "int8.cuh"

namespace blkq4 {
namespace int8 {

__device__ int g_rows_error = 0;  // 0 ok; otherwise (role << 8) | stage of the wait that gave up

namespace {

constexpr int kMaxParts = 8;  // CTAs a row

template <class T>
struct Pair;
template <>
struct Pair<__half> {
  using type = __half2;
};
template <>
struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
};
template <class T>
__device__ __forceinline__ typename Pair<T>::type as_pair(uint32_t v) {
  return *reinterpret_cast<typename Pair<T>::type*>(&v);
}
template <class P>
__device__ __forceinline__ uint32_t as_word(P v) {
  return *reinterpret_cast<uint32_t*>(&v);
}

// A chunk is 8 consecutive elements of a row, a thread's step, packed in four words.
template <class T>
__device__ __forceinline__ void unpack8(const uint32_t (&r)[4], float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2(r[i], T());
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// What L2 does with inputs that have been read.  Large ones make room first, so that what is written stays: 11008 x 4096 quantized 21.3 ->
// 18.7 us, 4095 x 8192 normed 25.7 -> 21.9.  Those that fit in L2 beside other things are kept, since they may be read again: 2048 x 4096 quantized
// 4.4 us time after time, 5.0 if its rows have made room.  A gate and its factor, which are read for this alone, always make room (4096 x 5504 20.1 ->
// 18.9 us); the inputs of a sum never do (4095 x 8192 36.4 us, 37.9 else).
enum Fetch { kKept, kOnce, kInOrder };  // `kInOrder`: kept, and in the order of the program among loads of kOnce
template <Fetch F>
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  if constexpr (F == kKept)
    v = *reinterpret_cast<const uint4*>(p);
  else if constexpr (F == kOnce)
    asm volatile("ld.global.cs.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  else
    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// VEC: every row begins on 16 bytes.  Zeros behind the end of the row.
template <class T, bool VEC, Fetch F = kKept>
__device__ __forceinline__ void load8(const T* row, int chunk, int cols, uint32_t (&r)[4]) {
  const T* src = row + (int64_t)chunk * 8;
  const uint16_t* one = reinterpret_cast<const uint16_t*>(src);
  if (VEC && chunk * 8 + 8 <= cols) {
    const uint4 u = load16<F>(src);
    r[0] = u.x, r[1] = u.y, r[2] = u.z, r[3] = u.w;
  } else if (!VEC && (reinterpret_cast<uintptr_t>(src) & 2u) == 0 && chunk * 8 + 8 <= cols) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = *reinterpret_cast<const uint32_t*>(one + 2 * i);
  } else if (!VEC && chunk > 0 && chunk * 8 + 9 <= cols) {  // the five words that it lies in
    uint32_t w[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = *reinterpret_cast<const uint32_t*>(one - 1 + 2 * i);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __funnelshift_r(w[i], w[i + 1], 16u);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = chunk * 8 + 2 * i < cols ? one[2 * i] : 0u, hi = chunk * 8 + 2 * i + 1 < cols ? one[2 * i + 1] : 0u;
      r[i] = lo | hi << 16;
    }
  }
}

template <class T, bool VEC>
__device__ __forceinline__ void store8(T* row, int chunk, int cols, const uint32_t (&r)[4]) {
  T* dst = row + (int64_t)chunk * 8;
  uint16_t* one = reinterpret_cast<uint16_t*>(dst);
  if (VEC && chunk * 8 + 8 <= cols) {
    *reinterpret_cast<uint4*>(dst) = make_uint4(r[0], r[1], r[2], r[3]);
  } else if (chunk * 8 + 8 <= cols) {  // words, between two halves of one where they do not begin on 4 bytes
    if (reinterpret_cast<uintptr_t>(dst) & 2u) {
      one[0] = (uint16_t)r[0];
#pragma unroll
      for (int i = 0; i < 3; ++i) *reinterpret_cast<uint32_t*>(one + 2 * i + 1) = __funnelshift_r(r[i], r[i + 1], 16u);
      one[7] = (uint16_t)(r[3] >> 16);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<uint32_t*>(one + 2 * i) = r[i];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (chunk * 8 + e < cols) one[e] = (uint16_t)(r[e / 2] >> (e % 2 * 16));
  }
}

// max(a, |b|, |c|), NaN if one of them is
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// What a thread holds of a chunk between the reduction and the quantization, and what it adds to the row's sums.  Plain rows
// stay packed, the others are t in fp32.
template <int OP, class T>
struct Chunk {
  float t[8];
  __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = t[e];
  }
};
template <class T>
struct Chunk<kQuant, T> {
  uint32_t r[4];
  __device__ __forceinline__ void values(float (&v)[8]) const { unpack8<T>(r, v); }
};
template <int OP, class T>
struct Sums {
  static constexpr bool kSquares = OP == kNorm || OP == kNormResidual;
  float top = 0.0f;   // max|t| so far (not of plain rows), NaN if a t is
  uint32_t top2 = 0;  // plain rows: of the even and of the odd elements
  float squares = 0.0f;

  __device__ __forceinline__ void take(Chunk<OP, T>& c) {
    if constexpr (OP == kQuant) {
#pragma unroll
      for (int i = 0; i < 4; ++i) top2 = as_word(__hmax2_nan(as_pair<T>(top2), __habs2(as_pair<T>(c.r[i]))));
    } else {
#pragma unroll
      for (int e = 0; e < 8; e += 2) top = max_abs(top, c.t[e], c.t[e + 1]);
    }
  }
  // As if a t had been NaN.
  __device__ __forceinline__ void spoil() {
    if constexpr (OP == kQuant) top2 = 0x7fff7fffu;
    else top = __uint_as_float(0x7fffffffu);
  }
  // Bits of max|t|: their order as integers puts infinities and NaN last.
  __device__ __forceinline__ uint32_t top_bits() const {
    if constexpr (OP == kQuant) {
      const float2 f = unpack2(top2, T());
      return __float_as_uint(max_abs(f.x, f.y, 0.0f));
    } else {
      return __float_as_uint(top);
    }
  }
};

// c = t of a chunk from its packed inputs; a: x or gate, b: residual or up, w: norm weight.
template <int OP, class T>
__device__ __forceinline__ void combine(Chunk<OP, T>& c, Sums<OP, T>& sums, uint32_t (&a)[4], const uint32_t (&b)[4], const uint32_t (&w)[4]) {
  if constexpr (OP == kQuant) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c.r[i] = a[i];
  } else if constexpr (OP == kSiluMul) {
    float u[8];
    unpack8<T>(a, c.t);
    unpack8<T>(b, u);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // g / (1 + 2^(-g log2 e)); 1 + an infinity has the reciprocal 0
      float p, r;
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(c.t[e] * -1.44269504f));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + p));
      c.t[e] = c.t[e] * r * u[e];
    }
  } else {
    float v[8];
    unpack8<T>(a, c.t);
    unpack8<T>(w, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sums.squares = fmaf(c.t[e], c.t[e], sums.squares);
      c.t[e] *= v[e];  // exact in fp32: T has 8 or 11 bits
    }
  }
  sums.take(c);
}
// The residual's sum is rounded to T once (packed addition: both are), and the norm reads what the next layer's residual will be.
template <class T>
__device__ __forceinline__ void add8(uint32_t (&a)[4], const uint32_t (&b)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = as_word(__hadd2(as_pair<T>(a[i]), as_pair<T>(b[i])));
}

// round(t * inverse), half to even, of |t * inverse| < 2^22: the sum's low mantissa bits are the integer.  The product is rounded
// by itself: 16-bit inputs often stand exactly half-way between two integers (t = max / 2 is 63.5 steps), and a product of the
// rounded inverse falls back on the tie where a fused one would always leave it to the side of the inverse's own error.  Gated
// values are no short numbers: there one instruction does (2048 x 28672 57.5 -> 56.9 us).
template <int OP>
__device__ __forceinline__ uint32_t rounded(float t, float inverse) {
  if (OP == kSiluMul) return __float_as_uint(fmaf(t, inverse, 12582912.0f));
  return __float_as_uint(__fadd_rn(__fmul_rn(t, inverse), 12582912.0f));
}

// What a row's largest |t| (its bits) says.  (Divisions are what costs most here: a thread has 16 or 32 elements to spread them over,
// so the row's scale is for one thread of it to compute.)
struct Scale {
  bool finite;
  float up, inverse;
};
__device__ __forceinline__ Scale scale_of(uint32_t top) {
  Scale s;
  // A row with an infinity or NaN has no scale that its other values could be told by: it is NaN as a whole.
  s.finite = top < 0x7f800000u;
  const float amax = s.finite ? __uint_as_float(top) : 0.0f;
  // 127 / amax is no float below 2^-121: such rows are scaled up by 2^64 first
  s.up = amax < 0x1p-64f ? 0x1p64f : 1.0f;
  s.inverse = amax > 0.0f ? __fdiv_rn(127.0f, amax * s.up) : 0.0f;
  return s;
}
template <bool SQUARES>
__device__ __forceinline__ void write_scale(const RowsParams& p, int64_t row, uint32_t top, float squares) {
  const float amax = __uint_as_float(top);
  float scale = __fdiv_rn(amax, 127.0f);
  bool known = top < 0x7f800000u;
  if (SQUARES) {
    // A mean of squares that is no normal float has lost bits that 1 / sqrt needs, or all of them; one that is infinite would make it 0.
    const float mean = __fdiv_rn(squares, (float)p.cols) + p.eps;
    known = known && squares < INFINITY && (top == 0 || mean >= 0x1p-126f);
    if (top > 0) scale *= __fdiv_rn(1.0f, __fsqrt_rn(mean));
  }
  p.scales[row] = known ? scale : __uint_as_float(0x7fc00000u);
}
template <int OP, class T>
__device__ __forceinline__ void write8(const Scale& s, int8_t* q, bool vec, int chunk, int cols, const Chunk<OP, T>& c) {
  float v[8];
  c.values(v);
  if (!s.finite || s.up != 1.0f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = s.finite ? v[e] * s.up : 0.0f;
  }
  uint32_t b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) b[e] = rounded<OP>(v[e], s.inverse);
  int8_t* dst = q + (int64_t)chunk * 8;
  if (vec && chunk * 8 + 8 <= cols) {
    uint2 o;
    o.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    o.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
    *reinterpret_cast<uint2*>(dst) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (chunk * 8 + e < cols) dst[e] = (int8_t)(b[e] & 0xffu);
  }
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  return v;
}

// A chunk's inputs.
template <int OP, class T, bool VEC, bool ONCE>
__device__ __forceinline__ void load_chunk(const RowsParams& p, int64_t row, int chunk, uint32_t (&a)[4], uint32_t (&b)[4],
                                           uint32_t (&w)[4]) {
  constexpr Fetch kInput = ONCE ? kOnce : kKept;
  load8<T, VEC, kInput>(reinterpret_cast<const T*>(p.a) + row * p.lda, chunk, p.cols, a);
  if constexpr (OP == kNormResidual || OP == kSiluMul)
    load8<T, VEC, kInput>(reinterpret_cast<const T*>(p.b) + row * p.ldb, chunk, p.cols, b);
  if constexpr (Sums<OP, T>::kSquares) load8<T, VEC, ONCE ? kInOrder : kKept>(reinterpret_cast<const T*>(p.w), chunk, p.cols, w);
}
template <int OP, class T, bool VEC>
__device__ __forceinline__ void take_chunk(const RowsParams& p, int64_t row, int chunk, uint32_t (&a)[4], const uint32_t (&b)[4],
                                           const uint32_t (&w)[4], Chunk<OP, T>& c, Sums<OP, T>& sums) {
  if constexpr (OP == kNormResidual) {
    add8<T>(a, b);
    store8<T, VEC>(reinterpret_cast<T*>(p.res_out) + row * p.ldr, chunk, p.cols, a);
  }
  combine(c, sums, a, b, w);
}
// One chunk of a row that is read twice.  `again`: the second pass, for which the sums are already in res_out (which may be x or
// the residual itself).
template <int OP, class T, bool VEC, bool ONCE>
__device__ __forceinline__ void chunk_of(const RowsParams& p, int64_t row, int chunk, bool again, Chunk<OP, T>& c, Sums<OP, T>& sums) {
  uint32_t a[4], b[4] = {}, w[4] = {};
  if (OP == kNormResidual && again) {
    load8<T, VEC>(reinterpret_cast<const T*>(p.res_out) + row * p.ldr, chunk, p.cols, a);
    load8<T, VEC>(reinterpret_cast<const T*>(p.w), chunk, p.cols, w);
    combine(c, sums, a, b, w);
  } else {
    load_chunk<OP, T, VEC, ONCE>(p, row, chunk, a, b, w);
    take_chunk<OP, T, VEC>(p, row, chunk, a, b, w, c, sums);
  }
}

// How the chunks of a row are dealt out.
enum Deal {
  kWarp,     // a warp a row, four rows a CTA
  kCta,      // a CTA a row
  kCluster,  // a row in equal parts to the CTAs of a cluster, which exchange their sums through distributed shared memory
  kLoop,     // a CTA a row, any number of chunks a thread, which are read twice
};

// blockDim.x threads a CTA, NV chunks a thread.
template <int OP, class T, bool VEC, int NV, int MAXT, Deal DEAL, bool ONCE>
__global__ void __launch_bounds__(MAXT) rows_kernel(const RowsParams p) {
  const int threads = DEAL == kWarp ? 32 : (int)blockDim.x, tid = DEAL == kWarp ? (int)threadIdx.x % 32 : (int)threadIdx.x;
  const int parts = DEAL == kCluster ? p.parts : 1, part = DEAL == kCluster ? (int)blockIdx.x % parts : 0;
  const int64_t row = DEAL == kWarp ? (int64_t)blockIdx.x * 4 + threadIdx.x / 32 : (int64_t)(blockIdx.x / (unsigned)parts);
  const int first = part * p.part_chunks + tid;
  if (DEAL == kCluster) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  griddep_wait();
  griddep_launch_dependents();
  if (DEAL == kWarp && row >= p.rows) return;  // whole warps

  constexpr bool kSquares = Sums<OP, T>::kSquares;
  Chunk<OP, T> c[NV];
  Sums<OP, T> sums;
  if constexpr (DEAL != kLoop) {
    // (a part's last threads have chunks of the next part behind theirs: no chunk at all is what lies behind the row)
    auto chunk = [&](int i) { return i * threads + tid < p.part_chunks ? first + i * threads : p.cols / 8 + 1; };
    if constexpr (OP == kQuant) {
#pragma unroll
      for (int i = 0; i < NV; ++i) chunk_of<OP, T, VEC, ONCE>(p, row, chunk(i), false, c[i], sums);
    } else {
      // All loads first: none can move ahead of a store of sums, which may be in the place of an input.  4095 x 8192 with a residual 46.7 ->
      // 36.4 us (6.5 TB/s), 16 x 8192 2.55 -> 2.05, silu_mul of 4096 x 5504 23.4 -> 20.1.
      uint32_t a[NV][4], b[NV][4], w[NV][4];
#pragma unroll
      for (int i = 0; i < NV; ++i) load_chunk<OP, T, VEC, ONCE>(p, row, chunk(i), a[i], b[i], w[i]);
#pragma unroll
      for (int i = 0; i < NV; ++i) take_chunk<OP, T, VEC>(p, row, chunk(i), a[i], b[i], w[i], c[i], sums);
    }
  } else {
    for (int k = tid; k * 8 < p.cols; k += threads) chunk_of<OP, T, VEC, ONCE>(p, row, k, false, c[0], sums);
  }
  uint32_t top = __reduce_max_sync(0xffffffffu, sums.top_bits());
  float squares = kSquares ? warp_sum(sums.squares) : 0.0f;
  if constexpr (DEAL != kWarp) {
    __shared__ uint32_t tops[32];
    __shared__ float all[32];
    const int lane = tid % 32, warps = threads / 32;
    if (lane == 0) {
      tops[tid / 32] = top;
      all[tid / 32] = squares;
    }
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < warps ? tops[lane] : 0u);
    if constexpr (kSquares) squares = warp_sum(lane < warps ? all[lane] : 0.0f);
    if constexpr (DEAL == kCluster) {
      __shared__ __align__(8) uint2 others[kMaxParts];
      asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // every CTA of the cluster has started
      if (tid < parts)
        asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(tc::map_to_cta(smem_u32(&others[part]), (uint32_t)tid)), "r"(top),
                     "r"(__float_as_uint(squares))
                     : "memory");
      tc::cluster_sync_all();
      const uint2 of = lane < parts ? others[lane] : make_uint2(0u, 0u);
      top = __reduce_max_sync(0xffffffffu, of.x);
      if constexpr (kSquares) squares = warp_sum(__uint_as_float(of.y));
    }
  }
  if (tid == 0 && part == 0) write_scale<kSquares>(p, row, top, squares);
  const Scale scale = scale_of(top);
  int8_t* q = p.q + row * p.ldq;
  if constexpr (DEAL != kLoop) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * threads + tid < p.part_chunks) write8(scale, q, p.q_vec, first + i * threads, p.cols, c[i]);
  } else {
    for (int k = tid; k * 8 < p.cols; k += threads) {
      chunk_of<OP, T, VEC, ONCE>(p, row, k, true, c[0], sums);
      write8(scale, q, p.q_vec, k, p.cols, c[0]);
    }
  }
}

template <int OP, class T, bool VEC, int NV, int MAXT, Deal DEAL>
std::string launch_instance(RowsParams p, int parts, cudaStream_t stream) {
  const int chunks = (p.cols + 7) / 8;
  p.parts = parts;
  p.part_chunks = (chunks + parts - 1) / parts;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(DEAL == kWarp ? ((unsigned)p.rows + 3) / 4 : (unsigned)p.rows * (unsigned)parts);
  cfg.blockDim = dim3((unsigned)(DEAL == kWarp ? 128 : DEAL == kLoop ? MAXT : ((p.part_chunks + NV - 1) / NV + 31) / 32 * 32));
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)parts;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = DEAL == kCluster ? 2 : 1;
  // see load16; a long row's second pass wants it kept
  constexpr bool kCanKeep = OP != kSiluMul || DEAL == kLoop, kCanDrop = VEC && OP != kNormResidual && DEAL != kLoop;
  const bool once = kCanDrop && (!kCanKeep || (int64_t)p.rows * p.cols * 2 > (32 << 20));
  cudaError_t e = once ? cudaLaunchKernelEx(&cfg, rows_kernel<OP, T, VEC, NV, MAXT, DEAL, kCanDrop>, p)
                       : cudaLaunchKernelEx(&cfg, rows_kernel<OP, T, VEC, NV, MAXT, DEAL, kCanDrop && !kCanKeep>, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? std::string() : std::string(cudaGetErrorString(e));
}

// ---- many wide rows ----
// A row of more than 20480 columns leaves an SM with one CTA, which loads nothing while it waits at its barrier; rows that do not begin
// on 16 bytes take several loads where others take one.  So there persistent CTAs have a producer warp that keeps bulk copies of the
// next rows under way into a ring in shared memory, while the other warps reduce and write the present one.  A stage holds the chunks of one step of all threads, of both inputs; copies
// begin and end on 16 bytes, whatever the row's place, and the threads shift what they read.  The elements of a row are dealt to
// threads and summed in the order of rows_kernel.
constexpr long long kWaitCycles = 4000000000ll;  // ~2 s
constexpr int kMaxStages = 8;

struct StreamParams {
  int stages, grid;
  uint32_t piece_bytes;  // of one input in a stage
};

// The 16 bytes that begin `behind` (even) bytes into the 32 of lo and hi.
__device__ __forceinline__ uint32_t pick(bool second, uint32_t a, uint32_t b) { return second ? b : a; }
__device__ __forceinline__ void shifted(const uint4& lo, const uint4& hi, uint32_t behind, uint32_t (&r)[4]) {
  const bool by8 = behind & 8u, by4 = behind & 4u, by2 = behind & 2u;
  const uint32_t a[6] = {pick(by8, lo.x, lo.z), pick(by8, lo.y, lo.w), pick(by8, lo.z, hi.x),
                         pick(by8, lo.w, hi.y), pick(by8, hi.x, hi.z), pick(by8, hi.y, hi.w)};
  uint32_t b[5];
#pragma unroll
  for (int i = 0; i < 5; ++i) b[i] = pick(by4, a[i], a[i + 1]);
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = __funnelshift_r(b[i], b[i + 1], by2 ? 16u : 0u);
}
// Copy of whole 16 bytes into shared memory, which complete on a barrier.
__device__ __forceinline__ void bulk_load(uint32_t dst, uint64_t src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
               "r"(bar)
               : "memory");
}
// Bytes [lo, hi) of one input's copy: whole 16 bytes around [start, end), but none outside the tensor; the elements that this leaves
// out at its two ends (of its first and last rows) are fetched one by one.
struct Window {
  uint64_t start, end, lo, hi;
};
__device__ __forceinline__ Window window_of(const void* base, int64_t ld, int rows, int cols, int64_t row, int first, int count) {
  const uint64_t b = reinterpret_cast<uint64_t>(base), e = b + 2ull * ((uint64_t)(rows - 1) * (uint64_t)ld + (uint64_t)cols);
  Window w;
  w.start = b + 2ull * ((uint64_t)row * (uint64_t)ld + (uint64_t)first);
  w.end = w.start + 2ull * (uint64_t)count;
  w.lo = w.start & ~15ull;
  w.hi = (w.end + 15ull) & ~15ull;
  if (w.lo < b) w.lo += 16;
  if (w.hi > e) w.hi -= 16;
  if (w.hi < w.lo) w.hi = w.lo;
  return w;
}

template <int OP, class T, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT) rows_stream_kernel(const RowsParams p, const StreamParams sp) {
  constexpr bool kTwo = OP == kNormResidual || OP == kSiluMul;
  constexpr bool kSquares = Sums<OP, T>::kSquares;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages];
  __shared__ uint32_t tops[2][32];
  __shared__ float all[2][32];
  __shared__ int abort_flag;
  const int threads = (int)blockDim.x - 32, tid = (int)threadIdx.x, warps = threads / 32;
  const int pieces = (p.cols + threads * 8 - 1) / (threads * 8);
  const uint32_t stage_bytes = sp.piece_bytes * (kTwo ? 2u : 1u), ring_u32 = smem_u32(ring);
  if (tid == 0) {
    for (int i = 0; i < sp.stages; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&empty[i]), (uint32_t)warps);
    }
    abort_flag = 0;
    mbar_init_fence();
  }
  __syncthreads();
  griddep_wait();
  griddep_launch_dependents();

  int s = 0;
  uint32_t parity = 0;
  auto advance = [&] {
    if (++s == sp.stages) s = 0, parity ^= 1u;
  };
  if (tid >= threads) {
    const int lane = tid - threads;
    for (int64_t row = blockIdx.x; row < p.rows; row += sp.grid) {
      for (int i = 0; i < pieces; ++i) {
        // (the first round finds fresh barriers: the phase before their first one is complete)
        const bool ok = mbar_wait_bounded(smem_u32(&empty[s]), parity ^ 1u, &abort_flag, &g_rows_error, 0x100 | s, kWaitCycles);
        if (__any_sync(0xffffffffu, !ok)) return;
        const int first = i * threads * 8, count = min(threads * 8, p.cols - first);
        uint8_t* stage = ring + s * stage_bytes;
        const Window a = window_of(p.a, p.lda, p.rows, p.cols, row, first, count);
        const Window b = kTwo ? window_of(p.b, p.ldb, p.rows, p.cols, row, first, count) : a;
        auto edges = [&](const Window& w, uint8_t* to) {
          if (w.lo > w.start || w.hi < w.end) {  // at most 7 elements at either end
            const uint64_t head = w.start + 2ull * (uint64_t)lane, tail = (w.hi > w.start ? w.hi : w.start) + 2ull * (uint64_t)(lane - 16);
            const uint64_t at = lane < 16 ? head : tail;
            if (at < w.end && (at < w.lo || at >= w.hi))
              *reinterpret_cast<uint16_t*>(to + (at - (w.start & ~15ull))) = *reinterpret_cast<const uint16_t*>(at);
          }
        };
        edges(a, stage);
        if (kTwo) edges(b, stage + sp.piece_bytes);
        __syncwarp();
        if (lane == 0) {
          const uint32_t bytes_a = (uint32_t)(a.hi - a.lo), bytes_b = kTwo ? (uint32_t)(b.hi - b.lo) : 0u;
          const uint32_t bar = smem_u32(&full[s]), to = ring_u32 + (uint32_t)s * stage_bytes;
          mbar_arrive_expect_tx(bar, bytes_a + bytes_b);
          if (bytes_a) bulk_load(to + (uint32_t)(a.lo - (a.start & ~15ull)), a.lo, bytes_a, bar);
          if (bytes_b) bulk_load(to + sp.piece_bytes + (uint32_t)(b.lo - (b.start & ~15ull)), b.lo, bytes_b, bar);
        }
        __syncwarp();
        advance();
      }
    }
    return;
  }

  const int lane = tid % 32;
  auto from_stage = [&](const uint8_t* piece, const void* base, int64_t ld, int64_t row, int chunk, uint32_t (&r)[4]) {
    const uint32_t behind = (uint32_t)(reinterpret_cast<uint64_t>(base) + 2ull * (uint64_t)row * (uint64_t)ld) & 15u;
    const uint4* at = reinterpret_cast<const uint4*>(piece + tid * 16);
    const uint4 lo = at[0];
    r[0] = lo.x, r[1] = lo.y, r[2] = lo.z, r[3] = lo.w;
    if (behind != 0) shifted(lo, at[1], behind, r);
    if (chunk * 8 + 8 > p.cols) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int left = p.cols - chunk * 8 - 2 * i;
        r[i] = left >= 2 ? r[i] : left == 1 ? r[i] & 0xffffu : 0u;
      }
    }
  };
  int buffer = 0;
  // 0 once a wait has given up: the rows that are left are NaN as a whole, like one with a NaN among its inputs, and no sums are stored
  // (later waits may pass on the phase before, with nothing new behind them).
  int stored = p.cols;
  for (int64_t row = blockIdx.x; row < p.rows; row += sp.grid, buffer ^= 1) {
    Chunk<OP, T> c[NV];
    Sums<OP, T> sums;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int chunk = i * threads + tid;
      uint32_t a[4] = {}, b[4] = {}, w[4] = {};
      if (i < pieces) {
        if (!mbar_wait_bounded(smem_u32(&full[s]), parity, &abort_flag, &g_rows_error, 0x200 | s, kWaitCycles)) stored = 0;
        const uint8_t* piece = ring + s * stage_bytes;
        from_stage(piece, p.a, p.lda, row, chunk, a);
        if constexpr (kTwo) from_stage(piece + sp.piece_bytes, p.b, p.ldb, row, chunk, b);
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&empty[s]));
        advance();
        if constexpr (OP == kNormResidual) {
          add8<T>(a, b);
          store8<T, false>(reinterpret_cast<T*>(p.res_out) + row * p.ldr, chunk, stored, a);
        }
        if constexpr (kSquares) load8<T, false>(reinterpret_cast<const T*>(p.w), chunk, p.cols, w);
      }
      combine(c[i], sums, a, b, w);
    }
    if (stored == 0) sums.spoil();
    uint32_t top = __reduce_max_sync(0xffffffffu, sums.top_bits());
    float squares = kSquares ? warp_sum(sums.squares) : 0.0f;
    if (lane == 0) {
      tops[buffer][tid / 32] = top;
      all[buffer][tid / 32] = squares;
    }
    // (the other pair of buffers is free again once every warp has come here)
    asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
    top = __reduce_max_sync(0xffffffffu, lane < warps ? tops[buffer][lane] : 0u);
    if constexpr (kSquares) squares = warp_sum(lane < warps ? all[buffer][lane] : 0.0f);
    if (tid == 0) write_scale<kSquares>(p, row, top, squares);
    const Scale scale = scale_of(top);
    int8_t* q = p.q + row * p.ldq;
#pragma unroll
    for (int i = 0; i < NV; ++i) write8(scale, q, p.q_vec, i * threads + tid, p.cols, c[i]);
  }
  if (*const_cast<volatile int*>(&abort_flag)) __nanosleep(50000);  // let copies in flight land
}

template <int OP, class T, int NV, int MAXT>
std::string launch_stream(const RowsParams& p, cudaStream_t stream) {
  constexpr int kInputs = OP == kNormResidual || OP == kSiluMul ? 2 : 1;
  const int threads = ((p.cols + 8 * NV - 1) / (8 * NV) + 31) / 32 * 32;
  StreamParams sp{};
  sp.piece_bytes = (uint32_t)threads * 16u + 16u;
  const uint32_t stage = sp.piece_bytes * kInputs;
  const int ctas = std::max(1, 1024 / (threads + 32));  // of 64 registers a thread
  sp.stages = (int)std::min<uint32_t>(kMaxStages, (uint32_t)(200 * 1024 / ctas) / stage);
  sp.grid = std::min(p.rows, ctas * sm_count());
  const uint32_t smem = (uint32_t)sp.stages * stage;
  static std::atomic<int> granted[64];
  cudaError_t e = ensure_dynamic_smem(rows_stream_kernel<OP, T, NV, MAXT>, smem, granted);
  if (e != cudaSuccess) return cudaGetErrorString(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)sp.grid);
  cfg.blockDim = dim3((unsigned)threads + 32u);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, rows_stream_kernel<OP, T, NV, MAXT>, p, sp);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? std::string() : std::string(cudaGetErrorString(e));
}

// Which thread sums which elements goes by the width alone, so that a row's result does not depend on the rows beside it.
template <int OP, class T, bool VEC>
std::string launch_by_width(const RowsParams& p, cudaStream_t stream) {
  if (p.cols <= 1024) return launch_instance<OP, T, VEC, 4, 128, kWarp>(p, 1, stream);
  if (OP == kQuant && p.cols <= 2048) return launch_instance<OP, T, VEC, 8, 128, kWarp>(p, 1, stream);
  if (p.cols <= 8192) {
    if constexpr (OP == kQuant || OP == kNorm) return launch_instance<OP, T, VEC, 4, 256, kCta>(p, 1, stream);
    else return launch_instance<OP, T, VEC, 2, 512, kCta>(p, 1, stream);
  }
  // Measured, us, the stream / a CTA a row: quantize 4096 x 11008 31.1 / 23.7, 4096 x 20480 56.4 / 47.6, 4096 x 22528 56.9 / 70.0; silu_mul 4096 x 11008
  // 49.6 / 38.0, 4096 x 18432 87 / 67, 4096 x 22528 95 / 112; with a residual 4096 x 16384 97 / 72, 4096 x 20480 113 / 101 (with up to 640 threads a second CTA
  // fits on the SM).  Rows that begin anywhere: 4096 x 9001 30.3 / 32.7, silu_mul 2000 x 20001 51.5 / 84.5.
  if (p.cols <= 31744 && p.rows > 4 * sm_count() && !(VEC && p.cols <= 20480)) return launch_stream<OP, T, 4, 1024>(p, stream);
  if (p.cols <= 32768) return launch_instance<OP, T, VEC, 4, 1024, kCta>(p, 1, stream);
  const int parts = (p.cols + 8191) / 8192;
  if (parts <= kMaxParts && (int64_t)p.rows * parts <= INT32_MAX) return launch_instance<OP, T, VEC, 2, 512, kCluster>(p, parts, stream);
  return launch_instance<OP, T, VEC, 1, 1024, kLoop>(p, 1, stream);
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

// Four bytes of q as two words of T(scale * q).
template <class T>
__device__ __forceinline__ void dequant4(uint32_t q, float scale, uint32_t& lo, uint32_t& hi) {
  const char4 b = *reinterpret_cast<const char4*>(&q);
  lo = pack2<T>(scale * (float)b.x, scale * (float)b.y);
  hi = pack2<T>(scale * (float)b.z, scale * (float)b.w);
}

// T(scale * q); `lanes` (a power of two) threads of a CTA share a row.  VEC: rows of q and of the output begin on 16 bytes, 16 values
// a step.  Else 8 values a step, those of 16 aligned bytes of the output: it has twice the bytes, and reads of q (by aligned 8
// bytes where its rows begin on them: q_vec) are the easier to shift.
template <class T, bool VEC>
__global__ void __launch_bounds__(256) dequant_kernel(int rows, int cols, int lanes, bool q_vec, const int8_t* q, int64_t ldq,
                                                      const float* scales, T* out, int64_t ldo) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t row = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
  if (row >= rows) return;
  const float scale = scales[row];
  q += row * ldq;
  out += row * ldo;
  if constexpr (VEC) {
    for (int c = threadIdx.x % lanes; c * 16 < cols; c += lanes) {
      if (c * 16 + 16 <= cols) {
        const uint4 u = *reinterpret_cast<const uint4*>(q + (int64_t)c * 16);
        uint4 lo, hi;
        dequant4<T>(u.x, scale, lo.x, lo.y);
        dequant4<T>(u.y, scale, lo.z, lo.w);
        dequant4<T>(u.z, scale, hi.x, hi.y);
        dequant4<T>(u.w, scale, hi.z, hi.w);
        uint4* dst = reinterpret_cast<uint4*>(out + (int64_t)c * 16);
        dst[0] = lo;
        dst[1] = hi;
      } else {
        for (int k = c * 16; k < cols; ++k) out[k] = from_float<T>(scale * (float)q[k]);
      }
    }
  } else {
    const int before = (int)(reinterpret_cast<uintptr_t>(out) & 15u) / 2;  // elements that the row's first 16 bytes lack
    const uint32_t shift = (uint32_t)(8 - before) % 8u * 8u;               // bits of q to drop from the 16 bytes it is read by
    for (int c = threadIdx.x % lanes; c * 8 - before < cols; c += lanes) {
      const int k0 = c * 8 - before, k1 = min(k0 + 8, cols);
      if (q_vec && k0 >= 0 && c * 8 + 8 <= cols) {
        const uint64_t hi = *reinterpret_cast<const uint64_t*>(q + (int64_t)c * 8);
        const uint64_t lo = before ? *reinterpret_cast<const uint64_t*>(q + (int64_t)(c - 1) * 8) : hi;
        const uint64_t v = shift ? lo >> shift | hi << (64u - shift) : lo;
        uint4 o;
        dequant4<T>((uint32_t)v, scale, o.x, o.y);
        dequant4<T>((uint32_t)(v >> 32), scale, o.z, o.w);
        *reinterpret_cast<uint4*>(out + k0) = o;
      } else {
        for (int k = max(k0, 0); k < k1; ++k) out[k] = from_float<T>(scale * (float)q[k]);
      }
    }
  }
}

template <class T>
std::string launch_dequant_typed(int rows, int cols, const int8_t* q, int64_t ldq, const float* scales, T* out, int64_t ldo,
                                 cudaStream_t stream) {
  const bool q_vec = reinterpret_cast<uintptr_t>(q) % 8 == 0 && ldq % 8 == 0;
  const bool vec = reinterpret_cast<uintptr_t>(q) % 16 == 0 && ldq % 16 == 0 && aligned(out, ldo, 16);
  int lanes = 1;
  while (lanes < 256 && lanes * (vec ? 16 : 8) < cols) lanes *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(((unsigned)rows + 256 / lanes - 1) / (256 / lanes));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, vec ? dequant_kernel<T, true> : dequant_kernel<T, false>, rows, cols, lanes, q_vec, q, ldq,
                                     scales, out, ldo);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? std::string() : std::string(cudaGetErrorString(e));
}

}  // namespace

int read_rows_error() {
  int v = 0;
  return cudaMemcpyFromSymbol(&v, g_rows_error, sizeof(int)) == cudaSuccess ? v : -1;
}
int clear_rows_error(cudaStream_t stream) {
  void* p = nullptr;
  if (cudaGetSymbolAddress(&p, g_rows_error) != cudaSuccess) return -1;
  return cudaMemsetAsync(p, 0, sizeof(int), stream) == cudaSuccess ? 0 : -1;
}

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
