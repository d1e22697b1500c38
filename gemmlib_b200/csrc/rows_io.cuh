// Loads and stores of 16-bit rows by chunks of 8 elements, wherever the rows begin: for the kernels that write 8-bit rows.
#pragma once

#include <cstdint>

#include "int8.cuh"

namespace blkq4 {
namespace int8 {

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
// -87 in the type's bits.
template <class T>
struct Far;
template <>
struct Far<__half> {
  static constexpr uint32_t bits = 0xd570u;
};
template <>
struct Far<__nv_bfloat16> {
  static constexpr uint32_t bits = 0xc2aeu;
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

// Chunks of rows that begin anywhere, in two calls: the first only loads, so that all loads of a thread are under way before the second uses any of
// them, and no branch keeps one chunk's from the next's.  w: the words that the chunk lies in, four or five, as far as they are within the row;
// off: whether the row begins in the middle of a word.  (load8 in their place, quantization in 8 bits floating point, us: rows 16000 x 2747 36 -> 33,
// their gate 66 -> 54, weights 48 -> 33.  Aligned pieces of 16 bytes, two a chunk, take fewer loads, and more instructions to pick the words:
// 41, 80 and 47.  The weighted sum's
// gradients, 8192 tokens of four, 4095 wide: 171 -> 144; the sum itself, whose rows begin differently, 96 -> 113, so it loads by load8.)
template <class T>
__device__ __forceinline__ int off_word(const T* row) {
  return (int)(reinterpret_cast<uintptr_t>(row) >> 1 & 1u);
}
template <class T>
__device__ __forceinline__ void load_words(const T* row, int off, int chunk, int cols, uint32_t (&w)[5]) {
  const uint32_t* word = reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint16_t*>(row) + (int64_t)chunk * 8 - off);
  const int left = cols - chunk * 8 + off;  // elements from the first word on
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = 2 * i + 2 <= left && (i > 0 || chunk > 0 || !off) && (i < 4 || off) ? word[i] : 0u;
}
template <class T>
__device__ __forceinline__ void take_words(const T* row, int off, int chunk, int cols, uint32_t (&w)[5], uint32_t (&r)[4]) {
  const int last = cols - 1 - chunk * 8;
  if ((chunk == 0 && off) || last < 8) {  // words of which a half is within the row
    const uint16_t* one = reinterpret_cast<const uint16_t*>(row) + (int64_t)chunk * 8;
    if (chunk == 0 && off && cols > 0) w[0] = (uint32_t)one[0] << 16;
    if (last >= 0 && last < 8 && ((last + off) & 1) == 0) {
      const uint32_t v = one[last];
#pragma unroll
      for (int i = 0; i < 5; ++i)
        if (2 * i == last + off) w[i] = v;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = __funnelshift_r(w[i], w[i + 1], off ? 16u : 0u);
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

// v = gate / (1 + exp(-gate)) * up of a chunk: g / (1 + p) * u with p = 2^(-g log2 e); 1 + an infinity has the reciprocal 0.
//
// FAR: gates below -87.3, whose p is beyond 2^126, are among them.  Their reciprocal is no normal float, and below -88.7 p is none either, while the
// product with a large u is one down to g = -181.  There 1 + p is p, and exp(g) is taken as exp(g / 4)^4, factor by factor: every product on the way
// is larger than the result, so none leaves the floats before it does.
template <class T, bool FAR>
__device__ __forceinline__ void silu_mul8(const uint32_t (&gate)[4], const uint32_t (&up)[4], float (&v)[8]) {
  float u[8];
  unpack8<T>(gate, v);
  unpack8<T>(up, u);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float p, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(v[e] * -1.44269504f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + p));
    const float t = v[e] * r * u[e];
    if (FAR && p > 0x1p126f) {
      const float h = expf(0.25f * v[e]);
      v[e] = u[e] * h * h * v[e] * h * h;
    } else {
      v[e] = t;
    }
  }
}
// Whether some of these gates may be as far.  Numbers of one sign are ordered as their bits are, the negative ones behind the others: what is behind
// -87 as an unsigned number of 16 bits is below it, or NaN.  (Two instructions a chunk and one branch for all of a thread's: 16000 x 2752 in 8 bits
// floating point 41.5 -> 42.0 us, 16000 x 2747 58.0 -> 57.6; the largest p of a chunk compared with 2^126, and a branch for each, 47.3 and 68.2.)
template <class T, int U>
__device__ __forceinline__ bool far_gates(const uint32_t (&gate)[U][4]) {
  constexpr uint32_t kFar = Far<T>::bits;
  uint32_t m = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) m = __vimax3_u16x2(__vimax3_u16x2(m, gate[u][0], gate[u][1]), gate[u][2], gate[u][3]);
  return max(m, m << 16) > (kFar << 16 | 0xffffu);
}

// max(a, |b|, |c|), NaN if one of them is
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

}  // namespace int8
}  // namespace blkq4
