// Tokens sorted by expert and back: the order of the choices, the rows of each expert behind one another, the weighted sum of a token's
// rows, and the gradients of both moves.
//
// Sort: a stable counting sort.  Every warp has a run of choices and a counter for each expert in shared memory; it goes through its run 32
// choices at a time, the lanes of one expert ranked among themselves, and counts; then the counters become the places where its choices of an expert
// begin (behind those of the experts, the CTAs and the warps before), and each choice's place is that and its rank.  Stable since runs, steps
// and lanes follow the choices' order; no atomic decides a place.  Up to 4096 choices are one CTA's; more are split over CTAs, whose counts a kernel before writes.
//
// Moves: bound by HBM and L2, 16 bytes a lane, a warp a stretch of a row.  The weighted sum is gathered (a token reads its rows, in the order
// of its choices, fp32), not scattered: no atomics, one rounding, the same result every time.  The gradient of the weighted sum reads y and the
// output's gradient once for both of its results.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <string>

#include "blkq4_tma.cuh"
#include "fp8.cuh"
#include "rows_io.cuh"

namespace blkq4 {
namespace experts {
namespace {

using namespace blkq4::int8;

// ---- sort ----
constexpr int kMaxWarps = 32;
constexpr int64_t kOneCta = 4096;  // (8192 choices: 12.1 us, by several CTAs 8.0; 4096: 8.7 and 8.6)
constexpr int kItems = 8;  // choices of a lane that are under way at a time

template <class Id>
__device__ __forceinline__ int key_of(const Id* ids, int64_t i, int n_experts) {
  const Id v = ids[i];
  return v >= 0 && v < (Id)n_experts ? (int)v : n_experts;
}

template <class Id>
__global__ void __launch_bounds__(1024) count_kernel(const Id* ids, int64_t n, int64_t chunk, int n_experts, int* counts) {
  extern __shared__ int own[];
  for (int e = threadIdx.x; e <= n_experts; e += blockDim.x) own[e] = 0;
  griddep_wait();
  griddep_launch_dependents();
  __syncthreads();
  const int64_t begin = (int64_t)blockIdx.x * chunk, end = min(n, begin + chunk);
  for (int64_t i = begin + threadIdx.x; i < end; i += blockDim.x) atomicAdd(&own[key_of(ids, i, n_experts)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e <= n_experts; e += blockDim.x) counts[(int64_t)blockIdx.x * (n_experts + 1) + e] = own[e];
}

// counts: [CTAs][n_experts + 1] of count_kernel, or null for a single CTA.  chunk: choices of a CTA, a multiple of its threads.
template <class Id>
__global__ void __launch_bounds__(1024) sort_kernel(const Id* ids, int64_t n, int64_t chunk, int n_experts, const int* counts, int* source,
                                                    int* places, int* offsets) {
  extern __shared__ int cells[];  // [warps][n_experts + 1]
  __shared__ int sums[kMaxWarps];
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, width = n_experts + 1;
  for (int i = threadIdx.x; i < warps * width; i += blockDim.x) cells[i] = 0;
  griddep_wait();
  griddep_launch_dependents();
  __syncthreads();
  const int64_t run = chunk / warps, begin = (int64_t)blockIdx.x * chunk + warp * run, end = min(n, begin + run);
  int* mine = cells + warp * width;
  // 32 choices at a time: how many of a choice's expert are ahead of it in the run, by the lanes that have the same one and the counter so far.
  // (The lanes by a vote for each bit of the number: the instruction that matches them takes a round for every expert among them, 8192 choices
  // of 32 experts 14.0 us instead of 12.1.)
  const int bits = 32 - __clz(width);
  auto take = [&](bool in, int key) {
    unsigned same = 0xffffffffu;
    for (int i = 0; i < bits; ++i) {
      const bool set = key >> i & 1;
      const unsigned with = __ballot_sync(0xffffffffu, set);
      same &= set ? with : ~with;
    }
    const int rank = __popc(same & ((1u << lane) - 1u));
    const int ahead = in ? mine[key] : 0;
    __syncwarp();
    if (in && rank == 0) mine[key] = ahead + __popc(same);
    __syncwarp();
    return ahead + rank;
  };
  int keys[kItems], ahead[kItems];
  auto load = [&](int64_t i0) {
#pragma unroll
    for (int t = 0; t < kItems; ++t) keys[t] = i0 + 32 * t + lane < end ? key_of(ids, i0 + 32 * t + lane, n_experts) : width;
  };
  const bool held = run <= 32 * kItems;  // the run stays in registers between its two passes
  for (int64_t i0 = begin; i0 < end; i0 += 32 * kItems) {
    load(i0);
#pragma unroll
    for (int t = 0; t < kItems; ++t)
      if (i0 + 32 * t < end) ahead[t] = take(keys[t] < width, keys[t]);
  }
  __syncthreads();
  int carry = 0;
  for (int e0 = 0; e0 < width; e0 += blockDim.x) {  // places of e0 + thread: behind all choices of the experts before
    const int e = e0 + threadIdx.x;
    int total = 0, before = 0;
    if (e < width) {
      if (counts) {
        for (unsigned b = 0; b < gridDim.x; ++b) {
          if (b == blockIdx.x) before = total;
          total += counts[(int64_t)b * width + e];
        }
      } else {
        for (int w = 0; w < warps; ++w) total += cells[w * width + e];
      }
    }
    int scan = total;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, scan, s);
      if (lane >= s) scan += v;
    }
    if (lane == 31) sums[warp] = scan;
    __syncthreads();
    int base = carry;
    for (int w = 0; w < warps; ++w) {
      if (w < warp) base += sums[w];
      carry += sums[w];
    }
    base += scan - total;
    if (e < width) {
      if (blockIdx.x == 0) offsets[e] = base;
      base += before;
      for (int w = 0; w < warps; ++w) {
        const int c = cells[w * width + e];
        cells[w * width + e] = base;
        base += c;
      }
    }
    __syncthreads();
  }
  for (int64_t i0 = begin; i0 < end; i0 += 32 * kItems) {
    if (!held) load(i0);
#pragma unroll
    for (int t = 0; t < kItems; ++t) {
      const int64_t i = i0 + 32 * t + lane;
      if (i0 + 32 * t >= end) break;
      const bool in = keys[t] < width;
      const int place = held ? (in ? mine[keys[t]] + ahead[t] : 0) : take(in, keys[t]);
      if (!in) continue;
      source[place] = (int)i;
      places[i] = keys[t] < n_experts ? place : -1;
    }
  }
}

// ---- moves ----
constexpr int kThreads = 128;

__device__ __forceinline__ float weight_at(const MoveParams& p, int64_t i) {
  if (p.weights_type == 2) return reinterpret_cast<const float*>(p.weights)[i];
  if (p.weights_type == kFp16) return __half2float(reinterpret_cast<const __half*>(p.weights)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.weights)[i]);
}
// The stretch of a row that a warp takes: U * 256 elements.
struct Part {
  int64_t row;
  int chunk;  // of the lane, its next ones 32 further on
};
__device__ __forceinline__ Part part_of(int parts, int U) {
  const int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  Part p;
  int part;
  if (i < 0xffffffffll) {
    p.row = (uint32_t)i / (uint32_t)parts;
    part = (int)((uint32_t)i % (uint32_t)parts);
  } else {
    p.row = i / parts;
    part = (int)(i % parts);
  }
  p.chunk = part * U * 32 + (threadIdx.x & 31);
  return p;
}
// The token of place p: -1 where it belongs to no expert.
__device__ __forceinline__ int choice_at(const MoveParams& p, int64_t place) {
  if (place >= *p.count) return -1;
  const int s = p.source[place];
  return s >= 0 && s < (int64_t)p.tokens * p.choices ? s : -1;
}

// Rows that begin anywhere are cut where the output's pieces of 16 bytes begin, so that all but a row's first and last are stored at once (8192
// tokens of four, 4095 wide: 126 -> 79 us).
template <class T, bool VEC, int U>
__global__ void __launch_bounds__(kThreads) gather_kernel(const MoveParams p, int parts) {
  griddep_wait();
  griddep_launch_dependents();
  const Part at = part_of(parts, U);
  if (at.row >= (int64_t)p.tokens * p.choices) return;
  const int choice = choice_at(p, at.row);
  const T* from = reinterpret_cast<const T*>(p.from) + (int64_t)(choice >= 0 ? choice / p.choices : 0) * p.ldf;
  T* to = reinterpret_cast<T*>(p.to) + at.row * p.ldt;
  uint32_t r[U][4] = {};
  if constexpr (VEC) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (choice >= 0 && (at.chunk + 32 * u) * 8 < p.cols) load8<T, VEC>(from, at.chunk + 32 * u, p.cols, r[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if ((at.chunk + 32 * u) * 8 < p.cols) store8<T, VEC>(to, at.chunk + 32 * u, p.cols, r[u]);
  } else {
    const int before = (int)(reinterpret_cast<uintptr_t>(to) / 2 & 7u), cols = p.cols + before;  // elements that the first piece lacks
    const int readable = choice >= 0 ? cols : 0;
    const T* cut = from - before;
    const int off = off_word(cut);
    uint32_t w[U][5] = {};
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at.chunk + 32 * u > 0) load_words(cut, off, at.chunk + 32 * u, readable, w[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = at.chunk + 32 * u;
      if (c * 8 >= cols) continue;
      if (c == 0) {
        const uint16_t* one = reinterpret_cast<const uint16_t*>(from);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < 8 - before && e < p.cols) reinterpret_cast<uint16_t*>(to)[e] = choice >= 0 ? one[e] : (uint16_t)0;
        continue;
      }
      take_words(cut, off, c, readable, w[u], r[u]);
      if (c * 8 + 8 <= cols) *reinterpret_cast<uint4*>(to - before + (int64_t)c * 8) = make_uint4(r[u][0], r[u][1], r[u][2], r[u][3]);
      else store8<T, false>(to - before, c, cols, r[u]);
    }
  }
}

template <class T, bool VEC, int U>
__global__ void __launch_bounds__(kThreads) combine_kernel(const MoveParams p, int parts) {
  griddep_wait();
  griddep_launch_dependents();
  const Part at = part_of(parts, U);
  if (at.row >= p.tokens) return;
  const int64_t first = at.row * p.choices, rows = (int64_t)p.tokens * p.choices;
  float sum[U][8] = {};
  constexpr int kAhead = 4;  // rows under way at a time
  for (int j0 = 0; j0 < p.choices; j0 += kAhead) {
    uint32_t r[kAhead][U][4] = {};
    float w[kAhead] = {};
    bool taken[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int place = j0 + j < p.choices ? p.places[first + j0 + j] : -1;
      taken[j] = place >= 0 && place < rows;
      if (taken[j]) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if ((at.chunk + 32 * u) * 8 < p.cols)
            load8<T, VEC>(reinterpret_cast<const T*>(p.from) + (int64_t)place * p.ldf, at.chunk + 32 * u, p.cols, r[j][u]);
        w[j] = p.weights ? weight_at(p, first + j0 + j) : 1.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (!taken[j]) continue;  // a choice that was dropped has no row, whatever its weight is
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[8];
        unpack8<T>(r[j][u], v);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[u][e] = fmaf(w[j], v[e], sum[u][e]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if ((at.chunk + 32 * u) * 8 >= p.cols) continue;
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = pack2<T>(sum[u][2 * i], sum[u][2 * i + 1]);
    store8<T, VEC>(reinterpret_cast<T*>(p.to) + at.row * p.ldt, at.chunk + 32 * u, p.cols, o);
  }
}

// A warp a place: to[p] = weight * d, dots[choice] = sum of y[p] * d, with d the row of the place's token; either may be left out (null), and its
// reads or writes with it (8192 tokens of four, 4096 wide: both 112 us, the first 69, the second 64).
template <class T, bool VEC>
__global__ void __launch_bounds__(kThreads) weigh_kernel(const MoveParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (row >= (int64_t)p.tokens * p.choices) return;
  const int lane = threadIdx.x & 31, choice = choice_at(p, row);
  const float w = choice >= 0 ? weight_at(p, choice) : 0.0f;
  const T* from = reinterpret_cast<const T*>(p.from) + (int64_t)(choice >= 0 ? choice / p.choices : 0) * p.ldf;
  const T* y = reinterpret_cast<const T*>(p.y) + row * p.ldy;
  T* to = reinterpret_cast<T*>(p.to) + row * p.ldt;
  const int chunks = (p.cols + 7) / 8, cols = choice >= 0 ? p.cols : 0;  // (of a place without an expert nothing is read)
  float dot = 0.0f;
  constexpr int kAhead = 4;
  for (int c0 = lane; c0 < chunks; c0 += 32 * kAhead) {
    uint32_t a[kAhead][4] = {}, b[kAhead][4] = {}, wa[VEC ? 1 : kAhead][5], wb[VEC ? 1 : kAhead][5];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int c = c0 + 32 * u;
      if constexpr (VEC) {
        if (choice >= 0 && c < chunks) {
          load8<T, VEC>(from, c, p.cols, a[u]);
          if (p.dots) load8<T, VEC>(y, c, p.cols, b[u]);
        }
      } else {
        load_words(from, off_word(from), c, cols, wa[u]);
        load_words(y, off_word(y), c, p.dots ? cols : 0, wb[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int c = c0 + 32 * u;
      if constexpr (!VEC) {
        take_words(from, off_word(from), c, cols, wa[u], a[u]);
        take_words(y, off_word(y), c, p.dots ? cols : 0, wb[u], b[u]);
      }
      if (c >= chunks) continue;
      float d[8], v[8];
      unpack8<T>(a[u], d);
      unpack8<T>(b[u], v);
      uint32_t o[4] = {};
#pragma unroll
      for (int e = 0; e < 8; ++e) dot = fmaf(d[e], v[e], dot);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (choice >= 0) o[i] = pack2<T>(w * d[2 * i], w * d[2 * i + 1]);
      if (p.to) store8<T, VEC>(to, c, p.cols, o);
    }
  }
  if (!p.dots) return;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
  if (lane == 0) {
    // (the choices of no expert stand behind the others in `source`)
    const int s = p.source[row];
    if (s >= 0 && s < (int64_t)p.tokens * p.choices) p.dots[s] = choice >= 0 ? dot : 0.0f;
  }
}

template <class... Params, class... Args>
std::string launch(void (*kernel)(Params...), int64_t ctas, int threads, size_t smem, cudaStream_t stream, Args... args) {
  if (ctas > 0x7fffffffll) return "too many rows";
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
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
bool rows_on_16(const void* ptr, int64_t ld, int64_t rows) {
  return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && (rows <= 1 || ld % 8 == 0);
}

struct SortPlan {
  int64_t ctas, chunk;
  int warps;
};
SortPlan plan_sort(int64_t n, int n_experts) {
  SortPlan s;
  // counters of all warps in shared memory
  const int most = n_experts < 1024 ? 32 : 16;
  if (n <= kOneCta) {
    s.ctas = 1;
    // a warp for 32 choices, or for as many counters
    s.warps = (int)std::min<int64_t>(most, std::max<int64_t>(n, n_experts + 1) / 32 + 1);
    s.chunk = (n + 32 * s.warps - 1) / (32 * s.warps) * (32 * s.warps);
  } else {
    s.warps = most;
    const int64_t step = 32 * s.warps;
    s.chunk = std::max<int64_t>(2 * step, ((n + 147) / 148 + step - 1) / step * step);
    s.ctas = (n + s.chunk - 1) / s.chunk;
  }
  return s;
}
template <class Id>
std::string sort_typed(const Id* ids, int64_t n, int n_experts, int* source, int* places, int* offsets, int* counts, cudaStream_t stream) {
  const SortPlan s = plan_sort(n, n_experts);
  const int threads = 32 * s.warps;
  const size_t smem = (size_t)s.warps * (n_experts + 1) * 4;
  static std::atomic<int> granted[64];
  if (smem > 40 * 1024) {
    cudaError_t e = ensure_dynamic_smem(sort_kernel<Id>, smem, granted);
    if (e != cudaSuccess) return cudaGetErrorString(e);
  }
  if (s.ctas > 1) {
    std::string e = launch(count_kernel<Id>, s.ctas, threads, (size_t)(n_experts + 1) * 4, stream, ids, n, s.chunk, n_experts, counts);
    if (!e.empty()) return e;
  }
  return launch(sort_kernel<Id>, s.ctas, threads, smem, stream, ids, n, s.chunk, n_experts, (const int*)(s.ctas > 1 ? counts : nullptr),
                source, places, offsets);
}

bool many_cols(int64_t rows, int cols) { return rows * cols >= 148 * 16 * 1024; }  // elements for 64 warps an SM, by stretches of 256

template <class T>
std::string gather_typed(const MoveParams& p, cudaStream_t stream) {
  const int64_t rows = (int64_t)p.tokens * p.choices;
  const bool vec = rows_on_16(p.from, p.ldf, p.tokens) && rows_on_16(p.to, p.ldt, rows);
  // four loads of a lane under way where there are enough of them for that
  const bool many = many_cols(rows, p.cols) && p.cols > 512;
  const int U = many ? 4 : 1, parts = (p.cols + (vec ? 0 : 7) + 256 * U - 1) / (256 * U);
  const int64_t ctas = (rows * parts + kThreads / 32 - 1) / (kThreads / 32);
  if (many)
    return vec ? launch(gather_kernel<T, true, 4>, ctas, kThreads, 0, stream, p, parts) : launch(gather_kernel<T, false, 4>, ctas, kThreads, 0, stream, p, parts);
  return vec ? launch(gather_kernel<T, true, 1>, ctas, kThreads, 0, stream, p, parts) : launch(gather_kernel<T, false, 1>, ctas, kThreads, 0, stream, p, parts);
}
template <class T>
std::string combine_typed(const MoveParams& p, cudaStream_t stream) {
  const bool vec = rows_on_16(p.from, p.ldf, (int64_t)p.tokens * p.choices) && rows_on_16(p.to, p.ldt, p.tokens);
  // two stretches a warp where that leaves enough of them: 8192 tokens of four, 4096 wide, 63.9 -> 57.3 us, but 16 of eight 2.9 -> 3.3; rows that
  // begin off 16 bytes take more registers and are slower by it, 4095 wide 96 -> 126 us
  const bool two = vec && many_cols(p.tokens, p.cols) && p.cols > 256;
  const int parts = (p.cols + 256 * (1 + two) - 1) / (256 * (1 + two));
  const int64_t ctas = ((int64_t)p.tokens * parts + kThreads / 32 - 1) / (kThreads / 32);
  if (two) return launch(combine_kernel<T, true, 2>, ctas, kThreads, 0, stream, p, parts);
  return vec ? launch(combine_kernel<T, true, 1>, ctas, kThreads, 0, stream, p, parts) : launch(combine_kernel<T, false, 1>, ctas, kThreads, 0, stream, p, parts);
}
template <class T>
std::string weigh_typed(const MoveParams& p, cudaStream_t stream) {
  const int64_t rows = (int64_t)p.tokens * p.choices, ctas = (rows + kThreads / 32 - 1) / (kThreads / 32);
  return rows_on_16(p.from, p.ldf, p.tokens) && (!p.dots || rows_on_16(p.y, p.ldy, rows)) && (!p.to || rows_on_16(p.to, p.ldt, rows))
             ? launch(weigh_kernel<T, true>, ctas, kThreads, 0, stream, p)
             : launch(weigh_kernel<T, false>, ctas, kThreads, 0, stream, p);
}

}  // namespace

size_t sort_workspace(int64_t n, int n_experts) {
  const SortPlan s = plan_sort(n, n_experts);
  return s.ctas > 1 ? (size_t)s.ctas * (n_experts + 1) * 4 : 0;
}
std::string launch_sort(const void* ids, bool wide, int64_t n, int n_experts, int* source, int* places, int* offsets, void* workspace,
                        cudaStream_t stream) {
  int* counts = reinterpret_cast<int*>(workspace);
  return wide ? sort_typed(reinterpret_cast<const long long*>(ids), n, n_experts, source, places, offsets, counts, stream)
              : sort_typed(reinterpret_cast<const int*>(ids), n, n_experts, source, places, offsets, counts, stream);
}
std::string launch_gather(Dtype dtype, const MoveParams& p, cudaStream_t stream) {
  return dtype == kFp16 ? gather_typed<__half>(p, stream) : gather_typed<__nv_bfloat16>(p, stream);
}
std::string launch_combine(Dtype dtype, const MoveParams& p, cudaStream_t stream) {
  return dtype == kFp16 ? combine_typed<__half>(p, stream) : combine_typed<__nv_bfloat16>(p, stream);
}
std::string launch_weigh(Dtype dtype, const MoveParams& p, cudaStream_t stream) {
  return dtype == kFp16 ? weigh_typed<__half>(p, stream) : weigh_typed<__nv_bfloat16>(p, stream);
}

}  // namespace experts
}  // namespace blkq4
