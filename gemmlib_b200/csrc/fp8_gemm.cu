// Product of e4m3 rows with an fp32 scale for each 128 k and e4m3 weights with one for each 128 x 128, for sm_100a:
//   out[m, n] = T(sum over blocks b of k of x_scale[m, b] * w_scale[n / 128, b] * (sum over k in b of x[m, k] w[n, k]) + bias[n])
// and the same for a layer of experts, where rows [offsets[e], offsets[e + 1]) have weight e.
//
// Both operands are K-major rows of bytes: TMA brings 128 k of a tile at a time into shared memory with the 128-byte swizzle, and tcgen05.mma
// (kind::f8f6f4, fp32 accumulators) multiplies them from there.  A step of the pipeline is a block of k, so the sum of a step is what the scales
// apply to: every step starts its accumulator anew in one of several buffers of tensor memory, from which warps take it, scale it and add it up
// in fp32 registers under the MMAs of the next steps.  The scales' product goes to a value with one multiply-add of its own.
//
// Two kernels.  fp8_rows_kernel (here): 128 weight rows (TMEM lanes) x 16 to 128 activation rows a tile, for few rows, where the weights'
// bytes are what counts.  fp8_wide_kernel (fp8_gemm_wide.cuh): 128 activation rows (TMEM lanes) x 256 weight rows, for many.
//
// Experts: the offsets are on the device and stay there.  Every CTA reads them once, counts the tiles of each expert, and walks through every
// gridDim-th tile of them all; so the launch does not depend on them.  They are read as a rising sequence within the rows (a value that is none
// is taken for the nearest that is), so that no offsets lead out of bounds.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstddef>
#include <cstdint>
#include <string>

#include "blkq4_common.cuh"
#include "blkq4_tc.cuh"
#include "blkq4_tma.cuh"
#include "fp8.cuh"
#include "ms_blkq4gemm.h"

namespace blkq4 {
namespace fp8 {

__device__ int g_fp8_error = 0;  // 0 ok; otherwise (role << 8) | stage of the wait that gave up

namespace {

using namespace blkq4::int8;
using tc::st_async_v4;
using tc::try_wait_cluster;

constexpr int kStepK = kBlock;              // k of a pipeline step: one 128-byte swizzle row, one scale
constexpr int kTileN = 128;                 // weight rows of a tile
constexpr uint32_t kWeightBytes = kTileN * kStepK;
constexpr long long kWaitCycles = 4000000000ll;  // ~2 s: far beyond any legitimate wait

__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int who) {
  return mbar_wait_bounded(bar, parity, abort_flag, &g_fp8_error, who, kWaitCycles);
}
// `wait` of a whole warp, with one answer for all of it.  abort_at: the flag's address in shared memory.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, uint32_t abort_at, int who) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const long long t0 = clock64();
  for (;;) {
    if (__all_sync(0xffffffffu, mbar_try_wait_hint(bar, parity, 1000u))) return true;
    const bool late = clock64() - t0 > kWaitCycles;
    int given_up;
    asm volatile("ld.volatile.shared.s32 %0, [%1];" : "=r"(given_up) : "r"(abort_at) : "memory");
    if (__any_sync(0xffffffffu, late || given_up != 0)) {
      if (late) {
        asm volatile("st.volatile.shared.s32 [%0], %1;" ::"r"(abort_at), "r"(1) : "memory");
        atomicCAS(&g_fp8_error, 0, who);
      }
      return false;
    }
  }
}
// `wait` on a barrier that other CTAs of the cluster arrive on.
__device__ __forceinline__ bool wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag, int who) {
  const long long t0 = clock64();
  while (!try_wait_cluster(bar, parity)) {
    if (*abort_flag) return false;
    if (clock64() - t0 > kWaitCycles) {
      *abort_flag = 1;
      atomicCAS(&g_fp8_error, 0, who);
      return false;
    }
  }
  return true;
}
// Instruction descriptor of kind::f8f6f4: fp32 accumulator (bits 4-5 = 1), e4m3 A and B (bits 7-9 and 10-12 = 0), both K-major,
// N >> 3 in bits 17-22, M >> 4 in bits 24-28.
__host__ __device__ constexpr uint32_t make_idesc_e4m3(int umma_m, int umma_n) {
  return (1u << 4) | ((uint32_t)(umma_n >> 3) << 17) | ((uint32_t)(umma_m >> 4) << 24);
}
// The four MMAs of a step: 32 k each, both operands two descriptor units (32 bytes) further on.  The first one starts the sum.
__device__ __forceinline__ void umma_e4m3_x4(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a0, a1, a2, a3, b0, b1, b2, b3;\n\t.reg .b32 x1, x2, x3, y1, y2, y3;\n\t"
      "setp.ne.b32 p, 0, 0;\n\t"
      "setp.eq.b32 q, 0, 0;\n\t"
      "add.u32 x1, %1, 2;\n\tadd.u32 x2, %1, 4;\n\tadd.u32 x3, %1, 6;\n\t"
      "add.u32 y1, %2, 2;\n\tadd.u32 y2, %2, 4;\n\tadd.u32 y3, %2, 6;\n\t"
      "mov.b64 a0, {%1, %3};\n\tmov.b64 a1, {x1, %3};\n\tmov.b64 a2, {x2, %3};\n\tmov.b64 a3, {x3, %3};\n\t"
      "mov.b64 b0, {%2, %3};\n\tmov.b64 b1, {y1, %3};\n\tmov.b64 b2, {y2, %3};\n\tmov.b64 b3, {y3, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a0, b0, %4, p;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a1, b1, %4, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a2, b2, %4, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a3, b3, %4, q;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc)
      : "memory");
}

// Groups of eight columns, 16 columns apart, there when it returns: loads and wait are one statement, so that no use of the registers can
// come between them.
__device__ __forceinline__ void tmem_ld_now(uint32_t taddr, uint32_t (&r)[1][8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0][0]), "=r"(r[0][1]), "=r"(r[0][2]), "=r"(r[0][3]), "=r"(r[0][4]), "=r"(r[0][5]), "=r"(r[0][6]), "=r"(r[0][7])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_now(uint32_t taddr, uint32_t (&r)[2][8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%16];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%17];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0][0]), "=r"(r[0][1]), "=r"(r[0][2]), "=r"(r[0][3]), "=r"(r[0][4]), "=r"(r[0][5]), "=r"(r[0][6]), "=r"(r[0][7]),
        "=r"(r[1][0]), "=r"(r[1][1]), "=r"(r[1][2]), "=r"(r[1][3]), "=r"(r[1][4]), "=r"(r[1][5]), "=r"(r[1][6]), "=r"(r[1][7])
      : "r"(taddr), "r"(taddr + 16u)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_now(uint32_t taddr, uint32_t (&r)[4][8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%32];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%33];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%16,%17,%18,%19,%20,%21,%22,%23}, [%34];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%24,%25,%26,%27,%28,%29,%30,%31}, [%35];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0][0]), "=r"(r[0][1]), "=r"(r[0][2]), "=r"(r[0][3]), "=r"(r[0][4]), "=r"(r[0][5]), "=r"(r[0][6]), "=r"(r[0][7]),
        "=r"(r[1][0]), "=r"(r[1][1]), "=r"(r[1][2]), "=r"(r[1][3]), "=r"(r[1][4]), "=r"(r[1][5]), "=r"(r[1][6]), "=r"(r[1][7]),
        "=r"(r[2][0]), "=r"(r[2][1]), "=r"(r[2][2]), "=r"(r[2][3]), "=r"(r[2][4]), "=r"(r[2][5]), "=r"(r[2][6]), "=r"(r[2][7]),
        "=r"(r[3][0]), "=r"(r[3][1]), "=r"(r[3][2]), "=r"(r[3][3]), "=r"(r[3][4]), "=r"(r[3][5]), "=r"(r[3][6]), "=r"(r[3][7])
      : "r"(taddr), "r"(taddr + 16u), "r"(taddr + 32u), "r"(taddr + 48u)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map),
      "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void prefetch_l2_3d(const CUtensorMap* map, int x, int y, int z) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(map), "r"(x), "r"(y), "r"(z) : "memory");
}
// Four bytes, or zeros in their place.
__device__ __forceinline__ void copy4(uint32_t dst, const float* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
}
// 16 bytes, of which the first `bytes` are copied and the others zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const float* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// Arrives on the barrier once this thread's copies so far have landed.
__device__ __forceinline__ void arrive_behind_copies(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

struct Params {
  int M, N;
  int n_tiles;
  int k_steps;
  int experts;
  const int* offsets;  // null: one weight
  int zero_rest;
  int split;       // CTAs of a tile: the cluster size; above 1 every CTA has one tile, and there are no offsets
  int k_per_cta;   // steps of each, the last one what is left
  int slice;       // activation rows whose sums one CTA of the cluster collects, a multiple of 8
  int stages;
  uint32_t exchange_bytes;  // behind the stages: what a CTA collects
  int early;       // weights may be copied before the kernels ahead in the stream have completed
  int pairs_of_columns;  // two neighbouring outputs of a row, from an even n on, may be stored at once
  void* out;
  int64_t ldo;
  const float* x_scales;
  int64_t ldxs;
  const float* w_scales;
  int64_t ldws, ws_stride;
  const void* bias;
};

// ---- which tiles there are ----
// begin(e): first row of expert e (begin(experts): the end); first(e): number of tile rows of the experts before e.  Shared memory, by addresses of
// 32 bits: the sums leave few registers.
__device__ __forceinline__ int lds(uint32_t at) {
  int v;
  asm volatile("ld.shared.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void sts(uint32_t at, int v) { asm volatile("st.shared.s32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
struct Experts {
  uint32_t begins, firsts;
  __device__ __forceinline__ int begin(int e) const { return lds(begins + 4u * (uint32_t)e); }
  __device__ __forceinline__ int first(int e) const { return lds(firsts + 4u * (uint32_t)e); }
};
__host__ __device__ constexpr uint32_t experts_bytes(int experts) { return 8u * (uint32_t)(experts + 1); }
// All threads of the CTA; behind griddep_wait where there are offsets.  `high`: rows of a tile.
__device__ __forceinline__ void count_tiles(const Experts& t, const int* offsets, int experts, int rows, int high) {
  if (offsets == nullptr) {
    if (threadIdx.x == 0) {
      sts(t.begins, 0), sts(t.begins + 4u, rows);
      sts(t.firsts, 0), sts(t.firsts + 4u, (rows + high - 1) / high);
    }
    __syncthreads();
    return;
  }
  for (int e = threadIdx.x; e <= experts; e += blockDim.x) sts(t.begins + 4u * (uint32_t)e, min(max(offsets[e], 0), rows));
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int top = 0, tiles = 0;  // of the experts before
    for (int e0 = 0; e0 <= experts; e0 += 32) {
      const int e = e0 + lane;
      int v = max(top, e <= experts ? t.begin(e) : 0);
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, v, s);
        if (lane >= s) v = max(v, o);
      }
      // tile rows of the expert before this one, which ends here
      int before = __shfl_up_sync(0xffffffffu, v, 1);
      if (lane == 0) before = top;
      int sum = e > 0 ? (v - before + high - 1) / high : 0;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, sum, s);
        if (lane >= s) sum += o;
      }
      if (e <= experts) {
        sts(t.begins + 4u * (uint32_t)e, v);
        sts(t.firsts + 4u * (uint32_t)e, tiles + sum);
      }
      top = __shfl_sync(0xffffffffu, v, 31);
      tiles += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  __syncthreads();
}
// The tiles of a CTA, every step-th.  An expert's tiles follow one another, those of one column of weight rows first.
struct Walk {
  Experts t;
  int tile, step, count, n_tiles, e;
  __device__ __forceinline__ Walk(const Experts& t, int experts, int n_tiles, int first, int step)
      : t(t), tile(first), step(step), count(t.first(experts) * n_tiles), n_tiles(n_tiles), e(0) {}
  // `high` rows a tile: m0 .. end
  __device__ __forceinline__ bool next(int high, int& expert, int& n_tile, int& m0, int& end) {
    if (tile >= count) return false;
    while (t.first(e + 1) * n_tiles <= tile) ++e;
    const int m_tiles = t.first(e + 1) - t.first(e), in = tile - t.first(e) * n_tiles;
    n_tile = in / m_tiles;
    expert = e;
    m0 = t.begin(e) + (in - n_tile * m_tiles) * high;
    end = min(t.begin(e + 1), m0 + high);
    tile += step;
    return true;
  }
};
// Rows of no expert, by some of the CTA's threads.
template <class T>
__device__ __forceinline__ void zero_rows(const Experts& t, int experts, int M, int N, T* out, int64_t ldo, int thread, int threads) {
  const int first = t.begin(0), behind = t.begin(experts), rest = M - behind;
  for (int i = blockIdx.x; i < first + rest; i += gridDim.x) {
    uint16_t* row = reinterpret_cast<uint16_t*>(out) + (int64_t)(i < first ? i : behind + i - first) * ldo;
    for (int n = thread; n < N; n += threads) row[n] = 0;
  }
}

constexpr int kMaxStages = 16, kMaxBuffers = 8, kScaleSlots = 8;
constexpr int kEpiWarps = 8, kXWarp = 2 + kEpiWarps, kScaleWarp = kXWarp + 1, kRowsThreads = 32 * (kScaleWarp + 1);
constexpr uint32_t kBarBytes = 1024;  // barriers, abort flag, TMEM address
constexpr uint32_t kSmemAlone = 200u * 1024, kSmemOfTwo = 100u * 1024;  // stages and exchange of a CTA alone on its SM, of one of two
__host__ __device__ constexpr uint32_t smem_room(int BN) { return BN <= 32 ? kSmemOfTwo : kSmemAlone; }

template <int BN>
struct RowsShape {
  static constexpr int kGroups = BN / 16;                 // of eight columns, of a warp
  static constexpr int kBuffers = BN <= 32 ? 128 / BN : 256 / BN;  // accumulators
  static constexpr uint32_t kColumns = BN * kBuffers;
  static constexpr uint32_t kStageBytes = kWeightBytes + BN * kStepK;
  static constexpr uint32_t kScaleBytes = kScaleSlots * BN * 4;
  static constexpr int kPerSm = BN <= 32 ? 2 : 1;
};

// The most that a plan asks for: what a kernel is allowed, once a device.  (Every caller allows the same, since a call replaces what one before allowed.)
__host__ __device__ constexpr uint32_t rows_most_smem(int BN) {
  return smem_room(BN) + (uint32_t)kScaleSlots * (uint32_t)BN * 4 + kBarBytes + experts_bytes(kMaxExperts) + 1024;
}

// Grid: the tiles of a walk, or tiles * split CTAs, those of a tile a cluster.
template <class T, int BN>
__global__ void __launch_bounds__(kRowsThreads, RowsShape<BN>::kPerSm)
fp8_rows_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const Params p) {
  using S = RowsShape<BN>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t exchange_at = (uint32_t)p.stages * S::kStageBytes, scales_at = exchange_at + p.exchange_bytes;
  const uint32_t bars_at = scales_at + S::kScaleBytes, bars = base + bars_at;
  uint8_t* bars_ptr = base_ptr + bars_at;
  auto full = [&](int s) { return bars + 16u * (uint32_t)s; };
  auto empty = [&](int s) { return bars + 16u * (uint32_t)s + 8u; };
  auto acc_full = [&](int b) { return bars + 16u * (uint32_t)(kMaxStages + b); };
  auto acc_empty = [&](int b) { return bars + 16u * (uint32_t)(kMaxStages + b) + 8u; };
  auto scale_full = [&](int s) { return bars + 16u * (uint32_t)(kMaxStages + kMaxBuffers + s); };
  auto scale_empty = [&](int s) { return bars + 16u * (uint32_t)(kMaxStages + kMaxBuffers + s) + 8u; };
  constexpr uint32_t kWords = 16u * (kMaxStages + kMaxBuffers + kScaleSlots);
  static_assert(kWords + 16 <= kBarBytes && rows_most_smem(BN) <= (BN <= 32 ? 113u : 227u) * 1024);
  const uint32_t exchanged = bars + kWords;
  const uint32_t abort_at = bars + kWords + 8u;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars_ptr + kWords + 8);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars_ptr + kWords + 12);
  const Experts table{bars + kBarBytes, bars + kBarBytes + 4u * (uint32_t)(p.experts + 1)};

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = (int)blockIdx.x % p.split, first_tile = (int)blockIdx.x / p.split, tile_step = (int)gridDim.x / p.split;
  const int ks0 = part * p.k_per_cta, steps = min(p.k_per_cta, p.k_steps - ks0);
  if (threadIdx.x == 0) {
    prefetch_tensormap(&tm_w);
    prefetch_tensormap(&tm_x);
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(full(i), 2);
      mbar_init(empty(i), 1);
    }
    for (int i = 0; i < S::kBuffers; ++i) {
      mbar_init(acc_full(i), 1);
      mbar_init(acc_empty(i), kEpiWarps);
    }
    for (int i = 0; i < kScaleSlots; ++i) {
      mbar_init(scale_full(i), 32);
      mbar_init(scale_empty(i), kEpiWarps);
    }
    mbar_init(exchanged, 1);
    *abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(S::kColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (p.offsets) griddep_wait();  // they are an operator's output
  tc::tc_fence_before();
  count_tiles(table, p.offsets, p.experts, p.M, BN);
  // of a split tile, the only one of its CTA
  const int split_rows = p.split > 1 ? min(BN, p.M - first_tile % table.first(1) * BN) : BN;
  const int first_row = min(split_rows, part * p.slice), end_row = min(split_rows, first_row + p.slice);  // whose sums end up here
  if (p.split > 1) {
    if (threadIdx.x == 0)
      mbar_arrive_expect_tx(exchanged, (uint32_t)((p.split - 1) * ((end_row - first_row + 3) / 4) * kTileN * 16));
    tc::cluster_sync_all();  // the others' barriers exist before anything is sent to them
  }
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  int expert, n_tile, m0, end;

  if (warp == 0) {  // ---- weights
    if (elect_one()) {
      Walk walk(table, p.experts, p.n_tiles, first_tile, tile_step);
      int s = 0;
      uint32_t parity = 1;  // (the first round finds fresh barriers: the phase before their first one is complete)
      auto copy = [&](int ks) {
        mbar_arrive_expect_tx(full(s), kWeightBytes);
        tma_load_3d(base + (uint32_t)s * S::kStageBytes, &tm_w, (ks0 + ks) * kStepK, n_tile * kTileN, expert, full(s));
        if (++s == p.stages) s = 0, parity ^= 1u;
      };
      bool first = true;
      while (walk.next(BN, expert, n_tile, m0, end)) {
        int ks = 0;
        if (first) {
          first = false;
          const int ahead = min(steps, p.stages);
          if (p.offsets) {
          } else if (p.early) {
            while (ks < ahead) copy(ks), ++ks;
          } else {  // at least on their way into L2, where a write that is still to come would find them
            for (int j = 0; j < ahead; ++j) prefetch_l2_3d(&tm_w, (ks0 + j) * kStepK, n_tile * kTileN, expert);
          }
          griddep_wait();
          griddep_launch_dependents();
        }
        for (; ks < steps; ++ks) {
          if (!wait(empty(s), parity, abort_flag, 0x100)) goto weights_done;
          copy(ks);
        }
      }
    weights_done:;
    }
  } else if (warp == kXWarp) {  // ---- activations
    if (elect_one()) {
      griddep_wait();
      Walk walk(table, p.experts, p.n_tiles, first_tile, tile_step);
      int s = 0;
      uint32_t parity = 1;
      while (walk.next(BN, expert, n_tile, m0, end)) {
        for (int ks = 0; ks < steps; ++ks) {
          if (!wait(empty(s), parity, abort_flag, 0x110)) goto x_done;
          mbar_arrive_expect_tx(full(s), BN * kStepK);
          tma_load_2d(base + (uint32_t)s * S::kStageBytes + kWeightBytes, &tm_x, (ks0 + ks) * kStepK, m0, full(s));
          if (++s == p.stages) s = 0, parity ^= 1u;
        }
      }
    x_done:;
    }
  } else if (warp == kScaleWarp) {  // ---- the activations' scales of a step: one of each row, a row of scales apart
    griddep_wait();
    Walk walk(table, p.experts, p.n_tiles, first_tile, tile_step);
    int s = 0;
    uint32_t parity = 1;
    while (walk.next(BN, expert, n_tile, m0, end)) {
      constexpr int kOwn = (BN + 31) / 32;
      const float* src[kOwn];
      bool in[kOwn];
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        in[i] = m0 + lane + 32 * i < end;
        src[i] = p.x_scales + (in[i] ? (int64_t)(m0 + lane + 32 * i) * p.ldxs + ks0 : 0);
      }
      for (int ks = 0; ks < steps; ++ks) {
        if (!wait(scale_empty(s), parity, abort_flag, 0x120)) goto scales_done;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          if (lane + 32 * i < BN) copy4(base + scales_at + (uint32_t)(s * BN + lane + 32 * i) * 4u, src[i], in[i]);
          src[i] += in[i];
        }
        arrive_behind_copies(scale_full(s));
        if (++s == kScaleSlots) s = 0, parity ^= 1u;
      }
    }
  scales_done:;
    __syncwarp();
  } else if (warp == 1) {  // ---- MMAs
    if (elect_one()) {
      griddep_wait();  // or the limit of the waits below would count the kernel ahead
      constexpr uint32_t idesc = make_idesc_e4m3(kTileN, BN);
      const uint64_t desc = tc::make_sw128_kmajor_desc(0);
      const uint32_t desc_hi = (uint32_t)(desc >> 32), desc_lo = (uint32_t)desc | ((base >> 4) & 0x3FFFu);
      Walk walk(table, p.experts, p.n_tiles, first_tile, tile_step);
      int s = 0, b = 0;
      uint32_t parity = 0, acc_parity = 1;
      while (walk.next(BN, expert, n_tile, m0, end)) {
        for (int ks = 0; ks < steps; ++ks) {
          if (!wait(acc_empty(b), acc_parity, abort_flag, 0x200)) goto mma_done;
          if (!wait(full(s), parity, abort_flag, 0x210)) goto mma_done;
          tc::tc_fence_after();
          const uint32_t lo = desc_lo + (uint32_t)s * (S::kStageBytes >> 4);
          umma_e4m3_x4(tmem + (uint32_t)(b * BN), lo, lo + (kWeightBytes >> 4), desc_hi, idesc);
          tc::umma_commit(empty(s));
          tc::umma_commit(acc_full(b));
          if (++s == p.stages) s = 0, parity ^= 1u;
          if (++b == S::kBuffers) b = 0, acc_parity ^= 1u;
        }
      }
    mma_done:;
    }
  } else {
    // ---- sums and outputs: a warp has the 32 weight rows n of its quarter of the TMEM lanes (by warp number mod 4), two warps share a
    // quarter on groups of 8 activation rows m (TMEM columns) in turn
    const int quarter = warp & 3, turn = (warp - 2) >> 2, n_l = quarter * 32 + lane;
    const uint32_t tmem_row = tmem + ((uint32_t)(quarter * 32) << 16) + 8u * (uint32_t)turn;
    const float* scales = reinterpret_cast<const float*>(base_ptr + scales_at) + 8 * turn;
    T* out = reinterpret_cast<T*>(p.out);
    griddep_wait();  // scales and the output belong to stream order
    Walk walk(table, p.experts, p.n_tiles, first_tile, tile_step);
    int s = 0, b = 0;
    uint32_t s_parity = 0, b_parity = 0;
    while (walk.next(BN, expert, n_tile, m0, end)) {
      const int n = n_tile * kTileN + n_l;
      const float* w_scale = p.w_scales + expert * p.ws_stride + n_tile * p.ldws + ks0;
      float bias = 0.0f;
      if (p.bias && n < p.N) bias = to_float(reinterpret_cast<const T*>(p.bias)[n]);
      float acc[S::kGroups][8];
#pragma unroll
      for (int g = 0; g < S::kGroups; ++g)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[g][j] = 0.0f;
      float next = w_scale[0];
#pragma unroll 1
      for (int ks = 0; ks < steps; ++ks) {
        const float ws = next;
        if (ks + 1 < steps) next = w_scale[ks + 1];
        if (!wait_warp(scale_full(s), s_parity, abort_at, 0x300) || !wait_warp(acc_full(b), b_parity, abort_at, 0x310)) goto sums_done;
        tc::tc_fence_after();
        constexpr int kAtOnce = S::kGroups < 4 ? S::kGroups : 4;
#pragma unroll
        for (int g0 = 0; g0 < S::kGroups; g0 += kAtOnce) {
          uint32_t r[kAtOnce][8];
          tmem_ld_now(tmem_row + (uint32_t)(b * BN + 16 * g0), r);
#pragma unroll
          for (int g = 0; g < kAtOnce; ++g) {
            const float4* sc = reinterpret_cast<const float4*>(scales + s * BN + 16 * (g0 + g));
            const float4 lo = sc[0], hi = sc[1];
            const float x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[g0 + g][j] = fmaf(__uint_as_float(r[g][j]), x[j] * ws, acc[g0 + g][j]);
          }
        }
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(acc_empty(b));
          mbar_arrive(scale_empty(s));
        }
        if (++s == kScaleSlots) s = 0, s_parity ^= 1u;
        if (++b == S::kBuffers) b = 0, b_parity ^= 1u;
      }

      // ---- the parts of a split tile: CTA o of the cluster collects the sums of activation rows [o * slice, (o + 1) * slice),
      // [part][4 rows][128 n][row], so that a lane moves 16 bytes and a warp 512 in a run; the bytes complete on the owner's barrier.  No
      // CTA can leave before all that is sent to it has arrived.  The owner adds its own sum and the others' in the order of the parts.
      if (p.split > 1) {
        const uint32_t part_words = (uint32_t)p.slice * kTileN;
#pragma unroll
        for (int g = 0; g < S::kGroups; ++g) {
          const int m = 8 * turn + 16 * g, o = m / p.slice;
          if (m >= split_rows || o == part) continue;
          const uint32_t at = (uint32_t)(part - (part > o)) * part_words + (uint32_t)((m - o * p.slice) * kTileN + n_l * 4);
          const uint32_t dst = tc::map_to_cta(base + exchange_at + at * 4u, (uint32_t)o), bar = tc::map_to_cta(exchanged, (uint32_t)o);
          uint32_t v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = __float_as_uint(acc[g][j]);
          st_async_v4(dst, bar, v[0], v[1], v[2], v[3]);
          if (m + 4 < split_rows) st_async_v4(dst + 4u * kTileN * 4u, bar, v[4], v[5], v[6], v[7]);
        }
        bool ok = true;
        if (end_row > first_row) ok = wait_cluster(exchanged, 0, abort_flag, 0x320);
        if (__any_sync(0xffffffffu, !ok)) goto sums_done;
        const float* parts = reinterpret_cast<const float*>(base_ptr + exchange_at) + n_l * 4;
#pragma unroll
        for (int g = 0; g < S::kGroups; ++g) {
          const int m = 8 * turn + 16 * g;
          if (m < first_row || m >= end_row) continue;
          float sum[8] = {};
          for (int q = 0; q < p.split; ++q) {
            if (q == part) {
#pragma unroll
              for (int j = 0; j < 8; ++j) sum[j] += acc[g][j];
              continue;
            }
            const float* at = parts + (q - (q > part)) * part_words + (m - first_row) * kTileN;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (m + 4 * h >= end_row) continue;
              const float4 v = *reinterpret_cast<const float4*>(at + 4 * h * kTileN);
              sum[4 * h] += v.x, sum[4 * h + 1] += v.y, sum[4 * h + 2] += v.z, sum[4 * h + 3] += v.w;
            }
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[g][j] = sum[j];
        }
      }
      const int first = p.split > 1 ? first_row : 0, last = p.split > 1 ? end_row : end - m0, odd = lane & 1;
#pragma unroll
      for (int g = 0; g < S::kGroups; ++g) {
        const int m = 8 * turn + 16 * g;
        if (m < first || m >= last) continue;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = acc[g][j] + bias;
        if (p.pairs_of_columns) {
          // lanes of an even and an odd n trade: the even one stores the even row's two values, the odd one the odd row's
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const float give = odd ? v[j] : v[j + 1], keep = odd ? v[j + 1] : v[j];
            const float got = __shfl_xor_sync(0xffffffffu, give, 1);
            const uint32_t both = odd ? pack2<T>(got, keep) : pack2<T>(keep, got);
            if (m + j + odd < last && n < p.N)  // N is even: n and its partner are inside together
              *reinterpret_cast<uint32_t*>(out + (int64_t)(m0 + m + j + odd) * p.ldo + (n & ~1)) = both;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (m + j < last && n < p.N) out[(int64_t)(m0 + m + j) * p.ldo + n] = from_float<T>(v[j]);
        }
      }
    }
    if (p.zero_rest) zero_rows<T>(table, p.experts, p.M, p.N, out, p.ldo, (int)threadIdx.x - 64, 32 * kEpiWarps);
  sums_done:;
  }
  __syncwarp();

  tc::tc_fence_before();
  __syncthreads();
  if (*abort_flag) {  // let copies in flight land, and the rest of the cluster give up or finish
    if (threadIdx.x == 0) __nanosleep(50000);
    __syncthreads();
    if (p.split > 1) tc::cluster_sync_all();
  }
  if (warp == 1) {
    tc::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kColumns) : "memory");
  }
}

#include "fp8_gemm_wide.cuh"

// ---- plans ----
struct RowsPlan {
  int BN, tiles, split, k_per_cta, slice, stages, ctas;
  uint32_t exchange_bytes, smem;
  float us;
};

// CTAs that run at a time in clusters of `split`, one on an SM: a cluster lies within one GPC, so that clusters of three and more leave SMs over.
int resident_ctas(int split, int sms) {
  static std::atomic<int> known[64][9];
  int dev = 0;
  if (split == 1 || cudaGetDevice(&dev) != cudaSuccess || dev >= 64) {
    cudaGetLastError();
    return sms;
  }
  std::atomic<int>& slot = known[dev][split];
  int ctas = slot.load(std::memory_order_relaxed);
  if (ctas > 0) return ctas;
  static std::atomic<int> granted[64];
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kRowsThreads);
  cfg.dynamicSmemBytes = rows_most_smem(64);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3((unsigned)(sms * split));
  int clusters = 0;
  if (ensure_dynamic_smem(fp8_rows_kernel<__half, 64>, cfg.dynamicSmemBytes, granted) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&clusters, fp8_rows_kernel<__half, 64>, &cfg) != cudaSuccess || clusters <= 0) {
    cudaGetLastError();
    clusters = sms / split;
  }
  ctas = clusters * split;
  slot.store(ctas, std::memory_order_relaxed);
  return ctas;
}

// The sizes of a problem as the plans see it: `groups` weights that have `M` rows each.
struct Problem {
  int M, N, K, groups, experts;
  bool dense;
  int64_t tile_rows(int high) const { return (int64_t)groups * ((M + high - 1) / high); }
  // the call's bytes, us at a TB/s; more where few SMs ask for them
  float bytes() const { return (float)groups * ((float)N * (float)K + (float)M * (float)K + 2.0f * (float)M * (float)N) * 1e-6f; }
  static float few(int64_t ctas, int sms) { return ctas < sms ? 1.3f - 0.3f * (float)ctas / (float)sms : 1.0f; }
};

// Estimates, us.  Launch and latencies; as the sides of a right angle, the steps of the busiest CTA (with its tiles' outputs) and the call's
// bytes; the exchange of split tiles; the beginning of further rounds.  Fitted to 2000 timings (M 1 to 2048, 300 x 300 to 28672 x 1024, every tile
// height, K in 1 to 8 parts; graphs of calls whose weights come from HBM): 11 % rms off for the kernel of few rows, 7 % for the other, and the
// choices by them are 0.7 % slower than the best of all that were timed.
RowsPlan plan_tiles(const Problem& q, int BN, int split, int sms) {
  RowsPlan t{};
  const int k_steps = (q.K + kStepK - 1) / kStepK, per_sm = BN <= 32 ? 2 : 1, rows = std::min(q.M, BN);
  t.BN = BN;
  t.k_per_cta = (k_steps + split - 1) / split;
  t.split = (k_steps + t.k_per_cta - 1) / t.k_per_cta;
  t.slice = t.split > 1 ? ((rows + t.split - 1) / t.split + 7) / 8 * 8 : BN;
  t.exchange_bytes = (uint32_t)(t.split - 1) * (uint32_t)t.slice * kTileN * 4;
  const uint32_t stage_bytes = kWeightBytes + (uint32_t)BN * kStepK;
  t.stages = t.exchange_bytes < smem_room(BN) ? std::min<int>(kMaxStages, (int)((smem_room(BN) - t.exchange_bytes) / stage_bytes)) : 0;
  t.smem = std::max((uint32_t)t.stages * stage_bytes + t.exchange_bytes + kScaleSlots * (uint32_t)BN * 4 + kBarBytes + experts_bytes(q.experts) + 1024,
                    BN <= 32 ? tc::kSmemOfFewColumns : tc::kSmemOfManyColumns);
  const int64_t tiles = q.tile_rows(BN) * ((q.N + kTileN - 1) / kTileN), all = tiles * t.split;
  const int64_t slots = (int64_t)per_sm * (t.split > 1 ? resident_ctas(t.split, sms) : sms), ctas = t.split > 1 ? all : std::min(all, slots);
  const int64_t rounds = (all + (t.split > 1 ? slots : ctas) - 1) / (t.split > 1 ? slots : ctas);
  const int together = (int)std::min<int64_t>(per_sm, (ctas + sms - 1) / sms);
  t.tiles = (int)std::min<int64_t>(tiles, INT32_MAX);
  t.ctas = (int)std::min<int64_t>(ctas, INT32_MAX);
  const float step = BN == 16 ? 0.22f * (float)together : BN == 32 ? std::max(0.296f, 0.201f * (float)together) : BN == 64 ? 0.294f : 0.47f;
  const float run = (float)rounds * (step * (float)t.k_per_cta + 0.0217f * (float)rows / (float)t.split);
  const float memory = q.bytes() / 7.4f * Problem::few(ctas, sms);
  t.us = 2.3f + std::sqrt(run * run + memory * memory) + 4.17f * (float)(rounds - 1);
  if (t.split > 1) t.us += 0.45f + 0.039f * (float)together * (float)(t.split - 1) / (float)t.split * (float)rows;
  return t;
}
float wide_us(const Problem& q, int sms) {
  const int64_t tiles = q.tile_rows(kWideM) * ((q.N + kWideN - 1) / kWideN), rounds = (tiles + sms - 1) / sms;
  const float run = (float)rounds * (0.373f * (float)((q.K + kStepK - 1) / kStepK) + 3.28f);
  const float memory = q.bytes() / 7.6f * Problem::few(tiles, sms);
  return 1.3f + std::sqrt(run * run + memory * memory);
}

struct Plan {
  bool wide;
  RowsPlan rows;  // if not
};
Plan plan_gemm(const Problem& q, int sms) {
  Plan p{};
  for (int BN : {16, 32, 64, 128}) {
    if (BN > 16 && BN >= 2 * q.M) break;
    for (int split : {1, 2, 3, 4, 6, 8}) {
      const int64_t all = q.tile_rows(BN) * ((q.N + kTileN - 1) / kTileN) * split;
      if (split > 1 && (!q.dense || split * 2 > (q.K + kStepK - 1) / kStepK || all > (BN <= 32 ? 2 : 1) * sms)) break;
      const RowsPlan t = plan_tiles(q, BN, split, sms);
      if (t.split == split && t.stages >= 3 && (p.rows.BN == 0 || t.us < p.rows.us)) p.rows = t;
    }
  }
  p.wide = q.M > 16 && wide_us(q, sms) < p.rows.us;
  return p;
}
// Experts: the offsets are on the device, so the plan takes it that every expert has as many rows as another.
Problem problem_of(int experts, int M, int N, int K, bool dense) {
  const int used = std::min(experts, M);
  return Problem{(M + used - 1) / used, N, K, used, experts, dense};
}

// ---- launches ----
// K-major rows of bytes `ld` apart.
bool encode_rows(CUtensorMap* map, const uint8_t* ptr, int64_t ld, int K, int rows, int box_rows) {
  TensorMapEncodeFn fn = tensor_map_encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {(cuuint32_t)kStepK, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// The weights of all experts: a tile that reaches beyond an expert's rows reads zeros there.
bool encode_weights(CUtensorMap* map, const GemmArgs& g, int box_rows) {
  TensorMapEncodeFn fn = tensor_map_encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {(cuuint64_t)g.K, (cuuint64_t)g.N, (cuuint64_t)g.experts};
  cuuint64_t strides[2] = {(cuuint64_t)g.ldw, (cuuint64_t)g.w_stride};
  cuuint32_t box[3] = {(cuuint32_t)kStepK, (cuuint32_t)box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(g.w), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int BN>
std::string launch_rows_kernel(const GemmArgs& g, const RowsPlan& r, unsigned flags, cudaStream_t stream) {
  CUtensorMap tm_x, tm_w;
  if (!encode_rows(&tm_x, g.x, g.ldx, g.K, g.M, BN) || !encode_weights(&tm_w, g, kTileN)) return "cuTensorMapEncodeTiled failed";
  Params p{};
  p.M = g.M; p.N = g.N;
  p.n_tiles = (g.N + kTileN - 1) / kTileN;
  p.k_steps = (g.K + kStepK - 1) / kStepK;
  p.experts = g.experts; p.offsets = g.offsets; p.zero_rest = g.zero_rest;
  p.split = r.split; p.k_per_cta = r.k_per_cta; p.slice = r.slice; p.stages = r.stages;
  p.exchange_bytes = r.exchange_bytes;
  p.early = (flags & BLKQ4_GEMM_EARLY_WEIGHT_FETCH) != 0;
  p.pairs_of_columns = reinterpret_cast<uintptr_t>(g.out) % 4 == 0 && g.ldo % 2 == 0 && g.N % 2 == 0;
  p.out = g.out; p.ldo = g.ldo;
  p.x_scales = g.x_scales; p.ldxs = g.ldxs;
  p.w_scales = g.w_scales; p.ldws = g.ldws; p.ws_stride = g.ws_stride;
  p.bias = g.bias;
  static std::atomic<int> granted[64];
  cudaError_t e = ensure_dynamic_smem(fp8_rows_kernel<T, BN>, rows_most_smem(BN), granted);
  if (e != cudaSuccess) return cudaGetErrorString(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)r.ctas);
  cfg.blockDim = dim3(kRowsThreads);
  cfg.dynamicSmemBytes = r.smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)r.split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = r.split > 1 ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, fp8_rows_kernel<T, BN>, tm_x, tm_w, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? std::string() : std::string(cudaGetErrorString(e));
}

template <class T>
std::string launch_wide_kernel(const GemmArgs& g, int ctas, unsigned flags, cudaStream_t stream) {
  WideParams p{};
  p.M = g.M; p.N = g.N;
  p.n_tiles = (g.N + kWideN - 1) / kWideN;
  p.k_steps = (g.K + kStepK - 1) / kStepK;
  p.experts = g.experts; p.offsets = g.offsets; p.zero_rest = g.zero_rest;
  p.early = (flags & BLKQ4_GEMM_EARLY_WEIGHT_FETCH) != 0;
  p.scales_on_16 = reinterpret_cast<uintptr_t>(g.x_scales) % 16 == 0 && (g.M == 1 || g.ldxs % 4 == 0);
  const auto begins_on = [&](int n) { return reinterpret_cast<uintptr_t>(g.out) % (2 * n) == 0 && (g.M == 1 || g.ldo % n == 0) && g.N % n == 0; };
  p.vector = begins_on(16) ? 16 : begins_on(8) ? 8 : 1;
  p.out = g.out; p.ldo = g.ldo;
  p.x_scales = g.x_scales; p.ldxs = g.ldxs;
  p.w_scales = g.w_scales; p.ldws = g.ldws; p.ws_stride = g.ws_stride;
  p.bias = g.bias;
  CUtensorMap tm_x, tm_w;
  if (!encode_rows(&tm_x, g.x, g.ldx, g.K, g.M, kWideM) || !encode_weights(&tm_w, g, kWideN)) return "cuTensorMapEncodeTiled failed";
  static std::atomic<int> granted[64];
  const uint32_t smem = wide_smem(g.experts);
  cudaError_t e = ensure_dynamic_smem(fp8_wide_kernel<T>, smem, granted);
  if (e != cudaSuccess) return cudaGetErrorString(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kWideThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, fp8_wide_kernel<T>, tm_x, tm_w, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? std::string() : std::string(cudaGetErrorString(e));
}

template <class T>
std::string launch_typed(const GemmArgs& g, unsigned flags, cudaStream_t stream) {
  const int sms = std::max(2, sm_count());
  // the plan of the latest problem: a function of the sizes alone
  struct Kept {
    int M = 0, N = 0, K = 0, experts = 0, sms = 0;
    bool dense = false;
    Plan plan;
  };
  static thread_local Kept kept[16];
  const bool dense = g.offsets == nullptr;
  Kept& k = kept[((unsigned)g.M * 31u + (unsigned)g.N * 7u + (unsigned)g.K) / 8u % 16u];
  if (k.M != g.M || k.N != g.N || k.K != g.K || k.experts != g.experts || k.dense != dense || k.sms != sms) {
    k.plan = plan_gemm(problem_of(g.experts, g.M, g.N, g.K, dense), sms);
    k.M = g.M, k.N = g.N, k.K = g.K, k.experts = g.experts, k.dense = dense, k.sms = sms;
  }
  // as many CTAs as there may be tiles
  const int high = k.plan.wide ? kWideM : k.plan.rows.BN, wide = k.plan.wide ? kWideN : kTileN;
  const int64_t tiles = ((int64_t)g.M / high + g.experts) * ((g.N + wide - 1) / wide);
  if (tiles > INT32_MAX) return "the problem has too many tiles";
  if (k.plan.wide) return launch_wide_kernel<T>(g, (int)std::min<int64_t>(sms, tiles), flags, stream);
  RowsPlan r = k.plan.rows;
  if (r.split == 1) r.ctas = (int)std::min<int64_t>((int64_t)(r.BN <= 32 ? 2 : 1) * sms, tiles);
  switch (r.BN) {
    case 16: return launch_rows_kernel<T, 16>(g, r, flags, stream);
    case 32: return launch_rows_kernel<T, 32>(g, r, flags, stream);
    case 64: return launch_rows_kernel<T, 64>(g, r, flags, stream);
    default: return launch_rows_kernel<T, 128>(g, r, flags, stream);
  }
}

}  // namespace

std::string launch_gemm(Dtype dtype, const GemmArgs& g, unsigned flags, cudaStream_t stream) {
  if (!g.offsets && gemv_takes(g.M, g.N, g.K)) return launch_gemv(dtype, g, flags, stream);
  return dtype == kFp16 ? launch_typed<__half>(g, flags, stream) : launch_typed<__nv_bfloat16>(g, flags, stream);
}

int read_gemm_error() {
  int v = 0;
  return cudaMemcpyFromSymbol(&v, g_fp8_error, sizeof(int)) == cudaSuccess ? v : -1;
}
int clear_gemm_error(cudaStream_t stream) {
  void* p = nullptr;
  if (cudaGetSymbolAddress(&p, g_fp8_error) != cudaSuccess) return -1;
  return cudaMemsetAsync(p, 0, sizeof(int), stream) == cudaSuccess ? 0 : -1;
}

}  // namespace fp8
}  // namespace blkq4

extern "C" int fp8_gemm_plan_sm100(int experts, int m, int n, int k, int* out8) {
  using namespace blkq4::fp8;
  if (!out8 || m <= 0 || n <= 0 || k <= 0 || m > (1 << 28) || n > (1 << 28) || k > (1 << 28) || experts < 0 || experts > kMaxExperts) return -1;
  for (int i = 0; i < 8; ++i) out8[i] = 0;
  if (experts == 0 && blkq4::fp8::gemv_takes(m, n, k)) {
    out8[0] = 2;
    return 0;
  }
  const int sms = blkq4::sm_count() > 0 ? blkq4::sm_count() : 148;
  const Plan p = plan_gemm(problem_of(std::max(1, experts), m, n, k, experts == 0), sms);
  const int k_steps = (k + kStepK - 1) / kStepK;
  if (p.wide) {
    const int v[8] = {1, kWideM, kWideN, 1, k_steps, kWideStages, (int)wide_smem(std::max(1, experts)), 512};
    std::copy(v, v + 8, out8);
  } else {
    const int v[8] = {0, p.rows.BN, kTileN, p.rows.split, p.rows.k_per_cta, p.rows.stages, (int)p.rows.smem, p.rows.BN <= 32 ? 128 : 256};
    std::copy(v, v + 8, out8);
  }
  return 0;
}
