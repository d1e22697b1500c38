// Product of int8 rows for sm_100a: out[m, n] = T(x_scale[m] * w_scale[n] * sum_k x[m, k] w[n, k] + bias[n]).
//
// Both operands are K-major rows of bytes as they lie in memory: TMA brings 128 k of a tile at a time into shared memory with
// the 128-byte swizzle, tcgen05.mma (kind::i8) multiplies them from there and adds in int32 in tensor memory.  The sums are exact,
// so neither the tiles nor the split of K show in the result; the two scales and the bias are applied in fp32 and the
// result is rounded once.
//
// Two kernels.  gemm_rows_kernel: 128 weight rows (TMEM lanes) x up to 256 activation rows per tile, so that few rows waste no weights'
// bandwidth; the K range of a tile is split over a cluster of CTAs, which exchange their int32 parts through distributed shared
// memory.  gemm_pair_kernel: 256 activation rows (TMEM lanes of two CTAs) x up to 256 weight rows per tile, persistent, for problems
// that fill the GPU with such tiles.
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
#include "int8.cuh"
#include "ms_blkq4gemm.h"

namespace blkq4 {
namespace int8 {

__device__ int g_int8_error = 0;  // 0 ok; otherwise (role << 8) | stage of the wait that gave up

namespace {

using tc::st_async_v4;
using tc::try_wait_cluster;

constexpr int kStepK = 128;                 // k of a pipeline step: one 128-byte swizzle row
constexpr int kTileN = 128;                 // weight rows of a tile
constexpr uint32_t kWeightBytes = kTileN * kStepK;
constexpr long long kWaitCycles = 4000000000ll;  // ~2 s: far beyond any legitimate wait

__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int who) {
  return mbar_wait_bounded(bar, parity, abort_flag, &g_int8_error, who, kWaitCycles);
}
// `wait` on a barrier that other CTAs of the cluster arrive on.
__device__ __forceinline__ bool wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag, int who) {
  const long long t0 = clock64();
  while (!try_wait_cluster(bar, parity)) {
    if (*abort_flag) return false;
    if (clock64() - t0 > kWaitCycles) {
      *abort_flag = 1;
      atomicCAS(&g_int8_error, 0, who);
      return false;
    }
  }
  return true;
}
// Instruction descriptor of kind::i8: int32 accumulator (bits 4-5 = 2), signed A and B (bits 7-9 and 10-12 = 1), both K-major,
// N >> 3 in bits 17-22, M >> 4 in bits 24-28.
__host__ __device__ inline uint32_t make_idesc_i8(int umma_m, int umma_n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(umma_n >> 3) << 17) | ((uint32_t)(umma_m >> 4) << 24);
}
// The four MMAs of a step: 32 k each, both operands two descriptor units (32 bytes) further on.
__device__ __forceinline__ void umma_i8_x4(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a0, a1, a2, a3, b0, b1, b2, b3;\n\t.reg .b32 x1, x2, x3, y1, y2, y3;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "setp.eq.b32 q, 0, 0;\n\t"
      "add.u32 x1, %1, 2;\n\tadd.u32 x2, %1, 4;\n\tadd.u32 x3, %1, 6;\n\t"
      "add.u32 y1, %2, 2;\n\tadd.u32 y2, %2, 4;\n\tadd.u32 y3, %2, 6;\n\t"
      "mov.b64 a0, {%1, %3};\n\tmov.b64 a1, {x1, %3};\n\tmov.b64 a2, {x2, %3};\n\tmov.b64 a3, {x3, %3};\n\t"
      "mov.b64 b0, {%2, %3};\n\tmov.b64 b1, {y1, %3};\n\tmov.b64 b2, {y2, %3};\n\tmov.b64 b3, {y3, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], a0, b0, %4, p;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], a1, b1, %4, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], a2, b2, %4, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], a3, b3, %4, q;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Eight columns, there when it returns: load and wait are one statement, so that no use of the registers can come between them.
__device__ __forceinline__ void tmem_ld_32x32b_x8_now(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(taddr)
      : "memory");
}
// Waits for this thread's loads from tensor memory; the registers they go to are named, so that no use of them moves ahead of it.
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[32]) {
  tc::tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}
__device__ __forceinline__ void prefetch_l2_2d(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}
// How two neighbouring outputs of a row may be stored at once: not; from every even n; in rows of even m from every even n, in the others
// from every odd one (contiguous rows of an odd length).
enum Stores { kSingle, kEven, kAlternate };

struct Params {
  int M, N;
  int BM;          // activation rows of a tile, a multiple of 16, <= 256
  int m_tiles;
  int k_steps;     // of a tile
  int split;       // CTAs of a tile: the cluster size
  int k_per_cta;   // steps of each, the last one what is left
  int slice;       // activation rows whose sums one CTA of the cluster collects, a multiple of 8
  int stages;
  uint32_t exchange_bytes;  // behind the stages: what a CTA collects
  int early;       // weights may be copied before the kernels ahead in the stream have completed
  uint32_t stage_bytes, tmem_cols;
  int stores;      // Stores
  void* out;
  int64_t ldo;
  const float* x_scales;
  const float* w_scales;
  const void* bias;
};

constexpr int kMaxStages = 16;
constexpr int kRowsEpiWarps = 8, kXWarp = 2 + kRowsEpiWarps, kRowsThreads = 32 * (kXWarp + 1);
constexpr uint32_t kBarBytes = 512 + 1024;  // full[], empty[], accumulator, exchange, abort flag, TMEM address; the activations' scales

// Grid: tiles * split CTAs, those of a tile a cluster.  The m tiles of a column tile follow one another.
template <class T>
__global__ void __launch_bounds__(kRowsThreads) gemm_rows_kernel(const __grid_constant__ CUtensorMap tm_x,
                                                             const __grid_constant__ CUtensorMap tm_w, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t exchange_at = (uint32_t)p.stages * p.stage_bytes, bars_at = exchange_at + p.exchange_bytes;
  const uint32_t bars = base + bars_at;
  uint8_t* bars_ptr = base_ptr + bars_at;
  auto full = [&](int s) { return bars + 16u * (uint32_t)s; };
  auto empty = [&](int s) { return bars + 16u * (uint32_t)s + 8u; };
  const uint32_t acc_full = bars + 16u * kMaxStages, exchanged = acc_full + 8u;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars_ptr + 16 * kMaxStages + 16);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars_ptr + 16 * kMaxStages + 20);
  float* x_scales = reinterpret_cast<float*>(bars_ptr + 512);

  const int tile = (int)blockIdx.x / p.split, part = (int)blockIdx.x % p.split;
  const int m0 = tile % p.m_tiles * p.BM, n0 = tile / p.m_tiles * kTileN;
  const int ks0 = part * p.k_per_cta, count = min(p.k_per_cta, p.k_steps - ks0);
  const int rows = min(p.BM, p.M - m0);
  const int first_row = min(rows, part * p.slice), end_row = min(rows, first_row + p.slice);  // whose sums end up here

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&tm_w);
    prefetch_tensormap(&tm_x);
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(full(i), 2);
      mbar_init(empty(i), 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(exchanged, 1);
    *abort_flag = 0;
    mbar_init_fence();
    if (p.split > 1) mbar_arrive_expect_tx(exchanged, (uint32_t)((p.split - 1) * ((end_row - first_row + 3) / 4) * kTileN * 16));
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(p.tmem_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  if (p.split > 1) tc::cluster_sync_all();  // the others' barriers exist before anything is sent to them
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // Two producers, each with its operand: one thread took 0.26 us for the two copies of a step, which set the pace of all
  // small problems (M = 64, 4096 x 4096, tiles of 32 rows, K whole: 11.7 -> 7.7 us).
  if (warp == 0 || warp == kXWarp) {
    if (elect_one()) {
      const bool is_w = warp == 0;
      const CUtensorMap* map = is_w ? &tm_w : &tm_x;
      const uint32_t tx = is_w ? kWeightBytes : (uint32_t)p.BM * kStepK;
      const int row = is_w ? n0 : m0, ahead = min(count, p.stages);
      uint32_t dst = base + (is_w ? 0u : kWeightBytes), bar = full(0), parity = 1;
      int k = ks0 * kStepK, i = 0;
      auto step = [&] {
        mbar_arrive_expect_tx(bar, tx);
        tma_load_2d(dst, map, k, row, bar);
        dst += p.stage_bytes, bar += 16u, k += kStepK, ++i;
      };
      if (is_w) {
        if (p.early) {
          while (i < ahead) step();
        } else {  // at least on their way into L2, where a write that is still to come would find them
          for (int j = 0; j < ahead; ++j) prefetch_l2_2d(map, k + j * kStepK, row);
        }
      }
      griddep_wait();
      griddep_launch_dependents();
      while (i < ahead) step();
      while (i < count) {
        dst -= (uint32_t)p.stages * p.stage_bytes, bar -= 16u * (uint32_t)p.stages, parity ^= 1u;
        const int end = min(count, i + p.stages);
        while (i < end) {
          if (!wait(bar + 8u, parity, abort_flag, 0x100)) goto producer_done;
          step();
        }
      }
    producer_done:;
    }
  } else if (warp == 1) {
    if (elect_one()) {
      griddep_wait();  // or the limit of the waits below would count the kernel ahead
      const uint32_t idesc = make_idesc_i8(kTileN, p.BM);
      const uint64_t desc = tc::make_sw128_kmajor_desc(0);
      const uint32_t desc_hi = (uint32_t)(desc >> 32), desc_lo = (uint32_t)desc;
      const uint32_t first = desc_lo | ((base >> 4) & 0x3FFFu), step = p.stage_bytes >> 4;
      uint32_t lo = first, bar = full(0), parity = 0;
      int left = p.stages;
      bool ok = true;
      for (int i = 0; i < count; ++i) {
        if (!wait(bar, parity, abort_flag, 0x200)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        umma_i8_x4(tmem, lo, lo + (kWeightBytes >> 4), desc_hi, idesc, i > 0);
        tc::umma_commit(bar + 8u);
        lo += step, bar += 16u;
        if (--left == 0) lo = first, bar = full(0), parity ^= 1u, left = p.stages;
      }
      if (ok) tc::umma_commit(acc_full);
    }
  }

  // ---- epilogue: a warp has the 32 weight rows n of its quarter of the TMEM lanes (by warp number mod 4), two warps share a
  // quarter on groups of 8 activation rows m (TMEM columns) in turn
  const int quarter = warp & 3, turn = (warp - 2) >> 2, n_l = quarter * 32 + lane, n = n0 + n_l;
  const uint32_t tmem_row = tmem + ((uint32_t)(quarter * 32) << 16);
  float w_scale = 0.0f, bias = 0.0f;
  const bool epilogue = warp >= 2 && warp < kXWarp;
  if (epilogue) {
    griddep_wait();  // scales of the activations and the output belong to stream order
    // fetched while the MMAs run: behind them, their latency would be the tail of a short call
    for (int i = (int)threadIdx.x - 64; i < rows; i += 32 * kRowsEpiWarps) x_scales[i] = p.x_scales[m0 + i];
    if (n < p.N) {
      w_scale = p.w_scales[n];
      if (p.bias) bias = to_float(reinterpret_cast<const T*>(p.bias)[n]);
    }
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kRowsEpiWarps) : "memory");
    wait(acc_full, 0, abort_flag, 0x300);
  }
  __syncwarp();
  auto dead = [&] { return __shfl_sync(0xffffffffu, *abort_flag, 0) != 0; };  // one answer a warp

  // ---- the parts of a split tile: CTA o of the cluster collects the sums of activation rows [o * slice, (o + 1) * slice),
  // [part][4 rows][128 n][row], so that a lane moves 16 bytes and a warp 512 in a run.  The bytes complete on the owner's
  // barrier, so that it waits for them alone: two barriers of the whole cluster took 0.8 us each (M = 64, 4096 x 4096 in four
  // parts 7.7 -> 6.8 us).  No CTA can leave before all that is sent to it has arrived.
  const uint32_t part_words = (uint32_t)p.slice * kTileN;
  if (p.split > 1 && epilogue && !dead()) {
    tc::tc_fence_after();
    int o = 0;  // owner of row m
    for (int m = turn * 8; m < rows; m += 16) {
      while (m >= (o + 1) * p.slice) ++o;
      if (o == part) continue;
      uint32_t r[8];
      tmem_ld_32x32b_x8_now(tmem_row + (uint32_t)m, r);
      const uint32_t at = (uint32_t)(part - (part > o)) * part_words + (uint32_t)((m - o * p.slice) * kTileN + n_l * 4);
      const uint32_t dst = tc::map_to_cta(base + exchange_at + at * 4u, (uint32_t)o), bar = tc::map_to_cta(exchanged, (uint32_t)o);
      st_async_v4(dst, bar, r[0], r[1], r[2], r[3]);
      if (m + 4 < rows) st_async_v4(dst + 4u * kTileN * 4u, bar, r[4], r[5], r[6], r[7]);
    }
    if (end_row > first_row) wait_cluster(exchanged, 0, abort_flag, 0x310);
  }
  __syncwarp();

  if (epilogue && !dead()) {
    tc::tc_fence_after();
    const int first = first_row, end = end_row;
    const uint32_t* parts = reinterpret_cast<const uint32_t*>(base_ptr + exchange_at) + n_l * 4;
    T* out = reinterpret_cast<T*>(p.out);
    const int odd = lane & 1;
    for (int m = first + turn * 8; m < end; m += 16) {
      uint32_t r[8];
      tmem_ld_32x32b_x8_now(tmem_row + (uint32_t)m, r);
      for (int q = 0; q < p.split - 1; ++q) {
        const uint32_t* at = parts + q * part_words + (m - first) * kTileN;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (m + 4 * h >= end) continue;
          const uint4 v = *reinterpret_cast<const uint4*>(at + 4 * h * kTileN);
          r[4 * h] += v.x, r[4 * h + 1] += v.y, r[4 * h + 2] += v.z, r[4 * h + 3] += v.w;
        }
      }
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = fmaf((float)(int)r[j] * x_scales[m + j], w_scale, bias);
      if (p.stores == kEven) {
        // lanes of an even and an odd n trade: the even one stores the even row's two values, the odd one the odd row's
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const float give = odd ? v[j] : v[j + 1], keep = odd ? v[j + 1] : v[j];
          const float got = __shfl_xor_sync(0xffffffffu, give, 1);
          const uint32_t both = odd ? pack2<T>(got, keep) : pack2<T>(keep, got);
          if (m + j + odd < end && n < p.N)  // N is even: n and its partner are inside together
            *reinterpret_cast<uint32_t*>(out + (int64_t)(m0 + m + j + odd) * p.ldo + (n & ~1)) = both;
        }
      } else if (p.stores == kAlternate) {
        // every second row begins inside a word: its words are the outputs of an odd n and the next one
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const float give = odd ? v[j] : v[j + 1], keep = odd ? v[j + 1] : v[j];
          const float got = __shfl_down_sync(0xffffffffu, give, 1);
          T* at = out + (int64_t)(m0 + m + j + odd) * p.ldo + n;
          if (m + j + odd < end && n < p.N) {
            if (lane < 31 && n + 1 < p.N) *reinterpret_cast<uint32_t*>(at) = pack2<T>(keep, got);
            else *at = from_float<T>(keep);
          }
          if (lane == 0 && m + j + 1 < end && n < p.N) at[p.ldo] = from_float<T>(v[j + 1]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (m + j < end && n < p.N) out[(int64_t)(m0 + m + j) * p.ldo + n] = from_float<T>(v[j]);
      }
    }
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
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
  }
}

// ---- pairs of CTAs ----
// A pair (cta_group::2) computes 256 x BN outputs: each CTA stages its 128 activation rows and its half of the BN weight rows,
// so that an SM reads 64 bytes of shared memory a cycle for the MMAs instead of 96 with a tile of its own, and every operand row
// crosses from L2 once a pair.  The MMAs of a tile run while the epilogue warps empty the other of two accumulators.
//   FULL[s]       of the even CTA (the leader): the bytes of both CTAs' copies; its MMA thread waits
//   EMPTY[s]      of each CTA, by a commit to both: the stage may be written again
//   ACC_FULL[b]   of each CTA, by a commit to both        ACC_EMPTY[b]   of the leader: the epilogue warps of both CTAs
constexpr int kEpiWarps = 8, kPairXWarp = 2 + kEpiWarps, kThreads = 32 * (kPairXWarp + 1);
constexpr int kPairM = 256, kPairMaxN = 256;
constexpr int kPairStages = 6;
constexpr uint32_t kPairHalfBytes = 128u * kStepK;            // one operand's rows of a stage, at most
constexpr uint32_t kPairStageBytes = 2 * kPairHalfBytes;
constexpr uint32_t kPairChunkBytes = 32u * 64u;               // 32 rows x 32 outputs
constexpr uint32_t kPairOutBytes = kEpiWarps * kPairChunkBytes;
constexpr uint32_t kPairScaleBytes = 2u * 2u * kPairMaxN * 4u;  // scales and biases of two tiles' columns
constexpr uint32_t kPairSmem = kPairStages * kPairStageBytes + kPairOutBytes + kPairScaleBytes + 512 + 1024;
static_assert(kPairSmem <= 227 * 1024 && kPairSmem >= tc::kSmemOfManyColumns);

struct PairParams {
  int M, N;
  int BN;  // weight rows of a tile, a multiple of 32, <= 256
  int m_tiles, n_tiles, k_steps;
  int group_m;  // m tiles that run side by side before the next column tiles
  int early;
  int bulk;     // outputs by TMA: rows of the output begin and end on 16 bytes
  void* out;
  int64_t ldo;
  const float* x_scales;
  const float* w_scales;
  const void* bias;
};

__device__ __forceinline__ void umma_i8_x4_pair(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc,
                                                uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a0, a1, a2, a3, b0, b1, b2, b3;\n\t.reg .b32 x1, x2, x3, y1, y2, y3;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "setp.eq.b32 q, 0, 0;\n\t"
      "add.u32 x1, %1, 2;\n\tadd.u32 x2, %1, 4;\n\tadd.u32 x3, %1, 6;\n\t"
      "add.u32 y1, %2, 2;\n\tadd.u32 y2, %2, 4;\n\tadd.u32 y3, %2, 6;\n\t"
      "mov.b64 a0, {%1, %3};\n\tmov.b64 a1, {x1, %3};\n\tmov.b64 a2, {x2, %3};\n\tmov.b64 a3, {x3, %3};\n\t"
      "mov.b64 b0, {%2, %3};\n\tmov.b64 b1, {y1, %3};\n\tmov.b64 b2, {y2, %3};\n\tmov.b64 b3, {y3, %3};\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], a0, b0, %4, p;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], a1, b1, %4, q;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], a2, b2, %4, q;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], a3, b3, %4, q;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives, once every earlier MMA of the pair has retired, on the barrier at this offset in both CTAs.
__device__ __forceinline__ void commit_both(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"((uint16_t)3)
      : "memory");
}
// Copy into this CTA's shared memory whose bytes complete on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar_cluster) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar_cluster)
      : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar_cluster) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster) : "memory");
}
// The tiles of a pair: every num_pairs-th.  Tiles run in bands of group_m m tiles, m fastest, so that those under way at a time
// share the rows of both operands in L2.
struct PairWalk {
  int tile, step, count, m_tiles, n_tiles, group_m;
  __device__ __forceinline__ PairWalk(const PairParams& p)
      : tile((int)(blockIdx.x >> 1)), step((int)(gridDim.x >> 1)), count(p.m_tiles * p.n_tiles), m_tiles(p.m_tiles),
        n_tiles(p.n_tiles), group_m(p.group_m) {}
  __device__ __forceinline__ bool next(int& m_tile, int& n_tile) {
    if (tile >= count) return false;
    const int band = tile / (group_m * n_tiles), first = band * group_m, high = min(group_m, m_tiles - first);
    const int in_band = tile - band * group_m * n_tiles;
    m_tile = first + in_band % high;
    n_tile = in_band / high;
    tile += step;
    return true;
  }
};

template <class T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
gemm_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                 const __grid_constant__ CUtensorMap tm_out, const PairParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
  constexpr uint32_t kOut = kPairStages * kPairStageBytes, kScales = kOut + kPairOutBytes, kBars = kScales + kPairScaleBytes;
  auto full = [&](int s) { return base + kBars + 16u * (uint32_t)s; };
  auto empty = [&](int s) { return base + kBars + 16u * (uint32_t)s + 8u; };
  auto acc_full = [&](int b) { return base + kBars + 16u * (uint32_t)(kPairStages + b); };
  auto acc_empty = [&](int b) { return base + kBars + 16u * (uint32_t)(kPairStages + b) + 8u; };
  constexpr uint32_t kWords = kBars + 16u * (kPairStages + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(base_ptr + kWords);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base_ptr + kWords + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = tc::cluster_ctarank();
  if (threadIdx.x == 0) {
    prefetch_tensormap(&tm_w);
    prefetch_tensormap(&tm_x);
    for (int i = 0; i < kPairStages; ++i) {
      mbar_init(full(i), 2);
      mbar_init(empty(i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full(i), 1);
      mbar_init(acc_empty(i), 2 * kEpiWarps);
    }
    *abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::cluster_sync_all();  // the other CTA's barriers exist before anything signals them
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0 || warp == kPairXWarp) {
    // two producers, each with its operand
    if (elect_one()) {
      const bool is_w = warp == 0;
      const CUtensorMap* map = is_w ? &tm_w : &tm_x;
      const int tile_rows = is_w ? p.BN : kPairM, off = (int)rank * (tile_rows >> 1);
      const uint32_t tx = (uint32_t)tile_rows * kStepK;  // of both CTAs
      const uint32_t dst = base + (is_w ? kPairHalfBytes : 0u), full_leader = tc::map_to_cta(full(0), 0);
      PairWalk walk(p);
      int m_tile, n_tile, s = 0;
      uint32_t parity = 1;  // (the first round finds fresh barriers: the phase before their first one is complete)
      auto copy = [&](int ks, int row) {
        if (rank == 0) mbar_arrive_expect_tx(full(s), tx);
        tma_load_pair(dst + s * kPairStageBytes, map, ks * kStepK, row, full_leader + 16u * (uint32_t)s);
        if (++s == kPairStages) s = 0, parity ^= 1u;
      };
      bool first = true;
      while (walk.next(m_tile, n_tile)) {
        const int row = (is_w ? n_tile : m_tile) * tile_rows + off;
        int ks = 0;
        if (first) {
          first = false;
          if (is_w) {
            const int ahead = min(p.k_steps, kPairStages);
            if (p.early) {
              while (ks < ahead) copy(ks, row), ++ks;
            } else {  // on its way into L2, where a write that is still to come would find it
              for (int j = 0; j < ahead; ++j) prefetch_l2_2d(map, j * kStepK, row);
            }
          }
          griddep_wait();
          griddep_launch_dependents();
        }
        for (; ks < p.k_steps; ++ks) {
          if (!wait(empty(s), parity, abort_flag, 0x1100 | s)) goto producer_done;
          copy(ks, row);
        }
      }
    producer_done:;
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      griddep_wait();  // or the limit of the waits below would count the kernel ahead
      const uint32_t idesc = make_idesc_i8(kPairM, p.BN);
      const uint64_t desc = tc::make_sw128_kmajor_desc(0);
      const uint32_t desc_hi = (uint32_t)(desc >> 32), desc_lo = (uint32_t)desc | ((base >> 4) & 0x3FFFu);
      PairWalk walk(p);
      int m_tile, n_tile, s = 0;
      uint32_t parity = 0;
      for (uint32_t t = 0; walk.next(m_tile, n_tile); ++t) {
        const uint32_t b = t & 1u;
        if (t >= 2 && !wait_cluster(acc_empty(b), ((t >> 1) - 1) & 1u, abort_flag, 0x1200 | b)) goto mma_done;
        tc::tc_fence_after();
        for (int ks = 0; ks < p.k_steps; ++ks) {
          if (!wait(full(s), parity, abort_flag, 0x1210 | s)) goto mma_done;
          tc::tc_fence_after();
          const uint32_t lo = desc_lo + s * (kPairStageBytes >> 4);
          umma_i8_x4_pair(tmem + b * kPairMaxN, lo, lo + (kPairHalfBytes >> 4), desc_hi, idesc, ks > 0);
          commit_both(empty(s));
          if (++s == kPairStages) s = 0, parity ^= 1u;
        }
        commit_both(acc_full(b));
      }
    mma_done:;
    }
  } else {
    // ---- epilogue: a warp has the 32 rows of its quarter of the lanes and every second chunk of 32 outputs, which it brings
    // to a staging block of its own (64-byte rows, their 16-byte pieces swizzled by the row as TMA's 64-byte swizzle has
    // them).  The next chunk is on its way from tensor memory while one is scaled and packed, and the block is waited for only then.
    // Four warps without this took 5.2 us a tile of 256 x 256, more than the MMAs of 2048 k; with eight, and a tile's scales fetched under the stores of
    // the one before, 4096 x 128 x 28672 (25 tiles a pair) takes 82 us.
    const int quarter = warp & 3, et = (int)threadIdx.x - 64;
    const uint32_t tmem_row = tmem + ((uint32_t)(quarter * 32) << 16);
    uint8_t* stage = base_ptr + kOut + (warp - 2) * kPairChunkBytes;
    const uint32_t stage_u32 = smem_u32(stage);
    T* out = reinterpret_cast<T*>(p.out);
    griddep_wait();
    PairWalk walk(p);
    int m_tile, n_tile;
    bool more = walk.next(m_tile, n_tile);
    // a tile's scales and biases, fetched while the tile before it is stored: one column a thread, its row's scale a lane
    float w_scale = 0.0f, bias = 0.0f, x_scale = 0.0f;
    auto fetch = [&] {
      const int n = n_tile * p.BN + et, m = m_tile * kPairM + (int)rank * 128 + quarter * 32 + lane;
      const bool in = et < p.BN && n < p.N;
      w_scale = in ? p.w_scales[n] : 0.0f;
      bias = in && p.bias ? to_float(reinterpret_cast<const T*>(p.bias)[n]) : 0.0f;
      x_scale = m < p.M ? p.x_scales[m] : 0.0f;
    };
    static_assert(32 * kEpiWarps >= kPairMaxN);
    if (more) fetch();
    for (uint32_t t = 0; more; ++t) {
      const uint32_t b = t & 1u;
      const int n0 = n_tile * p.BN, row0 = m_tile * kPairM + (int)rank * 128 + quarter * 32;
      const float row_scale = x_scale;
      // for all warps; the buffer of the tile before last is free, since every warp has passed the barrier of the last one
      float* scales = reinterpret_cast<float*>(base_ptr + kScales) + b * 2 * kPairMaxN;
      float* biases = scales + kPairMaxN;
      scales[et] = w_scale;
      biases[et] = bias;
      asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
      more = walk.next(m_tile, n_tile);
      if (more) fetch();
      const bool ok = wait_cluster(acc_full(b), (t >> 1) & 1u, abort_flag, 0x1300 | b);
      if (__any_sync(0xffffffffu, !ok)) continue;  // on to the barriers of the tiles that are left, so that no warp waits for another
      tc::tc_fence_after();
      const uint32_t acc = tmem_row + b * kPairMaxN;
      uint32_t next[32];
      int c0 = 32 * ((warp - 2) >> 2);
      tc::tmem_ld_32x32b_x32(acc + (uint32_t)c0, next);
      for (; c0 < p.BN; c0 += 64) {
        uint32_t r[32];
        tmem_ld_wait_for(next);
#pragma unroll
        for (int i = 0; i < 32; ++i) r[i] = next[i];
        if (c0 + 64 < p.BN) {
          tc::tmem_ld_32x32b_x32(acc + (uint32_t)c0 + 64u, next);
        } else {  // all of the accumulator that is this warp's is in registers: the MMAs of the tile after next may have it
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_cluster(tc::map_to_cta(acc_empty(b), 0));
        }
        uint32_t v[16];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const float4 s4 = *reinterpret_cast<const float4*>(scales + c0 + q * 4);
          const float4 b4 = *reinterpret_cast<const float4*>(biases + c0 + q * 4);
          const uint32_t* a = r + q * 4;
          v[q * 2] = pack2<T>(fmaf((float)(int)a[0] * row_scale, s4.x, b4.x), fmaf((float)(int)a[1] * row_scale, s4.y, b4.y));
          v[q * 2 + 1] = pack2<T>(fmaf((float)(int)a[2] * row_scale, s4.z, b4.z), fmaf((float)(int)a[3] * row_scale, s4.w, b4.w));
        }
        if (p.bulk && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the last store has read the block
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<uint4*>(stage + lane * 64 + ((q ^ ((lane >> 1) & 3)) * 16)) =
              make_uint4(v[q * 4], v[q * 4 + 1], v[q * 4 + 2], v[q * 4 + 3]);
        if (p.bulk) {
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            if (row0 < p.M && n0 + c0 < p.N)
              asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(&tm_out), "r"(n0 + c0),
                           "r"(row0), "r"(stage_u32)
                           : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {
          __syncwarp();
          const int n = n0 + c0 + lane;
          T* at = out + (int64_t)row0 * p.ldo + n;
          const uint8_t* from[4];  // the lane's output in rows of each swizzle
#pragma unroll
          for (int i = 0; i < 4; ++i) from[i] = stage + ((lane >> 3) ^ i) * 16 + (lane & 7) * 2;
          if (row0 + 32 <= p.M && n0 + c0 + 32 <= p.N) {  // (with its tests in every row: 4000 x 640 x 19999 126 us, 103 without)
#pragma unroll
            for (int row = 0; row < 32; ++row, at += p.ldo) *at = *reinterpret_cast<const T*>(from[(row >> 1) & 3] + row * 64);
          } else {
#pragma unroll 8
            for (int row = 0; row < 32; ++row, at += p.ldo) {
              const T o = *reinterpret_cast<const T*>(from[(row >> 1) & 3] + row * 64);
              if (n < p.N && row0 + row < p.M) *at = o;
            }
          }
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  __syncwarp();

  // neither CTA frees tensor memory or leaves while the other may still signal it
  tc::tc_fence_before();
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) __nanosleep(50000);  // let copies in flight land
  __syncthreads();
  tc::cluster_sync_all();
  if (warp == 1) {
    tc::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// ---- plans ----
struct RowsPlan {
  int BM, m_tiles, n_tiles, split, k_per_cta, slice, stages;
  uint32_t stage_bytes, exchange_bytes, smem;
  float us;
};
constexpr uint32_t kSmemAlone = 222u * 1024, kSmemOfTwo = 110u * 1024;  // stages and exchange of a CTA alone on its SM, of one of two

// The most that a plan asks for, once a device.
template <class T>
cudaError_t allow_smem() {
  static std::atomic<int> granted[64];
  return ensure_dynamic_smem(gemm_rows_kernel<T>, kSmemAlone + kBarBytes + 1024, granted);
}

// CTAs that run at a time in clusters of `split`, `per_sm` on an SM: a cluster lies within one GPC, so that clusters of three and
// more leave SMs over.  (The occupancy query answers one CTA an SM for every kernel that allocates tensor memory; two do run.)
int resident_ctas(int split, int per_sm, int sms) {
  static std::atomic<int> known[64][9];
  int dev = 0;
  if (split == 1 || cudaGetDevice(&dev) != cudaSuccess || dev >= 64) {
    cudaGetLastError();
    return sms * per_sm;
  }
  std::atomic<int>& slot = known[dev][split];
  int ctas = slot.load(std::memory_order_relaxed);
  if (ctas > 0) return ctas * per_sm;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kRowsThreads);
  cfg.dynamicSmemBytes = kSmemAlone + kBarBytes + 1024;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3((unsigned)(sms * split));
  int clusters = 0;
  if (allow_smem<__half>() != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&clusters, gemm_rows_kernel<__half>, &cfg) != cudaSuccess || clusters <= 0) {
    cudaGetLastError();
    clusters = sms / split;
  }
  ctas = clusters * split;
  slot.store(ctas, std::memory_order_relaxed);
  return ctas * per_sm;
}

// All bytes of a call at 7.3 TB/s.
float call_us(int M, int N, int K) { return 0.136e-6f * ((float)N * (float)K + (float)M * (float)K + 2.0f * (float)M * (float)N); }

// The height of tiles and the split of K with the least estimated time.  The estimate, us: 2.3 for a launch and its latencies; as
// the sides of a right angle, the bytes that the busiest SM copies at 130 GB/s (90 where operand rows do not all begin on 32 bytes,
// `sectors`: pitches of 5008 / 5024 / 5120 bytes, 4096 x 5001 x 8192: 136 / 115 / 109 us) and the call's bytes at 7.3 TB/s (5.2
// where few SMs ask for them); 0.26 for an exchange and its bytes at 23 GB/s an SM; 0.011 a row of the epilogue; 0.45 a further
// round of CTAs.  Fitted to 1100 timings (M 8 to 512, 1024 x 1024 to 8192 x 28672, tiles of 16 to 256 rows, K in 1 to 8 parts):
// 16 % rms off, and its choices 2 % slower than the best of all that were timed.
RowsPlan plan_rows(int M, int N, int K, bool sectors, int sms) {
  const int n_tiles = (N + kTileN - 1) / kTileN, k_steps = (K + kStepK - 1) / kStepK;
  const float call = call_us(M, N, K);
  RowsPlan best{};
  int last = 0;
  for (int cap : {256, 192, 128, 96, 64, 48, 32}) {
    const int m_tiles = (M + cap - 1) / cap;
    if (m_tiles == last) continue;
    last = m_tiles;
    const int BM = ((M + m_tiles - 1) / m_tiles + 15) / 16 * 16, rows = std::min(M, BM);
    const int64_t tiles = (int64_t)m_tiles * n_tiles;
    const uint32_t stage_bytes = kWeightBytes + (uint32_t)BM * kStepK;
    for (int want : {1, 2, 3, 4, 6, 8}) {
      if (want > 1 && (want > k_steps / 2 || tiles * want > 2 * sms)) break;
      const int k_per_cta = (k_steps + want - 1) / want, split = (k_steps + k_per_cta - 1) / k_per_cta;
      if (split != want) continue;
      const int64_t ctas = tiles * split;
      const int per_sm = BM <= 128 && ctas > sms ? 2 : 1;
      const int64_t room = resident_ctas(split, per_sm, sms), rounds = (ctas + room - 1) / room;
      const float busiest = (float)(rounds == 1 ? (ctas + sms - 1) / sms : rounds * per_sm);
      const float copy = (sectors ? 7.8e-6f : 1.1e-5f) * busiest * (float)k_per_cta * (float)stage_bytes;
      const float all = ctas < sms ? call * (1.4f - 0.4f * (float)ctas / (float)sms) : call;
      float us = 2.3f + 0.45f * (float)(rounds - 1) + std::sqrt(copy * copy + all * all) +
                 0.0108f * busiest * (float)rows / (float)split;
      if (split > 1) us += 0.26f + 4.3e-5f * busiest * (float)(split - 1) / (float)split * (float)rows * 512.0f;
      RowsPlan t{BM, m_tiles, n_tiles, split, k_per_cta, 0, 0, stage_bytes, 0, 0, us};
      t.slice = split > 1 ? ((rows + split - 1) / split + 7) / 8 * 8 : BM;
      t.exchange_bytes = (uint32_t)(split - 1) * (uint32_t)t.slice * kTileN * 4;
      t.stages = std::min<int>(kMaxStages, (int)(((per_sm == 2 ? kSmemOfTwo : kSmemAlone) - t.exchange_bytes) / stage_bytes));
      t.smem = std::max((uint32_t)t.stages * stage_bytes + t.exchange_bytes + kBarBytes + 1024,
                        BM <= 128 ? tc::kSmemOfFewColumns : tc::kSmemOfManyColumns);
      if (t.stages >= 3 && (best.BM == 0 || us < best.us)) best = t;
    }
  }
  return best;
}

struct PairPlan {
  int BN, m_tiles, n_tiles, pairs;
  float us;
};
// The width of tiles that leaves the least work to the slowest pair.  The estimate, us: 3.8 for a launch and its latencies; 0.1 + 0.0009 BN a
// step (the copies of a pair's two operands set the pace: 100 GB/s an SM), at least 0.8 + 0.0095 BN a tile for its epilogue, and the call's bytes,
// as above; 1 more where outputs are stored one by one.  Measured / estimated: 512 x 4096 x 4096 BN = 128 11.8 / 11.3; 1000 x 4096 x 4096
// 256 16.3 / 15.3; 192 x 4096 x 11008 160 14.4 / 14.3; 256 x 8192 x 28672 224 54 / 55; 2048 x 4096 x 11008 256 58.9 / 57.4; 4096 x 128 x 28672 256
// 82 / 93.
PairPlan plan_pairs(int M, int N, int K, bool bulk, bool sectors, int sms) {
  const int pairs = std::max(1, sms / 2), k_steps = (K + kStepK - 1) / kStepK;
  const float call = call_us(M, N, K);
  PairPlan best{};
  for (int BN = 256; BN >= 128; BN -= 32) {
    PairPlan t{BN, (M + kPairM - 1) / kPairM, (N + BN - 1) / BN, 0, 0.0f};
    const int64_t tiles = (int64_t)t.m_tiles * t.n_tiles, rounds = (tiles + pairs - 1) / pairs;
    t.pairs = (int)std::min<int64_t>(pairs, tiles);
    const float copy = (float)rounds * std::max((float)k_steps * (0.1f + 0.0009f * (float)BN) * (sectors ? 1.0f : 1.4f), 0.8f + 0.0095f * (float)BN);
    t.us = 3.8f + std::sqrt(copy * copy + call * call) + (bulk ? 0.0f : 1.0f);
    if (best.BN == 0 || t.us < best.us) best = t;
  }
  return best;
}

struct Plan {
  bool pair;
  RowsPlan rows;
  PairPlan pairs;
};
Plan plan_gemm(int M, int N, int K, bool bulk, bool sectors, int sms) {
  Plan p{};
  p.pairs = plan_pairs(M, N, K, bulk, sectors, sms);
  p.pair = M > 512 && (int64_t)p.pairs.m_tiles * p.pairs.n_tiles >= sms / 2;
  if (p.pair) return p;
  p.rows = plan_rows(M, N, K, sectors, sms);
  p.pair = p.pairs.us < p.rows.us;
  return p;
}

// ---- launches ----
// K-major rows of bytes `ld` apart.
bool encode_rows(CUtensorMap* map, const int8_t* ptr, int64_t ld, int K, int rows, int box_rows) {
  TensorMapEncodeFn fn = tensor_map_encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {(cuuint32_t)kStepK, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(ptr), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T>
std::string launch_rows_gemm(const GemmArgs& g, const RowsPlan& r, unsigned flags, cudaStream_t stream) {
  CUtensorMap tm_x, tm_w;
  if (!encode_rows(&tm_x, g.x, g.ldx, g.K, g.M, r.BM) || !encode_rows(&tm_w, g.w, g.ldw, g.K, g.N, kTileN))
    return "cuTensorMapEncodeTiled failed";
  Params p{};
  p.M = g.M; p.N = g.N;
  p.BM = r.BM; p.m_tiles = r.m_tiles;
  p.k_steps = (g.K + kStepK - 1) / kStepK;
  p.split = r.split; p.k_per_cta = r.k_per_cta; p.slice = r.slice; p.stages = r.stages;
  p.exchange_bytes = r.exchange_bytes;
  p.early = (flags & BLKQ4_GEMM_EARLY_WEIGHT_FETCH) != 0;
  p.stage_bytes = r.stage_bytes;
  p.tmem_cols = 32;
  while ((int)p.tmem_cols < r.BM) p.tmem_cols *= 2;
  p.stores = reinterpret_cast<uintptr_t>(g.out) % 4 != 0 ? kSingle : g.ldo % 2 != 0 ? kAlternate : g.N % 2 == 0 ? kEven : kSingle;
  p.out = g.out; p.ldo = g.ldo;
  p.x_scales = g.x_scales; p.w_scales = g.w_scales; p.bias = g.bias;
  cudaError_t e = allow_smem<T>();
  if (e != cudaSuccess) return cudaGetErrorString(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(r.m_tiles * r.n_tiles * r.split));
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
  e = cudaLaunchKernelEx(&cfg, gemm_rows_kernel<T>, tm_x, tm_w, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? std::string() : std::string(cudaGetErrorString(e));
}

// Outputs by TMA: rows that begin and end on 16 bytes (a store writes the whole of the 16 bytes in which the tensor's rows end, and
// what lies behind them in a wider matrix is not this call's).
bool stores_in_bulk(const GemmArgs& g) {
  return reinterpret_cast<uintptr_t>(g.out) % 16 == 0 && g.ldo % 8 == 0 && g.N % 8 == 0;
}

template <class T>
std::string launch_pairs(const GemmArgs& g, const PairPlan& t, unsigned flags, cudaStream_t stream) {
  PairParams p{};
  p.M = g.M; p.N = g.N;
  p.BN = t.BN; p.m_tiles = t.m_tiles; p.n_tiles = t.n_tiles;
  p.k_steps = (g.K + kStepK - 1) / kStepK;
  p.group_m = 8;
  p.early = (flags & BLKQ4_GEMM_EARLY_WEIGHT_FETCH) != 0;
  p.bulk = stores_in_bulk(g);
  p.out = g.out; p.ldo = g.ldo;
  p.x_scales = g.x_scales; p.w_scales = g.w_scales; p.bias = g.bias;
  CUtensorMap tm_x, tm_w, tm_out;
  bool ok = encode_rows(&tm_x, g.x, g.ldx, g.K, g.M, 128) && encode_rows(&tm_w, g.w, g.ldw, g.K, g.N, t.BN / 2);
  if (p.bulk) {
    TensorMapEncodeFn fn = tensor_map_encode_fn();
    cuuint64_t dims[2] = {(cuuint64_t)g.N, (cuuint64_t)g.M};
    cuuint64_t strides[1] = {(cuuint64_t)g.ldo * 2};
    cuuint32_t box[2] = {32, 32}, estr[2] = {1, 1};
    ok = ok && fn(&tm_out, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, g.out, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  } else {
    tm_out = tm_x;
  }
  if (!ok) return "cuTensorMapEncodeTiled failed";
  static std::atomic<int> granted[64];
  cudaError_t e = ensure_dynamic_smem(gemm_pair_kernel<T>, kPairSmem, granted);
  if (e != cudaSuccess) return cudaGetErrorString(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2u * (unsigned)t.pairs);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kPairSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, gemm_pair_kernel<T>, tm_x, tm_w, tm_out, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? std::string() : std::string(cudaGetErrorString(e));
}

template <class T>
std::string launch_typed(const GemmArgs& g, unsigned flags, cudaStream_t stream) {
  const int sms = std::max(2, sm_count());
  // the plan of the latest problem: a function of the sizes alone
  struct Kept {
    int M = 0, N = 0, K = 0, sms = 0;
    bool bulk = false, sectors = false;
    Plan plan;
  };
  static thread_local Kept kept[16];
  const bool bulk = stores_in_bulk(g), sectors = g.ldx % 32 == 0 && g.ldw % 32 == 0;
  Kept& k = kept[((unsigned)g.M * 31u + (unsigned)g.N * 7u + (unsigned)g.K) / 8u % 16u];
  if (k.M != g.M || k.N != g.N || k.K != g.K || k.bulk != bulk || k.sectors != sectors || k.sms != sms) {
    k.plan = plan_gemm(g.M, g.N, g.K, bulk, sectors, sms);
    k.M = g.M, k.N = g.N, k.K = g.K, k.bulk = bulk, k.sectors = sectors, k.sms = sms;
  }
  return k.plan.pair ? launch_pairs<T>(g, k.plan.pairs, flags, stream) : launch_rows_gemm<T>(g, k.plan.rows, flags, stream);
}

}  // namespace

std::string launch_gemm(Dtype dtype, const GemmArgs& g, unsigned flags, cudaStream_t stream) {
  if (gemv_takes(g.M, g.N, g.K)) return launch_gemv(dtype, g, flags, stream);
  return dtype == kFp16 ? launch_typed<__half>(g, flags, stream) : launch_typed<__nv_bfloat16>(g, flags, stream);
}

int read_gemm_error() {
  int v = 0;
  return cudaMemcpyFromSymbol(&v, g_int8_error, sizeof(int)) == cudaSuccess ? v : -1;
}
int clear_gemm_error(cudaStream_t stream) {
  void* p = nullptr;
  if (cudaGetSymbolAddress(&p, g_int8_error) != cudaSuccess) return -1;
  return cudaMemsetAsync(p, 0, sizeof(int), stream) == cudaSuccess ? 0 : -1;
}

}  // namespace int8
}  // namespace blkq4

extern "C" int int8_gemm_plan_sm100(int m, int n, int k, int* out8) {
  using namespace blkq4::int8;
  if (!out8 || m <= 0 || n <= 0 || k <= 0 || m > (1 << 28) || n > (1 << 28) || k > kMaxK) return -1;
  for (int i = 0; i < 8; ++i) out8[i] = 0;
  if (gemv_takes(m, n, k)) return 0;
  const int sms = blkq4::sm_count() > 0 ? blkq4::sm_count() : 148;
  const Plan p = plan_gemm(m, n, k, n % 8 == 0, true, sms);
  const int k_steps = (k + kStepK - 1) / kStepK;
  if (p.pair) {
    const int v[8] = {2, kPairM, p.pairs.BN, p.pairs.m_tiles * p.pairs.n_tiles, 1, k_steps, kPairStages, (int)kPairSmem};
    std::copy(v, v + 8, out8);
  } else {
    const int v[8] = {1, p.rows.BM, kTileN, p.rows.m_tiles * p.rows.n_tiles, p.rows.split, p.rows.k_per_cta, p.rows.stages, (int)p.rows.smem};
    std::copy(v, v + 8, out8);
  }
  return 0;
}
