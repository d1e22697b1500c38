// Product of e4m3 rows for many of them: part of fp8_gemm.cu.
//
// A CTA computes 128 x 256 outputs.  A step's 128 x 256 sums leave tensor memory under the MMAs of the next step, which go to the other one of
// two accumulators; eight warps (a quarter of the lanes and half of the columns each) hold the outputs' sums in registers, 128 a thread.  A lane
// is an activation row and has one scale of a step, and the 128 columns of a weight's scale are the warp's: the product of the two is taken
// once a step, and a sum costs half a packed multiply-add.
//
// What sets the pace is the way of an accumulator: its MMAs (512 cycles), their completion's way to the warps, the loads and half of the
// additions (128 sums and 128 loaded values would not fit a thread's registers), and the way back.  So everything that does not have to be on
// it is not: scales go by four steps, additions that are left come before the wait for the next sums, arrivals are no branches.  Shared memory
// is nearly as long at work: 96 bytes a cycle for the MMAs' operands and as many for the copies, 770 cycles a step at 128 bytes.  As pairs of CTAs
// (cta_group::2, 256 x 256 outputs, 128 bytes of shared memory a cycle), with the same warps, the way is longer by that to the other CTA and
// back: 2048 x 8192 x 4096 65.6 us instead of 62.9, 4096 x 8192 x 28672 847 instead of 800.
#pragma once

// Warps 0 to 3: weights, MMAs, activations, scales; the other two warpgroups: the sums, whose threads hold 128 of them.  So those take 232
// registers and leave 40 to the first: 128 * 40 + 256 * 232 are the 384 * 168 that the block is launched with.  (With fewer, a few are spilled to
// local memory, which has next to no L1 beside this shared memory: a reload takes 300 cycles of a step's 600.)
constexpr int kWideXWarp = 2, kWideScaleWarp = 3, kWideSumWarp = 4, kWideThreads = 32 * (kWideSumWarp + kEpiWarps);
constexpr int kWideM = 128, kWideN = 256;
constexpr uint32_t kWideXBytes = kWideM * kStepK, kWideStageBytes = kWideXBytes + kWideN * kStepK;
constexpr int kWideStages = 4;
constexpr int kWideChunks = kWideN / 64;  // of 32 columns, of a warp
constexpr uint32_t kWideBarBytes = 256;
// Scales go by four steps: [128 rows][4] and [2 blocks of 128 columns][4].
constexpr int kWideSlots = 4;
constexpr uint32_t kWideSlotBytes = (kWideM + 2) * 16;
constexpr uint32_t kWideChunkBytes = 32u * 64u;  // 32 rows x 32 outputs, of a warp
constexpr uint32_t wide_smem(int experts) {
  return kWideStages * kWideStageBytes + kEpiWarps * kWideChunkBytes + kWideSlots * kWideSlotBytes + kWideBarBytes +
         8u * (uint32_t)(experts + 1) + 1024;
}
static_assert(wide_smem(kMaxExperts) <= 227 * 1024 && wide_smem(1) >= tc::kSmemOfManyColumns);

struct WideParams {
  int M, N;
  int n_tiles, k_steps;
  int experts;
  const int* offsets;
  int zero_rest;
  int early;
  int scales_on_16;  // every row of the activations' scales begins on 16 bytes
  int vector;  // outputs that may be stored at once: rows begin and end on as many
  void* out;
  int64_t ldo;
  const float* x_scales;
  int64_t ldxs;
  const float* w_scales;
  int64_t ldws, ws_stride;
  const void* bias;
};

// An arrival of the first lane, without a branch.
__device__ __forceinline__ void arrive_lane0(uint32_t bar) {
  asm volatile("{\n\t.reg .pred p;\n\t.reg .u32 l;\n\tmov.u32 l, %%laneid;\n\tsetp.eq.u32 p, l, 0;\n\t@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(bar)
               : "memory");
}
// Waits for this thread's loads from tensor memory; the registers they go to are named, so that no use of them moves ahead of it.
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[32]) {
  tc::tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}
// acc += t * s of two neighbouring columns
__device__ __forceinline__ void add_scaled2(float& a0, float& a1, uint32_t t0, uint32_t t1, float s) {
  asm("{\n\t.reg .b64 a, t, s;\n\t"
      "mov.b64 a, {%0, %1};\n\tmov.b64 t, {%2, %3};\n\tmov.b64 s, {%4, %4};\n\t"
      "fma.rn.f32x2 a, t, s, a;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "r"(t0), "r"(t1), "f"(s));
}

// The tiles of a CTA: every gridDim-th.  An expert's tiles run in bands of 16 tile rows, rows fastest, so that those under way at a time share the
// rows of both operands in L2.
struct WideWalk {
  Experts t;
  int tile, e;
  __device__ __forceinline__ explicit WideWalk(const Experts& t) : t(t), tile((int)blockIdx.x), e(0) {}
  __device__ __forceinline__ bool next(int experts, int n_tiles, int& expert, int& n_tile, int& m0, int& end) {
    if (tile >= t.first(experts) * n_tiles) return false;
    while (t.first(e + 1) * n_tiles <= tile) ++e;
    constexpr int kBand = 16;
    const int m_tiles = t.first(e + 1) - t.first(e), in = tile - t.first(e) * n_tiles;
    const int band = in / (kBand * n_tiles), high = min(kBand, m_tiles - band * kBand), in_band = in - band * kBand * n_tiles;
    n_tile = in_band / high;
    expert = e;
    m0 = t.begin(e) + (band * kBand + in_band - n_tile * high) * kWideM;
    end = t.begin(e + 1);
    tile += (int)gridDim.x;
    return true;
  }
};
__device__ __forceinline__ float4 lds4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}

// Two lanes that differ in one bit (BIT) of their number: the one without it keeps a and gets the other's a for its b; the one with it keeps b and
// gets the other's b for its a.
template <int BIT>
__device__ __forceinline__ void trade(uint32_t (&a)[8], uint32_t (&b)[8], int lane) {
  const bool has = lane & BIT;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t got = __shfl_xor_sync(0xffffffffu, has ? a[j] : b[j], BIT);
    a[j] = has ? got : a[j];
    b[j] = has ? b[j] : got;
  }
}

template <class T>
__global__ void __launch_bounds__(kWideThreads, 1)
fp8_wide_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const WideParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
  constexpr uint32_t kOut = kWideStages * kWideStageBytes, kSlots = kOut + kEpiWarps * kWideChunkBytes;
  constexpr uint32_t kBars = kSlots + kWideSlots * kWideSlotBytes;
  auto full = [&](int s) { return base + kBars + 16u * (uint32_t)s; };
  auto empty = [&](int s) { return base + kBars + 16u * (uint32_t)s + 8u; };
  auto acc_full = [&](int b) { return base + kBars + 16u * (uint32_t)(kWideStages + b); };
  auto acc_empty = [&](int b) { return base + kBars + 16u * (uint32_t)(kWideStages + b) + 8u; };
  auto scale_full = [&](int s) { return base + kBars + 16u * (uint32_t)(kWideStages + 2 + s); };
  auto scale_empty = [&](int s) { return base + kBars + 16u * (uint32_t)(kWideStages + 2 + s) + 8u; };
  constexpr uint32_t kWords = kBars + 16u * (kWideStages + 2 + kWideSlots);
  static_assert(kWords + 8 <= kBars + kWideBarBytes);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(base_ptr + kWords);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base_ptr + kWords + 4);
  const Experts table{base + kBars + kWideBarBytes, base + kBars + kWideBarBytes + 4u * (uint32_t)(p.experts + 1)};

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&tm_w);
    prefetch_tensormap(&tm_x);
    for (int i = 0; i < kWideStages; ++i) {
      mbar_init(full(i), 2);
      mbar_init(empty(i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full(i), 1);
      mbar_init(acc_empty(i), kEpiWarps);
    }
    for (int i = 0; i < kWideSlots; ++i) {
      mbar_init(scale_full(i), 32);
      mbar_init(scale_empty(i), kEpiWarps);
    }
    *abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (p.offsets) griddep_wait();  // they are an operator's output
  tc::tc_fence_before();
  count_tiles(table, p.offsets, p.experts, p.M, kWideM);
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  int expert, n_tile, m0, end;
  WideWalk walk(table);

  if (warp < kWideSumWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0 || warp == kWideXWarp) {
      // two producers, each with its operand
      if (elect_one()) {
        const bool is_w = warp == 0;
        const uint32_t tx = is_w ? kWideN * kStepK : kWideXBytes, dst = base + (is_w ? kWideXBytes : 0u);
        int s = 0;
        uint32_t parity = 1;  // (the first round finds fresh barriers: the phase before their first one is complete)
        auto copy = [&](int ks) {
          mbar_arrive_expect_tx(full(s), tx);
          const uint32_t to = dst + (uint32_t)s * kWideStageBytes;
          if (is_w) tma_load_3d(to, &tm_w, ks * kStepK, n_tile * kWideN, expert, full(s));
          else tma_load_2d(to, &tm_x, ks * kStepK, m0, full(s));
          if (++s == kWideStages) s = 0, parity ^= 1u;
        };
        bool first = true;
        while (walk.next(p.experts, p.n_tiles, expert, n_tile, m0, end)) {
          int ks = 0;
          if (first) {
            first = false;
            if (is_w && !p.offsets) {
              const int ahead = min(p.k_steps, kWideStages);
              if (p.early) {
                while (ks < ahead) copy(ks), ++ks;
              } else {  // on its way into L2, where a write that is still to come would find it
                for (int j = 0; j < ahead; ++j) prefetch_l2_3d(&tm_w, j * kStepK, n_tile * kWideN, expert);
              }
            }
            griddep_wait();
            griddep_launch_dependents();
          }
          for (; ks < p.k_steps; ++ks) {
            if (!wait(empty(s), parity, abort_flag, 0x1100 | s)) goto producer_done;
            copy(ks);
          }
        }
      producer_done:;
      }
    } else if (warp == 1) {
      if (elect_one()) {
        griddep_wait();  // or the limit of the waits below would count the kernel ahead
        constexpr uint32_t idesc = make_idesc_e4m3(kWideM, kWideN);
        const uint64_t desc = tc::make_sw128_kmajor_desc(0);
        const uint32_t desc_hi = (uint32_t)(desc >> 32), desc_lo = (uint32_t)desc | ((base >> 4) & 0x3FFFu);
        int s = 0, b = 0;
        uint32_t parity = 0, acc_parity = 1;
        while (walk.next(p.experts, p.n_tiles, expert, n_tile, m0, end)) {
          for (int ks = 0; ks < p.k_steps; ++ks) {
            if (!wait(full(s), parity, abort_flag, 0x1210 | s)) goto mma_done;
            if (!wait(acc_empty(b), acc_parity, abort_flag, 0x1200 | b)) goto mma_done;
            tc::tc_fence_after();
            const uint32_t lo = desc_lo + (uint32_t)s * (kWideStageBytes >> 4);
            umma_e4m3_x4(tmem + (uint32_t)(b * kWideN), lo, lo + (kWideXBytes >> 4), desc_hi, idesc);
            tc::umma_commit(acc_full(b));
            tc::umma_commit(empty(s));
            if (++s == kWideStages) s = 0, parity ^= 1u;
            if (++b == 2) b = 0, acc_parity ^= 1u;
          }
        }
      mma_done:;
      }
    } else {
      griddep_wait();
      int s = 0;
      uint32_t parity = 1;
      while (walk.next(p.experts, p.n_tiles, expert, n_tile, m0, end)) {
        for (int ks = 0; ks < p.k_steps; ks += 4) {
          if (!wait(scale_empty(s), parity, abort_flag, 0x1120)) goto scales_done;
          const uint32_t dst = base + kSlots + (uint32_t)s * kWideSlotBytes;
          const int left = p.k_steps - ks;
#pragma unroll 1
          for (int i = lane; i < kWideM; i += 32) {
            const bool in = m0 + i < end;
            const float* src = p.x_scales + (in ? (int64_t)(m0 + i) * p.ldxs + ks : 0);
            if (p.scales_on_16 && left >= 4) {
              copy16(dst + (uint32_t)i * 16u, src, in ? 16u : 0u);
            } else {
#pragma unroll
              for (int q = 0; q < 4; ++q) copy4(dst + (uint32_t)i * 16u + 4u * (uint32_t)q, src + (in && q < left ? q : 0), in && q < left);
            }
          }
          if (lane < 8) {
            const int block = min(n_tile * (kWideN / kBlock) + lane / 4, (p.N - 1) / kBlock);
            const bool in = lane % 4 < left;
            copy4(dst + kWideM * 16u + (uint32_t)lane * 4u,
                  p.w_scales + expert * p.ws_stride + (int64_t)block * p.ldws + (in ? ks + lane % 4 : 0), in);
          }
          arrive_behind_copies(scale_full(s));
          if (++s == kWideSlots) s = 0, parity ^= 1u;
        }
      }
    scales_done:
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    // ---- sums and outputs: a warp has the 32 rows of its quarter of the lanes and half of the columns, in chunks of 32
    constexpr int kChunks = kWideChunks;
    const int quarter = warp & 3, half = (warp - kWideSumWarp) >> 2;
    const uint32_t tmem_row = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * kBlock);
    griddep_wait();
    int slot = 0, b = 0;
    uint32_t parity = 0, slot_parity = 0;
    while (walk.next(p.experts, p.n_tiles, expert, n_tile, m0, end)) {
      float acc[kChunks][32];
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int j = 0; j < 32; ++j) acc[c][j] = 0.0f;
      // The scales of four steps at once, and well ahead of their use: shared memory is busy with the MMAs' operands, and a load from it takes
      // 250 to 500 cycles.
      float4 x, w;
      auto next_scales = [&] {
        if (!wait_warp(scale_full(slot), slot_parity, base + kWords, 0x1310)) return false;
        const uint32_t scales = base + kSlots + (uint32_t)slot * kWideSlotBytes;
        x = lds4(scales + (uint32_t)(quarter * 32 + lane) * 16u), w = lds4(scales + (uint32_t)(kWideM + half) * 16u);
        __syncwarp();
        arrive_lane0(scale_empty(slot));
        if (++slot == kWideSlots) slot = 0, slot_parity ^= 1u;
        return true;
      };
      uint32_t r[2][32];
      auto load = [&](int c) { tc::tmem_ld_32x32b_x32(tmem_row + (uint32_t)(b * kWideN + 32 * c), r[c % 2]); };
      auto add = [&](int c, float s) {
#pragma unroll
        for (int j = 0; j < 32; j += 2) add_scaled2(acc[c][j], acc[c][j + 1], r[c % 2][j], r[c % 2][j + 1], s);
      };
#pragma unroll 1
      for (int ks = 0; ks < p.k_steps; ++ks) {
        if (ks % 4 == 0 && !next_scales()) goto sums_done;
        if (!wait_warp(acc_full(b), parity, base + kWords, 0x1300)) goto sums_done;
        tc::tc_fence_after();
        load(0);
        load(1);
        tmem_ld_wait_for(r[0]);
        tmem_ld_wait_for(r[1]);
        const float s = x.x * w.x;
        x = make_float4(x.y, x.z, x.w, 0.0f), w = make_float4(w.y, w.z, w.w, 0.0f);
        add(0, s);
        load(2);
        add(1, s);
        load(3);
        tmem_ld_wait_for(r[0]);
        tmem_ld_wait_for(r[1]);
        // all of the step's sums are in registers: the MMAs may have the accumulator again
        tc::tc_fence_before();
        __syncwarp();
        arrive_lane0(acc_empty(b));
        if (++b == 2) b = 0, parity ^= 1u;
        add(2, s);
        add(3, s);
      }
      const int n0 = n_tile * kWideN + half * kBlock, row0 = m0 + quarter * 32;
      uint8_t* stage = base_ptr + kOut + (warp - kWideSumWarp) * kWideChunkBytes;
      T* out = reinterpret_cast<T*>(p.out);
      if (p.bias) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const float mine = n0 + 32 * c + lane < p.N ? to_float(reinterpret_cast<const T*>(p.bias)[n0 + 32 * c + lane]) : 0.0f;
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[c][j] += __shfl_sync(0xffffffffu, mine, j);
        }
      }
      if (p.vector > 1) {
        // A lane has a row's outputs.  Stored as they are, 32 bytes a lane, an instruction would touch 32 lines, one a cycle, and a tile's
        // outputs take 2000 cycles, for which the MMAs have to wait.  So four lanes trade first: of 64 columns each gets a quarter, of its
        // own row and of the three others'; an instruction then stores whole lines of eight rows.
#pragma unroll
        for (int c = 0; c < kChunks; c += 2) {
          uint32_t v[4][8];  // 16 columns each
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[q][j] = pack2<T>(acc[c + q / 2][16 * (q % 2) + 2 * j], acc[c + q / 2][16 * (q % 2) + 2 * j + 1]);
          trade<1>(v[0], v[1], lane);
          trade<1>(v[2], v[3], lane);
          trade<2>(v[0], v[2], lane);
          trade<2>(v[1], v[3], lane);
          const int n = n0 + 32 * c + 16 * (lane & 3), row = row0 + (lane & ~3);
          T* at = out + (int64_t)row * p.ldo + n;
          if (n < p.N) {
#pragma unroll
            for (int q = 0; q < 4; ++q, at += p.ldo) {
              if (row + q >= end) continue;
              if (p.vector == 16) {  // N is a multiple of it
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(v[q][0]), "r"(v[q][1]), "r"(v[q][2]),
                             "r"(v[q][3]), "r"(v[q][4]), "r"(v[q][5]), "r"(v[q][6]), "r"(v[q][7])
                             : "memory");
              } else {
                *reinterpret_cast<uint4*>(at) = make_uint4(v[q][0], v[q][1], v[q][2], v[q][3]);
                if (n + 8 < p.N) *reinterpret_cast<uint4*>(at + 8) = make_uint4(v[q][4], v[q][5], v[q][6], v[q][7]);
              }
            }
          }
        }
      } else {
        // rows that begin anywhere: through a block of the warp's own, so that neighbouring lanes have neighbouring outputs of a row
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const int n = n0 + 32 * c;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float* a = acc[c] + 8 * q;
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((q ^ ((lane >> 1) & 3)) * 16)) =
                make_uint4(pack2<T>(a[0], a[1]), pack2<T>(a[2], a[3]), pack2<T>(a[4], a[5]), pack2<T>(a[6], a[7]));
          }
          __syncwarp();
          T* at = out + (int64_t)row0 * p.ldo + n + lane;
          const uint8_t* from[4];  // the lane's output in rows of each place of its piece
#pragma unroll
          for (int i = 0; i < 4; ++i) from[i] = stage + ((lane >> 3) ^ i) * 16 + (lane & 7) * 2;
          if (row0 + 32 <= end && n + 32 <= p.N) {
#pragma unroll
            for (int i = 0; i < 32; ++i, at += p.ldo) *at = *reinterpret_cast<const T*>(from[(i >> 1) & 3] + i * 64);
          } else {
#pragma unroll 8
            for (int i = 0; i < 32; ++i, at += p.ldo) {
              const T o = *reinterpret_cast<const T*>(from[(i >> 1) & 3] + i * 64);
              if (n + lane < p.N && row0 + i < end) *at = o;
            }
          }
          __syncwarp();  // all have read the block
        }
      }
    }
    if (p.zero_rest) zero_rows<T>(table, p.experts, p.M, p.N, reinterpret_cast<T*>(p.out), p.ldo, (int)threadIdx.x - 32 * kWideSumWarp, 32 * kEpiWarps);
  sums_done:;
  }
  __syncwarp();

  tc::tc_fence_before();
  __syncthreads();
  if (*abort_flag) {  // let copies in flight land
    if (threadIdx.x == 0) __nanosleep(50000);
    __syncthreads();
  }
  if (warp == 1) {
    tc::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}
